// The 8-bit cache: tokens in (with the position rotation on the way) and out again as 16-bit values.
//
// Both directions are bound by memory: a token of one head is 512 B of 16-bit keys and values and 256 B of codes.
// Work unit: one block of 32 tokens of one head, keys by four warps and values by the other four, a block of threads
// walking over heads so that the tokens' angle table (64-bit products, sine, cosine) is made once.
//
// Codes: 127 x / max|x| to the nearest, halves away from zero, as floor(x * inv + 1/2) with inv = 127 / max|x| raised
// by 2^-21.  x and max|x| are 16-bit numbers, so the quotient is a half exactly or at least 2^-12 of it away (2^-13 per
// power of two that the quotient is below 127); 32-bit rounding stays below a quarter of that, and the raise, which
// is above the rounding and below that distance, sends exact halves outward on both sides of zero.
#include "decode.cuh"
#include "kv8.cuh"
#include "rotary.cuh"

namespace kitty {

struct AppendArgs {
  kitty_kv8_layer L;
  kitty_rotary_plan pl;
  const void *k, *v, *q;
  void *q_out;
  int64_t ks[3], vs[3], qs[3];
  const int32_t *start, *counts;
  int32_t T, h_q, heads;          // heads: key heads of a block of threads
};

__device__ __forceinline__ void half_barrier(int half) {
  asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
}

// Four floats -> four codes (two's complement bytes) in one word.
__device__ __forceinline__ uint32_t kv8_codes4(const float *x, float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(__fadd_rd(fmaf(x[i], inv, 0.5f), 12582912.0f));
  return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}

template <typename T, int MODE>
__global__ void __launch_bounds__(256) kv8_append_kernel(const __grid_constant__ AppendArgs a) {
  using U = RotUnits<T, MODE>;
  constexpr bool HALF = MODE == ROT_HALF || MODE == ROT_HALF_SCALAR;
  constexpr uint32_t INF16 = sizeof(T) == 2 && __is_same(T, __half) ? 0x7c00u : 0x7f80u;
  __shared__ __align__(16) float2 tab[MODE == ROT_NONE ? 1 : KV8_BLOCK][HD / 2];
  __shared__ __align__(16) uint8_t vt[HD][36];
  __shared__ __align__(16) T stage[HALF ? KV8_BLOCK : 1][HD + 8];
  __shared__ uint32_t red[2][8];
  const kitty_kv8_layer &L = a.L;
  const int b = blockIdx.z, cap = L.max_page * PAGE;
  const int raw = a.start[b];
  int n = a.counts != nullptr ? a.counts[b] : a.T;
  int s = raw;
  bool bad = n < 0 || n > a.T || s < 0 || s > cap;
  n = min(max(n, 0), a.T);
  if (s < 0 || s > cap) s = 0, n = 0;
  if (n > cap - s) n = cap - s, bad = true;
  if (bad && threadIdx.x == 0) atomicOr(L.status, KITTY_KV8_BAD_LENGTH);
  const int end = s + n, fb = s / KV8_BLOCK, eb = end / KV8_BLOCK;
  const int h0 = blockIdx.y * a.heads, h1 = min(h0 + a.heads, L.h_kv);
  const int r = a.pl.rotary_dim, np = r / 2;
  const int half = threadIdx.x >> 7, tid = threadIdx.x & 127;

  auto process = [&](int blk, bool kv, bool rows_q) {
    const int t0 = blk * KV8_BLOCK - s;                 // input index of the block's first token
    if constexpr (MODE != ROT_NONE) {
      const int last = rows_q ? a.T : n;
      for (int i = threadIdx.x; i < KV8_BLOCK * np; i += 256) {
        const int tk = i / np, p = i - tk * np;
        if (t0 + tk >= 0 && t0 + tk < last) tab[tk][U::slot(p, r)] = rot_angle(a.pl, static_cast<int64_t>(raw) + t0 + tk, p);
      }
      __syncthreads();
    }
    if (kv) {
      const int tk = tid >> 2, t = tid & 3, warp = tid >> 5;
      const int i = t0 + tk;
      const bool full = (blk + 1) * KV8_BLOCK <= end;
      const bool fresh = i >= 0 && i < n, kept = i < 0 && full;
      const bool turn = MODE != ROT_NONE && half == 0 && fresh;
      // A thread holds channels 16t .. 16t+15 and 64+16t .. 64+16t+15 of its token: for a fully rotated head in halves,
      // and for neighbouring pairs, both members of sixteen pairs, whose angles stay in registers over the heads.
      const bool in_regs = !HALF || r == HD;
      float cs[16], sn[16];
      if constexpr (MODE != ROT_NONE) {
        if (turn && in_regs) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int p = HALF ? 16 * t + e : 8 * t + (e & 7) + 32 * (e >> 3);
            const float2 x = p < np ? tab[tk][U::slot(p, r)] : make_float2(1.f, 0.f);
            cs[e] = x.x;
            sn[e] = x.y;
          }
        }
      }
      const int64_t page = full ? kv8_page(L, b, blk) : -1;
      T *tail = static_cast<T *>(half ? L.tail_v : L.tail_k);
      const int64_t *st = half ? a.vs : a.ks;
      const T *in = static_cast<const T *>(half ? a.v : a.k) + b * st[0] + i * st[2];
      for (int h = h0; h < h1; ++h) {
        T *trow = tail + ((static_cast<int64_t>(b) * L.h_kv + h) * KV8_BLOCK + tk) * HD;
        uint4 w[4] = {};
        if (fresh || kept) {
          const T *src = fresh ? in + h * st[1] : trow;
#pragma unroll
          for (int c = 0; c < 4; ++c) w[c] = *reinterpret_cast<const uint4 *>(src + (c >> 1) * 64 + t * 16 + (c & 1) * 8);
        }
        if constexpr (MODE != ROT_NONE) {
          if (turn && in_regs) {
            float x[4][8];
#pragma unroll
            for (int c = 0; c < 4; ++c) Vec8<T>::unpack(w[c], x[c]);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if constexpr (HALF) {
                const float u = x[e >> 3][e & 7], v = x[2 + (e >> 3)][e & 7];
                x[e >> 3][e & 7] = fmaf(u, cs[e], -v * sn[e]);
                x[2 + (e >> 3)][e & 7] = fmaf(v, cs[e], u * sn[e]);
              } else {
                float &u = x[e >> 2][(2 * e) & 7], &v = x[e >> 2][(2 * e + 1) & 7];
                if (8 * t + (e & 7) + 32 * (e >> 3) < np) {      // an untouched pair may hold infinities
                  const float u0 = u;
                  u = fmaf(u0, cs[e], -v * sn[e]);
                  v = fmaf(v, cs[e], u0 * sn[e]);
                }
              }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              Piece<T> p;
#pragma unroll
              for (int e = 0; e < 8; ++e) p.f[e] = x[c][e];
              w[c] = p.pack();
            }
          }
          if constexpr (HALF) {
            if (r != HD && half == 0) {        // a pair's members are in two threads of the token's four
#pragma unroll
              for (int c = 0; c < 4; ++c)
                *reinterpret_cast<uint4 *>(&stage[tk][(c >> 1) * 64 + t * 16 + (c & 1) * 8]) = w[c];
              __syncwarp();
              if (turn) {
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                  Piece<T> p;
                  p.unpack(w[c]);
#pragma unroll
                  for (int e = 0; e < 8; ++e) {
                    const int d = (c >> 1) * 64 + t * 16 + (c & 1) * 8 + e;
                    if (d < r) {
                      const int q = d < np ? d : d - np;
                      const float2 z = tab[tk][U::slot(q, r)];
                      const float o = to_f32<T>(stage[tk][d < np ? d + np : d - np]);
                      p.f[e] = d < np ? fmaf(p.f[e], z.x, -o * z.y) : fmaf(p.f[e], z.x, o * z.y);
                    }
                  }
                  w[c] = p.pack();
                }
              }
              __syncwarp();
            }
          }
        }
        if (!full) {
          if (fresh) {
#pragma unroll
            for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4 *>(trow + (c >> 1) * 64 + t * 16 + (c & 1) * 8) = w[c];
          }
          continue;
        }
        // largest magnitude of the block: 16-bit patterns without the sign order like the numbers
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          m = __vmaxu2(m, w[c].x & 0x7fff7fffu);
          m = __vmaxu2(m, w[c].y & 0x7fff7fffu);
          m = __vmaxu2(m, w[c].z & 0x7fff7fffu);
          m = __vmaxu2(m, w[c].w & 0x7fff7fffu);
        }
        m = max(m & 0xffffu, m >> 16);
        m = __reduce_max_sync(0xffffffffu, m);
        uint32_t *rd = red[h & 1] + 4 * half;
        if ((tid & 31) == 0) rd[warp] = m;
        half_barrier(half);
        m = max(max(rd[0], rd[1]), max(rd[2], rd[3]));
        const uint16_t mb = static_cast<uint16_t>(m);
        const float top = to_f32<T>(*reinterpret_cast<const T *>(&mb));
        float scale, inv;
        float pre = 1.0f;
        if (m >= INF16) scale = __uint_as_float(0x7fc00000u), inv = 0.0f;
        else if (m == 0) scale = 1.0f, inv = 0.0f;
        else {
          if (top < 0x1p-100f) pre = 0x1p100f;           // keeps the reciprocal in range
          scale = __fdiv_rn(top, 127.0f);
          inv = __fdiv_rn(127.0f, top * pre) * (1.0f + 0x1p-21f);
        }
        uint8_t *rec = page >= 0 ? kv8_record(L, page, h, blk & 3) : nullptr;
        if (rec != nullptr && tid == 0) *reinterpret_cast<float *>(rec + KV8_OFF_SCALE + 4 * half) = scale;
        uint4 code[2];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float x[8];
          Vec8<T>::unpack(w[c], x);
          if (pre != 1.0f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= pre;
          }
          const uint32_t lo = kv8_codes4(x, inv), hi = kv8_codes4(x + 4, inv);
          if (c & 1) code[c >> 1].z = lo, code[c >> 1].w = hi;
          else code[c >> 1].x = lo, code[c >> 1].y = hi;
        }
        if (half == 0) {
          if (rec != nullptr) {
            const int i4 = (tk >> 1) & 3, g = 2 * (tk >> 3) + (tk & 1);
            uint8_t *o = rec + i4 * 1024 + (4 * g + t) * 16;
            *reinterpret_cast<uint4 *>(o) = code[0];
            *reinterpret_cast<uint4 *>(o + 512) = code[1];
          }
        } else {
          // values go out with their tokens side by side
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t q4[4] = {code[c].x, code[c].y, code[c].z, code[c].w};
#pragma unroll
            for (int e = 0; e < 16; ++e) vt[64 * c + 16 * t + e][tk] = static_cast<uint8_t>(q4[e >> 2] >> (8 * (e & 3)));
          }
          half_barrier(half);
          if (rec != nullptr) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int p = tid + 128 * j, x = p >> 5, g = (p >> 2) & 7, tt = p & 3;
              const uint32_t *r0 = reinterpret_cast<const uint32_t *>(&vt[16 * x + g][8 * tt]);
              const uint32_t *r1 = reinterpret_cast<const uint32_t *>(&vt[16 * x + 8 + g][8 * tt]);
              *reinterpret_cast<uint4 *>(rec + KV8_OFF_V + p * 16) = make_uint4(r0[0], r0[1], r1[0], r1[1]);
            }
          }
        }
      }
    }
    if constexpr (MODE != ROT_NONE) {
      if (rows_q) {
        constexpr int LPR = U::VEC ? (MODE == ROT_HALF ? 8 : 16) : 32;
        const int q0 = static_cast<int>(static_cast<int64_t>(a.h_q) * blockIdx.y / gridDim.y);
        const int q1 = static_cast<int>(static_cast<int64_t>(a.h_q) * (blockIdx.y + 1) / gridDim.y);
        const int first = max(0, -t0), toks = min(KV8_BLOCK, a.T - t0) - first, nh = q1 - q0;
        const int nu = U::turned(r) + U::copied(r);
        for (int row = threadIdx.x / LPR; row < toks * nh; row += 256 / LPR) {
          const int tk = first + row / nh, h = q0 + row % nh;
          const T *src = static_cast<const T *>(a.q) + b * a.qs[0] + h * a.qs[1] + (t0 + tk) * a.qs[2];
          T *dst = static_cast<T *>(a.q_out) + ((static_cast<int64_t>(b) * a.h_q + h) * a.T + t0 + tk) * HD;
          for (int u = threadIdx.x % LPR; u < nu; u += LPR) {
            RotUnit<T, MODE> x;
            x.load(src, u, r);
            x.store(dst, u, r, tab[tk]);
          }
        }
      }
    }
    __syncthreads();
  };

  const int blk = fb + blockIdx.x;
  const bool full = (blk + 1) * KV8_BLOCK <= end;
  const bool kv = n > 0 && (full || (blockIdx.x == 0 && eb == fb));
  const bool rows_q = MODE != ROT_NONE && a.h_q > 0 && blk * KV8_BLOCK - s < a.T;
  if (kv || rows_q) process(blk, kv, rows_q);
  // The open block that the call leaves behind overwrites the tails, which the first block reads: the same threads do
  // both, one after the other.
  if (blockIdx.x == 0 && n > 0 && eb > fb && end % KV8_BLOCK != 0) process(eb, true, false);
}

struct ExpandArgs {
  kitty_kv8_layer L;
  const int32_t *lengths, *start;
  void *k_out, *v_out;
  int32_t n;
};

template <typename T>
__device__ __forceinline__ void expand16(uint4 codes, float scale, uint4 (&out)[2]) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    Piece<T> p;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      p.f[e] = static_cast<float>(static_cast<int8_t>(w[2 * c + (e >> 2)] >> (8 * (e & 3)))) * scale;
    out[c] = p.pack();
  }
}

template <typename T>
__global__ void __launch_bounds__(256) kv8_expand_kernel(const __grid_constant__ ExpandArgs a) {
  __shared__ __align__(16) uint8_t vt[KV8_BLOCK][HD + 16];
  const kitty_kv8_layer &L = a.L;
  const int b = blockIdx.z, h = blockIdx.y, cap = L.max_page * PAGE;
  const int len = kv8_clamp_len(L, a.lengths[b]);
  int s = a.start != nullptr ? a.start[b] : 0;
  if (s < 0 || s > cap) {
    atomicOr(L.status, KITTY_KV8_BAD_LENGTH);
    s = cap;                                            // nothing held there: zeros
  }
  const int blk = s / KV8_BLOCK + blockIdx.x, t0 = blk * KV8_BLOCK - s;    // output index of the block's first token
  if (t0 >= a.n) return;
  const bool full = (blk + 1) * KV8_BLOCK <= len;
  const int64_t page = full ? kv8_page(L, b, blk) : -1;
  const int64_t bh = static_cast<int64_t>(b) * L.h_kv + h;
  T *ko = static_cast<T *>(a.k_out) + bh * a.n * HD, *vo = static_cast<T *>(a.v_out) + bh * a.n * HD;
  auto put = [&](T *base, int tk, int ch, const uint4 (&x)[2]) {
    const int i = t0 + tk;
    if (i < 0 || i >= a.n) return;
    uint4 *o = reinterpret_cast<uint4 *>(base + static_cast<int64_t>(i) * HD + ch);
    o[0] = x[0];
    o[1] = x[1];
  };
  uint4 x[2] = {};
  if (full && page >= 0) {
    const uint8_t *rec = kv8_record(L, page, h, blk & 3);
    const uint4 kc = *reinterpret_cast<const uint4 *>(rec + threadIdx.x * 16);
    const uint4 vc = *reinterpret_cast<const uint4 *>(rec + KV8_OFF_V + threadIdx.x * 16);
    const float2 sc = *reinterpret_cast<const float2 *>(rec + KV8_OFF_SCALE);
    const int g = (threadIdx.x >> 2) & 7, t = threadIdx.x & 3;
    expand16<T>(kc, sc.x, x);
    put(ko, kv8_key_token(threadIdx.x >> 6, g), ((threadIdx.x >> 5) & 1) * 64 + 16 * t, x);
    const uint32_t w[4] = {vc.x, vc.y, vc.z, vc.w};
    const int ch = 16 * (threadIdx.x >> 5) + g;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      vt[8 * t + e][ch] = static_cast<uint8_t>(w[e >> 2] >> (8 * (e & 3)));
      vt[8 * t + e][ch + 8] = static_cast<uint8_t>(w[2 + (e >> 2)] >> (8 * (e & 3)));
    }
    __syncthreads();
    const int tk = threadIdx.x >> 3, c = (threadIdx.x & 7) * 16;
    expand16<T>(*reinterpret_cast<const uint4 *>(&vt[tk][c]), sc.y, x);
    put(vo, tk, c, x);
  } else {
    const int tk = threadIdx.x >> 3, c = (threadIdx.x & 7) * 16;
    const bool held = !full && blk * KV8_BLOCK + tk < len;      // an open block's token; a skipped page gives zeros
    const int64_t at = (bh * KV8_BLOCK + tk) * HD + c;
    for (int side = 0; side < 2; ++side) {
      if (held) {
        const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(side ? L.tail_v : L.tail_k) + at);
        x[0] = src[0];
        x[1] = src[1];
      }
      put(side ? vo : ko, tk, c, x);
    }
  }
}

template <typename T>
int launch_append(const AppendArgs &a, int mode, dim3 grid, cudaStream_t s) {
  switch (mode) {
    case ROT_HALF: kv8_append_kernel<T, ROT_HALF><<<grid, 256, 0, s>>>(a); break;
    case ROT_INTER: kv8_append_kernel<T, ROT_INTER><<<grid, 256, 0, s>>>(a); break;
    case ROT_HALF_SCALAR: kv8_append_kernel<T, ROT_HALF_SCALAR><<<grid, 256, 0, s>>>(a); break;
    case ROT_INTER_SCALAR: kv8_append_kernel<T, ROT_INTER_SCALAR><<<grid, 256, 0, s>>>(a); break;
    default: kv8_append_kernel<T, ROT_NONE><<<grid, 256, 0, s>>>(a); break;
  }
  return cudaGetLastError() == cudaSuccess ? KITTY_OK : KITTY_E_CUDA;
}

}  // namespace kitty

using namespace kitty;

extern "C" int kitty_kv8_append(const kitty_kv8_layer *layer, const void *key, const void *value,
                                const int64_t *strides, const int32_t *start, const int32_t *counts, int32_t B,
                                int32_t T, const kitty_rotary_plan *rotary, const void *query, void *q_out,
                                int32_t h_q, void *stream) {
  int rc = check_kv8_layer(layer);
  if (rc != KITTY_OK) return rc;
  if (!strides || B < 0 || T < 0 || h_q < 0 || B > layer->max_bs) return KITTY_E_BADARG;
  if (rotary != nullptr && (rc = check_rotary_plan(rotary)) != KITTY_OK) return rc;
  if (h_q > 0 && rotary == nullptr) return KITTY_E_BADARG;
  if (B == 0 || T == 0) return KITTY_OK;
  if (h_q > 0 && (!query || !q_out)) return KITTY_E_BADARG;
  if (!key || !value || !start) return KITTY_E_BADARG;
  AppendArgs a{};
  a.L = *layer;
  if (rotary != nullptr) a.pl = *rotary;
  else a.pl.rotary_dim = 0;
  a.k = key;
  a.v = value;
  a.q = query;
  a.q_out = q_out;
  if ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15) return KITTY_E_BADARG;
  if (h_q > 0 && ((reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(q_out)) & 15)) return KITTY_E_BADARG;
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = strides[i];
    a.vs[i] = strides[3 + i];
    a.qs[i] = strides[6 + i];
    if (a.ks[i] % 8 != 0 || a.vs[i] % 8 != 0 || (h_q > 0 && a.qs[i] % 8 != 0)) return KITTY_E_BADARG;
  }
  a.start = start;
  a.counts = counts;
  a.T = T;
  a.h_q = h_q;
  const int64_t blocks = (static_cast<int64_t>(T) + 2 * KV8_BLOCK - 2) / KV8_BLOCK;   // that T tokens can touch
  if (B > 65535 || T > (1 << 30)) return KITTY_E_BADSHAPE;
  // Heads are spread over blocks of threads until there are four per multiprocessor; the rest share an angle table.
  int64_t split = (4 * static_cast<int64_t>(sm_count()) + blocks * B - 1) / (blocks * B);
  if (split > layer->h_kv) split = layer->h_kv;
  a.heads = static_cast<int32_t>((layer->h_kv + split - 1) / split);
  split = (layer->h_kv + a.heads - 1) / a.heads;
  if (split > 65535) return KITTY_E_BADSHAPE;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(split), static_cast<unsigned>(B));
  const int mode = rotary != nullptr ? rot_mode(*rotary, 2) : ROT_NONE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return layer->dtype == KITTY_F16 ? launch_append<__half>(a, mode, grid, s) : launch_append<__nv_bfloat16>(a, mode, grid, s);
}

extern "C" int kitty_kv8_expand(const kitty_kv8_layer *layer, const int32_t *lengths, const int32_t *start,
                                void *k_out, void *v_out, int32_t B, int32_t n, void *stream) {
  const int rc = check_kv8_layer(layer);
  if (rc != KITTY_OK) return rc;
  if (B < 0 || n < 0 || B > layer->max_bs) return KITTY_E_BADARG;
  if (B == 0 || n == 0) return KITTY_OK;
  if (!lengths || !k_out || !v_out) return KITTY_E_BADARG;
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) return KITTY_E_BADARG;
  if (B > 65535 || layer->h_kv > 65535 || n > (1 << 30)) return KITTY_E_BADSHAPE;
  ExpandArgs a{*layer, lengths, start, k_out, v_out, n};
  const int64_t blocks = (static_cast<int64_t>(n) + 2 * KV8_BLOCK - 2) / KV8_BLOCK;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(layer->h_kv), static_cast<unsigned>(B));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (layer->dtype == KITTY_F16) kv8_expand_kernel<__half><<<grid, 256, 0, s>>>(a);
  else kv8_expand_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? KITTY_OK : KITTY_E_CUDA;
}
