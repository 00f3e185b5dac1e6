// The 8-bit cache: tokens in (with the position rotation on the way) and out again as 16-bit values.
//
// Both directions are bound by memory: a token of one head is 512 B of 16-bit keys and values and 256 B of codes.
// Work unit: one block of 32 tokens of one head, keys by four warps and values by the other four, a block of threads
// walking over heads so that the tokens' angle table (64-bit products, sine, cosine) is made once.
//
// Codes: 127 x / max|x| to the nearest, halves away from zero, as floor(x * inv + 1/2) with inv = 127 / max|x| raised
// by 2^-21.  x and max|x| are 16-bit numbers, so the quotient is a half exactly or at least 2^-12 of it away (2^-13 per
// power of two that the quotient is below 127); the 32-bit rounding of inv stays below a quarter of that, and the raise,
// which is above the rounding and below that distance, sends exact halves outward on both sides of zero.  The floor costs
// nothing: the multiply-add has 49152.5 as its addend and rounds down, so its result is a multiple of 2^-8 and the code
// is the second byte of the number.
#include "decode.cuh"
#include "kv8.cuh"
#include "overlap.cuh"
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
  for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(__fmaf_rd(x[i], inv, 49152.5f));
  return __byte_perm(__byte_perm(w[0], w[1], 0x0051), __byte_perm(w[2], w[3], 0x0051), 0x5410);
}

// The angle table of the append kernel: entries of the 32 tokens side by side in the order in which the four threads of
// a key token hold its channels (thread t: channels 16t .. 16t + 15 and 64 + 16t ... as sixteen pairs), two pairs a word.
// Pairs in halves of a fully rotated head: pair 16t + e; neighbouring pairs: 8t + e, then 32 + 8t + e - 8.  A partly
// rotated head in halves keeps the first form, its pairs in order.
template <typename T, int MODE>
struct BlockTable {
  using U = RotUnits<T, MODE>;
  static constexpr bool INTER = MODE == ROT_INTER || MODE == ROT_INTER_SCALAR;
  const float4 *tab;       // [8][128]
  int tk;
  // word and half of pair p of token tk
  static __device__ __forceinline__ int word(int p, int tk) {
    const int t = INTER ? (p >> 3) & 3 : p >> 4, e = INTER ? (p & 7) + 8 * (p >> 5) : p & 15;
    return (e >> 1) * 128 + 4 * tk + t;
  }
  __device__ __forceinline__ float4 pairs(int p) const { return tab[word(p, tk)]; }          // p even: pairs p, p + 1
  __device__ __forceinline__ float4 two(int u, int k) const { return pairs(u * U::PV + 2 * k); }
  __device__ __forceinline__ float2 one(int p) const {
    const float4 x = pairs(p & ~1);
    return p & 1 ? make_float2(x.z, x.w) : make_float2(x.x, x.y);
  }
};

// 4 x 4 bytes the other way round: byte j of out[i] = byte i of in[j].
__device__ __forceinline__ void transpose4(const uint32_t (&in)[4], uint32_t (&out)[4]) {
  const uint32_t a = __byte_perm(in[0], in[1], 0x5140), b = __byte_perm(in[2], in[3], 0x5140);
  const uint32_t c = __byte_perm(in[0], in[1], 0x7362), d = __byte_perm(in[2], in[3], 0x7362);
  out[0] = __byte_perm(a, b, 0x5410);
  out[1] = __byte_perm(a, b, 0x7632);
  out[2] = __byte_perm(c, d, 0x5410);
  out[3] = __byte_perm(c, d, 0x7632);
}

// Scale of a block whose largest magnitude has the 16-bit pattern m, and the factor that takes its numbers to codes.
template <typename T>
__device__ __forceinline__ float kv8_scale(uint32_t m, float &inv, float &pre) {
  constexpr uint32_t INF16 = __is_same(T, __half) ? 0x7c00u : 0x7f80u;
  pre = 1.0f;
  inv = 0.0f;
  if (m >= INF16) return __uint_as_float(0x7fc00000u);
  if (m == 0) return 1.0f;
  const uint16_t mb = static_cast<uint16_t>(m);
  const float top = to_f32<T>(*reinterpret_cast<const T *>(&mb));
  if (top < 0x1p-100f) pre = 0x1p100f;                  // keeps the reciprocal in range
  inv = __fdiv_rn(127.0f, top * pre) * (1.0f + 0x1p-21f);
  return __fdiv_rn(top, 127.0f);
}

__device__ __forceinline__ uint32_t max_abs16(uint32_t m, uint32_t w) { return __vmaxu2(m, w & 0x7fff7fffu); }

// Blocks of threads per multiprocessor: four (64 registers, which keeps 212 bytes a thread of the rotating half form in
// local memory, 12 of the plain one) hide more of the memory's latency than three (80 registers: 60 bytes and none).  Between
// events, from a cold L2, 8 heads: 4 x 4096 rotated tokens 30.7 against 34.8 us, as they are 26.6 against 30.7, 3 x 2000
// rotated 20.5 against 22.4.  The scalar forms have more state and take two.
template <int MODE>
constexpr int APPEND_BLOCKS = MODE == ROT_NONE || MODE == ROT_HALF || MODE == ROT_INTER ? 4 : 2;

// A block walks over the heads with the next head's loads in flight
// behind the current one's work.  Warps 0-3 take the keys, a token per four threads (both members of a pair in one
// thread, angles from the shared table); warps 4-7 the values, eight tokens a warp, four channels a thread, so that the
// tokens of a channel end up side by side in registers.
template <typename T, int MODE>
__global__ void __launch_bounds__(256, APPEND_BLOCKS<MODE>) kv8_append_kernel(const __grid_constant__ AppendArgs a) {
  using U = RotUnits<T, MODE>;
  constexpr bool HALF = MODE == ROT_HALF || MODE == ROT_HALF_SCALAR;
  __shared__ __align__(16) float4 tab[MODE == ROT_NONE ? 1 : 8 * 128];
  __shared__ __align__(16) uint8_t vt[KV8_OFF_V];
  __shared__ __align__(16) T stage[HALF ? KV8_BLOCK : 1][HD + 8];
  __shared__ uint32_t red[2][8];
  const kitty_kv8_layer &L = a.L;
  const int b = blockIdx.z, cap = L.max_page * PAGE;
  int n = a.counts != nullptr ? a.counts[b] : a.T;
  int s = a.start[b];
  bool bad = n < 0 || n > a.T || s < 0 || s > cap;
  n = min(max(n, 0), a.T);
  if (s < 0 || s > cap) s = 0, n = 0;
  if (n > cap - s) n = cap - s, bad = true;
  if (bad && threadIdx.x == 0) atomicOr(L.status, KITTY_KV8_BAD_LENGTH);
  const int end = s + n, fb = s / KV8_BLOCK, eb = end / KV8_BLOCK;
  const int h0 = blockIdx.y * a.heads, h1 = min(h0 + a.heads, L.h_kv);
  const int r = a.pl.rotary_dim, np = r / 2;
  const int half = threadIdx.x >> 7, tid = threadIdx.x & 127, warp = tid >> 5, lane = tid & 31;

  auto process = [&](int blk, bool kv, bool rows_q) {
    const int t0 = blk * KV8_BLOCK - s;                 // input index of the block's first token
    const bool full = blk < eb;
    const int64_t tail_row = static_cast<int64_t>(b) * L.h_kv * KV8_BLOCK * HD;
    // keys: thread t of token tk holds chunks of eight channels, chunk c from 16t + 8 (c & 1) + 64 (c >> 1)
    const int tk = tid >> 2, t = tid & 3, ik = t0 + tk;
    const bool fresh = ik >= 0 && ik < n, kept = ik < 0 && full;
    const bool whole = t0 >= 0 && t0 + KV8_BLOCK <= n;  // all tokens of the block come with the call
    auto channel = [&](int c) { return (c >> 1) * 64 + 16 * t + (c & 1) * 8; };
    T *tail_k = static_cast<T *>(L.tail_k) + tail_row + tk * HD;
    const T *in_k = static_cast<const T *>(a.k) + b * a.ks[0] + ik * a.ks[2] + 16 * t;
    auto fetch_k = [&](int h, uint4 (&w)[4]) {
      if (whole) {
        const T *src = in_k + h * a.ks[1];
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = *reinterpret_cast<const uint4 *>(src + (c >> 1) * 64 + (c & 1) * 8);
        return;
      }
      const T *src = fresh ? static_cast<const T *>(a.k) + b * a.ks[0] + h * a.ks[1] + ik * a.ks[2]
                           : tail_k + static_cast<int64_t>(h) * KV8_BLOCK * HD;
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] = fresh || kept ? *reinterpret_cast<const uint4 *>(src + channel(c)) : make_uint4(0, 0, 0, 0);
    };
    // values: a warp's lane holds four channels of eight tokens
    const int iv = t0 + 8 * warp;
    T *tail_v = static_cast<T *>(L.tail_v) + tail_row + 8 * warp * HD + 4 * lane;
    const T *in_v = static_cast<const T *>(a.v) + b * a.vs[0] + iv * a.vs[2] + 4 * lane;
    auto fetch_v = [&](int h, uint4 (&w)[4]) {
      const T *in = in_v + h * a.vs[1];
      uint2 z[8];
      if (whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = *reinterpret_cast<const uint2 *>(in + j * a.vs[2]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = iv + j;
          z[j] = make_uint2(0, 0);
          if (i >= 0 && i < n) z[j] = *reinterpret_cast<const uint2 *>(in + j * a.vs[2]);
          else if (i < 0 && full) z[j] = *reinterpret_cast<const uint2 *>(tail_v + (static_cast<int64_t>(h) * KV8_BLOCK + j) * HD);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] = make_uint4(z[2 * c].x, z[2 * c].y, z[2 * c + 1].x, z[2 * c + 1].y);
    };
    uint4 w[4];
    if (kv) {                                           // on their way while the angles are made
      if (half == 0) fetch_k(h0, w);
      else fetch_v(h0, w);
    }
    if constexpr (MODE != ROT_NONE) {
      // a thread makes the angles of one pair and eight tokens: one sine and cosine at a multiple of eight, and the steps
      static_assert(256 * ROT_STEPS == KV8_BLOCK * (HD / 2) && KV8_BLOCK % ROT_STEPS == 0);
      const int last = rows_q ? a.T : n, p = threadIdx.x % (HD / 2), tk = threadIdx.x / (HD / 2) * ROT_STEPS;
      if (p < np) {
        const double2 base = rot_base(a.pl, static_cast<int64_t>(blk) * KV8_BLOCK + tk, p);
#pragma unroll
        for (int i = 0; i < ROT_STEPS; ++i)
          if (t0 + tk + i >= 0 && t0 + tk + i < last)
            reinterpret_cast<float2 *>(tab)[2 * BlockTable<T, MODE>::word(p, tk + i) + (p & 1)] = rot_step(a.pl, base, i, p);
      }
      __syncthreads();
    }
    const int64_t page = kv && full ? kv8_page(L, b, blk) : -1;
    if (kv && half == 0) {
      const bool turn = MODE != ROT_NONE && fresh;
      const BlockTable<T, MODE> table{tab, tk};
      for (int h = h0; h < h1; ++h) {
        uint4 nx[4];
        if (h + 1 < h1) fetch_k(h + 1, nx);
        if constexpr (MODE != ROT_NONE) {
          if (HALF && r != HD) {                // a pair's members are in two threads of the token's four
#pragma unroll
            for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4 *>(&stage[tk][channel(c)]) = w[c];
            __syncwarp();
            if (turn) {
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const int d = channel(c);
                if (d >= r) continue;
                Piece<T> x;
                x.unpack(w[c]);
                if constexpr (MODE == ROT_HALF) {       // whole chunks on either side
                  Piece<T> y;
                  y.unpack(*reinterpret_cast<const uint4 *>(&stage[tk][d < np ? d + np : d - np]));
                  const float sg = d < np ? -1.0f : 1.0f;
                  const int p = d < np ? d : d - np;
#pragma unroll
                  for (int e = 0; e < 8; e += 2) {
                    const float4 z = table.pairs(p + e);
                    x.f[e] = fmaf(x.f[e], z.x, sg * (y.f[e] * z.y));
                    x.f[e + 1] = fmaf(x.f[e + 1], z.z, sg * (y.f[e + 1] * z.w));
                  }
                } else {
#pragma unroll
                  for (int e = 0; e < 8; ++e)
                    if (d + e < r) {
                      const bool first = d + e < np;
                      const float2 z = table.one(first ? d + e : d + e - np);
                      const float o = to_f32<T>(stage[tk][first ? d + e + np : d + e - np]);
                      x.f[e] = fmaf(x.f[e], z.x, first ? -o * z.y : o * z.y);
                    }
                }
                w[c] = x.pack();
              }
            }
            __syncwarp();
          } else if (turn) {
#pragma unroll
            for (int c = 0; c < (HALF ? 2 : 4); ++c) {
              Piece<T> x;
              x.unpack(w[c]);
              if constexpr (HALF) {             // channels 16t + e and 64 + 16t + e: both here
                Piece<T> y;
                y.unpack(w[c + 2]);
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                  const float4 z = table.pairs(16 * t + 8 * c + e);
                  const float x0 = x.f[e], y0 = y.f[e], x1 = x.f[e + 1], y1 = y.f[e + 1];
                  x.f[e] = fmaf(x0, z.x, -y0 * z.y);
                  y.f[e] = fmaf(y0, z.x, x0 * z.y);
                  x.f[e + 1] = fmaf(x1, z.z, -y1 * z.w);
                  y.f[e + 1] = fmaf(y1, z.z, x1 * z.w);
                }
                w[c + 2] = y.pack();
              } else {
                const int p = channel(c) / 2;
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                  const float4 z = table.pairs(p + e);
                  const float x0 = x.f[2 * e], x1 = x.f[2 * e + 1], x2 = x.f[2 * e + 2], x3 = x.f[2 * e + 3];
                  if (p + e < np) {             // an untouched pair may hold infinities
                    x.f[2 * e] = fmaf(x0, z.x, -x1 * z.y);
                    x.f[2 * e + 1] = fmaf(x1, z.x, x0 * z.y);
                  }
                  if (p + e + 1 < np) {
                    x.f[2 * e + 2] = fmaf(x2, z.z, -x3 * z.w);
                    x.f[2 * e + 3] = fmaf(x3, z.z, x2 * z.w);
                  }
                }
              }
              w[c] = x.pack();
            }
          }
        }
        if (!full) {
          if (fresh) {
            T *o = tail_k + static_cast<int64_t>(h) * KV8_BLOCK * HD;
#pragma unroll
            for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4 *>(o + channel(c)) = w[c];
          }
        } else {
          // largest magnitude of the block: 16-bit patterns without the sign order like the numbers
          uint32_t m = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) m = max_abs16(max_abs16(max_abs16(max_abs16(m, w[c].x), w[c].y), w[c].z), w[c].w);
          m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
          if (lane == 0) red[h & 1][warp] = m;
          half_barrier(0);
          m = max(max(red[h & 1][0], red[h & 1][1]), max(red[h & 1][2], red[h & 1][3]));
          float inv, pre;
          const float scale = kv8_scale<T>(m, inv, pre);
          if (page >= 0) {
            uint8_t *rec = kv8_record(L, page, h, blk & 3);
            if (tid == 0) *reinterpret_cast<float *>(rec + KV8_OFF_SCALE) = scale;
            uint8_t *o = rec + ((tk >> 1) & 3) * 1024 + (4 * (2 * (tk >> 3) + (tk & 1)) + t) * 16;
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              uint32_t code[4];
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                Piece<T> x;
                x.unpack(w[c + y]);
                if (pre != 1.0f) {
#pragma unroll
                  for (int e = 0; e < 8; ++e) x.f[e] *= pre;
                }
                code[2 * y] = kv8_codes4(x.f, inv);
                code[2 * y + 1] = kv8_codes4(x.f + 4, inv);
              }
              *reinterpret_cast<uint4 *>(o + (c >> 1) * 512) = make_uint4(code[0], code[1], code[2], code[3]);
            }
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = nx[c];
      }
    } else if (kv) {
      for (int h = h0; h < h1; ++h) {
        uint4 nx[4];
        if (h + 1 < h1) fetch_v(h + 1, nx);
        if (!full) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint4 z = w[j >> 1];
            if (iv + j >= 0 && iv + j < n)
              *reinterpret_cast<uint2 *>(tail_v + (static_cast<int64_t>(h) * KV8_BLOCK + j) * HD) = j & 1 ? make_uint2(z.z, z.w) : make_uint2(z.x, z.y);
          }
        } else {
          uint32_t m = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) m = max_abs16(max_abs16(max_abs16(max_abs16(m, w[c].x), w[c].y), w[c].z), w[c].w);
          m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
          if (lane == 0) red[h & 1][4 + warp] = m;
          half_barrier(1);
          m = max(max(red[h & 1][4], red[h & 1][5]), max(red[h & 1][6], red[h & 1][7]));
          float inv, pre;
          const float scale = kv8_scale<T>(m, inv, pre);
          uint32_t out[2][4];                   // [tokens 4y .. 4y + 3][channel 4 lane + j]
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t code[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint4 q4 = w[2 * y + (j >> 1)];
              const uint2 z = j & 1 ? make_uint2(q4.z, q4.w) : make_uint2(q4.x, q4.y);
              T v4[4];
              memcpy(v4, &z, 8);
              float x[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = to_f32<T>(v4[e]);
              if (pre != 1.0f) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] *= pre;
              }
              code[j] = kv8_codes4(x, inv);
            }
            transpose4(code, out[y]);
          }
          // channel c: piece row c / 16, half (c / 8) % 2, lane 4 (c % 8) + the tokens' eight (the warp); the lane's place in
          // its row is turned by the row, so that the eight rows a warp writes to fall on different banks
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = 4 * lane + j;
            *reinterpret_cast<uint2 *>(vt + (c >> 4) * 512 + ((4 * (c & 7) + warp) ^ (c >> 4)) * 16 + ((c >> 3) & 1) * 8) = make_uint2(out[0][j], out[1][j]);
          }
          half_barrier(1);
          if (page >= 0) {
            uint8_t *rec = kv8_record(L, page, h, blk & 3);
            if (tid == 0) *reinterpret_cast<float *>(rec + KV8_OFF_SCALE + 4) = scale;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int p = tid + 128 * j;
              *reinterpret_cast<uint4 *>(rec + KV8_OFF_V + p * 16) = *reinterpret_cast<const uint4 *>(vt + (p ^ (p >> 5)) * 16);
            }
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = nx[c];
      }
    }
    if constexpr (MODE != ROT_NONE) {
      if (rows_q) {
        constexpr int LPR = U::VEC ? (MODE == ROT_HALF ? 8 : 16) : 32, ROWS = 4;
        const int q0 = static_cast<int>(static_cast<int64_t>(a.h_q) * blockIdx.y / gridDim.y);
        const int q1 = static_cast<int>(static_cast<int64_t>(a.h_q) * (blockIdx.y + 1) / gridDim.y);
        const int first = max(0, -t0), toks = min(KV8_BLOCK, a.T - t0) - first, nh = q1 - q0;
        const int nu = U::turned(r) + U::copied(r);
        constexpr int STEP = 256 / LPR;
        for (int base = threadIdx.x / LPR; base < toks * nh; base += STEP * ROWS)
          for (int u = threadIdx.x % LPR; u < nu; u += LPR) {
            RotUnit<T, MODE> x[ROWS];
#pragma unroll
            for (int j = 0; j < ROWS; ++j) {
              const int row = base + j * STEP, tk = first + row / nh, h = q0 + row % nh;
              if (row < toks * nh)
                x[j].load(static_cast<const T *>(a.q) + b * a.qs[0] + h * a.qs[1] + (t0 + tk) * a.qs[2], u, r);
            }
#pragma unroll
            for (int j = 0; j < ROWS; ++j) {
              const int row = base + j * STEP, tk = first + row / nh, h = q0 + row % nh;
              if (row < toks * nh)
                x[j].store(static_cast<T *>(a.q_out) + ((static_cast<int64_t>(b) * a.h_q + h) * a.T + t0 + tk) * HD, u, r,
                           BlockTable<T, MODE>{tab, tk});
            }
          }
      }
    }
    __syncthreads();
  };

  const int blk = fb + blockIdx.x;               // start and T may be 2^30 each: the token behind the block can pass 2^31
  const bool kv = n > 0 && (blk < eb || (blockIdx.x == 0 && eb == fb));
  const bool rows_q = MODE != ROT_NONE && a.h_q > 0 && static_cast<int>(blockIdx.x) * KV8_BLOCK - s % KV8_BLOCK < a.T;
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

// Sixteen codes -> 16-bit values.  A code + 128 in the low byte of 2^23 is a float that is 2^23 + 128 too large: a byte
// shuffle and an exact subtraction in place of the conversion unit, which makes sixteen a clock.
template <typename T>
__device__ __forceinline__ void expand16(uint4 codes, float scale, uint4 (&out)[2]) {
  const uint32_t w[4] = {codes.x ^ 0x80808080u, codes.y ^ 0x80808080u, codes.z ^ 0x80808080u, codes.w ^ 0x80808080u};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    Piece<T> p;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      p.f[e] = (__uint_as_float(__byte_perm(w[2 * c + (e >> 2)], 0x4b000000u, 0x7440 | (e & 3))) - 8388736.0f) * scale;
    out[c] = p.pack();
  }
}

// A block of threads per (block of tokens, head); values first, whose way through shared memory is the longer one.
// Two or four heads a block, their records in flight together, took 17.5 and 19.2 us where this takes 16.8 (4 x 4096 tokens,
// 8 heads; 15.4 at the copy bandwidth).
template <typename T>
__global__ void __launch_bounds__(256) kv8_expand_kernel(const __grid_constant__ ExpandArgs a) {
  // rows of 148 bytes: eight rows on is eight banks on, so the four token groups of a warp write to different banks
  __shared__ __align__(16) uint8_t vt[KV8_BLOCK][HD + 20];
  const kitty_kv8_layer &L = a.L;
  const int b = blockIdx.z, h = blockIdx.y, cap = L.max_page * PAGE;
  const int len = kv8_clamp_len(L, a.lengths[b]);
  int s = a.start != nullptr ? a.start[b] : 0;
  if (s < 0 || s > cap) {
    atomicOr(L.status, KITTY_KV8_BAD_LENGTH);
    s = cap;                                            // nothing held there: zeros
  }
  const int blk = s / KV8_BLOCK + blockIdx.x;
  const int t0 = static_cast<int>(blockIdx.x) * KV8_BLOCK - s % KV8_BLOCK;     // output index of the block's first token
  if (t0 >= a.n) return;
  const bool full = blk < len / KV8_BLOCK;
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
  const int tk = threadIdx.x >> 3, c = (threadIdx.x & 7) * 16;
  uint4 x[2] = {};
  if (full && page >= 0) {
    const uint8_t *rec = kv8_record(L, page, h, blk & 3);
    const uint4 vc = *reinterpret_cast<const uint4 *>(rec + KV8_OFF_V + threadIdx.x * 16);
    const uint4 kc = *reinterpret_cast<const uint4 *>(rec + threadIdx.x * 16);
    const float2 sc = *reinterpret_cast<const float2 *>(rec + KV8_OFF_SCALE);
    const int g = (threadIdx.x >> 2) & 7, t = threadIdx.x & 3, ch = 16 * (threadIdx.x >> 5) + g;
    const uint32_t w[4] = {vc.x, vc.y, vc.z, vc.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      vt[8 * t + e][ch] = static_cast<uint8_t>(w[e >> 2] >> (8 * (e & 3)));
      vt[8 * t + e][ch + 8] = static_cast<uint8_t>(w[2 + (e >> 2)] >> (8 * (e & 3)));
    }
    expand16<T>(kc, sc.x, x);
    put(ko, kv8_key_token(threadIdx.x >> 6, g), ((threadIdx.x >> 5) & 1) * 64 + 16 * t, x);
    __syncthreads();
    const uint32_t *vw = reinterpret_cast<const uint32_t *>(&vt[tk][c]);
    expand16<T>(make_uint4(vw[0], vw[1], vw[2], vw[3]), sc.y, x);
    put(vo, tk, c, x);
  } else {
    const bool held = !full && blk == len / KV8_BLOCK && tk < len % KV8_BLOCK;      // an open block's token; a skipped page gives zeros
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
  if (h_q > 0) {
    constexpr int64_t ROW = HD * 2;
    const Rows turned{q_out, {B, h_q, T}, {h_q * T * ROW, T * ROW, ROW}, ROW};
    const void *in[3] = {key, value, query};
    for (int x = 0; x < 3; ++x) {
      const int64_t *st = strides + 3 * x;
      const Rows read{in[x], {B, x < 2 ? layer->h_kv : h_q, T}, {st[0] * 2, st[1] * 2, st[2] * 2}, ROW};
      if (!(x == 2 && same_rows(turned, read)) && rows_meet(turned, read)) return KITTY_E_OVERLAP;
    }
  }
  a.start = start;
  a.counts = counts;
  a.T = T;
  a.h_q = h_q;
  const int64_t blocks = (static_cast<int64_t>(T) + 2 * KV8_BLOCK - 2) / KV8_BLOCK;   // that T tokens can touch
  if (B > 65535 || T > (1 << 30)) return KITTY_E_BADSHAPE;
  // Heads are spread over blocks of threads until there are three per multiprocessor; the rest share an angle table.
  // From a cold L2, in us, by the blocks asked for per multiprocessor (8 heads; q: with 32 query heads):
  //                    1     2     3     4
  //   4 x 4096        27.8  27.9  27.9  29.8
  //   3 x 2000        26.0  20.8  19.5  22.4
  //   16 x 512, q     56.0  47.2  47.3  60.5
  //   1 x 4096, q     33.5  32.4  30.0  30.0
  // (taken with a slower way to the angles, 26.9 in place of 27.9 since.)
  int64_t split = (3 * static_cast<int64_t>(sm_count()) + blocks * B - 1) / (blocks * B);
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
  const int64_t bytes = static_cast<int64_t>(B) * layer->h_kv * n * HD * 2;
  if (rows_meet({k_out, {1, 1, 1}, {}, bytes}, {v_out, {1, 1, 1}, {}, bytes})) return KITTY_E_OVERLAP;
  ExpandArgs a{*layer, lengths, start, k_out, v_out, n};
  const int64_t blocks = (static_cast<int64_t>(n) + 2 * KV8_BLOCK - 2) / KV8_BLOCK;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(layer->h_kv), static_cast<unsigned>(B));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (layer->dtype == KITTY_F16) kv8_expand_kernel<__half><<<grid, 256, 0, s>>>(a);
  else kv8_expand_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? KITTY_OK : KITTY_E_CUDA;
}
