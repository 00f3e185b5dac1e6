// Attention over a whole prompt on the tcgen05 tensor cores: causal or full, grouped heads, dense or packed sequences.
//
//   o_i = sum_j softmax_j(scaling * q_i . k_j) v_j,   j < min(keys, i + 1 + keys - queries)
//
// Bound by the tensor cores (4 * 128 operations per visible pair and query head) and, on the same scale, by the 16
// exponentials a multiprocessor makes per clock: a 128 x 128 tile costs 1024 clocks of either.  One block of threads
// per multiprocessor works on TWO query tiles of 128 rows that share the key head's keys and values, so that the tensor
// cores multiply for one while the other takes its exponentials.  The (row tile, head) pairs of a key head are numbered
// row tile first: the two tiles of a block are neighbouring heads of the same rows (or neighbouring rows), see nearly
// the same keys, and read every key and value tile once.
//
//   warps 0-3, 4-7   softmax of tile A / B: thread = row.  Logits come from tensor memory, the weights go back to the
//                    same columns as 16-bit numbers, as the left operand of the second product.
//   warp 8           tiled bulk copies: both query tiles, then key and value tiles through a ring of 32 KB stages
//   warp 9           issues the products; tensor memory: logits A, B and accumulators A, B, 128 columns each
//
// The running maximum is kept in the logits' own units and allowed to lag: the accumulator is rescaled only when a row's
// maximum has grown by more than 2^8, by the softmax threads themselves (the product before is complete by then: the
// commit that announces new logits also covers it).  Weights up to 256 fit the 16-bit types, sums are 32-bit.
// Weights are rounded to the inputs' type for the second product (half a step, 2^-9 for bf16, of independent sign, as
// large as the rounding of the output itself).
//
// Keys that a row does not see: their logits are replaced before the maximum is taken, so keys may hold anything.  Their
// values enter the product with weight zero, and zero times infinity or NaN is NaN: a row that ends up with a value that
// is not finite is looked at again, and computed without the matrix units if one of its unseen values is the cause.
#include <cuda.h>

#include "decode.cuh"
#include "tcgen05.cuh"

namespace kitty {

constexpr int PT = 128;                        // rows of a query tile, keys of a key tile
constexpr int TILE_BYTES = PT * HD * 2;        // 32 KB
constexpr int KV_STAGES = 5;
constexpr int PROMPT_SMEM = (2 + KV_STAGES) * TILE_BYTES + 1024;
constexpr int PROMPT_THREADS = 384;            // three groups of four warps; warps 10 and 11 only hand over registers
constexpr float LAG = 8.0f;                    // log2 of how far a maximum may lag

struct PromptArgs {
  const void *q, *k, *v;
  void *out;
  int64_t qs[3], ks[3], vs[3];                 // element strides (batch, head, token)
  const int32_t *q_lens, *k_lens, *cu_q, *cu_k;
  int32_t *status;
  int32_t B, Lq, Lk, G, h_kv, pairs, causal, zero_rest;
  float c;                                     // scaling * log2 e
};

struct Seq {
  int b;              // batch coordinate
  int q0, nq, k0, nk; // first row and rows of its queries and keys
  int rows;           // rows of the output it owns (nq, or Lq for a padded row of a batch)
  int64_t out0;       // its first output row
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// Keys that row i of a sequence sees.
__device__ __forceinline__ int key_limit(const Seq &s, int i, int causal) {
  if (i >= s.nq) return 0;
  return causal ? clampi(i + 1 + s.nk - s.nq, 0, s.nk) : s.nk;
}

// One row again, by one warp, without the matrix units: only keys that the row sees are touched.
template <typename T>
__device__ __noinline__ void repair_row(const PromptArgs &a, const Seq &s, int row, int head, int limit, int touched) {
  const int lane = threadIdx.x & 31;
  const int hk = head / a.G;
  const T *k = static_cast<const T *>(a.k) + s.b * a.ks[0] + hk * a.ks[1] + s.k0 * a.ks[2] + 4 * lane;
  const T *v = static_cast<const T *>(a.v) + s.b * a.vs[0] + hk * a.vs[1] + s.k0 * a.vs[2] + 4 * lane;
  auto load4 = [](const T *p, float (&x)[4]) {
    T t[4];
    *reinterpret_cast<uint2 *>(t) = *reinterpret_cast<const uint2 *>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = to_f32<T>(t[e]);
  };
  bool cause = false;
  float x[4];
  for (int j = limit; j < touched; ++j) {
    load4(v + j * a.vs[2], x);
#pragma unroll
    for (int e = 0; e < 4; ++e) cause |= !(fabsf(x[e]) < INFINITY);
  }
  if (!__any_sync(0xffffffffu, cause)) return;
  float q[4], acc[4] = {}, m = -INFINITY, l = 0.0f;
  load4(static_cast<const T *>(a.q) + s.b * a.qs[0] + head * a.qs[1] + (static_cast<int64_t>(s.q0) + row) * a.qs[2] + 4 * lane, q);
  for (int j = 0; j < limit; ++j) {
    load4(k + j * a.ks[2], x);
    float d = q[0] * x[0] + q[1] * x[1] + q[2] * x[2] + q[3] * x[3];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    d *= a.c;
    const float mn = fmaxf(m, d), ref = mn == -INFINITY ? 0.0f : mn;
    const float f = ex2(m - ref), p = ex2(d - ref);
    load4(v + j * a.vs[2], x);
    l = l * f + p;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = acc[e] * f + p * x[e];
    m = mn;
  }
  T o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(acc[e] / l);
  T *dst = static_cast<T *>(a.out) + ((s.out0 + row) * static_cast<int64_t>(a.G) * a.h_kv + head) * HD + 4 * lane;
  *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(o);
}

template <typename T>
__global__ void __launch_bounds__(PROMPT_THREADS, 1)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                       const __grid_constant__ CUtensorMap mv, const __grid_constant__ PromptArgs a) {
  constexpr bool BF16 = __is_same(T, __nv_bfloat16);
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_q, bar_full[KV_STAGES], bar_empty[KV_STAGES], bar_s[2], bar_p[2], bar_o[2], bar_end;
  __shared__ uint32_t tmem_base;
  __shared__ int item_seq, item_pair;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;

  // ---- which sequence, key head and pair of tiles
  Seq s;
  int h, pair;
  if (a.cu_q == nullptr) {
    const int sh = blockIdx.x % (a.B * a.h_kv);
    pair = a.pairs - 1 - blockIdx.x / (a.B * a.h_kv);      // the longest rows first
    s.b = sh / a.h_kv;
    h = sh % a.h_kv;
    s.q0 = s.k0 = 0;
    s.nq = a.q_lens != nullptr ? clampi(a.q_lens[s.b], 0, a.Lq) : a.Lq;
    s.nk = a.k_lens != nullptr ? clampi(a.k_lens[s.b], 0, a.Lk) : a.Lk;
    s.rows = a.Lq;
    s.out0 = static_cast<int64_t>(s.b) * a.Lq;
  } else {
    h = blockIdx.x % a.h_kv;
    const int want = blockIdx.x / a.h_kv;
    if (warp == 0) {
      const int nseq = a.B + (a.zero_rest ? 1 : 0);
      int base = 0, found = -1, fp = 0;
      for (int i0 = 0; i0 < nseq && found < 0; i0 += 32) {
        const int i = i0 + lane;
        int np = 0;
        if (i < nseq) {
          const int lo = clampi(a.cu_q[i], 0, a.Lq), hi = i < a.B ? clampi(a.cu_q[i + 1], lo, a.Lq) : a.Lq;
          np = ((hi - lo + PT - 1) / PT * a.G + 1) / 2;
        }
        int inc = np;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int t = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, want < base + inc);
        if (hit) {
          const int l = __ffs(hit) - 1;
          const int upto = __shfl_sync(0xffffffffu, inc, l), n1 = __shfl_sync(0xffffffffu, np, l);
          found = i0 + l;
          fp = n1 - 1 - (want - (base + upto - n1));       // the longest rows first
        }
        base += __shfl_sync(0xffffffffu, inc, 31);
      }
      if (lane == 0) item_seq = found, item_pair = fp;
    }
    __syncthreads();
    const int i = item_seq;
    if (i < 0) return;                                      // the grid covers the most that Lq rows can need
    pair = item_pair;
    s.b = 0;
    s.q0 = clampi(a.cu_q[i], 0, a.Lq);
    s.nq = (i < a.B ? clampi(a.cu_q[i + 1], s.q0, a.Lq) : a.Lq) - s.q0;
    s.k0 = s.nk = 0;
    if (i < a.B) {
      const int32_t *cu = a.cu_k != nullptr ? a.cu_k : a.cu_q;
      s.k0 = clampi(cu[i], 0, a.Lk);
      s.nk = clampi(cu[i + 1], s.k0, a.Lk) - s.k0;
    }
    s.rows = s.nq;
    s.out0 = s.q0;
  }
  const int tiles = (s.rows + PT - 1) / PT * a.G;           // (row tile, head) pairs of the key head
  int row0[2], head[2], nblk[2];
  bool live[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int f = 2 * pair + x;
    live[x] = f < tiles;
    row0[x] = f / a.G * PT;
    head[x] = h * a.G + f % a.G;
    const int last = min(row0[x] + PT, s.nq) - 1;
    nblk[x] = live[x] && last >= row0[x] ? (key_limit(s, last, a.causal) + PT - 1) / PT : 0;
  }
  const int n = max(nblk[0], nblk[1]);

  if (n > 0) {
    if (warp == 9) tmem_alloc(smem_u32(&tmem_base), 512);
    if (threadIdx.x == 0) {
      mbar_init(smem_u32(&bar_q), 1);
      for (int i = 0; i < KV_STAGES; ++i) mbar_init(smem_u32(&bar_full[i]), 1), mbar_init(smem_u32(&bar_empty[i]), 1);
      for (int x = 0; x < 2; ++x) mbar_init(smem_u32(&bar_s[x]), 1), mbar_init(smem_u32(&bar_p[x]), PT), mbar_init(smem_u32(&bar_o[x]), 1);
      mbar_init(smem_u32(&bar_end), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  const uint32_t tmem = n > 0 ? tmem_base : 0;
  const uint32_t q_addr = smem, kv_addr = smem + 2 * TILE_BYTES;
  auto give_up = [&] {
    if (a.status != nullptr) atomicExch(a.status, 1);
  };

  // 384 threads start with 168 registers; the softmax threads take what the other group gives up (2 * 232 + 40 = 3 * 168)
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 8) {
      if (lane == 0 && n > 0) {
        const uint32_t bq = smem_u32(&bar_q);
        mbar_expect_tx(bq, (nblk[0] > 0 ? TILE_BYTES : 0) + (nblk[1] > 0 ? TILE_BYTES : 0));
        for (int x = 0; x < 2; ++x)
          if (nblk[x] > 0)
            for (int c = 0; c < 2; ++c)
              tma_load_4d(q_addr + x * TILE_BYTES + c * (TILE_BYTES / 2), &mq, bq, 64 * c, s.q0 + row0[x], head[x], s.b);
        int i = 0;
        bool ok = true;
        for (; i < 2 * n; ++i) {
          const int st = i % KV_STAGES, round = i / KV_STAGES;
          if (round > 0 && !mbar_wait(smem_u32(&bar_empty[st]), (round - 1) & 1)) {
            give_up();
            ok = false;
            break;
          }
          const uint32_t bf = smem_u32(&bar_full[st]);
          mbar_expect_tx(bf, TILE_BYTES);
          const CUtensorMap *m = (i & 1) ? &mv : &mk;
          for (int c = 0; c < 2; ++c)
            tma_load_4d(kv_addr + st * TILE_BYTES + c * (TILE_BYTES / 2), m, bf, 64 * c, s.k0 + (i >> 1) * PT, h, s.b);
        }
        if (!ok)                                              // leave no copy in flight behind
          for (int j = max(0, i - KV_STAGES); j < i; ++j) mbar_wait(smem_u32(&bar_full[j % KV_STAGES]), (j / KV_STAGES) & 1);
      }
    } else if (warp == 9) {
      if (lane == 0 && n > 0) {
        constexpr uint32_t ID_S = umma_idesc(BF16, PT, PT, false), ID_O = umma_idesc(BF16, PT, HD, true);
        bool ok = true;
        auto wait = [&](uint64_t &bar, int phase) {
          if (ok && !mbar_wait(smem_u32(&bar), phase & 1)) {
            ok = false;
            give_up();
          }
          tc_fence_after();
          return ok;
        };
        // logits of tile x against key tile j: contraction over 128 channels, 16 at a time, two swizzled halves
        auto logits = [&](int x, int j) {
          const uint32_t qa = umma_lo(q_addr + x * TILE_BYTES, 16);
          const uint32_t ka = umma_lo(kv_addr + (2 * j % KV_STAGES) * TILE_BYTES, 16);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t off = ((kk >> 2) * (TILE_BYTES / 2) + (kk & 3) * 32) >> 4;
            umma_ss(tmem + x * PT, qa + off, umma_hi(1024), ka + off, umma_hi(1024), ID_S, kk > 0);
          }
          umma_commit(smem_u32(&bar_s[x]));
        };
        // accumulator of tile x += weights x value tile j: contraction over 128 keys, 16 at a time
        auto values = [&](int x, int j) {
          const uint32_t va = umma_lo(kv_addr + ((2 * j + 1) % KV_STAGES) * TILE_BYTES, TILE_BYTES / 2);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ts(tmem + 2 * PT + x * HD, tmem + x * PT + kk * 8, va + (kk * 2048 >> 4), umma_hi(1024), ID_O, j > 0 || kk > 0);
          if (j + 1 == (x ? nblk[1] : nblk[0])) umma_commit(smem_u32(&bar_o[x]));
        };
        wait(bar_q, 0);
        if (wait(bar_full[0], 0)) {
#pragma unroll 1
          for (int x = 0; x < 2; ++x)
            if ((x ? nblk[1] : nblk[0]) > 0) logits(x, 0);
          umma_commit(smem_u32(&bar_empty[0]));
        }
        for (int j = 0; j < n && ok; ++j) {
          const int sv = (2 * j + 1) % KV_STAGES, sk = (2 * j + 2) % KV_STAGES;
          if (!wait(bar_full[sv], (2 * j + 1) / KV_STAGES)) break;
#pragma unroll 1
          for (int x = 0; x < 2 && ok; ++x) {
            const int nb = x ? nblk[1] : nblk[0];
            if (j < nb) {
              if (!wait(bar_p[x], j)) break;
              values(x, j);
            }
            if (x == 1) umma_commit(smem_u32(&bar_empty[sv]));
            if (j + 1 < n) {
              if (x == 0 && !wait(bar_full[sk], (2 * j + 2) / KV_STAGES)) break;
              if (j + 1 < nb) logits(x, j + 1);
              if (x == 1) umma_commit(smem_u32(&bar_empty[sk]));
            }
          }
        }
        // every product is complete before the tensor memory is given back
        umma_commit(smem_u32(&bar_end));
        mbar_wait(smem_u32(&bar_end), 0);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int x = warp >> 2;
    const uint32_t at = tmem + (static_cast<uint32_t>(warp & 3) << 21);     // the warp's 32 lanes
    const uint32_t ts = at + x * PT, to = at + 2 * PT + x * HD;
    const int row = row0[x] + (threadIdx.x & 127);
    const int limit = key_limit(s, row, a.causal);
    const int nb = nblk[x];
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    // keys that every row of the tile sees need no comparison
    const int all = key_limit(s, min(row0[x], s.nq - 1), a.causal);
    for (int j = 0; j < nb; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_s[x]), j & 1));
      if (!ok) break;
      tc_fence_after();
      float v[PT];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld32(ts + 32 * i, v + 32 * i);
      tmem_wait_ld();
      if ((j + 1) * PT > all) {
        const int seen = limit - j * PT;
#pragma unroll
        for (int i = 0; i < PT; ++i) v[i] = i < seen ? v[i] : -INFINITY;
      }
      float t0 = -INFINITY, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
#pragma unroll
      for (int i = 0; i < PT; i += 8) {
        t0 = fmaxf(t0, fmaxf(v[i], v[i + 1]));
        t1 = fmaxf(t1, fmaxf(v[i + 2], v[i + 3]));
        t2 = fmaxf(t2, fmaxf(v[i + 4], v[i + 5]));
        t3 = fmaxf(t3, fmaxf(v[i + 6], v[i + 7]));
      }
      const float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
      const bool grow = (top - m) * a.c > LAG || m == -INFINITY;
      if (j == 0) {
        m = top;
      } else if (__any_sync(0xffffffffu, grow)) {
        const float mn = grow ? fmaxf(m, top) : m;
        const float f = grow ? ex2((m - (mn == -INFINITY ? 0.0f : mn)) * a.c) : 1.0f;
        m = mn;
        l *= f;
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          float o[32];
          tmem_ld32(to + 32 * i, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= f;
          tmem_st32(to + 32 * i, reinterpret_cast<const uint32_t *>(o));
        }
      }
      const float mc = m == -INFINITY ? 0.0f : m * a.c;
      float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const int e = 64 * half + 2 * i;
          const float p0 = ex2(fmaf(v[e], a.c, -mc)), p1 = ex2(fmaf(v[e + 1], a.c, -mc));
          const float p2 = ex2(fmaf(v[e + 2], a.c, -mc)), p3 = ex2(fmaf(v[e + 3], a.c, -mc));
          s0 += p0;
          s1 += p1;
          s2 += p2;
          s3 += p3;
          if constexpr (BF16) {
            __nv_bfloat162 x0 = __floats2bfloat162_rn(p0, p1), x1 = __floats2bfloat162_rn(p2, p3);
            w[i] = *reinterpret_cast<uint32_t *>(&x0);
            w[i + 1] = *reinterpret_cast<uint32_t *>(&x1);
          } else {
            w[i] = pack_h2(p0, p1);
            w[i + 1] = pack_h2(p2, p3);
          }
        }
        tmem_st32(ts + 32 * half, w);
      }
      l += (s0 + s1) + (s2 + s3);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(smem_u32(&bar_p[x]));
    }
    if (nb > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_o[x]), 0));
    if (!ok) give_up();
    if (live[x] && ok) {
      tc_fence_after();
      const bool mine = row < s.rows;
      const float inv = limit > 0 ? 1.0f / l : 0.0f;
      T *dst = static_cast<T *>(a.out) + ((s.out0 + row) * static_cast<int64_t>(a.G) * a.h_kv + head[x]) * HD;
      bool odd = false;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        float o[32];
        if (nb > 0) {
          tmem_ld32(to + 32 * i, o);
          tmem_wait_ld();
        }
        uint4 w[4];
        T *t = reinterpret_cast<T *>(w);
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float y = limit > 0 ? o[e] * inv : 0.0f;
          odd |= !(fabsf(y) < INFINITY);
          t[e] = from_f32<T>(y);
        }
        if (mine) {
#pragma unroll
          for (int e = 0; e < 4; ++e) reinterpret_cast<uint4 *>(dst + 32 * i)[e] = w[e];
        }
      }
      unsigned again = __ballot_sync(0xffffffffu, odd && mine);
      while (again) {
        const int r = __ffs(again) - 1;
        again &= again - 1;
        const int touched = min(nb * PT, a.Lk - s.k0);
        repair_row<T>(a, s, __shfl_sync(0xffffffffu, row, r), head[x], __shfl_sync(0xffffffffu, limit, r), touched);
      }
    }
    tc_fence_before();
  }
  if (n > 0) {
    __syncthreads();
    __syncwarp();
    tc_fence_after();
    if (warp == 9) tmem_free(tmem, 512);
  }
}

// Token rows of one head as boxes of 128 rows x 64 channels in the 128-byte swizzle; what lies outside reads as zero.
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static std::atomic<EncodeTiled> known{nullptr};
  EncodeTiled f = known.load(std::memory_order_acquire);
  if (f == nullptr) {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess)
      return nullptr;
    f = reinterpret_cast<EncodeTiled>(p);
    known.store(f, std::memory_order_release);
  }
  return f;
}

bool make_map(CUtensorMap *m, const void *base, bool bf16, int64_t T, int64_t H, int64_t B, const int64_t *st) {
  EncodeTiled enc = encode_tiled();
  if (enc == nullptr) return false;
  const cuuint64_t dims[4] = {HD, static_cast<cuuint64_t>(T), static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(B)};
  // a dimension of size one is never stepped along: any legal stride will do
  const cuuint64_t str[3] = {T > 1 ? static_cast<cuuint64_t>(st[2]) * 2 : 2 * HD, H > 1 ? static_cast<cuuint64_t>(st[1]) * 2 : 2 * HD,
                             B > 1 ? static_cast<cuuint64_t>(st[0]) * 2 : 2 * HD};
  const cuuint32_t box[4] = {64, PT, 1, 1}, es[4] = {1, 1, 1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(base),
             dims, str, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
int launch_prompt(const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, const PromptArgs &a, unsigned grid,
                  cudaStream_t s) {
  static PerDeviceOnce once;
  const int rc = per_device_once(once, [] {
    return cudaFuncSetAttribute(prompt_attn_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, PROMPT_SMEM) == cudaSuccess
               ? KITTY_OK
               : KITTY_E_CUDA;
  });
  if (rc != KITTY_OK) return rc;
  prompt_attn_kernel<T><<<grid, PROMPT_THREADS, PROMPT_SMEM, s>>>(mq, mk, mv, a);
  return cudaGetLastError() == cudaSuccess ? KITTY_OK : KITTY_E_CUDA;
}

}  // namespace kitty

using namespace kitty;

extern "C" int kitty_prompt_attn(const void *q, const void *k, const void *v, int dtype, const int64_t *strides,
                                 int32_t B, int64_t Lq, int64_t Lk, int32_t h_q, int32_t h_kv, float scaling,
                                 int causal, const int32_t *q_lens, const int32_t *k_lens, const int32_t *cu_q,
                                 const int32_t *cu_k, void *out, int zero_rest, int32_t *status, void *stream) {
  if (!strides || B < 0 || Lq < 0 || Lk < 0 || h_q <= 0 || h_kv <= 0 || h_q % h_kv != 0) return KITTY_E_BADARG;
  if (dtype != KITTY_F16 && dtype != KITTY_BF16) return KITTY_E_BADARG;
  if (!(scaling > 0.0f) || !(scaling < INFINITY)) return KITTY_E_BADARG;
  if (Lq > (1 << 30) || Lk > (1 << 30)) return KITTY_E_BADSHAPE;
  const bool packed = cu_q != nullptr;
  if (Lq == 0 || (B == 0 && !packed)) return KITTY_OK;
  if (!q || !out || (Lk > 0 && (!k || !v))) return KITTY_E_BADARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out)) & 15)
    return KITTY_E_BADARG;
  PromptArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  int64_t *st[3] = {a.qs, a.ks, a.vs};
  const int64_t size[3][3] = {{packed ? 1 : B, h_q, Lq}, {packed ? 1 : B, h_kv, Lk}, {packed ? 1 : B, h_kv, Lk}};
  for (int x = 0; x < 3; ++x)
    for (int i = 0; i < 3; ++i) {
      st[x][i] = packed && i == 0 ? 0 : strides[3 * x + i];
      // a copy's strides are positive multiples of 16 bytes below 2^40
      if (size[x][i] > 1 && (st[x][i] <= 0 || st[x][i] % 8 != 0 || st[x][i] >= (1ll << 39))) return KITTY_E_BADARG;
    }
  a.q_lens = packed ? nullptr : q_lens;
  a.k_lens = packed ? nullptr : k_lens;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.status = status;
  a.B = B;
  a.Lq = static_cast<int32_t>(Lq);
  a.Lk = static_cast<int32_t>(Lk);
  a.G = h_q / h_kv;
  a.h_kv = h_kv;
  a.causal = causal != 0;
  a.zero_rest = zero_rest != 0;
  a.c = scaling * 1.4426950408889634f;
  int64_t grid;
  if (packed) {
    const int64_t nseq = static_cast<int64_t>(B) + a.zero_rest;
    grid = (((Lq / PT + nseq) * a.G + 1) / 2 + nseq) * h_kv;      // most pairs of tiles that nseq sequences can need
  } else {
    a.pairs = static_cast<int32_t>(((Lq + PT - 1) / PT * a.G + 1) / 2);
    grid = static_cast<int64_t>(a.pairs) * B * h_kv;
  }
  if (grid > 0x7fffffff || (Lq + PT) / PT * a.G > 0x7fffffff) return KITTY_E_BADSHAPE;
  if (grid == 0) return KITTY_OK;
  const bool bf16 = dtype == KITTY_BF16;
  CUtensorMap mq, mk, mv;
  // without keys nothing is copied through their maps; they only have to be well formed
  if (!make_map(&mq, q, bf16, Lq, h_q, packed ? 1 : B, a.qs)) return KITTY_E_CUDA;
  if (Lk == 0) mk = mv = mq;
  else if (!make_map(&mk, k, bf16, Lk, h_kv, packed ? 1 : B, a.ks) || !make_map(&mv, v, bf16, Lk, h_kv, packed ? 1 : B, a.vs))
    return KITTY_E_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return bf16 ? launch_prompt<__nv_bfloat16>(mq, mk, mv, a, static_cast<unsigned>(grid), s)
              : launch_prompt<__half>(mq, mk, mv, a, static_cast<unsigned>(grid), s);
}
