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
//   warps 10, 11     take what is not finite out of value tiles that some row does not see all of, half a tile each
//
// The running maximum is kept in the logits' own units and allowed to lag: the accumulator is rescaled only when a row's
// maximum has grown by more than 2^8, by the softmax threads themselves (the product before is complete by then: the
// commit that announces new logits also covers it).  Weights up to 256 fit the 16-bit types, sums are 32-bit.  fp16 weights
// are held 2^7 times as large (up to 2^15, of 65504): those below 2^-32 of the largest round to nothing, which costs a
// million of them together 2^-13, and not those below 2^-25, which counted in the sum but were missing from the product
// (0.1 % with 32768 keys behind a dominant one).
// The matrix unit itself adds with 32 bits but cuts off what lies some 2^-25 below the accumulator, always towards zero:
// measured, a row loses about 2^-26 of its result per key of a part (one key of weight 1 and the rest at 2^-20, all values
// between 1 and 2: 0.04 % with 32768 keys, 0.08 % with 65536; equal weights in fp16 0.005 and 0.02 %), less where values
// change sign.  Half a step of the output is 0.05 % in fp16 and 0.4 % in bf16.  The sums are 32-bit additions that round.
// Weights are rounded to the inputs' type for the second product (half a step, 2^-9 for bf16, of independent sign, as
// large as the rounding of the output itself).
//
// Keys that a row does not see: their logits are replaced before the maximum is taken, so keys may hold anything.  Their
// values enter the product with weight zero, and zero times infinity or NaN is NaN.  So in the value tiles that some row
// of the two query tiles does not see all of (three at most: the diagonal, or the last one), infinities and NaN become
// zeros in shared memory before the product, and the keys that held one are noted.  A row that sees such a key has them
// added to its accumulator at the end: what is not finite stays so under any weight, so the sum of the numbers
// themselves is the result.  Padding, the next sequence of a packed batch and later tokens cost no more for what they hold.  The
// two warps look at a tile while the step before it runs: 4 x 4096 tokens take 468 us with them, 469 without (asked for
// only when the tile's own step began, and with a test per word instead of a multiply-add, 487).
#include <cuda.h>

#include "decode.cuh"
#include "overlap.cuh"
#include "tcgen05.cuh"

namespace kitty {

constexpr int PT = 128;                        // rows of a query tile, keys of a key tile
constexpr int TILE_BYTES = PT * HD * 2;        // 32 KB
constexpr int KV_STAGES = 5;
constexpr int PROMPT_SMEM = (2 + KV_STAGES) * TILE_BYTES + 1024;
constexpr int PROMPT_THREADS = 384;            // three groups of four warps
constexpr int CLEAN_TILES = 3;                 // value tiles of an item that some row does not see all of, at most
constexpr float LAG = 8.0f;                    // log2 of how far a maximum may lag
template <typename T>
constexpr float SHIFT = __is_same(T, __half) ? 7.0f : 0.0f;      // log2 of the weight of a maximum

// A wait for something that comes once an item lasts as long as its key tiles do (1.5 us each): their number is added to the
// limit.
__device__ __forceinline__ unsigned long long item_limit(int tiles) { return WAIT_LIMIT_NS + 20000ull * tiles; }

struct PromptArgs {
  const void *q, *k, *v;
  void *out;
  int64_t qs[3], ks[3], vs[3];                 // element strides (batch, head, token)
  const int32_t *q_lens, *k_lens, *cu_q, *cu_k;
  int32_t *status;
  float *part;                                 // splits > 1: [splits][rows][h_q][128] accumulators,
  float2 *part_ml;                             // [splits][rows][h_q] (maximum in base 2, sum; sum -1: sees nothing); sums
                                               // and accumulators are 2^SHIFT times as large, all of them
  int64_t rows;                                // output rows of one head
  int32_t B, Lq, Lk, G, h_kv, pairs, causal, zero_rest, splits, items;
  float c;                                     // scaling * log2 e
};

// ---- two 32-bit floats at a time
__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 un2(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Largest of three; NaN if one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x of two numbers (finite, below 2^16) on the multiply-add pipe: x = whole + f with |f| <= 1/2, 2^f by a polynomial of
// degree four fitted for the least largest relative error (2.6e-6 = 2^-18.6), the whole part added to the exponent.
// Below 2^-126 the result stays there: a weight of 1e-38.
__device__ __forceinline__ uint64_t ex2_poly2(uint64_t x2) {
  float2 x = un2(x2);
  x2 = pk2(fmaxf(x.x, -126.0f), fmaxf(x.y, -126.0f));
  const uint64_t magic = pk2(12582912.0f, 12582912.0f), unmagic = pk2(-12582912.0f, -12582912.0f);
  const uint64_t t = add2(x2, magic);                       // whole part in the low bits
  const uint64_t f = fma2(add2(t, unmagic), pk2(-1.0f, -1.0f), x2);
  uint64_t p = fma2(f, pk2(0.00957009f, 0.00957009f), pk2(0.0559179f, 0.0559179f));
  p = fma2(p, f, pk2(0.24024745f, 0.24024745f));
  p = fma2(p, f, pk2(0.69312181f, 0.69312181f));
  p = fma2(p, f, pk2(0.99999926f, 0.99999926f));
  const float2 pf = un2(p), tf = un2(t);
  return pk2(__uint_as_float(__float_as_uint(pf.x) + (__float_as_uint(tf.x) << 23)),
             __uint_as_float(__float_as_uint(pf.y) + (__float_as_uint(tf.y) << 23)));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(uint64_t p) {
  const float2 f = un2(p);
  if constexpr (__is_same(T, __nv_bfloat16)) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t *>(&x);
  } else {
    return pack_h2(f.x, f.y);
  }
}

// Weights of 64 logits, 2^(v c - mc + SHIFT), as 16-bit pairs; returns their sum.  POLY: every eighth pair goes through the
// polynomial, which takes some of the load off the 16-a-clock exponential unit (for finite logits only): 1.36 PFLOP/s
// over long unmasked rows; with none, a quarter or three eighths of them 1.35, 1.30 and 1.28.
template <typename T, bool POLY>
__device__ __forceinline__ uint64_t weights64(const float *v, uint64_t c2, uint64_t nmc2, uint32_t (&w)[32]) {
  uint64_t sum[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint64_t x = fma2(pk2(v[2 * i], v[2 * i + 1]), c2, nmc2);
    uint64_t p;
    if (POLY && (i & 7) == 7) {
      p = ex2_poly2(x);
    } else {
      const float2 f = un2(x);
      p = pk2(ex2(f.x), ex2(f.y));
    }
    sum[i & 1] = add2(sum[i & 1], p);
    w[i] = pack2<T>(p);
  }
  return add2(sum[0], sum[1]);
}

// Four 16-byte words of a thread's row, the same of its three neighbours: after the exchange a thread holds one word of
// each of the four rows, and a store covers 64 consecutive bytes of eight rows (16 of 32 rows it would be otherwise: four
// times the passes through the memory pipe, 5000 clocks an item).  dst: the thread's own row, `stride` elements to the next.
template <typename E>
__device__ __forceinline__ void store_quad(uint4 (&w)[4], E *dst, int64_t stride, int row, int rows) {
  const int q = threadIdx.x & 3;
#pragma unroll
  for (int bit = 1; bit <= 2; bit <<= 1)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int lo = bit == 1 ? 2 * n : n, hi = lo + bit;
      uint4 x = q & bit ? w[lo] : w[hi];
      x.x = __shfl_xor_sync(0xffffffffu, x.x, bit);
      x.y = __shfl_xor_sync(0xffffffffu, x.y, bit);
      x.z = __shfl_xor_sync(0xffffffffu, x.z, bit);
      x.w = __shfl_xor_sync(0xffffffffu, x.w, bit);
      if (q & bit) w[lo] = x;
      else w[hi] = x;
    }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (row - q + k < rows) *reinterpret_cast<uint4 *>(dst + (k - q) * stride + q * (16 / static_cast<int>(sizeof(E)))) = w[k];
}

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

// What an item's value tiles held that is not finite.
struct Odd {
  uint32_t rows[2][4 * CLEAN_TILES];   // by half of the channels: bits of the keys, from key tile0 * 128 on
  const void *v;                       // the first of the sequence's value rows
  int tile0, nk;
};

// x * 0 + acc on two 16-bit numbers: NaN from the first x on that is not finite.
template <typename T>
__device__ __forceinline__ uint32_t stain2(uint32_t x, uint32_t acc) {
  if constexpr (__is_same(T, __half)) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(x), "r"(0));
  else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(x), "r"(0));
  return acc;
}

// Half a value tile (128 rows of 128 bytes) in shared memory, by one warp: numbers that are not finite become zero, and
// the bits of their rows are set in `rows`.
template <typename T>
__device__ __forceinline__ void clear_odd_values(uint32_t half, uint32_t *rows) {
  constexpr uint32_t EXP = __is_same(T, __half) ? 0x7c007c00u : 0x7f807f80u, ONE = __is_same(T, __half) ? 0x04000400u : 0x00800080u;
  // an exponent of all ones, and only that, carries into the sign's place
  auto odd = [](uint32_t x) { return ((x & EXP) + ONE) & 0x80008000u; };
  auto load = [](uint32_t at, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  };
  const int lane = threadIdx.x & 31;
  const uint32_t at = half + lane * 16;
  uint32_t acc[4] = {};
#pragma unroll 1
  for (int i = 0; i < 32; i += 8) {
    uint32_t w[8][4];
#pragma unroll
    for (int y = 0; y < 8; ++y) load(at + (i + y) * 512, w[y]);
#pragma unroll
    for (int y = 0; y < 8; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = stain2<T>(w[y][e], acc[e]);
  }
  if (!__any_sync(0xffffffffu, (odd(acc[0]) | odd(acc[1]) | odd(acc[2]) | odd(acc[3])) != 0)) return;
#pragma unroll 1
  for (int i = 0; i < 32; ++i) {
    uint32_t w[4];
    load(at + i * 512, w);
    if (odd(w[0]) | odd(w[1]) | odd(w[2]) | odd(w[3])) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] &= ~((odd(w[e]) >> 15) * 0xffffu);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + i * 512), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
      const int row = 4 * i + (lane >> 3);
      atomicOr(rows + (row >> 5), 1u << (row & 31));
    }
  }
}

// Adds what clear_odd_values() took out, as far as the thread's row sees it, to the row's accumulator.  The keys are the
// same for all rows of a warp, which read them together.
template <typename T>
__device__ __noinline__ void add_odd_values(const Odd &odd, int64_t stride, uint32_t acc, int limit) {
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    float o[32];
    tmem_ld32(acc + 32 * i, o);
    tmem_wait_ld();
#pragma unroll 1
    for (int y = 0; y < 4 * CLEAN_TILES; ++y) {
      uint32_t m = odd.rows[0][y] | odd.rows[1][y];
      while (m) {
        const int key = odd.tile0 * PT + 32 * y + __ffs(m) - 1;
        m &= m - 1;
        if (key >= odd.nk) break;
        const T *row = static_cast<const T *>(odd.v) + key * stride + 32 * i;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float x[8];
          Vec8<T>::load(row + 8 * c, x);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (key < limit && !(fabsf(x[e]) < INFINITY)) o[8 * c + e] += x[e];
        }
      }
    }
    tmem_st32(acc + 32 * i, reinterpret_cast<const uint32_t *>(o));
  }
  tmem_wait_st();
}

// One piece of work of a block: a pair of query tiles of one key head against its key tiles (or the z-th part of them).
struct Item {
  Seq s;
  int h, pair, z;
  int j0, n;          // first key tile and their number
  int nb[2];          // how many of them each tile sees
  int clean;          // the first of them that some row does not see all of (n: none)
  int more;           // 0: there is no further item
};

// Row tile and head of query tile x of an item; the key tiles that its last row sees (0: none, or no such tile).
__device__ __forceinline__ int tile_of(const PromptArgs &a, const Seq &s, int h, int pair, int x, int &row0, int &head) {
  const int f = 2 * pair + x;
  row0 = f / a.G * PT;
  head = h * a.G + f % a.G;
  const int last = min(row0 + PT, s.nq) - 1;
  return f < (s.rows + PT - 1) / PT * a.G && last >= row0 ? (key_limit(s, last, a.causal) + PT - 1) / PT : 0;
}

// Rows of packed sequence i (i = a.B: the rows behind the last sequence).
__device__ __forceinline__ void packed_rows(const PromptArgs &a, int i, int &lo, int &hi) {
  lo = clampi(a.cu_q[i], 0, a.Lq);
  hi = i < a.B ? clampi(a.cu_q[i + 1], lo, a.Lq) : a.Lq;
}
__device__ __forceinline__ int packed_pairs(const PromptArgs &a, int i) {
  int lo, hi;
  packed_rows(a, i, lo, hi);
  return ((hi - lo + PT - 1) / PT * a.G + 1) / 2;
}

// Work item number `id` (by one warp); false when the packed sequences have no such item.
__device__ __forceinline__ bool find_item(const PromptArgs &a, int id, Item &w) {
  const int lane = threadIdx.x & 31;
  w.z = id % a.splits;
  id /= a.splits;
  Seq &s = w.s;
  if (a.cu_q == nullptr) {
    const int sh = id % (a.B * a.h_kv);
    w.pair = a.pairs - 1 - id / (a.B * a.h_kv);             // the longest rows first
    s.b = sh / a.h_kv;
    w.h = sh % a.h_kv;
    s.q0 = s.k0 = 0;
    s.nq = a.q_lens != nullptr ? clampi(a.q_lens[s.b], 0, a.Lq) : a.Lq;
    s.nk = a.k_lens != nullptr ? clampi(a.k_lens[s.b], 0, a.Lk) : a.Lk;
    s.rows = a.Lq;
    s.out0 = static_cast<int64_t>(s.b) * a.Lq;
  } else {
    w.h = id % a.h_kv;
    const int want = id / a.h_kv, nseq = a.B + (a.zero_rest ? 1 : 0);
    int seq = -1;
    if (nseq <= 64) {
      // The longest rows of all sequences first.  level(p) = pairs with number p or above, over all sequences; the item
      // is one of those with the largest p for which level(p) is above its own number.
      const int n0 = lane < nseq ? packed_pairs(a, lane) : 0, n1 = lane + 32 < nseq ? packed_pairs(a, lane + 32) : 0;
      auto level = [&](int p) { return __reduce_add_sync(0xffffffffu, max(n0 - p, 0) + max(n1 - p, 0)); };
      if (level(0) <= want) return false;
      int lo = 0, hi = __reduce_max_sync(0xffffffffu, max(n0, n1));      // level(lo) > want >= level(hi)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (level(mid) > want) lo = mid;
        else hi = mid;
      }
      const int r = want - level(hi);                       // the r-th sequence that has a pair lo
      const unsigned b0 = __ballot_sync(0xffffffffu, n0 > lo), b1 = __ballot_sync(0xffffffffu, n1 > lo);
      const int c0 = __popc(b0);
      seq = r < c0 ? static_cast<int>(__fns(b0, 0, r + 1)) : 32 + static_cast<int>(__fns(b1, 0, r - c0 + 1));
      w.pair = lo;
    } else {
      // many sequences: one after the other
      int base = 0;
      for (int i0 = 0; i0 < nseq && seq < 0; i0 += 32) {
        const int np = i0 + lane < nseq ? packed_pairs(a, i0 + lane) : 0;
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
          seq = i0 + l;
          w.pair = n1 - 1 - (want - (base + upto - n1));
        }
        base += __shfl_sync(0xffffffffu, inc, 31);
      }
      if (seq < 0) return false;
    }
    s.b = 0;
    int hi;
    packed_rows(a, seq, s.q0, hi);
    s.nq = hi - s.q0;
    s.k0 = s.nk = 0;
    if (seq < a.B) {
      const int32_t *cu = a.cu_k != nullptr ? a.cu_k : a.cu_q;
      s.k0 = clampi(cu[seq], 0, a.Lk);
      s.nk = clampi(cu[seq + 1], s.k0, a.Lk) - s.k0;
    }
    s.rows = s.nq;
    s.out0 = s.q0;
  }
  int row0, head;
  const int all0 = tile_of(a, s, w.h, w.pair, 0, row0, head), all1 = tile_of(a, s, w.h, w.pair, 1, row0, head);
  const int most = max(all0, all1);
  w.j0 = static_cast<int>(static_cast<int64_t>(most) * w.z / a.splits);
  w.n = static_cast<int>(static_cast<int64_t>(most) * (w.z + 1) / a.splits) - w.j0;
  w.nb[0] = min(max(all0 - w.j0, 0), w.n);
  w.nb[1] = min(max(all1 - w.j0, 0), w.n);
  // rows of the two tiles see 255 keys more than their first row at most, which are in CLEAN_TILES tiles
  w.clean = w.n;
  for (int x = 0; x < 2; ++x)
    if (w.nb[x] > 0) {
      tile_of(a, s, w.h, w.pair, x, row0, head);
      w.clean = min(w.clean, max(key_limit(s, row0, a.causal) / PT - w.j0, 0));
    }
  w.more = 1;
  return true;
}

template <typename T>
__global__ void __launch_bounds__(PROMPT_THREADS, 1)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                       const __grid_constant__ CUtensorMap mv, const __grid_constant__ PromptArgs a) {
  constexpr bool BF16 = __is_same(T, __nv_bfloat16);
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_q, bar_q_free, bar_full[KV_STAGES], bar_empty[KV_STAGES], bar_s[2], bar_p[2][2], bar_o[2],
      bar_item[2], bar_item_free[2], bar_turn[2], bar_clean[2], bar_odd[2], bar_odd_free[2], bar_end;
  __shared__ uint32_t tmem_base;
  __shared__ Item items[2];
  __shared__ Odd odd[2];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  if (warp == 9) tmem_alloc(smem_u32(&tmem_base), 512);
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar_q), 1);
    mbar_init(smem_u32(&bar_q_free), 1);
    for (int i = 0; i < KV_STAGES; ++i) mbar_init(smem_u32(&bar_full[i]), 1), mbar_init(smem_u32(&bar_empty[i]), 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_u32(&bar_s[x]), 1);
      mbar_init(smem_u32(&bar_p[x][0]), 4);
      mbar_init(smem_u32(&bar_p[x][1]), 4);
      mbar_init(smem_u32(&bar_o[x]), 1);
      mbar_init(smem_u32(&bar_item[x]), 1);
      mbar_init(smem_u32(&bar_item_free[x]), 11);           // all warps but the copying one
      mbar_init(smem_u32(&bar_turn[x]), 1);
      mbar_init(smem_u32(&bar_clean[x]), 2);
      mbar_init(smem_u32(&bar_odd[x]), 2);
      mbar_init(smem_u32(&bar_odd_free[x]), 8);
    }
    mbar_init(smem_u32(&bar_end), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  const uint32_t q_addr = smem, kv_addr = smem + 2 * TILE_BYTES;
  auto give_up = [&] {
    if (a.status != nullptr) atomicExch(a.status, 1);
  };
  // the c-th item of this block, as the copying warp has published it
  auto next_item = [&](int c, Item &w) {
    const bool ok = __all_sync(0xffffffffu, mbar_wait_asleep(smem_u32(&bar_item[c & 1]), (c >> 1) & 1));
    if (!ok) return false;
    w = items[c & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&bar_item_free[c & 1]));
    return w.more != 0;
  };

  // 384 threads start with 168 registers; the softmax threads take what the other group gives up (2 * 224 + 56 = 3 * 168)
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 8) {
      // ---- copies, and the list of items: items are numbered from the most work to the least, and the blocks take them
      // in turn, there and back (first to last, last to first, ...), which leaves every block about the same
      uint32_t pos = 0;                                     // key and value tiles requested so far
      int published = 0, loaded = 0;
      bool ok = true;
      auto publish = [&](const Item &w) {
        const int c = published++;
        if (c >= 2) ok = __all_sync(0xffffffffu, mbar_wait_asleep(smem_u32(&bar_item_free[c & 1]), ((c >> 1) - 1) & 1));
        if (ok && lane == 0) {
          items[c & 1] = w;
          mbar_arrive(smem_u32(&bar_item[c & 1]));
        }
        __syncwarp();
      };
      for (int k = 0; ok && static_cast<int64_t>(k) * gridDim.x < a.items; ++k) {
        const int id = k * gridDim.x + (k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        Item w;
        if (id >= a.items || !find_item(a, id, w)) continue;
        publish(w);
        if (!ok || w.n == 0) continue;
        if (elect_one()) {
          // the query tiles' place is free when the last logits of the item before are complete
          if (loaded > 0) ok = mbar_wait_asleep(smem_u32(&bar_q_free), (loaded - 1) & 1);
          if (ok) {
            const uint32_t bq = smem_u32(&bar_q);
            mbar_expect_tx(bq, (w.nb[0] > 0 ? TILE_BYTES : 0) + (w.nb[1] > 0 ? TILE_BYTES : 0));
            for (int x = 0; x < 2; ++x) {
              int row0, head;
              tile_of(a, w.s, w.h, w.pair, x, row0, head);
              if (w.nb[x] > 0)
                for (int c = 0; c < 2; ++c)
                  tma_load_4d(q_addr + x * TILE_BYTES + c * (TILE_BYTES / 2), &mq, bq, 64 * c, w.s.q0 + row0, head, w.s.b);
            }
          }
          uint32_t at = pos;
          for (int i = 0; i < 2 * w.n && ok; ++i, ++at) {
            const uint32_t st = at % KV_STAGES, round = at / KV_STAGES;
            if (round > 0 && !mbar_wait_asleep(smem_u32(&bar_empty[st]), (round - 1) & 1)) {
              ok = false;
              break;
            }
            const uint32_t bf = smem_u32(&bar_full[st]);
            mbar_expect_tx(bf, TILE_BYTES);
            const CUtensorMap *m = (i & 1) ? &mv : &mk;
            for (int c = 0; c < 2; ++c)
              tma_load_4d(kv_addr + st * TILE_BYTES + c * (TILE_BYTES / 2), m, bf, 64 * c, w.s.k0 + (w.j0 + (i >> 1)) * PT, w.h, w.s.b);
          }
          if (!ok) {                                        // leave no copy in flight behind
            give_up();
            mbar_wait_asleep(smem_u32(&bar_q), loaded & 1);
            for (uint32_t j = at > KV_STAGES ? at - KV_STAGES : 0; j < at; ++j)
              mbar_wait_asleep(smem_u32(&bar_full[j % KV_STAGES]), (j / KV_STAGES) & 1);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        pos += 2 * w.n;
        ++loaded;
      }
      Item end{};
      if (ok) publish(end);
    } else if (warp == 9) {
      // ---- products.  The issuing thread's instructions are the pace of the block: a straight line of them would miss the
      // instruction cache at every step (the softmax code fills it), so everything is in short loops.
      constexpr uint32_t ID_S = umma_idesc(BF16, PT, PT, false), ID_O = umma_idesc(BF16, PT, HD, true);
      constexpr uint32_t STAGE = TILE_BYTES >> 4;             // in units of a descriptor's address
      const uint32_t full = smem_u32(&bar_full[0]), empty = smem_u32(&bar_empty[0]);
      const uint32_t ready = smem_u32(&bar_s[0]), weights = smem_u32(&bar_p[0][0]), done = smem_u32(&bar_o[0]);
      const uint32_t q_lo = umma_lo(q_addr, 16), k_lo = umma_lo(kv_addr, 16), v_lo = umma_lo(kv_addr, TILE_BYTES / 2);
      uint32_t pos = 0, step0 = 0, step1 = 0, cleaned = 0;  // tiles read, weights of either query tile taken, tiles cleaned so far
      int loaded = 0;
      bool ok = true;
      Item w;
      for (int c = 0; ok && next_item(c, w); ++c) {
        if (w.n == 0) continue;
        const int n = w.n, nb0 = w.nb[0], nb1 = w.nb[1], clean = w.clean;
        if (elect_one()) {
          uint32_t st = pos % KV_STAGES, ph = pos / KV_STAGES & 1;      // ring position of the next tile
          auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = ok && mbar_wait_asleep(bar, parity);
            tc_fence_after();
            return ok;
          };
          auto advance = [&] {
            if (++st == KV_STAGES) st = 0, ph ^= 1;
          };
          // logits of tile x: contraction over 128 channels, 16 at a time, two swizzled halves
          auto logits = [&](uint32_t x, uint32_t stage) {
            uint32_t ql = q_lo + x * STAGE, kl = k_lo + stage * STAGE;
#pragma unroll 1
            for (int y = 0; y < 2; ++y) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_ss(tmem + x * PT, ql + 2 * k, umma_hi(1024), kl + 2 * k, umma_hi(1024), ID_S, (y | k) != 0);
              ql += STAGE / 2;
              kl += STAGE / 2;
            }
            umma_commit(ready + 8 * x);
          };
          // Value tile j is to be cleaned: said a step early, so that it is done when the step's weights are there.  The next
          // tile may be asked for, and done, before this thread sees that this one is, but not the one after it: two barriers
          // either way.
          auto ask = [&](int j) { mbar_arrive(smem_u32(&bar_turn[(cleaned + (j - clean)) & 1])); };
          wait(smem_u32(&bar_q), loaded & 1);
          if (clean == 0) ask(0);
          if (wait(full + 8 * st, ph)) {
#pragma unroll 1
            for (int x = 0; x < 2; ++x)
              if ((x ? nb1 : nb0) > 0) logits(x, st);
            umma_commit(empty + 8 * st);
            if (n == 1) umma_commit(smem_u32(&bar_q_free));
            advance();
          }
#pragma unroll 1
          for (int j = 0; j < n && ok; ++j) {
            const uint32_t sv = st;
            if (!wait(full + 8 * sv, ph)) break;
            if (j + 1 >= clean && j + 1 < n) ask(j + 1);
            if (j >= clean) {
              const uint32_t at = cleaned + (j - clean);
              if (!wait(smem_u32(&bar_clean[at & 1]), (at >> 1) & 1)) break;
            }
            advance();
            const bool more = j + 1 < n;
#pragma unroll 1
            for (int x = 0; x < 2 && ok; ++x) {
              const int nb = x ? nb1 : nb0;
              if (j < nb) {
                // accumulator of tile x += weights x value tile j: contraction over 128 keys, 16 at a time
                uint32_t vl = v_lo + sv * STAGE, pa = tmem + x * PT;
                uint32_t bar = weights + 16 * x;
                const uint32_t parity = ((x ? step1 : step0) + j) & 1;
#pragma unroll 1
                for (int y = 0; y < 2; ++y) {
                  if (!wait(bar, parity)) break;
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    umma_ts(tmem + 2 * PT + x * HD, pa + 8 * k, vl + (2048 >> 4) * k, umma_hi(1024), ID_O, (j | y | k) != 0);
                  vl += 4 * (2048 >> 4);
                  pa += 32;
                  bar += 8;
                }
                if (!ok) break;
                if (j + 1 == nb) umma_commit(done + 8 * x);
              }
              if (x == 1) umma_commit(empty + 8 * sv);
              if (more) {
                if (x == 0 && !wait(full + 8 * st, ph)) break;
                if (j + 1 < nb) logits(x, st);
                if (x == 1) {
                  umma_commit(empty + 8 * st);
                  if (j + 2 == n) umma_commit(smem_u32(&bar_q_free));
                }
              }
            }
            if (more) advance();
          }
          if (!ok) give_up();
        }
        ok = __all_sync(0xffffffffu, ok);
        pos += 2 * n;
        step0 += nb0;
        step1 += nb1;
        cleaned += n - clean;
        ++loaded;
      }
      // every product is complete before the tensor memory is given back
      if (elect_one()) {
        umma_commit(smem_u32(&bar_end));
        mbar_wait_asleep(smem_u32(&bar_end), 0);
      }
      __syncwarp();
    } else {
      // ---- values that are not finite, in the tiles that the issuing warp asks for
      uint32_t pos = 0, cleaned = 0;
      bool ok = true;
      Item w;
      for (int c = 0; ok && next_item(c, w); ++c) {
        // the softmax warps are done with the words of the item before last
        if (c >= 2) ok = __all_sync(0xffffffffu, mbar_wait_asleep(smem_u32(&bar_odd_free[c & 1]), ((c >> 1) - 1) & 1));
        if (!ok) break;
        Odd &o = odd[c & 1];
        uint32_t *rows = o.rows[warp - 10];
        if (lane < 4 * CLEAN_TILES) rows[lane] = 0;
        if (warp == 10 && lane == 0) {
          o.v = static_cast<const T *>(a.v) + w.s.b * a.vs[0] + w.h * a.vs[1] + w.s.k0 * a.vs[2];
          o.tile0 = w.j0 + w.clean;
          o.nk = w.s.nk;
        }
        __syncwarp();
        for (int j = w.clean; j < w.n; ++j, ++cleaned) {
          const uint32_t at = pos + 2 * j + 1, st = at % KV_STAGES;
          ok = __all_sync(0xffffffffu, mbar_wait_asleep(smem_u32(&bar_turn[cleaned & 1]), (cleaned >> 1) & 1, item_limit(w.n)) &&
                                           mbar_wait_asleep(smem_u32(&bar_full[st]), at / KV_STAGES & 1));
          if (!ok) break;
          clear_odd_values<T>(kv_addr + st * TILE_BYTES + (warp - 10) * (TILE_BYTES / 2), rows + 4 * (j - w.clean));
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the product reads what was written here
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_clean[cleaned & 1]));
        }
        if (ok && lane == 0) mbar_arrive(smem_u32(&bar_odd[c & 1]));
        pos += 2 * w.n;
      }
      if (!ok) give_up();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int x = warp >> 2;
    const uint32_t at = tmem + (static_cast<uint32_t>(warp & 3) << 21);     // the warp's 32 lanes
    const uint32_t ts = at + x * PT, to = at + 2 * PT + x * HD;
    const uint64_t c2 = pk2(a.c, a.c);
    uint32_t step = 0, outs = 0;             // tiles of logits and accumulators taken so far
    bool ok = true;
    Item w_;
    for (int count = 0; ok && next_item(count, w_); ++count) {
      const Seq s = w_.s;
      const int j0 = w_.j0, nb = x ? w_.nb[1] : w_.nb[0];
      int row0, head;
      tile_of(a, s, w_.h, w_.pair, x, row0, head);
      const bool live = 2 * w_.pair + x < (s.rows + PT - 1) / PT * a.G;
      const int z = w_.z;
      const int row = row0 + (threadIdx.x & 127);
      const int limit = key_limit(s, row, a.causal);
      float m = -INFINITY, l = 0.0f;
      // keys that every row of the tile sees need no comparison
      const int all = key_limit(s, min(row0, s.nq - 1), a.causal);
      for (int j = 0; j < nb; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait_asleep(smem_u32(&bar_s[x]), (step + j) & 1));
        if (!ok) break;
        tc_fence_after();
        float v[PT];
        tmem_ld32(ts, v);
        tmem_ld32(ts + 32, v + 32);
        tmem_wait_ld();
        tmem_ld32(ts + 64, v + 64);
        tmem_ld32(ts + 96, v + 96);
        const bool masked = (j0 + j + 1) * PT > all;
        const int seen = limit - (j0 + j) * PT;
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        uint32_t w[32];
        uint64_t sum = 0;
        bool settled = false;
        auto announce = [&](int half) {
          tmem_st32(ts + 32 * half, w);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_p[x][half]));      // one arrival a warp: arrivals at one address queue up
        };
        auto largest = [&](int half) {
#pragma unroll
          for (int i = 64 * half; i < 64 * half + 64; i += 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = max3(t[e], v[i + 2 * e], v[i + 2 * e + 1]);
          }
        };
        if (j > 0 && !masked) {
          // The maximum so far is mostly the one to use: the first weights are taken with it while the tile's own maximum
          // is found, and count if no row has outgrown it (nor met a NaN, which this comparison does not pass).
          const float nmc = fmaf(-m, a.c, SHIFT<T>);
          const uint64_t nmc2 = pk2(nmc, nmc);
          sum = weights64<T, true>(v, c2, nmc2, w);
          largest(0);
          tmem_wait_ld();
          largest(1);
          const float top = max3(max3(t[0], t[1], t[2]), t[3], t[3]);
          settled = __all_sync(0xffffffffu, (top - m) * a.c <= LAG);
          if (settled) {
            announce(0);
            sum = add2(sum, weights64<T, true>(v + 64, c2, nmc2, w));
            announce(1);
          }
        }
        if (!settled) {
          tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int i = 0; i < PT; ++i) v[i] = i < seen ? v[i] : -INFINITY;
          }
          t[0] = t[1] = t[2] = t[3] = -INFINITY;
          largest(0);
          largest(1);
          const float top = max3(max3(t[0], t[1], t[2]), t[3], t[3]);
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
          const float nmc = m == -INFINITY ? 0.0f : fmaf(-m, a.c, SHIFT<T>);
          const uint64_t nmc2 = pk2(nmc, nmc);
          sum = weights64<T, false>(v, c2, nmc2, w);
          announce(0);
          sum = add2(sum, weights64<T, false>(v + 64, c2, nmc2, w));
          announce(1);
        }
        const float2 sf = un2(sum);
        l += sf.x + sf.y;
      }
      if (nb > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait_asleep(smem_u32(&bar_o[x]), outs & 1));
      step += nb;
      outs += nb > 0;
      tc_fence_after();
      // a tile that sees fewer keys than its neighbour, or none, waits here for the item's end
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_asleep(smem_u32(&bar_odd[count & 1]), (count >> 1) & 1, item_limit(w_.n)));
      if (ok) {
        const Odd &o = odd[count & 1];
        const bool some = lane < 4 * CLEAN_TILES && (o.rows[0][lane] | o.rows[1][lane]) != 0;
        if (__any_sync(0xffffffffu, some) && nb > 0) add_odd_values<T>(o, a.vs[2], to, limit);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_odd_free[count & 1]));
      }
      if (live && ok) {
        const bool mine = row < s.rows;
        const int64_t at_out = (s.out0 + row) * static_cast<int64_t>(a.G) * a.h_kv + head;
        const int64_t stride = static_cast<int64_t>(a.G) * a.h_kv * HD;      // from a row of the output to the next
        if (a.splits == 1) {
          const float inv = limit > 0 ? 1.0f / l : 0.0f;
          T *dst = static_cast<T *>(a.out) + at_out * HD;
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
              t[e] = from_f32<T>(limit > 0 ? o[e] * inv : 0.0f);
            }
            store_quad(w, dst + 32 * i, stride, row, s.rows);
          }
        } else if (mine) {
          // a part of the keys: the accumulator as it is, the maximum and the sum; no accumulator without a sum
          const int64_t pa = z * a.rows * a.G * a.h_kv + at_out;
          const bool some = limit > j0 * PT && nb > 0;
          a.part_ml[pa] = limit == 0 ? make_float2(-INFINITY, -1.0f) : some ? make_float2(m == -INFINITY ? m : m * a.c, l) : make_float2(-INFINITY, 0.0f);
        }
        if (a.splits > 1 && nb > 0) {
          float *dst = a.part + (z * a.rows * a.G * a.h_kv + at_out) * HD;
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            float o[32];
            tmem_ld32(to + 32 * i, o);
            tmem_wait_ld();
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint4 w[4];
              memcpy(w, o + 16 * y, 64);
              store_quad(w, dst + 32 * i + 16 * y, stride, row, s.rows);
            }
          }
        }
      }
    }
    if (!ok) give_up();
    tc_fence_before();
  }
  __syncthreads();
  __syncwarp();
  tc_fence_after();
  if (warp == 9) tmem_free(tmem, 512);
}

// Joins the parts of split keys: one warp per (row, query head), four channels a lane.
template <typename T>
__global__ void __launch_bounds__(256) prompt_join_kernel(const __grid_constant__ PromptArgs a) {
  const int64_t n = a.rows * a.G * a.h_kv;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  dep_wait();
  if (at >= n) return;
  if (a.cu_q != nullptr && !a.zero_rest) {       // rows of no sequence are left as they are
    const int64_t row = at / (a.G * a.h_kv);
    if (row >= a.cu_q[a.B] || row < a.cu_q[0]) return;
  }
  // the parts' maxima and sums, a part per lane
  float m = -INFINITY, l = 0.0f, acc[4] = {};
  for (int z0 = 0; z0 < a.splits; z0 += 32) {
    const float2 ml = z0 + lane < a.splits ? a.part_ml[(z0 + lane) * n + at] : make_float2(-INFINITY, 0.0f);
    float top = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.0f : mn;
    const float f = ex2(m - ref);
    l *= f;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= f;
    m = mn;
    const float w = ml.y == 0.0f ? 0.0f : ex2(ml.x - ref);
    for (int i = 0; i < min(32, a.splits - z0); ++i) {
      const float li = __shfl_sync(0xffffffffu, ml.y, i), wi = __shfl_sync(0xffffffffu, w, i);
      if (li < 0.0f) {                            // a row that sees nothing says so in every part
        l = -1.0f;
        break;
      }
      if (li == 0.0f) continue;
      const float4 x = *reinterpret_cast<const float4 *>(a.part + ((z0 + i) * n + at) * HD + 4 * lane);
      l = fmaf(li, wi, l);
      acc[0] = fmaf(x.x, wi, acc[0]);
      acc[1] = fmaf(x.y, wi, acc[1]);
      acc[2] = fmaf(x.z, wi, acc[2]);
      acc[3] = fmaf(x.w, wi, acc[3]);
    }
    if (l < 0.0f) break;
  }
  T o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(l < 0.0f ? 0.0f : acc[e] / l);
  *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + at * HD + 4 * lane) = *reinterpret_cast<const uint2 *>(o);
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

// Pairs of tiles of a call (packed: the most that its sequences can need).
int64_t prompt_pairs(bool packed, int64_t B, int64_t Lq, int64_t G, bool rest) {
  if (!packed) return ((Lq + PT - 1) / PT * G + 1) / 2 * B;
  const int64_t nseq = B + rest;
  return ((Lq / PT + nseq) * G + 1) / 2 + nseq;
}

// In how many parts the keys are cut.  Unit: the time of one key tile against a pair of query tiles; a block of threads
// costs FIXED of them besides its tiles, and joining parts costs a launch and the parts' way through memory.  With it
// 1, 16 and 128 rows over 131072 keys (32 query heads, 8 key heads) take 212, 214 and 226 us, launch and join included, from a
// cold L2, which is 2.6 times the keys' and values' way through memory: a tile takes its time whatever rows it has.
int prompt_splits(bool packed, int64_t B, int64_t Lq, int64_t Lk, int64_t h_kv, int64_t G, bool causal) {
  constexpr double FIXED = 2.5, JOIN = 3.0;
  if (Lq == 0 || Lk == 0 || B == 0) return 1;
  const int64_t sms = sm_count();
  const int64_t nseq = packed ? B : 1;
  const double nq = static_cast<double>(Lq) / nseq, nk = static_cast<double>(Lk) / nseq;     // of one sequence
  const double longest = ceil(nk / PT);
  const double mean = causal ? fmax(1.0, (nk - fmin(nq, nk) / 2) / PT) : longest;
  const double items = ceil(ceil(nq / PT) * G / 2) * h_kv * B;
  const double traffic = static_cast<double>(packed ? Lq : B * Lq) * h_kv * G * (HD + 2) * 8 / 6.5e12 / 1.3e-6;   // tiles' time, per part
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 64 && s <= longest; ++s) {
    const double work = items * s * (mean / s + FIXED);
    // equal blocks run in whole waves; unequal ones (longest first) fill in, but the longest is the least there is
    double t = mean > 0.8 * longest ? ceil(items * s / sms) * (mean / s + FIXED) : fmax(work / sms, longest / s + FIXED);
    if (s > 1) t += JOIN + traffic * s;
    if (s == 1 || t < 0.95 * least) {
      best = s;
      least = t;
    }
  }
  return best;
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
  if (cudaGetLastError() != cudaSuccess) return KITTY_E_CUDA;
  if (a.splits == 1) return KITTY_OK;
  const int64_t rows = a.rows * a.G * a.h_kv;
  const cudaError_t e = launch_after(prompt_join_kernel<T>, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0, s, a);
  return (e == cudaSuccess && cudaGetLastError() == cudaSuccess) ? KITTY_OK : KITTY_E_CUDA;
}

}  // namespace kitty

using namespace kitty;

extern "C" int64_t kitty_prompt_workspace_bytes(int32_t B, int64_t Lq, int64_t Lk, int32_t h_q, int32_t h_kv, int causal,
                                                int packed) {
  if (B < 0 || Lq < 0 || Lk < 0 || h_q <= 0 || h_kv <= 0 || h_q % h_kv != 0) return KITTY_E_BADARG;
  if (Lq > (1 << 30) || Lk > (1 << 30)) return KITTY_E_BADSHAPE;
  const int s = prompt_splits(packed != 0, B, Lq, Lk, h_kv, h_q / h_kv, causal != 0);
  return s == 1 ? 0 : (packed ? Lq : B * Lq) * h_q * s * (HD + 2) * 4;
}

extern "C" int kitty_prompt_attn(const void *q, const void *k, const void *v, int dtype, const int64_t *strides,
                                 int32_t B, int64_t Lq, int64_t Lk, int32_t h_q, int32_t h_kv, float scaling,
                                 int causal, const int32_t *q_lens, const int32_t *k_lens, const int32_t *cu_q,
                                 const int32_t *cu_k, void *out, int zero_rest, int32_t *status, void *workspace,
                                 int64_t workspace_bytes, void *stream) {
  if (!strides || B < 0 || Lq < 0 || Lk < 0 || h_q <= 0 || h_kv <= 0 || h_q % h_kv != 0) return KITTY_E_BADARG;
  if (dtype != KITTY_F16 && dtype != KITTY_BF16) return KITTY_E_BADARG;
  if (!(scaling > 0.0f) || !(scaling * 1.4426950408889634f < INFINITY)) return KITTY_E_BADARG;
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
  a.rows = packed ? Lq : B * Lq;
  a.splits = 1;
  if (workspace != nullptr) {
    const int64_t need = kitty_prompt_workspace_bytes(B, Lq, Lk, h_q, h_kv, causal, packed);
    if (workspace_bytes < need) return KITTY_E_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return KITTY_E_BADARG;
    if (need > 0) {
      a.splits = prompt_splits(packed, B, Lq, Lk, h_kv, a.G, a.causal);
      a.part = static_cast<float *>(workspace);
      a.part_ml = reinterpret_cast<float2 *>(a.part + a.splits * a.rows * h_q * HD);
    }
  }
  const int64_t row = static_cast<int64_t>(h_q) * HD * 2;
  const Rows written{out, {packed ? 1 : B, Lq, h_q}, {Lq * row, row, HD * 2}, HD * 2};
  const void *in[3] = {q, k, v};
  for (int x = 0; x < 3; ++x)
    if (rows_meet(written, {in[x], {size[x][0], size[x][1], size[x][2]}, {st[x][0] * 2, st[x][1] * 2, st[x][2] * 2}, HD * 2}))
      return KITTY_E_OVERLAP;
  const int64_t pairs = prompt_pairs(packed, B, Lq, a.G, a.zero_rest);
  if (!packed) a.pairs = static_cast<int32_t>(B > 0 ? pairs / B : 0);
  const int64_t items = pairs * h_kv * a.splits;
  if (items > 0x3fffffff || (Lq + PT) / PT * a.G > 0x7fffffff) return KITTY_E_BADSHAPE;
  if (items == 0) return KITTY_OK;
  a.items = static_cast<int32_t>(items);
  const unsigned grid = static_cast<unsigned>(items < sm_count() ? items : sm_count());
  const bool bf16 = dtype == KITTY_BF16;
  CUtensorMap mq, mk, mv;
  // without keys nothing is copied through their maps; they only have to be well formed
  if (!make_map(&mq, q, bf16, Lq, h_q, packed ? 1 : B, a.qs)) return KITTY_E_CUDA;
  if (Lk == 0) mk = mv = mq;
  else if (!make_map(&mk, k, bf16, Lk, h_kv, packed ? 1 : B, a.ks) || !make_map(&mv, v, bf16, Lk, h_kv, packed ? 1 : B, a.vs))
    return KITTY_E_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return bf16 ? launch_prompt<__nv_bfloat16>(mq, mk, mv, a, grid, s)
              : launch_prompt<__half>(mq, mk, mv, a, grid, s);
}
