// Decode attention over the 8-bit cache: one query token per sequence.
//
// Bound by memory (256 B of codes per token and key head against 4 * group * 128 operations), so the kernel is built
// around an even, uninterrupted stream.  The blocks of 32 tokens of all (sequence, key head) rows form one long line of
// units; every warp of a grid that fills the machine takes an equal, contiguous stretch of it, whatever the lengths
// (they are read on the device, so a captured launch stays valid as sequences grow).  A warp keeps a ring of block
// records in flight with bulk copies (one 8208-byte copy per unit) and needs no other warp until the end.  A row that
// several warps share is joined by a second kernel from their (accumulator, maximum, sum) partials, in a fixed order.
//
// Arithmetic of a unit: whole-number matrix products (mma.m16n8k32, 8-bit operands, exact 32-bit sums) on the stored
// bytes as they are; records hold them in operand order, so every shared-memory read is one conflict-free 16-byte word
// per lane.  The other operand is a 16-bit fixed-point number in two bytes, 256 hi + lo, which are two of the tile's
// sixteen rows (eight heads):
//   logits   query elements in units of (largest of the head) / 32512: off by at most 1/65024 of the head's largest
//   weights  in units of (largest of the block's 32 tokens) / 32512: off by at most 1/65024 of that one, so a far larger
//            weight elsewhere in the sequence costs nothing
// Scales, exponentials, sums and accumulators are 32-bit floats.  Conversions of the codes to 16-bit floats, which an
// fp16 product needs, cost twice the instructions in all and held the kernel at 79 % of the copy bandwidth.
// tcgen05 has no use here: 16 of 128 tile rows would be filled.
#include "kv8.cuh"
#include "overlap.cuh"
#include "paged_core.cuh"

namespace kitty {

constexpr int KV8_WARPS = 12;           // per block of threads, one block per multiprocessor
constexpr int KV8_STAGES = 2;
constexpr int KV8_MAX_SMS = 160;        // the workspace is sized for this many
constexpr int KV8_WORKERS_MAX = KV8_MAX_SMS * KV8_WARPS;
constexpr float KV8_FIX = 32512.0f;     // 127 * 256: both bytes of a fixed-point number stay in -128 .. 127
constexpr float KV8_MAGIC = 12582912.0f;   // 1.5 * 2^23: x + this has the whole number x in its low bits

struct Kv8AttnArgs {
  kitty_kv8_layer L;
  const int32_t *lengths;
  const void *q;
  void *out;
  float *partials;       // [workers + B*h_kv][G][PART]
  int32_t *prefix;       // [B + 1] units before each sequence (of one head)
  float scale_log2;
  int32_t B, G, workers;
};

// Worker w takes units kv8_first_unit(w) .. kv8_first_unit(w + 1) - 1: a part each, the first units % workers one more.
__device__ __forceinline__ int kv8_first_unit(int w, int units, int workers) {
  return w * (units / workers) + min(w, units % workers);
}
__device__ __forceinline__ int kv8_worker_of(int u, int units, int workers) {
  const int q = units / workers, r = units % workers;
  return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q;
}

__device__ __forceinline__ void imma(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four fixed-point numbers (in the low bits of the words) -> their high and low bytes.
__device__ __forceinline__ void fix_bytes(const float *x, uint32_t &hi, uint32_t &lo) {
  uint32_t v[4], y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = __float_as_uint(x[e]);
    y[e] = v[e] + 128u;
  }
  lo = __byte_perm(__byte_perm(v[0], v[1], 0x0040), __byte_perm(v[2], v[3], 0x0040), 0x5410);
  hi = __byte_perm(__byte_perm(y[0], y[1], 0x0051), __byte_perm(y[2], y[3], 0x0051), 0x5410);
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma_t(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (__is_same(T, __half)) {
    mma16816(c, a0, a1, a2, a3, b0, b1);
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack_t(float lo, float hi) {
  T t[2] = {from_f32<T>(lo), from_f32<T>(hi)};
  uint32_t r;
  memcpy(&r, t, 4);
  return r;
}

// Place of a unit: sequence, key head, block, the number of units of the sequence's rows and the tokens it holds.
struct Kv8Cursor {
  int b, h, blk, nblk, len;
  __device__ __forceinline__ void enter(const Kv8AttnArgs &a, const int32_t *prefix) {
    nblk = prefix[b + 1] - prefix[b];
    len = max(0, min(a.lengths[b], a.L.max_page * PAGE));
  }
  __device__ __forceinline__ int tokens() const { return min(KV8_BLOCK, len - blk * KV8_BLOCK); }
  __device__ __forceinline__ void seek(int u, const Kv8AttnArgs &a, const int32_t *prefix) {
    // prefix[b] * h_kv <= u < prefix[b + 1] * h_kv
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] * a.L.h_kv <= u) lo = mid;
      else hi = mid;
    }
    b = lo;
    enter(a, prefix);
    const int rest = u - prefix[b] * a.L.h_kv;
    h = rest / nblk;
    blk = rest - h * nblk;
  }
  // true when the next unit belongs to another row
  template <bool ROW>
  __device__ __forceinline__ bool next(const Kv8AttnArgs &a, const int32_t *prefix) {
    if (++blk < nblk) return false;
    if (ROW) return true;
    blk = 0;
    if (++h == a.L.h_kv) {
      h = 0;
      do {
        ++b;
      } while (b < a.B && prefix[b + 1] == prefix[b]);
      if (b < a.B) enter(a, prefix);
    }
    return true;
  }
};

// MT: 1 for groups of up to 8 query heads, 2 for up to 16 (two matrix tiles).  At 168 registers the even split keeps 80
// bytes a thread in local memory with MT 1 and 280 with MT 2 (32 x 32768 tokens, 2 key heads: 120 us for groups of 8, 142
// for groups of 16, 82 at the copy bandwidth).
// ROW 0: the even split over the machine described above, W = KV8_WARPS.  ROW 1 (see kv8_by_row): a block
// of threads per row, whose W warps share the row's blocks and join their parts in shared memory: no line of units to
// find one's place in, no second kernel.
template <typename T, int MT, int W, bool ROW>
__global__ void __launch_bounds__(W * 32, W == 4 ? 3 : 1) kv8_attn_kernel(const __grid_constant__ Kv8AttnArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[W][KV8_STAGES];
  __shared__ int32_t scan[W];
  __shared__ int32_t skipped[W][KV8_STAGES];      // stages without a record
  __shared__ float2 parts[ROW ? W : 1][MAX_GROUP];        // maximum and sum of each warp's part
  int32_t *prefix = reinterpret_cast<int32_t *>(smem + W * KV8_STAGES * KV8_REC);
  const kitty_kv8_layer &L = a.L;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int H = L.h_kv, B = a.B, G = a.G;

  if (lane == 0) {
    for (int s = 0; s < KV8_STAGES; ++s) mbar_init(smem_u32(&bars[warp][s]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  Kv8Cursor cur;
  int u0, u1, worker = 0;
  if constexpr (ROW) {
    cur.b = blockIdx.x / H;
    cur.h = blockIdx.x % H;
    cur.len = kv8_clamp_len(L, a.lengths[cur.b]);
    cur.nblk = (cur.len + KV8_BLOCK - 1) / KV8_BLOCK;
    u0 = cur.nblk * warp / W;
    u1 = cur.nblk * (warp + 1) / W;
    cur.blk = u0;
    __syncwarp();
  } else {
    // units before each sequence: every block of threads scans the lengths
    const int per = (B + W * 32 - 1) / (W * 32), i0 = min(B, per * static_cast<int>(threadIdx.x));
    const int i1 = min(B, i0 + per);
    int sum = 0;
    for (int i = i0; i < i1; ++i) {
      const int c = (kv8_clamp_len(L, a.lengths[i]) + KV8_BLOCK - 1) / KV8_BLOCK;
      prefix[i + 1] = c;
      sum += c;
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    int base = inc - sum;
    for (int w = 0; w < warp; ++w) base += scan[w];
    for (int i = i0; i < i1; ++i) prefix[i + 1] = base += prefix[i + 1];
    if (threadIdx.x == 0) prefix[0] = 0;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i <= B; i += W * 32) a.prefix[i] = prefix[i];
    dep_release();
    const int units = prefix[B] * H;
    // neighbouring workers sit on different multiprocessors, so that a few units spread over all of them
    worker = warp * gridDim.x + blockIdx.x;
    if (units == 0) return;
    u0 = kv8_first_unit(worker, units, a.workers);
    u1 = kv8_first_unit(worker + 1, units, a.workers);
    if (u0 >= u1) return;
    cur.seek(u0, a, prefix);
  }

  const uint8_t *ring_p = smem + warp * KV8_STAGES * KV8_REC;
  const uint32_t ring = smem_u32(ring_p);
  Kv8Cursor ahead = cur;
  int ua = u0;
  int64_t page = 0;                        // page row of the unit that is requested next, looked up a unit early
  auto look_up = [&] {
    if (lane == 0 && ua < u1 && ahead.tokens() == KV8_BLOCK) page = kv8_page(L, ahead.b, ahead.blk);
  };
  // request the unit `ahead`: the record of a whole block, or the 16-bit values of an open one
  auto request = [&](int stage) {
    if (lane == 0) {
      const uint32_t bar = smem_u32(&bars[warp][stage]);
      const bool whole = ahead.tokens() == KV8_BLOCK;
      skipped[warp][stage] = whole && page < 0;
      if (!whole) {
        constexpr uint32_t BYTES = KV8_BLOCK * HD * sizeof(T);
        mbar_expect_tx(bar, BYTES);
        bulk_g2s(ring + stage * KV8_REC, static_cast<const T *>(L.tail_v) + (static_cast<int64_t>(ahead.b) * H + ahead.h) * KV8_BLOCK * HD,
                 BYTES, bar);
      } else if (page >= 0) {
        mbar_expect_tx(bar, KV8_REC);
        bulk_g2s(ring + stage * KV8_REC, kv8_record(L, page, ahead.h, ahead.blk & 3), KV8_REC, bar);
      } else {
        mbar_expect_tx(bar, 0);
      }
    }
    ahead.template next<ROW>(a, prefix);
    ++ua;
    look_up();
  };
  look_up();
  for (int s = 0; s < KV8_STAGES; ++s)
    if (ua < u1) request(s);

  uint32_t qa[MT][4][4];      // [tile][32 channels][operand]: rows g = high bytes of head g (+ 8), rows g + 8 = low bytes
  float acc[16][2 * MT], mx[MT], sum[MT], qs[MT];
  bool fresh = true, from_start = false;
  int stage = 0, phase = 0;
  for (int u = u0; u < u1; ++u) {
    if (fresh) {
      fresh = false;
      from_start = cur.blk == 0;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int head = g + 8 * m;
        uint4 w[4] = {};
        if (head < G) {
          const T *qp = static_cast<const T *>(a.q) + (static_cast<int64_t>(cur.b) * H * G + cur.h * G + head) * HD + 16 * t;
#pragma unroll
          for (int c = 0; c < 4; ++c) w[c] = *reinterpret_cast<const uint4 *>(qp + (c >> 1) * 64 + (c & 1) * 8);
        }
        float x[4][8], top = 0.0f;
        bool odd = false;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          Vec8<T>::unpack(w[c], x[c]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            top = fmaxf(top, fabsf(x[c][e]));
            odd |= !(fabsf(x[c][e]) < INFINITY);
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        odd = (__ballot_sync(0xffffffffu, odd) >> (lane & 28) & 15u) != 0;
        // the largest element is brought to [1, 2) by a power of two first, which keeps its reciprocal in range
        int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
        ex = max(-100, min(100, ex));
        const float down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
        const float inv = top > 0.0f && !odd ? KV8_FIX / (top * down) * down : 0.0f;
        qs[m] = odd ? __uint_as_float(0x7fc00000u) : a.scale_log2 * (top / KV8_FIX);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            float z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = fmaf(x[ks][4 * o + e], inv, KV8_MAGIC);
            fix_bytes(z, qa[m][ks][2 * o], qa[m][ks][2 * o + 1]);
          }
        mx[m] = -INFINITY;
        sum[m] = 0.0f;
      }
#pragma unroll
      for (int n = 0; n < 16; ++n)
#pragma unroll
        for (int e = 0; e < 2 * MT; ++e) acc[n][e] = 0.0f;
    }
    const int cnt = cur.tokens();
    const bool packed = cnt == KV8_BLOCK;
    if (!mbar_wait(smem_u32(&bars[warp][stage]), phase)) {
      if (lane == 0) atomicOr(L.status, KITTY_KV8_TIMEOUT);
      for (int v = u; v < ua; ++v) {          // leave no copy of this warp in flight behind
        mbar_wait(smem_u32(&bars[warp][stage]), phase);
        if (++stage == KV8_STAGES) stage = 0, phase ^= 1;
      }
      if (ROW) break;                          // the block's barrier is still to come
      return;
    }
    const uint8_t *rec = ring_p + stage * KV8_REC;
    float p[4][2 * MT];           // logits, then weights: tile i, columns 2t, 2t+1 of head g (and g + 8)
    float vscale = 1.0f;
    if (packed) {
      const float2 sc = *reinterpret_cast<const float2 *>(rec + KV8_OFF_SCALE);
      vscale = sc.y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int c[MT][4] = {};
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint4 w = *reinterpret_cast<const uint4 *>(rec + i * 1024 + hf * 512 + lane * 16);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            imma(c[m], qa[m][2 * hf], w.x, w.y);
            imma(c[m], qa[m][2 * hf + 1], w.z, w.w);
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int e = 0; e < 2; ++e) p[i][2 * m + e] = static_cast<float>(c[m][e] * 256 + c[m][2 + e]) * (sc.x * qs[m]);
      }
    } else {
      // open block: 16-bit keys straight from memory, the query in its own type
      const T *kt = static_cast<const T *>(L.tail_k) + (static_cast<int64_t>(cur.b) * H + cur.h) * KV8_BLOCK * HD + 16 * t;
      const T *qp = static_cast<const T *>(a.q) + (static_cast<int64_t>(cur.b) * H * G + cur.h * G) * HD + 16 * t;
      float c[4][4] = {};
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        const int off = (ch >> 1) * 64 + (ch & 1) * 8;
        uint4 q0 = {}, q1 = {}, k4[4] = {};
        if (g < G) q0 = *reinterpret_cast<const uint4 *>(qp + g * HD + off);
        if (MT == 2 && g + 8 < G) q1 = *reinterpret_cast<const uint4 *>(qp + (g + 8) * HD + off);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (kv8_key_token(i, g) < cnt) k4[i] = *reinterpret_cast<const uint4 *>(kt + kv8_key_token(i, g) * HD + off);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mma_t<T>(c[i], q0.x, q1.x, q0.y, q1.y, k4[i].x, k4[i].y);
          mma_t<T>(c[i], q0.z, q1.z, q0.w, q1.w, k4[i].z, k4[i].w);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2 * MT; ++e)
          p[i][e] = 8 * t + 2 * i + (e & 1) < cnt ? c[i][e] * a.scale_log2 : -INFINITY;
    }
    const bool skip = skipped[warp][stage] != 0;
    if (skip) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2 * MT; ++e) p[i][e] = -INFINITY;
      vscale = 0.0f;
    }
    // The block's own maximum and weights, and the running maximum and sum (base 2).  A maximum stays -infinity as long as
    // nothing but skipped blocks was met; of tokens whose logits are all -infinity it is the lowest number.
    float corr[MT], part[MT];
    bool moved = false;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float top = fmaxf(fmaxf(fmaxf(p[0][2 * m], p[0][2 * m + 1]), fmaxf(p[1][2 * m], p[1][2 * m + 1])),
                        fmaxf(fmaxf(p[2][2 * m], p[2][2 * m + 1]), fmaxf(p[3][2 * m], p[3][2 * m + 1])));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (!skip) top = fmaxf(top, -3.402823466e38f);
      const float own = top == -INFINITY ? 0.0f : top;
      const float mn = fmaxf(mx[m], top), ref = mn == -INFINITY ? 0.0f : mn;
      corr[m] = ex2(mx[m] - ref);
      part[m] = top == -INFINITY ? 0.0f : ex2(top - ref);
      moved |= corr[m] != 1.0f;
      mx[m] = mn;
      float add = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i][2 * m] = ex2(p[i][2 * m] - own);
        p[i][2 * m + 1] = ex2(p[i][2 * m + 1] - own);
        add += p[i][2 * m] + p[i][2 * m + 1];
      }
      sum[m] = fmaf(sum[m], corr[m], add * part[m]);
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < 16; ++n)
#pragma unroll
        for (int e = 0; e < 2 * MT; ++e) acc[n][e] *= corr[e >> 1];
    }
    if (packed) {
      uint32_t pa[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          float z[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) z[e] = fmaf(p[2 * o + (e >> 1)][2 * m + (e & 1)], KV8_FIX, KV8_MAGIC);
          fix_bytes(z, pa[m][2 * o], pa[m][2 * o + 1]);
        }
        part[m] *= vscale * (1.0f / KV8_FIX);
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const uint4 w = *reinterpret_cast<const uint4 *>(rec + KV8_OFF_V + x * 512 + lane * 16);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          int c0[4] = {}, c1[4] = {};
          imma(c0, pa[m], w.x, w.y);
          imma(c1, pa[m], w.z, w.w);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            acc[2 * x][2 * m + e] = fmaf(static_cast<float>(c0[e] * 256 + c0[2 + e]), part[m], acc[2 * x][2 * m + e]);
            acc[2 * x + 1][2 * m + e] = fmaf(static_cast<float>(c1[e] * 256 + c1[2 + e]), part[m], acc[2 * x + 1][2 * m + e]);
          }
        }
      }
    } else {
      // 16-bit values of the open block, in the stage; weights as a sum of two 16-bit numbers, so that the bf16 form loses
      // nothing; tokens behind the last one are nothing, whatever they hold
      uint32_t hi[4][MT], lo[4][MT], keep[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tk = 8 * t + 2 * i;
        keep[i] = (tk < cnt ? 0x0000ffffu : 0u) | (tk + 1 < cnt ? 0xffff0000u : 0u);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const float p0 = p[i][2 * m], p1 = p[i][2 * m + 1];
          const float r0 = to_f32<T>(from_f32<T>(p0)), r1 = to_f32<T>(from_f32<T>(p1));
          hi[i][m] = pack_t<T>(r0, r1);
          lo[i][m] = pack_t<T>(p0 - r0, p1 - r1);
        }
      }
      // lane l names row l % 8 of matrix l / 8: the token that row 2t' + e of tile i stands for
      const int mi = lane >> 3, mr = lane & 7;
      const uint32_t row = ring + stage * KV8_REC + kv8_key_token(mi, mr) * HD * sizeof(T);
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        float c[4] = {};
        uint32_t bv[4];
        ldmatrix4_trans(bv, row + n * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) bv[i] &= keep[i];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          mma_t<T>(c, hi[2 * s][0], MT == 2 ? hi[2 * s][MT - 1] : 0, hi[2 * s + 1][0], MT == 2 ? hi[2 * s + 1][MT - 1] : 0,
                   bv[2 * s], bv[2 * s + 1]);
          mma_t<T>(c, lo[2 * s][0], MT == 2 ? lo[2 * s][MT - 1] : 0, lo[2 * s + 1][0], MT == 2 ? lo[2 * s + 1][MT - 1] : 0,
                   bv[2 * s], bv[2 * s + 1]);
        }
#pragma unroll
        for (int e = 0; e < 2 * MT; ++e) acc[n][e] = fmaf(c[e], part[e >> 1], acc[n][e]);
      }
    }
    // the stage is read: request the unit that comes KV8_STAGES later into it
    __syncwarp();
    if (ua < u1) request(stage);
    if (++stage == KV8_STAGES) stage = 0, phase ^= 1;
    const int b = cur.b, h = cur.h;
    const bool ends = cur.template next<ROW>(a, prefix);
    if (!ROW && (ends || u + 1 == u1)) {
      fresh = true;
      const bool all = from_start && ends;          // the whole row: no one else has a part of it
      const int64_t row = static_cast<int64_t>(b) * H + h;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float s = sum[m];
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        const int head = g + 8 * m;
        if (head < G && all) {
          T *o = static_cast<T *>(a.out) + (row * G + head) * HD + 2 * t;
          const float inv = mx[m] == -INFINITY ? 0.0f : 1.0f / s;       // every block skipped: zeros
#pragma unroll
          for (int n = 0; n < 16; ++n)
            *reinterpret_cast<uint32_t *>(o + 8 * n) = pack_t<T>(acc[n][2 * m] * inv, acc[n][2 * m + 1] * inv);
        } else if (head < G) {
          float *o = a.partials + ((worker + row) * G + head) * PART;
#pragma unroll
          for (int n = 0; n < 16; ++n)
            *reinterpret_cast<float2 *>(o + 8 * n + 2 * t) = make_float2(acc[n][2 * m], acc[n][2 * m + 1]);
          if (t == 0) *reinterpret_cast<float2 *>(o + HD) = make_float2(mx[m], s);
        }
      }
    }
  }
  if constexpr (ROW) {
    // the warps' parts, each in its own ring (all its copies are done): accumulators [head][128], (maximum, sum) beside
    float *mine = reinterpret_cast<float *>(smem + warp * KV8_STAGES * KV8_REC);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int head = g + 8 * m;
      float s = u0 < u1 ? sum[m] : 0.0f;
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      if (head < G) {
        if (t == 0) parts[warp][head] = make_float2(u0 < u1 ? mx[m] : -INFINITY, s);
        if (u0 < u1) {
#pragma unroll
          for (int n = 0; n < 16; ++n)
            *reinterpret_cast<float2 *>(mine + head * HD + 8 * n + 2 * t) = make_float2(acc[n][2 * m], acc[n][2 * m + 1]);
        }
      }
    }
    __syncthreads();
    T *out = static_cast<T *>(a.out) + static_cast<int64_t>(blockIdx.x) * G * HD;
    for (int i = threadIdx.x; i < G * HD / 2; i += W * 32) {
      const int head = i / (HD / 2);
      float top = -INFINITY, l = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, parts[w][head].x);
      const bool none = top == -INFINITY;                                // no token, or every block skipped
      if (none) top = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (cur.nblk * w / W == cur.nblk * (w + 1) / W) continue;      // a warp without blocks
        const float2 p = parts[w][head];
        const float wgt = ex2(p.x - top);
        const float2 v = *reinterpret_cast<const float2 *>(smem + w * KV8_STAGES * KV8_REC + i * sizeof(float2));
        l = fmaf(p.y, wgt, l);
        x = fmaf(v.x, wgt, x);
        y = fmaf(v.y, wgt, y);
      }
      const float inv = none ? 0.0f : 1.0f / l;
      *reinterpret_cast<uint32_t *>(out + 2 * i) = pack_t<T>(x * inv, y * inv);
    }
  }
}

// Workers that share the row of (sequence b, key head h): first and last; false when nothing is left to do (one worker
// had the whole row and has written it).
__device__ __forceinline__ bool kv8_shared_row(const Kv8AttnArgs &a, int b, int h, int &w0, int &w1, int &nblk) {
  const int H = a.L.h_kv, units = a.prefix[a.B] * H, before = a.prefix[b] * H;
  nblk = a.prefix[b + 1] - a.prefix[b];
  w0 = w1 = 0;
  if (nblk == 0) return true;
  const int f = before + h * nblk;
  w0 = kv8_worker_of(f, units, a.workers);
  w1 = kv8_worker_of(f + nblk - 1, units, a.workers);
  return w0 != w1;
}

// Joins the partials of rows that several workers share, weights 2^(max - largest max) in 32 bits, partials in the order
// of the workers.  Two shapes, by how many partials a row can have (about workers / rows + 2):
// many rows, few partials: a warp per (sequence, query head), four channels a lane.
template <typename T>
__global__ void __launch_bounds__(256) kv8_join_rows_kernel(const __grid_constant__ Kv8AttnArgs a) {
  const int H = a.L.h_kv, G = a.G, hq = H * G;
  const int at = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  dep_wait();
  if (at >= a.B * hq) return;
  const int b = at / hq, head = at % hq, h = head / G;
  int w0, w1, nblk;
  if (!kv8_shared_row(a, b, h, w0, w1, nblk)) return;
  T *out = static_cast<T *>(a.out) + static_cast<int64_t>(at) * HD + 4 * lane;
  float m = -INFINITY, l = 0.0f, acc[4] = {};
  const float *p = a.partials + ((static_cast<int64_t>(b) * H + h) * G + head % G) * PART;
  const int64_t step = static_cast<int64_t>(G) * PART;
  if (nblk > 0)
    for (int w = w0; w <= w1; w += 4) {
      float2 ml[4], v[4][2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ml[j] = make_float2(-INFINITY, 0.0f);
        v[j][0] = v[j][1] = make_float2(0.0f, 0.0f);
        if (w + j <= w1) {
          const float *o = p + (w + j) * step;
          ml[j] = *reinterpret_cast<const float2 *>(o + HD);
          v[j][0] = *reinterpret_cast<const float2 *>(o + 4 * lane);
          v[j][1] = *reinterpret_cast<const float2 *>(o + 4 * lane + 2);
        }
      }
      const float mn = fmaxf(fmaxf(m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x));
      const float ref = mn == -INFINITY ? 0.0f : mn, f = ex2(m - ref);
      l *= f;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float g = ex2(ml[j].x - ref);
        l = fmaf(ml[j].y, g, l);
        acc[0] = fmaf(v[j][0].x, g, acc[0]);
        acc[1] = fmaf(v[j][0].y, g, acc[1]);
        acc[2] = fmaf(v[j][1].x, g, acc[2]);
        acc[3] = fmaf(v[j][1].y, g, acc[3]);
      }
      m = mn;
    }
  const float inv = m == -INFINITY ? 0.0f : 1.0f / l;      // no token, or every block skipped: zeros
  uint2 o;
  o.x = pack_t<T>(acc[0] * inv, acc[1] * inv);
  o.y = pack_t<T>(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<uint2 *>(out) = o;
}

// few rows, many partials: a block per (sequence, query head); thread s first turns the maximum of partial s into its
// weight, while every thread already has its channel of the first partials of its group in flight.
template <typename T, int KV8_JOIN_GROUPS>
__global__ void __launch_bounds__(HD * KV8_JOIN_GROUPS) kv8_join_kernel(const __grid_constant__ Kv8AttnArgs a) {
  constexpr int NT = HD * KV8_JOIN_GROUPS, NW = NT / 32;
  __shared__ float wgt[NT], red[KV8_JOIN_GROUPS][HD], wm[NW], wl[NW];
  const int H = a.L.h_kv, G = a.G, hq = H * G;
  const int b = blockIdx.x / hq, head = blockIdx.x % hq, h = head / G;
  const int c = threadIdx.x & (HD - 1), grp = threadIdx.x / HD, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  dep_wait();
  int w0, w1, nblk;
  if (!kv8_shared_row(a, b, h, w0, w1, nblk)) return;
  const float *p = a.partials + ((static_cast<int64_t>(b) * H + h + w0) * G + head % G) * PART;
  const int64_t step = static_cast<int64_t>(G) * PART;
  const int n = nblk > 0 ? w1 - w0 + 1 : 0;
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  for (int s0 = 0; s0 < n; s0 += NT) {               // one pass unless a row has over a thousand partials
    const int nn = min(NT, n - s0);
    constexpr int U = 2 * KV8_JOIN_GROUPS;
    float v[U];
    auto fetch = [&](int s) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int sj = s + j * KV8_JOIN_GROUPS;
        v[j] = sj < nn ? p[(s0 + sj) * step + c] : 0.0f;
      }
    };
    fetch(grp);
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (static_cast<int>(threadIdx.x) < nn) ml = *reinterpret_cast<const float2 *>(p + (s0 + threadIdx.x) * step + HD);
    float top = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    __syncthreads();
    if (lane == 0) wm[warp] = top;
    __syncthreads();
    float mn = m;
#pragma unroll
    for (int i = 0; i < NW; ++i) mn = fmaxf(mn, wm[i]);
    const float ref = mn == -INFINITY ? 0.0f : mn, f = ex2(m - ref), g = ex2(ml.x - ref);
    m = mn;
    wgt[threadIdx.x] = g;
    float part = ml.y * g;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (lane == 0) wl[warp] = part;
    __syncthreads();
    l *= f;
#pragma unroll
    for (int i = 0; i < NW; ++i) l += wl[i];
    acc *= f;
    for (int s = grp; s < nn; s += U * KV8_JOIN_GROUPS) {
      if (s != grp) fetch(s);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int sj = s + j * KV8_JOIN_GROUPS;
        acc = fmaf(v[j], sj < nn ? wgt[sj] : 0.0f, acc);
      }
    }
  }
  red[grp][c] = acc;
  __syncthreads();
  if (grp != 0) return;
  float tot = 0.0f;
#pragma unroll
  for (int i = 0; i < KV8_JOIN_GROUPS; ++i) tot += red[i][c];
  static_cast<T *>(a.out)[static_cast<int64_t>(blockIdx.x) * HD + c] = from_f32<T>(m == -INFINITY ? 0.0f : tot / l);
}

template <typename T, int MT, int W, bool ROW>
int start_kv8_attn(const Kv8AttnArgs &a, int blocks, cudaStream_t s) {
  static PerDeviceOnce once;
  constexpr int RING = W * KV8_STAGES * KV8_REC;
  const int rc = per_device_once(once, [] {
    return cudaFuncSetAttribute(kv8_attn_kernel<T, MT, W, ROW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                RING + (ROW ? 0 : (KITTY_KV8_MAX_BATCH + 1) * 4)) == cudaSuccess
               ? KITTY_OK
               : KITTY_E_CUDA;
  });
  if (rc != KITTY_OK) return rc;
  kv8_attn_kernel<T, MT, W, ROW><<<blocks, W * 32, RING + (ROW ? 0 : (a.B + 1) * 4), s>>>(a);
  return cudaGetLastError() == cudaSuccess ? KITTY_OK : KITTY_E_CUDA;
}

// Whether a call gives every row a block of threads.  Lengths are on the device: the rule goes by what a row can hold, so a
// short row in a cache with room for a long one is split and joined (1 x 517 tokens, 8 heads: 6.8 us on the device with room
// for 640, 10.5 with room for 32768; 16 x 517: 7.3 and 15.3).
// Up to 1024 tokens a row, while there are at most four rows per multiprocessor: 8 rows of 640 tokens 8.2 us (11.0 evenly
// split and joined), 256 rows of 1024 16.5 (20.1), but 1024 rows of 640 46.9 (44.5).  Up to 4096, from a row per
// multiprocessor or nearly on: 128 rows of 4096 26 us (39), 1024 rows of 4096 174 (186), but 8 rows of 4096 20 (12).
bool kv8_by_row(int64_t rows, int max_page) {
  const int sms = sm_count();
  return max_page <= 8 ? rows <= 4 * sms : max_page <= 32 && rows >= sms - sms / 4;
}

template <typename T, int MT>
int launch_kv8_attn(const Kv8AttnArgs &a, int blocks, cudaStream_t s) {
  const int rows = a.B * a.L.h_kv;
  // Eight warps a row; four (three blocks to a multiprocessor) for short rows when there are more than multiprocessors:
  // 256 rows of 640 tokens 12.4 us, 14.7 with eight; 256 rows of 2048 32.6, 30.7 with eight.
  if (kv8_by_row(rows, a.L.max_page))
    return a.L.max_page > 8 || rows <= blocks ? start_kv8_attn<T, MT, 8, true>(a, rows, s)
                                              : start_kv8_attn<T, MT, 4, true>(a, rows, s);
  const int rc = start_kv8_attn<T, MT, KV8_WARPS, false>(a, blocks, s);
  if (rc != KITTY_OK) return rc;
  // From 256 rows of about one length on a row has nine partials or fewer (1776 workers): folded by a warp each (1024 rows:
  // 5 us, 25 us as blocks).  Below, a block each: 1024 threads for a few rows of hundreds of partials (8 rows of 222: 9 us,
  // 16 us with 512 threads), 512 threads when there are more blocks than multiprocessors (64 rows of 28: 7 us, 11 us with
  // 1024).  The rule goes by the number of rows, which the host knows, not by their lengths: a long row among hundreds of
  // short ones has hundreds of partials that one warp folds (40 sequences, 8 heads, one of 131072 tokens and 39 of 500:
  // 120 us in all, 81 for as many tokens evenly spread; 256 rows, one of 131072: 157).
  const int heads = rows * a.G;
  cudaError_t e;
  if (rows >= 256) e = launch_after(kv8_join_rows_kernel<T>, dim3((heads + 7) / 8), dim3(256), 0, s, a);
  else if (heads > blocks) e = launch_after(kv8_join_kernel<T, 4>, dim3(heads), dim3(HD * 4), 0, s, a);
  else e = launch_after(kv8_join_kernel<T, 8>, dim3(heads), dim3(HD * 8), 0, s, a);
  return (e == cudaSuccess && cudaGetLastError() == cudaSuccess) ? KITTY_OK : KITTY_E_CUDA;
}

int64_t kv8_prefix_bytes(int B) { return (static_cast<int64_t>(B) + 1 + 3) / 4 * 16; }

}  // namespace kitty

using namespace kitty;

extern "C" int64_t kitty_kv8_workspace_bytes(int32_t B, int32_t h_kv, int32_t h_q, int32_t max_page) {
  if (B < 0 || h_kv <= 0 || h_q <= 0 || max_page <= 0 || h_q % h_kv != 0) return KITTY_E_BADARG;
  if (h_q / h_kv > MAX_GROUP || B > KITTY_KV8_MAX_BATCH) return KITTY_E_BADSHAPE;
  if (kv8_by_row(static_cast<int64_t>(B) * h_kv, max_page)) return 0;
  return kv8_prefix_bytes(B) + (KV8_WORKERS_MAX + static_cast<int64_t>(B) * h_kv) * (h_q / h_kv) * PART * 4;
}

extern "C" int kitty_kv8_attn(const kitty_kv8_layer *layer, const int32_t *lengths, const void *query, int32_t B,
                              int32_t h_q, float scaling, void *out, void *workspace, int64_t workspace_bytes,
                              void *stream) {
  const int rc = check_kv8_layer(layer);
  if (rc != KITTY_OK) return rc;
  const int64_t need = kitty_kv8_workspace_bytes(B, layer->h_kv, h_q, layer->max_page);
  if (need < 0) return static_cast<int>(need);
  if (B > layer->max_bs) return KITTY_E_BADARG;
  if (B == 0) return KITTY_OK;
  if (!lengths || !query || !out || (need > 0 && !workspace)) return KITTY_E_BADARG;
  if ((reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return KITTY_E_BADARG;
  if (workspace_bytes < need) return KITTY_E_WORKSPACE;
  const int64_t bytes = static_cast<int64_t>(B) * h_q * HD * 2;
  if (out != query && rows_meet({out, {1, 1, 1}, {}, bytes}, {query, {1, 1, 1}, {}, bytes})) return KITTY_E_OVERLAP;
  // units are counted in 32 bits
  if (static_cast<int64_t>(B) * layer->max_page * 4 > 0x7fffffff / layer->h_kv) return KITTY_E_BADSHAPE;
  const int sms = sm_count() < KV8_MAX_SMS ? sm_count() : KV8_MAX_SMS;
  Kv8AttnArgs a{};
  a.L = *layer;
  a.lengths = lengths;
  a.q = query;
  a.out = out;
  if (need > 0) {
    a.prefix = static_cast<int32_t *>(workspace);
    a.partials = reinterpret_cast<float *>(static_cast<char *>(workspace) + kv8_prefix_bytes(B));
  }
  a.scale_log2 = scaling * 1.4426950408889634f;
  a.B = B;
  a.G = h_q / layer->h_kv;
  a.workers = sms * KV8_WARPS;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (layer->dtype == KITTY_F16)
    return a.G > 8 ? launch_kv8_attn<__half, 2>(a, sms, s) : launch_kv8_attn<__half, 1>(a, sms, s);
  return a.G > 8 ? launch_kv8_attn<__nv_bfloat16, 2>(a, sms, s) : launch_kv8_attn<__nv_bfloat16, 1>(a, sms, s);
}
