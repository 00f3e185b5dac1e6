// Decode attention over the 8-bit cache: one query token per sequence.
//
// Bound by memory (256 B of codes per token and key head against 4 * group * 128 operations), so the kernel is built
// around an even, uninterrupted stream.  The blocks of 32 tokens of all (sequence, key head) rows form one long line of
// units; every warp of a grid that fills the machine takes an equal, contiguous stretch of it, whatever the lengths
// (they are read on the device, so a captured launch stays valid as sequences grow).  A warp keeps a ring of block
// records in flight with bulk copies (one 8208-byte copy per unit) and needs no other warp until the end.  A row that
// several warps share is joined by a second kernel from their (accumulator, maximum, sum) partials, in a fixed order.
//
// Arithmetic of a unit: 16 matrix rows = query heads, contraction over 16 channels or 16 tokens at a time
// (mma.m16n8k16, fp16 operands, 32-bit sums).  A code byte becomes the fp16 number 1024 + byte by placing it in the low
// mantissa bits; subtracting 1152 leaves the whole number exactly.  Records hold the bytes in operand order, so every
// shared-memory read is one conflict-free 16-byte word per lane, and no transposing step is needed anywhere.  The key
// scale multiplies the block's logits, the value scale the block's products, both in 32 bits.
// The tensor units need neither tcgen05 nor shared-memory operands here: 16 of 128 tile rows would be used, and the
// operands are made in registers.
#include "kv8.cuh"
#include "paged_core.cuh"

namespace kitty {

constexpr int KV8_WARPS = 8;            // per block of threads, one block per multiprocessor
constexpr int KV8_STAGES = 3;
constexpr int KV8_MAX_SMS = 160;        // the workspace is sized for this many
constexpr int KV8_WORKERS_MAX = KV8_MAX_SMS * KV8_WARPS;

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

__device__ __forceinline__ int64_t kv8_first_unit(int64_t w, int64_t units, int64_t workers) { return w * units / workers; }
__device__ __forceinline__ int64_t kv8_worker_of(int64_t u, int64_t units, int64_t workers) {
  return ((u + 1) * workers - 1) / units;
}

// Two code bytes of a word (sel 0x4140: bytes 0, 1; 0x4342: bytes 2, 3) as exact fp16 whole numbers.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t code2(uint32_t w) {
  const uint32_t r = __byte_perm(w, 0x64646464u, SEL);
  const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&r), __float2half2_rn(1152.0f));
  return *reinterpret_cast<const uint32_t *>(&d);
}

__device__ __forceinline__ void mma16816_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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
  const int32_t *lengths;
  int cap;
  __device__ __forceinline__ void enter(const int32_t *prefix) {
    nblk = prefix[b + 1] - prefix[b];
    len = max(0, min(lengths[b], cap));
  }
  __device__ __forceinline__ int tokens() const { return min(KV8_BLOCK, len - blk * KV8_BLOCK); }
  __device__ __forceinline__ void seek(int64_t u, const int32_t *prefix, int B, int H) {
    // prefix[b] * H <= u < prefix[b + 1] * H
    int lo = 0, hi = B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (static_cast<int64_t>(prefix[mid]) * H <= u) lo = mid;
      else hi = mid;
    }
    b = lo;
    enter(prefix);
    const int64_t rest = u - static_cast<int64_t>(prefix[b]) * H;
    h = static_cast<int>(rest / nblk);
    blk = static_cast<int>(rest % nblk);
  }
  // true when the next unit belongs to another row
  __device__ __forceinline__ bool next(const int32_t *prefix, int B, int H) {
    if (++blk < nblk) return false;
    blk = 0;
    if (++h == H) {
      h = 0;
      do {
        ++b;
      } while (b < B && prefix[b + 1] == prefix[b]);
      if (b < B) enter(prefix);
    }
    return true;
  }
};

// MT: 1 for groups of up to 8 query heads (matrix rows 8..15 idle), 2 for up to 16.
template <typename T, int MT>
__global__ void __launch_bounds__(KV8_WARPS * 32, 1) kv8_attn_kernel(const __grid_constant__ Kv8AttnArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[KV8_WARPS][KV8_STAGES];
  __shared__ int32_t scan[KV8_WARPS];
  __shared__ int32_t skipped[KV8_WARPS][KV8_STAGES];      // stages without a record
  uint8_t *ring_all = smem;
  int32_t *prefix = reinterpret_cast<int32_t *>(smem + KV8_WARPS * KV8_STAGES * KV8_REC);
  const kitty_kv8_layer &L = a.L;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int H = L.h_kv, B = a.B, G = a.G;

  if (lane == 0) {
    for (int s = 0; s < KV8_STAGES; ++s) mbar_init(smem_u32(&bars[warp][s]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  dep_wait();
  // units before each sequence: every block of threads scans the lengths
  {
    const int per = (B + KV8_WARPS * 32 - 1) / (KV8_WARPS * 32), i0 = min(B, per * static_cast<int>(threadIdx.x));
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
      for (int i = threadIdx.x; i <= B; i += KV8_WARPS * 32) a.prefix[i] = prefix[i];
  }
  dep_release();
  const int64_t units = static_cast<int64_t>(prefix[B]) * H;
  const int64_t worker = static_cast<int64_t>(blockIdx.x) * KV8_WARPS + warp;
  if (units == 0) return;
  const int64_t u0 = kv8_first_unit(worker, units, a.workers), u1 = kv8_first_unit(worker + 1, units, a.workers);
  if (u0 >= u1) return;

  const uint32_t ring = smem_u32(ring_all) + warp * KV8_STAGES * KV8_REC;
  const uint8_t *ring_p = ring_all + warp * KV8_STAGES * KV8_REC;
  // request the record of a unit; an open block has none (its 16-bit tokens are read when their turn comes)
  auto request = [&](const Kv8Cursor &c, int stage) {
    if (lane == 0) {
      const uint32_t bar = smem_u32(&bars[warp][stage]);
      const int64_t page = c.tokens() == KV8_BLOCK ? kv8_page(L, c.b, c.blk) : -1;
      skipped[warp][stage] = page < 0;
      if (page >= 0) {
        mbar_expect_tx(bar, KV8_REC);
        bulk_g2s(ring + stage * KV8_REC, kv8_record(L, page, c.h, c.blk & 3), KV8_REC, bar);
      } else {
        mbar_expect_tx(bar, 0);
      }
    }
  };
  Kv8Cursor cur, ahead;
  cur.lengths = a.lengths;
  cur.cap = L.max_page * PAGE;
  cur.seek(u0, prefix, B, H);
  ahead = cur;
  int64_t ua = u0;
  for (int s = 0; s < KV8_STAGES; ++s)
    if (ua < u1) {
      request(ahead, s);
      ahead.next(prefix, B, H);
      ++ua;
    }

  uint32_t qa[8][4];          // query heads as matrix rows g (and g + 8), fp16, scaled by a power of two
  float acc[16][2 * MT], mx[MT], sum[MT], qs[MT];
  bool fresh = true;
  int stage = 0, phase = 0;
  for (int64_t u = u0; u < u1; ++u) {
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int head = g + 8 * m;
        uint4 w[4] = {};
        if (head < G) {
          const T *qp = static_cast<const T *>(a.q) + (static_cast<int64_t>(cur.b) * H * G + cur.h * G + head) * HD + 16 * t;
#pragma unroll
          for (int c = 0; c < 4; ++c) w[c] = *reinterpret_cast<const uint4 *>(qp + (c >> 1) * 64 + (c & 1) * 8);
        }
        // a power of two brings the row's largest element to [1, 2): bf16 values then fit fp16 exactly, except those
        // 2^-14 and more below the largest, which lose low bits that are 2^-24 of it at most
        float top = 0.0f;
        float x[4][8];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          Vec8<T>::unpack(w[c], x[c]);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[c][e]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
        ex = max(-100, min(100, ex));
        const float down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
        qs[m] = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const float *z = &x[ks >> 1][(ks & 1) * 4];
          qa[ks][m] = pack_h2(z[0] * down, z[1] * down);
          qa[ks][2 + m] = pack_h2(z[2] * down, z[3] * down);
          if (MT == 1) qa[ks][1] = qa[ks][3] = 0;
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
    const uint32_t bar = smem_u32(&bars[warp][stage]);
    if (!mbar_wait(bar, phase)) {
      if (lane == 0) atomicOr(L.status, KITTY_KV8_TIMEOUT);
      for (int64_t v = u; v < ua; ++v) {          // leave no copy of this warp in flight behind
        mbar_wait(smem_u32(&bars[warp][stage]), phase);
        if (++stage == KV8_STAGES) stage = 0, phase ^= 1;
      }
      return;
    }
    float p[4][2 * MT];           // logits, then weights: tile i, columns 2t, 2t+1 of rows g (and g + 8)
    const uint8_t *rec = ring_p + stage * KV8_REC;
    const bool packed = cnt == KV8_BLOCK;
    const bool valid = !packed || skipped[warp][stage] == 0;
    float vscale = 1.0f;
    if (packed) {
      const float2 sc = *reinterpret_cast<const float2 *>(rec + KV8_OFF_SCALE);
      vscale = sc.y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float c[4];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint4 w4 = *reinterpret_cast<const uint4 *>(rec + i * 1024 + hf * 512 + lane * 16);
          const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t b0 = code2<0x4140>(w[j]), b1 = code2<0x4342>(w[j]);
            if (hf == 0 && j == 0) mma16816_zero(c, qa[0], b0, b1);
            else mma16816(c, qa[4 * hf + j][0], qa[4 * hf + j][1], qa[4 * hf + j][2], qa[4 * hf + j][3], b0, b1);
          }
        }
#pragma unroll
        for (int e = 0; e < 2 * MT; ++e) p[i][e] = c[e] * (sc.x * qs[e >> 1]);
      }
    } else {
      // open block: 16-bit keys straight from memory, the query in its own type
      const int64_t at = ((static_cast<int64_t>(cur.b) * H + cur.h) * KV8_BLOCK) * HD;
      const T *kt = static_cast<const T *>(L.tail_k) + at;
      const T *qp = static_cast<const T *>(a.q) + (static_cast<int64_t>(cur.b) * H * G + cur.h * G) * HD + 16 * t;
      float c[4][4] = {};
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        const int off = (ch >> 1) * 64 + (ch & 1) * 8;
        uint4 q0 = {}, q1 = {};
        if (g < G) q0 = *reinterpret_cast<const uint4 *>(qp + g * HD + off);
        if (MT == 2 && g + 8 < G) q1 = *reinterpret_cast<const uint4 *>(qp + (g + 8) * HD + off);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tk = kv8_key_token(i, g);
          uint4 k4 = {};
          if (tk < cnt) k4 = *reinterpret_cast<const uint4 *>(kt + tk * HD + 16 * t + off);
          mma_t<T>(c[i], q0.x, q1.x, q0.y, q1.y, k4.x, k4.y);
          mma_t<T>(c[i], q0.z, q1.z, q0.w, q1.w, k4.z, k4.w);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2 * MT; ++e)
          p[i][e] = 8 * t + 2 * i + (e & 1) < cnt ? c[i][e] * a.scale_log2 : -INFINITY;
    }
    if (!valid) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2 * MT; ++e) p[i][e] = -INFINITY;
      vscale = 0.0f;
    }
    // running maximum and sum (base 2)
    float corr[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(p[i][2 * m], p[i][2 * m + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float mn = fmaxf(mx[m], top);
      const float ref = mn == -INFINITY ? 0.0f : mn;
      corr[m] = ex2(mx[m] - ref);
      mx[m] = mn;
      float add = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i][2 * m] = ex2(p[i][2 * m] - ref);
        p[i][2 * m + 1] = ex2(p[i][2 * m + 1] - ref);
        add += p[i][2 * m] + p[i][2 * m + 1];
      }
      sum[m] = sum[m] * corr[m] + add;
    }
    bool moved = corr[0] != 1.0f;
    if (MT == 2) moved |= corr[MT - 1] != 1.0f;
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < 16; ++n)
#pragma unroll
        for (int e = 0; e < 2 * MT; ++e) acc[n][e] *= corr[e >> 1];
    }
    if (packed) {
      uint32_t pa[2][4];        // weights as matrix rows, 16 tokens each
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        pa[s][0] = pack_h2(p[2 * s][0], p[2 * s][1]);
        pa[s][2] = pack_h2(p[2 * s + 1][0], p[2 * s + 1][1]);
        pa[s][1] = MT == 2 ? pack_h2(p[2 * s][2 * MT - 2], p[2 * s][2 * MT - 1]) : 0;
        pa[s][3] = MT == 2 ? pack_h2(p[2 * s + 1][2 * MT - 2], p[2 * s + 1][2 * MT - 1]) : 0;
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const uint4 w4 = *reinterpret_cast<const uint4 *>(rec + KV8_OFF_V + x * 512 + lane * 16);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float c[4];
          mma16816_zero(c, pa[0], code2<0x4140>(w[2 * y]), code2<0x4342>(w[2 * y]));
          mma16816(c, pa[1][0], pa[1][1], pa[1][2], pa[1][3], code2<0x4140>(w[2 * y + 1]), code2<0x4342>(w[2 * y + 1]));
#pragma unroll
          for (int e = 0; e < 2 * MT; ++e) acc[2 * x + y][e] = fmaf(vscale, c[e], acc[2 * x + y][e]);
        }
      }
    } else {
      // 16-bit values of the open block; weights as a sum of two 16-bit numbers, so that the bf16 form loses nothing
      const int64_t at = ((static_cast<int64_t>(cur.b) * H + cur.h) * KV8_BLOCK) * HD;
      const T *vp = static_cast<const T *>(L.tail_v) + at;
      uint32_t hi[4][MT], lo[4][MT];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const float p0 = p[i][2 * m], p1 = p[i][2 * m + 1];
          const float r0 = to_f32<T>(from_f32<T>(p0)), r1 = to_f32<T>(from_f32<T>(p1));
          hi[i][m] = pack_t<T>(r0, r1);
          lo[i][m] = pack_t<T>(p0 - r0, p1 - r1);
        }
#pragma unroll 4
      for (int n = 0; n < 16; ++n) {
        float c[4] = {};
        uint32_t bv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tk = 8 * t + 2 * i;
          uint16_t e0 = 0, e1 = 0;
          if (tk < cnt) e0 = *reinterpret_cast<const uint16_t *>(vp + tk * HD + 8 * n + g);
          if (tk + 1 < cnt) e1 = *reinterpret_cast<const uint16_t *>(vp + (tk + 1) * HD + 8 * n + g);
          bv[i] = e0 | static_cast<uint32_t>(e1) << 16;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          mma_t<T>(c, hi[2 * s][0], MT == 2 ? hi[2 * s][MT - 1] : 0, hi[2 * s + 1][0], MT == 2 ? hi[2 * s + 1][MT - 1] : 0,
                   bv[2 * s], bv[2 * s + 1]);
          mma_t<T>(c, lo[2 * s][0], MT == 2 ? lo[2 * s][MT - 1] : 0, lo[2 * s + 1][0], MT == 2 ? lo[2 * s + 1][MT - 1] : 0,
                   bv[2 * s], bv[2 * s + 1]);
        }
#pragma unroll
        for (int n2 = 0; n2 < 16; ++n2)
          if (n2 == n) {
#pragma unroll
            for (int e = 0; e < 2 * MT; ++e) acc[n2][e] += c[e];
          }
      }
    }
    // the stage is read: request the unit that comes KV8_STAGES later into it
    __syncwarp();
    if (ua < u1) {
      request(ahead, stage);
      ahead.next(prefix, B, H);
      ++ua;
    }
    if (++stage == KV8_STAGES) stage = 0, phase ^= 1;
    const int row = cur.b * H + cur.h;
    const bool ends = cur.next(prefix, B, H);
    if (ends || u + 1 == u1) {
      fresh = true;
      float *dst = a.partials + (worker + row) * G * PART;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float s = sum[m];
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        const int head = g + 8 * m;
        if (head < G) {
          float *o = dst + head * PART;
#pragma unroll
          for (int n = 0; n < 16; ++n)
            *reinterpret_cast<float2 *>(o + 8 * n + 2 * t) = make_float2(acc[n][2 * m], acc[n][2 * m + 1]);
          if (t == 0) *reinterpret_cast<float2 *>(o + HD) = make_float2(mx[m], s);
        }
      }
    }
  }
}

// Joins the partials of one (sequence, query head): four groups of 128 threads, a channel each, take every fourth
// partial; weights 2^(max - largest max) in 32 bits.
template <typename T>
__global__ void __launch_bounds__(512) kv8_join_kernel(const __grid_constant__ Kv8AttnArgs a) {
  __shared__ float red[4][HD], ms[4][2];
  const int H = a.L.h_kv, G = a.G, hq = H * G;
  const int b = blockIdx.x / hq, head = blockIdx.x % hq, h = head / G;
  const int c = threadIdx.x & 127, grp = threadIdx.x >> 7;
  dep_wait();
  dep_release();
  const int64_t units = static_cast<int64_t>(a.prefix[a.B]) * H;
  const int64_t before = static_cast<int64_t>(a.prefix[b]) * H, nblk = a.prefix[b + 1] - a.prefix[b];
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  if (nblk > 0) {
    const int64_t f = before + h * nblk;
    const int64_t w0 = kv8_worker_of(f, units, a.workers), w1 = kv8_worker_of(f + nblk - 1, units, a.workers);
    const float *p = a.partials + ((b * static_cast<int64_t>(H) + h) * G + head % G) * PART;
    const int64_t step = static_cast<int64_t>(G) * PART;
    for (int64_t w = w0 + grp; w <= w1; w += 16) {       // four of the group's partials at once
      float pm[4], pl[4], pv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t wj = w + 4 * j;
        pm[j] = -INFINITY;
        pl[j] = pv[j] = 0.0f;
        // a worker without units has no partial
        if (wj <= w1 && kv8_first_unit(wj, units, a.workers) < kv8_first_unit(wj + 1, units, a.workers)) {
          const float *o = p + wj * step;
          const float2 x = *reinterpret_cast<const float2 *>(o + HD);
          pm[j] = x.x;
          pl[j] = x.y;
          pv[j] = o[c];
        }
      }
      float mn = m;
#pragma unroll
      for (int j = 0; j < 4; ++j) mn = fmaxf(mn, pm[j]);
      const float ref = mn == -INFINITY ? 0.0f : mn;
      const float f0 = ex2(m - ref);
      l *= f0;
      acc *= f0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float wgt = ex2(pm[j] - ref);
        l = fmaf(pl[j], wgt, l);
        acc = fmaf(pv[j], wgt, acc);
      }
      m = mn;
    }
  }
  red[grp][c] = acc;
  if (c == 0) ms[grp][0] = m, ms[grp][1] = l;
  __syncthreads();
  if (grp != 0) return;
  float mn = fmaxf(fmaxf(ms[0][0], ms[1][0]), fmaxf(ms[2][0], ms[3][0]));
  if (mn == -INFINITY) mn = 0.0f;
  float tot = 0.0f, ls = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float wgt = ex2(ms[i][0] - mn);
    tot = fmaf(red[i][c], wgt, tot);
    ls = fmaf(ms[i][1], wgt, ls);
  }
  static_cast<T *>(a.out)[static_cast<int64_t>(blockIdx.x) * HD + c] = from_f32<T>(nblk > 0 ? tot / ls : 0.0f);
}

template <typename T, int MT>
int launch_kv8_attn(const Kv8AttnArgs &a, int blocks, int smem, cudaStream_t s) {
  static PerDeviceOnce once;
  const int rc = per_device_once(once, [] {
    return cudaFuncSetAttribute(kv8_attn_kernel<T, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                KV8_WARPS * KV8_STAGES * KV8_REC + (KITTY_KV8_MAX_BATCH + 1) * 4) == cudaSuccess
               ? KITTY_OK
               : KITTY_E_CUDA;
  });
  if (rc != KITTY_OK) return rc;
  kv8_attn_kernel<T, MT><<<blocks, KV8_WARPS * 32, smem, s>>>(a);
  if (cudaGetLastError() != cudaSuccess) return KITTY_E_CUDA;
  const cudaError_t e = launch_after(kv8_join_kernel<T>, dim3(a.B * a.L.h_kv * a.G), dim3(512), 0, s, a);
  return (e == cudaSuccess && cudaGetLastError() == cudaSuccess) ? KITTY_OK : KITTY_E_CUDA;
}

int64_t kv8_prefix_bytes(int B) { return (static_cast<int64_t>(B) + 1 + 3) / 4 * 16; }

}  // namespace kitty

using namespace kitty;

extern "C" int64_t kitty_kv8_workspace_bytes(int32_t B, int32_t h_kv, int32_t h_q) {
  if (B < 0 || h_kv <= 0 || h_q <= 0 || h_q % h_kv != 0) return KITTY_E_BADARG;
  if (h_q / h_kv > MAX_GROUP || B > KITTY_KV8_MAX_BATCH) return KITTY_E_BADSHAPE;
  return kv8_prefix_bytes(B) + (KV8_WORKERS_MAX + static_cast<int64_t>(B) * h_kv) * (h_q / h_kv) * PART * 4;
}

extern "C" int kitty_kv8_attn(const kitty_kv8_layer *layer, const int32_t *lengths, const void *query, int32_t B,
                              int32_t h_q, float scaling, void *out, void *workspace, int64_t workspace_bytes,
                              void *stream) {
  const int rc = check_kv8_layer(layer);
  if (rc != KITTY_OK) return rc;
  const int64_t need = kitty_kv8_workspace_bytes(B, layer->h_kv, h_q);
  if (need < 0) return static_cast<int>(need);
  if (B > layer->max_bs) return KITTY_E_BADARG;
  if (B == 0) return KITTY_OK;
  if (!lengths || !query || !out || !workspace) return KITTY_E_BADARG;
  if ((reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return KITTY_E_BADARG;
  if (workspace_bytes < need) return KITTY_E_WORKSPACE;
  // units are counted in 32 bits per head
  if (static_cast<int64_t>(B) * layer->max_page * 4 > 0x7fffffff) return KITTY_E_BADSHAPE;
  const int sms = sm_count() < KV8_MAX_SMS ? sm_count() : KV8_MAX_SMS;
  Kv8AttnArgs a{};
  a.L = *layer;
  a.lengths = lengths;
  a.q = query;
  a.out = out;
  a.prefix = static_cast<int32_t *>(workspace);
  a.partials = reinterpret_cast<float *>(static_cast<char *>(workspace) + kv8_prefix_bytes(B));
  a.scale_log2 = scaling * 1.4426950408889634f;
  a.B = B;
  a.G = h_q / layer->h_kv;
  a.workers = sms * KV8_WARPS;
  const int smem = KV8_WARPS * KV8_STAGES * KV8_REC + (B + 1) * 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (layer->dtype == KITTY_F16)
    return a.G > 8 ? launch_kv8_attn<__half, 2>(a, sms, smem, s) : launch_kv8_attn<__half, 1>(a, sms, smem, s);
  return a.G > 8 ? launch_kv8_attn<__nv_bfloat16, 2>(a, sms, smem, s) : launch_kv8_attn<__nv_bfloat16, 1>(a, sms, smem, s);
}
