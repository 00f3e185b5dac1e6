// Rotary positions: the angle table of a few tokens and the rotation of one head row.
//
// Pair p of a head (p < rotary_dim / 2) is turned by angle = position * w_p:
//   (x1, x2) -> factor * (x1 cos - x2 sin, x2 cos + x1 sin)
// with channels (p, p + rotary_dim/2) ("half") or (2p, 2p + 1) ("interleaved"); channels from rotary_dim on keep
// their value.  The plan holds w_p in TURNS per position (w_p / 2 pi, 64 bits): position * turns loses its whole part
// exactly in 64 bits, and an angle is off by 2^-51 of the position times w at most (a 32-bit product is off by 0.004 rad
// at position 100000).  Sine and cosine are 64-bit too: those of the position's multiple of eight are computed, those of
// the rest come from the plan's table of eight small steps and are turned on with four multiplications.  (A table of 32
// steps has a block of 32 tokens compute a quarter of the sines, but in a quarter of its threads and with four times the
// loads: 4 x 4096 tokens appended in 27.8 us against 26.9 from a cold L2.)  Both, times the plan's factor, round to 32 bits
// once, to half a step; a factor other than 1 is itself a 32-bit number, half a step off at most.  (With 32-bit sines the
// turned keys were off by up to 2^-22, and four times as many of them fell on the other side of a rounding to 16 bits as
// with exact ones.)  The rotation itself is two fused multiply-adds in 32 bits, rounded once to the data type.
#pragma once

#include "common.cuh"

namespace kitty {

enum RotMode { ROT_HALF = 0, ROT_INTER = 1, ROT_HALF_SCALAR = 2, ROT_INTER_SCALAR = 3, ROT_NONE = 4 };

// How a head row is cut into units: a unit of the vector modes is one 16-byte piece (interleaved) or the two pieces
// that hold both halves of its pairs (half); scalar modes take one pair per unit (rotary_dim that does not split into
// whole pieces).  Channels from rotary_dim on are copied: one by one up to the next piece, then piece by piece.
template <typename T, int MODE>
struct RotUnits {
  static constexpr int V = 16 / sizeof(T);                       // channels of a piece
  static constexpr int PV = MODE == ROT_HALF ? V : MODE == ROT_INTER ? V / 2 : 1;   // pairs of a unit
  static constexpr bool VEC = MODE == ROT_HALF || MODE == ROT_INTER;
  static __device__ __forceinline__ int turned(int r) { return r / 2 / PV; }        // units that turn pairs
  static __device__ __forceinline__ int loose(int r) { return VEC ? 0 : (V - r % V) % V; }      // channels copied singly
  static __device__ __forceinline__ int copied(int r) { return loose(r) + (HD - r) / V; }
};

// The angle table of a block of threads in the order of the rotary kernel's units: token by token (64 entries each), the
// pairs of all units two by two, so that a row of threads reads consecutive 16-byte words.
template <typename T, int MODE>
struct RotTable {
  using U = RotUnits<T, MODE>;
  const float2 *tab;       // the token's entries
  int nt;
  static __device__ __forceinline__ int slot(int p, int nt) {
    if (U::PV == 1) return p;
    const int u = p / U::PV, e = p % U::PV;
    return ((e >> 1) * nt + u) * 2 + (e & 1);
  }
  // pairs 2k and 2k + 1 of unit u
  __device__ __forceinline__ float4 two(int u, int k) const { return *reinterpret_cast<const float4 *>(tab + (k * nt + u) * 2); }
  __device__ __forceinline__ float2 one(int p) const { return tab[p]; }
};

constexpr int ROT_STEPS = 8;

// Factor times cosine and sine of pair p at a multiple of eight, and with the remaining steps turned on.
__device__ __forceinline__ double2 rot_base(const kitty_rotary_plan &pl, int64_t pos, int p) {
  double t = static_cast<double>(pos) * pl.turns[p];
  t -= rint(t);
  double s, c;
  sincospi(t + t, &s, &c);
  return make_double2(c * pl.factor, s * pl.factor);
}
__device__ __forceinline__ float2 rot_step(const kitty_rotary_plan &pl, double2 base, int step, int p) {
  const double2 z = reinterpret_cast<const double2 *>(pl.steps)[step * (pl.rotary_dim / 2) + p];
  return make_float2(static_cast<float>(fma(base.x, z.x, -base.y * z.y)), static_cast<float>(fma(base.y, z.x, base.x * z.y)));
}
__device__ __forceinline__ float2 rot_angle(const kitty_rotary_plan &pl, int64_t pos, int p) {
  const int step = static_cast<int>(pos & (ROT_STEPS - 1));
  return rot_step(pl, rot_base(pl, pos - step, p), step, p);
}

template <typename T>
struct Piece {          // 16 bytes as 32-bit floats
  static constexpr int V = 16 / sizeof(T);
  float f[V];
  __device__ __forceinline__ void unpack(uint4 w) {
    if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
    } else {
      Vec8<T>::unpack(w, f);
    }
  }
  __device__ __forceinline__ uint4 pack() const {
    uint4 w;
    T *t = reinterpret_cast<T *>(&w);
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = from_f32<T>(f[i]);
    return w;
  }
};

// One unit of a head row in flight: load() requests its channels, store() turns them by the token's table row and
// writes them.  `row` / `out` may be the same memory: a unit reads all it needs before it writes, and units are
// disjoint.
template <typename T, int MODE>
struct RotUnit {
  using U = RotUnits<T, MODE>;
  uint4 a, b;
  T s0, s1;

  __device__ __forceinline__ void load(const T *row, int u, int r) {
    const int nt = U::turned(r);
    if constexpr (U::VEC) {
      if (u < nt) {
        const T *p = row + (MODE == ROT_HALF ? u * U::V : 2 * u * U::PV);
        a = *reinterpret_cast<const uint4 *>(p);
        if constexpr (MODE == ROT_HALF) b = *reinterpret_cast<const uint4 *>(p + r / 2);
      } else {
        a = *reinterpret_cast<const uint4 *>(row + r + (u - nt) * U::V);
      }
    } else {
      if (u < nt) {
        s0 = row[MODE == ROT_HALF_SCALAR ? u : 2 * u];
        s1 = row[MODE == ROT_HALF_SCALAR ? u + r / 2 : 2 * u + 1];
      } else if (u < nt + U::loose(r)) {
        s0 = row[r + (u - nt)];
      } else {
        a = *reinterpret_cast<const uint4 *>(row + r + U::loose(r) + (u - nt - U::loose(r)) * U::V);
      }
    }
  }
  template <typename Table>
  __device__ __forceinline__ void store(T *out, int u, int r, const Table &tab) const {
    const int nt = U::turned(r);
    if constexpr (MODE == ROT_HALF) {
      if (u < nt) {
        Piece<T> x, y;
        x.unpack(a);
        y.unpack(b);
#pragma unroll
        for (int e = 0; e < U::V; e += 2) {
          const float4 cs = tab.two(u, e >> 1);
          const float x0 = x.f[e], y0 = y.f[e], x1 = x.f[e + 1], y1 = y.f[e + 1];
          x.f[e] = fmaf(x0, cs.x, -y0 * cs.y);
          y.f[e] = fmaf(y0, cs.x, x0 * cs.y);
          x.f[e + 1] = fmaf(x1, cs.z, -y1 * cs.w);
          y.f[e + 1] = fmaf(y1, cs.z, x1 * cs.w);
        }
        *reinterpret_cast<uint4 *>(out + u * U::V) = x.pack();
        *reinterpret_cast<uint4 *>(out + u * U::V + r / 2) = y.pack();
      } else {
        *reinterpret_cast<uint4 *>(out + r + (u - nt) * U::V) = a;
      }
    } else if constexpr (MODE == ROT_INTER) {
      if (u < nt) {
        Piece<T> x;
        x.unpack(a);
#pragma unroll
        for (int e = 0; e < U::PV; e += 2) {
          const float4 cs = tab.two(u, e >> 1);
          const float x0 = x.f[2 * e], x1 = x.f[2 * e + 1], x2 = x.f[2 * e + 2], x3 = x.f[2 * e + 3];
          x.f[2 * e] = fmaf(x0, cs.x, -x1 * cs.y);
          x.f[2 * e + 1] = fmaf(x1, cs.x, x0 * cs.y);
          x.f[2 * e + 2] = fmaf(x2, cs.z, -x3 * cs.w);
          x.f[2 * e + 3] = fmaf(x3, cs.z, x2 * cs.w);
        }
        *reinterpret_cast<uint4 *>(out + u * U::V) = x.pack();
      } else {
        *reinterpret_cast<uint4 *>(out + r + (u - nt) * U::V) = a;
      }
    } else {
      if (u < nt) {
        const float2 cs = tab.one(u);
        const float x0 = to_f32<T>(s0), x1 = to_f32<T>(s1);
        out[MODE == ROT_HALF_SCALAR ? u : 2 * u] = from_f32<T>(fmaf(x0, cs.x, -x1 * cs.y));
        out[MODE == ROT_HALF_SCALAR ? u + r / 2 : 2 * u + 1] = from_f32<T>(fmaf(x1, cs.x, x0 * cs.y));
      } else if (u < nt + U::loose(r)) {
        out[r + (u - nt)] = s0;
      } else {
        *reinterpret_cast<uint4 *>(out + r + U::loose(r) + (u - nt - U::loose(r)) * U::V) = a;
      }
    }
  }
};

// Mode of a plan for elements of `esize` bytes.
inline int rot_mode(const kitty_rotary_plan &p, int esize) {
  const int v = 16 / esize;
  if (p.layout == KITTY_ROPE_HALF) return p.rotary_dim % (2 * v) == 0 ? ROT_HALF : ROT_HALF_SCALAR;
  return p.rotary_dim % v == 0 ? ROT_INTER : ROT_INTER_SCALAR;
}

inline int check_rotary_plan(const kitty_rotary_plan *p) {
  if (p == nullptr || p->turns == nullptr || p->steps == nullptr) return KITTY_E_BADARG;
  if (reinterpret_cast<uintptr_t>(p->steps) & 15) return KITTY_E_BADARG;
  if (p->rotary_dim < 2 || p->rotary_dim > HD || p->rotary_dim % 2 != 0) return KITTY_E_BADSHAPE;
  if (p->layout != KITTY_ROPE_HALF && p->layout != KITTY_ROPE_INTERLEAVED) return KITTY_E_BADARG;
  return KITTY_OK;
}

}  // namespace kitty
