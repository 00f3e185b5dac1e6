// Rotary positions of whole prompts and of single tokens: query and key heads in one launch.
//
// Bound by memory: every element is read once and written once (4 bytes of traffic per 16-bit element).  A block takes
// a few tokens of one sequence and many heads, computes the tokens' angle table once (the 64-bit products and the sine
// and cosine are shared by all heads) and streams the head rows through registers.
#include "rotary.cuh"

#include "decode.cuh"
#include "overlap.cuh"

namespace kitty {

struct RotArgs {
  kitty_rotary_plan pl;
  const void *in[2];
  void *out[2];
  int64_t is[2][3], os[2][3];      // element strides (batch, head, token) of query / key and of their outputs
  const int64_t *pos;
  int64_t pos_b;
  int32_t T, h_q, h_all, tt, hc, tiles;
};

constexpr int ROT_TOK = 8;         // tokens of a block's table

// LPR threads per head row, UPT units of a row per thread; each thread keeps ROWS rows in flight.
template <typename T, int MODE, int LPR, int UPT, int ROWS>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotArgs a) {
  using U = RotUnits<T, MODE>;
  __shared__ __align__(16) float2 tab[ROT_TOK][HD / 2];
  const int r = a.pl.rotary_dim, np = r / 2;
  const int b = blockIdx.x / a.tiles, t0 = (blockIdx.x % a.tiles) * a.tt;
  const int ntok = min(a.tt, a.T - t0);
  const int h0 = blockIdx.y * a.hc, nh = min(a.hc, a.h_all - h0);
  const int rows = ntok * nh;
  const int nt = U::turned(r), nu = nt + U::copied(r);
  const int lane = threadIdx.x % LPR, row0 = threadIdx.x / LPR;
  constexpr int STEP = 256 / LPR;

  auto locate = [&](int row, const T *&src, T *&dst, int &tok) {
    tok = row / nh;
    int h = h0 + row - tok * nh;
    const int s = h >= a.h_q;
    if (s) h -= a.h_q;
    const int64_t t = t0 + tok;
    src = static_cast<const T *>(a.in[s]) + b * a.is[s][0] + h * a.is[s][1] + t * a.is[s][2];
    dst = static_cast<T *>(a.out[s]) + b * a.os[s][0] + h * a.os[s][1] + t * a.os[s][2];
  };
  for (int i = threadIdx.x; i < ntok * np; i += 256) {
    const int tok = i / np, p = i - tok * np;
    tab[tok][RotTable<T, MODE>::slot(p, nt)] = rot_angle(a.pl, a.pos[b * a.pos_b + t0 + tok], p);
  }
  __syncthreads();
  for (int base = row0; base < rows; base += STEP * ROWS) {
    RotUnit<T, MODE> x[ROWS][UPT];
    T *dst[ROWS];
    int tok[ROWS];
    for (int u0 = lane; u0 < nu; u0 += LPR * UPT) {            // one pass, but for the scalar modes
#pragma unroll
      for (int j = 0; j < ROWS; ++j)
        if (base + j * STEP < rows) {
          const T *src;
          locate(base + j * STEP, src, dst[j], tok[j]);
#pragma unroll
          for (int k = 0; k < UPT; ++k)
            if (u0 + k * LPR < nu) x[j][k].load(src, u0 + k * LPR, r);
        }
#pragma unroll
      for (int j = 0; j < ROWS; ++j)
        if (base + j * STEP < rows) {
#pragma unroll
          for (int k = 0; k < UPT; ++k)
            if (u0 + k * LPR < nu) x[j][k].store(dst[j], u0 + k * LPR, r, RotTable<T, MODE>{tab[tok[j]], nt});
        }
    }
  }
}

template <typename T>
int launch_rotary(const RotArgs &a, dim3 grid, cudaStream_t s) {
  constexpr int LPR = sizeof(T) == 2 ? 8 : 16;
  switch (rot_mode(a.pl, sizeof(T))) {
    case ROT_HALF:
      // units of a full-width head: 8 (16 bit) or 16 (32 bit); a partly rotated head has up to twice as many
      if (a.pl.rotary_dim == HD) rotary_kernel<T, ROT_HALF, LPR, 1, 2><<<grid, 256, 0, s>>>(a);
      else rotary_kernel<T, ROT_HALF, LPR, 2, 2><<<grid, 256, 0, s>>>(a);
      break;
    case ROT_INTER: rotary_kernel<T, ROT_INTER, LPR, 2, 2><<<grid, 256, 0, s>>>(a); break;
    case ROT_HALF_SCALAR: rotary_kernel<T, ROT_HALF_SCALAR, 16, 2, 2><<<grid, 256, 0, s>>>(a); break;
    default: rotary_kernel<T, ROT_INTER_SCALAR, 16, 2, 2><<<grid, 256, 0, s>>>(a); break;
  }
  return cudaGetLastError() == cudaSuccess ? KITTY_OK : KITTY_E_CUDA;
}

}  // namespace kitty

using namespace kitty;

extern "C" int kitty_rows_overlap(const void *x, const int64_t *x_sizes, const int64_t *x_steps, const void *y,
                                  const int64_t *y_sizes, const int64_t *y_steps, int64_t run) {
  return rows_meet({x, {x_sizes[0], x_sizes[1], x_sizes[2]}, {x_steps[0], x_steps[1], x_steps[2]}, run},
                   {y, {y_sizes[0], y_sizes[1], y_sizes[2]}, {y_steps[0], y_steps[1], y_steps[2]}, run});
}

extern "C" int kitty_rotary(const kitty_rotary_plan *plan, const void *q, const void *k, const int64_t *positions,
                            int64_t pos_stride_b, void *q_out, void *k_out, int dtype, int32_t B, int32_t T,
                            int32_t h_q, int32_t h_kv, const int64_t *strides, void *stream) {
  const int rc = check_rotary_plan(plan);
  if (rc != KITTY_OK) return rc;
  if (!strides || B < 0 || T < 0 || h_q < 0 || h_kv < 0 || pos_stride_b < 0) return KITTY_E_BADARG;
  if (dtype < KITTY_F16 || dtype > KITTY_F32) return KITTY_E_BADARG;
  if (B == 0 || T == 0 || h_q + h_kv == 0) return KITTY_OK;
  if (!positions || (h_q && (!q || !q_out)) || (h_kv && (!k || !k_out))) return KITTY_E_BADARG;
  const int esize = dtype == KITTY_F32 ? 4 : 2;
  RotArgs a{};
  a.pl = *plan;
  const void *in[2] = {q, k};
  void *out[2] = {q_out, k_out};
  for (int s = 0; s < 2; ++s) {
    a.in[s] = in[s];
    a.out[s] = out[s];
    if ((reinterpret_cast<uintptr_t>(in[s]) | reinterpret_cast<uintptr_t>(out[s])) & 15) return KITTY_E_BADARG;
    for (int i = 0; i < 3; ++i) {
      a.is[s][i] = strides[s * 3 + i];
      a.os[s][i] = strides[6 + s * 3 + i];
      if ((s ? h_kv : h_q) != 0 && ((a.is[s][i] * esize) % 16 != 0 || (a.os[s][i] * esize) % 16 != 0)) return KITTY_E_BADARG;
    }
  }
  Rows rows[2][2];                 // [query, key][in, out]
  for (int s = 0; s < 2; ++s) {
    const int64_t h = s ? h_kv : h_q;
    for (int o = 0; o < 2; ++o) {
      const int64_t *st = strides + 3 * s + 6 * o;
      rows[s][o] = {o ? a.out[s] : a.in[s], {B, h, T}, {st[0] * esize, st[1] * esize, st[2] * esize}, HD * esize};
    }
  }
  for (int s = 0; s < 2; ++s)
    if ((!same_rows(rows[s][1], rows[s][0]) && rows_meet(rows[s][1], rows[s][0])) || rows_meet(rows[s][1], rows[1 - s][0]))
      return KITTY_E_OVERLAP;
  if (rows_meet(rows[0][1], rows[1][1])) return KITTY_E_OVERLAP;
  a.pos = positions;
  a.pos_b = pos_stride_b;
  a.T = T;
  a.h_q = h_q;
  a.h_all = h_q + h_kv;
  a.tt = T < ROT_TOK ? T : ROT_TOK;
  a.tiles = static_cast<int32_t>((static_cast<int64_t>(T) + a.tt - 1) / a.tt);
  const int64_t blocks = static_cast<int64_t>(B) * a.tiles;
  if (blocks > 0x7fffffff) return KITTY_E_BADSHAPE;
  // Few tokens: spread the heads over blocks too, at least four heads each.
  int split = 1;
  const int want = 2 * sm_count();
  if (blocks < want) split = static_cast<int>((want + blocks - 1) / blocks);
  const int most = (a.h_all + 3) / 4;
  if (split > most) split = most;
  a.hc = (a.h_all + split - 1) / split;
  split = (a.h_all + a.hc - 1) / a.hc;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(split));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == KITTY_F16) return launch_rotary<__half>(a, grid, s);
  if (dtype == KITTY_BF16) return launch_rotary<__nv_bfloat16>(a, grid, s);
  return launch_rotary<float>(a, grid, s);
}
