// Block records of the 8-bit cache (layout in the public header) and the conversions of its codes.
#pragma once

#include "common.cuh"

namespace kitty {

constexpr int KV8_BLOCK = KITTY_KV8_BLOCK;      // tokens that share a scale
constexpr int KV8_REC = KITTY_KV8_RECORD;
constexpr int KV8_OFF_V = KV8_BLOCK * HD;       // 4096
constexpr int KV8_OFF_SCALE = 2 * KV8_OFF_V;    // 8192: key scale, value scale

// Token of key piece (i, lane group g): pieces of equal i hold the eight tokens whose logits one 8-column matrix tile
// produces, and the tokens of value byte 2i + e of lane t (8t + 2i + e) are the ones that land in that lane's columns.
__host__ __device__ constexpr int kv8_key_token(int i, int g) { return 8 * (g >> 1) + 2 * i + (g & 1); }

__device__ __forceinline__ uint8_t *kv8_record(const kitty_kv8_layer &L, int64_t page, int h, int block) {
  return L.pages + ((page * L.h_kv + h) * 4 + block) * KV8_REC;
}

// Page row of block `blk` of batch row b, or -1 (and the status bit) when the table entry is out of range.
__device__ __forceinline__ int64_t kv8_page(const kitty_kv8_layer &L, int b, int blk) {
  const int64_t p = L.page_table[static_cast<int64_t>(b) * L.max_page + (blk >> 2)];
  if (p < 0 || p >= L.num_pages) {
    atomicOr(L.status, KITTY_KV8_BAD_PAGE);
    return -1;
  }
  return p;
}

__device__ __forceinline__ int kv8_clamp_len(const kitty_kv8_layer &L, int n) {
  const int cap = L.max_page * PAGE;
  if (n < 0 || n > cap) {
    atomicOr(L.status, KITTY_KV8_BAD_LENGTH);
    return n < 0 ? 0 : cap;
  }
  return n;
}

inline int check_kv8_layer(const kitty_kv8_layer *L) {
  if (L == nullptr || !L->pages || !L->tail_k || !L->tail_v || !L->page_table || !L->status) return KITTY_E_BADARG;
  if (L->head_dim != HD) return KITTY_E_BADSHAPE;
  if (L->dtype != KITTY_F16 && L->dtype != KITTY_BF16) return KITTY_E_BADARG;
  if (L->max_bs <= 0 || L->max_page <= 0 || L->num_pages <= 0 || L->h_kv <= 0) return KITTY_E_BADARG;
  if (L->max_page > (1 << 30) / PAGE) return KITTY_E_BADSHAPE;        // token positions are 32-bit
  if ((reinterpret_cast<uintptr_t>(L->pages) | reinterpret_cast<uintptr_t>(L->tail_k) |
       reinterpret_cast<uintptr_t>(L->tail_v)) & 15)
    return KITTY_E_BADARG;
  return KITTY_OK;
}

}  // namespace kitty
