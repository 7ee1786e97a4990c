// The paged bf16 KV cache: what the kernels that write, read, attend and evict it share.
//
// A page is 64 slots of every kv head of one layer, K and V each [kv_heads][64 * hd] in the 64-slot block layout of common.h
// (k_off, v_off): what a page holds of one kv head is the MFMA operands of one 64-key block, 128 hd bytes in one run, so a page
// never ends inside a tile and the attention needs one table word a block.
// A batch (SsdPagedBatch): sequence s owns rows [row_begin[s], row_begin[s + 1]) of the packed operands; row i of its n sits at slot
// lengths[s] - n + i.
#pragma once
#include "common.h"

#include <initializer_list>

namespace ssd {

constexpr int PAGE = 64;

struct PagedBatch {
  const int* table;
  int64_t ld_table;
  int table_cols, n_seq, rows_max;
  const int *row_begin, *lengths;
};

struct PagedCache {
  bf16_t *k, *v;
  int pages, kv;
};

// Rows [r0, r0 + n) of sequence s; row i sits at slot first + i (below 0: nowhere).
struct PagedRows {
  int r0, n, first;
};
__device__ __forceinline__ PagedRows paged_rows(const PagedBatch& b, int s, int M) {
  const int lo = b.row_begin ? b.row_begin[s] : s, hi = b.row_begin ? b.row_begin[s + 1] : s + 1;
  PagedRows r;
  r.r0 = min(max(lo, 0), M);
  const int all = min(max(hi, r.r0), M) - r.r0;
  r.n = min(all, b.rows_max);
  r.first = min(max(b.lengths[s], 0), 1 << 30) - all;
  return r;
}

__device__ __forceinline__ float paged_max_lanes(float v) {  // over the four 16-lane groups
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float paged_sum_lanes(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Key of a block that lane group g holds in element e of score tile kt.
__device__ __forceinline__ int paged_key(int kt, int g, int e) { return (kt >> 1) * 32 + 8 * g + (kt & 1) * 4 + e; }

// A block that not every column of a tile attends whole: a V value that is not finite must reach the columns that attend its slot and
// no other (0 * NaN is NaN), and a slot behind the last one may hold anything. So such values are taken out of the operand, and
// the first slot that held one is noted for its dim; as columns attend all slots up to their last, those whose last slot is not
// before it get NaN in the end.
// x: 8 slots of one dim, the first of them `slot`.
__device__ __forceinline__ bool paged_not_finite(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ u32x4_t paged_take_out(u32x4_t x, int slot, int* first_bad) {
  int at = INT32_MAX;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    if ((x[i] & 0x7f800000u) == 0x7f800000u) at = slot + 2 * i + 1, x[i] &= 0xffffu;
    if ((x[i] & 0x7f80u) == 0x7f80u) at = slot + 2 * i, x[i] &= 0xffff0000u;
  }
  if (at != INT32_MAX) atomicMin(first_bad, at);
  return x;
}

// Page of slots 64 p .. 64 p + 63 of sequence s, or -1: none of the pool's.
__device__ __forceinline__ int paged_page(const PagedBatch& b, int s, int p, int pages) {
  const int id = b.table[s * b.ld_table + p];
  return (uint32_t)id < (uint32_t)pages ? id : -1;
}

// A launch holds at most 2^32 - 1 threads.
__host__ inline bool paged_grid_too_large(int64_t workgroups, int threads) { return workgroups > (int64_t)UINT32_MAX / threads; }

// Product of sizes, INT64_MAX / 2 if that is less (a sum of two such does not wrap either).
__host__ inline int64_t paged_product(std::initializer_list<int64_t> sizes) {
  int64_t p = 1;
  for (const int64_t n : sizes)
    if (__builtin_mul_overflow(p, n, &p) || p > INT64_MAX / 2) return n == 0 ? 0 : INT64_MAX / 2;
  return p;
}

// Host checks of the descriptors; 0, or the code of the error they set.
int paged_check(const SsdPagedKv* c, const SsdPagedBatch* b, const char* what);
inline PagedBatch paged_batch(const SsdPagedBatch* b) {
  return PagedBatch{b->table, b->ld_table, b->table_cols, b->n_seq, b->rows_max, b->row_begin, b->lengths};
}

// Adds up every row's records of its length's groups of grp_keys keys (O in ws_o [row][head][group][head_dim], (m, l) in ws_ml) into out.
int paged_join(const PagedBatch& b, int M, int heads, int head_dim, int l_cap, int grp_keys, int n_grps, float* ws_o, float2* ws_ml,
               bf16_t* out, int64_t ldo, hipStream_t stream);

}  // namespace ssd
