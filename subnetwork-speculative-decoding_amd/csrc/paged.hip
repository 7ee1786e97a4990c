// The paged bf16 KV cache's write and read-back, and its eviction by received weight (layout in paged.h).
#include "paged.h"

#include <algorithm>
#include <cstdlib>

namespace ssd {

int paged_check(const SsdPagedKv* c, const SsdPagedBatch* b, const char* what) {
  if (!c || !b) return set_error(SSD_EINVAL, "%s: null descriptor", what);
  if (!c->k || !c->v || (b->n_seq > 0 && (!b->table || !b->lengths))) return set_error(SSD_EINVAL, "%s: null pointer", what);
  if (((uintptr_t)c->k & 15) || ((uintptr_t)c->v & 15)) return set_error(SSD_EINVAL, "%s: the cache must be 16-byte aligned", what);
  if (c->head_dim != 64 && c->head_dim != 128) return set_error(SSD_EINVAL, "%s: head_dim %d unsupported (64, 128)", what, c->head_dim);
  if (c->pages < 1 || c->kv_heads < 1) return set_error(SSD_EINVAL, "%s: bad pages=%d kv_heads=%d", what, c->pages, c->kv_heads);
  if (b->n_seq < 0 || b->rows_max < 0 || b->table_cols < 1 || b->ld_table < b->table_cols)
    return set_error(SSD_EINVAL, "%s: bad n_seq=%d rows_max=%d table_cols=%d ld_table=%lld", what, b->n_seq, b->rows_max, b->table_cols,
                     (long long)b->ld_table);
  if (b->table_cols > 1 << 24) return set_error(SSD_ERANGE, "%s: %d pages a sequence > 2^24", what, b->table_cols);
  if (!b->row_begin && b->rows_max > 1) return set_error(SSD_EINVAL, "%s: several rows a sequence need row_begin", what);
  return SSD_OK;
}

struct PagedRowArgs {
  PagedBatch b;
  PagedCache c;
  bf16_t *k, *v;  // rows [M][kv * hd]
  int64_t ldk, ldv;
  int M, page_sets;  // page_sets: most pages that one sequence's rows touch
};

// Workgroup (sequence, page its rows touch, kv head), at most 64 rows. K pieces of 8 dims go to their place as they are;
// V turns through LDS, so that 8 slots of a dim leave as one 16-byte store where the page takes all 8.
// What bounds it: latency for a step's rows (a workgroup a row and kv head); for prompts bytes: 4096 rows of 8 heads of 128, 34 MB
// read and written, 7 us (4.8 TB/s).
template <int HD>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedRowArgs a) {
  constexpr int PC = HD / 8, LD = HD + 2;  // 16-byte pieces a row; LDS row stride: two-byte reads of a column spread over banks
  __shared__ bf16_t vs[PAGE * LD];
  const int kvh = blockIdx.x % a.c.kv, u = blockIdx.x / a.c.kv, s = u / a.page_sets;
  const PagedRows r = paged_rows(a.b, s, a.M);
  const int begin = max(r.first, 0), end = r.first + r.n;  // slots
  const int p = begin / PAGE + u % a.page_sets, lo = max(begin, p * PAGE), hi = min(end, p * PAGE + PAGE);
  if (lo >= hi || p >= a.b.table_cols) return;  // uniform, as is the page
  const int page = paged_page(a.b, s, p, a.c.pages);
  if (page < 0) return;
  const size_t at = ((size_t)page * a.c.kv + kvh) * PAGE * HD;
  const int row0 = r.r0 - r.first;  // row of slot t: row0 + t
  for (int i = threadIdx.x; i < (hi - lo) * PC; i += 256) {
    const int t = lo + i / PC, d = i % PC * 8;
    const uint4 kx = *(const uint4*)(a.k + (row0 + t) * a.ldk + kvh * HD + d);
    const uint4 vx = *(const uint4*)(a.v + (row0 + t) * a.ldv + kvh * HD + d);
    *(uint4*)(a.c.k + at + k_off(t & 63, d, HD)) = kx;
    uint32_t* dst = (uint32_t*)(vs + (t & 63) * LD + d);
    dst[0] = vx.x, dst[1] = vx.y, dst[2] = vx.z, dst[3] = vx.w;
  }
  __syncthreads();
  const int l = lo & 63, n = hi - lo, g0 = l >> 3, groups = ((l + n - 1) >> 3) - g0 + 1;
  for (int i = threadIdx.x; i < groups * HD; i += 256) {
    const int d = i % HD, o = (g0 + i / HD) * 8;
    bf16_t* dst = a.c.v + at + v_off(o, d, HD);
    if (o >= l && o + 8 <= l + n) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = vs[(o + 2 * e) * LD + d] | (uint32_t)vs[(o + 2 * e + 1) * LD + d] << 16;
      *(uint4*)dst = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      for (int e = max(l - o, 0); e < min(8, l + n - o); ++e) dst[e] = vs[(o + e) * LD + d];
    }
  }
}

// The same workgroups the other way; slots without a page read as zeros.
template <int HD>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedRowArgs a) {
  constexpr int PC = HD / 8, LD = HD + 2;
  __shared__ bf16_t vs[PAGE * LD];
  const int kvh = blockIdx.x % a.c.kv, u = blockIdx.x / a.c.kv, s = u / a.page_sets;
  const PagedRows r = paged_rows(a.b, s, a.M);
  // page 0's workgroup also takes rows before slot 0
  const int p0 = max(r.first, 0) / PAGE, p = p0 + u % a.page_sets;
  if (p == p0 && r.first < 0) {
    const int n = min(-r.first, r.n);
    for (int i = threadIdx.x; i < n * PC; i += 256) {
      const int64_t row = r.r0 + i / PC;
      const int d = kvh * HD + i % PC * 8;
      *(uint4*)(a.k + row * a.ldk + d) = make_uint4(0, 0, 0, 0);
      *(uint4*)(a.v + row * a.ldv + d) = make_uint4(0, 0, 0, 0);
    }
  }
  const int lo = max(r.first, p * PAGE), hi = min(r.first + r.n, p * PAGE + PAGE);
  if (lo >= hi) return;
  const int page = p < a.b.table_cols ? paged_page(a.b, s, p, a.c.pages) : -1;
  const size_t at = ((size_t)max(page, 0) * a.c.kv + kvh) * PAGE * HD;
  const int l = lo & 63, n = hi - lo, g0 = l >> 3, groups = ((l + n - 1) >> 3) - g0 + 1;
  if (page >= 0)
    for (int i = threadIdx.x; i < groups * HD; i += 256) {
      const int d = i % HD, o = (g0 + i / HD) * 8;
      const uint4 x = *(const uint4*)(a.c.v + at + v_off(o, d, HD));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) vs[(o + e) * LD + d] = (bf16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
  __syncthreads();
  const int64_t row0 = (int64_t)r.r0 - r.first;
  for (int i = threadIdx.x; i < n * PC; i += 256) {
    const int t = lo + i / PC, d = i % PC * 8;
    uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
    if (page >= 0) {
      kx = *(const uint4*)(a.c.k + at + k_off(t & 63, d, HD));
      const uint32_t* src = (const uint32_t*)(vs + (t & 63) * LD + d);
      vx = make_uint4(src[0], src[1], src[2], src[3]);
    }
    *(uint4*)(a.k + (row0 + t) * a.ldk + kvh * HD + d) = kx;
    *(uint4*)(a.v + (row0 + t) * a.ldv + kvh * HD + d) = vx;
  }
}

static int paged_rows_call(const SsdPagedKv* c, const SsdPagedBatch* b, uint16_t* k, int64_t ldk, uint16_t* v, int64_t ldv, int M,
                           bool write, hipStream_t stream) {
  const char* what = write ? "paged_write" : "paged_read";
  if (int rc = paged_check(c, b, what)) return rc;
  if (M < 0) return set_error(SSD_EINVAL, "%s: bad M=%d", what, M);
  if (M == 0 || b->n_seq == 0 || b->rows_max == 0) return SSD_OK;
  if (!k || !v) return set_error(SSD_EINVAL, "%s: null pointer", what);
  const int64_t cols = (int64_t)c->kv_heads * c->head_dim;
  if (((uintptr_t)k & 15) || ((uintptr_t)v & 15) || ldk % 8 || ldv % 8 || ldk < cols || ldv < cols)
    return set_error(SSD_EINVAL, "%s: k/v rows must be 16-byte aligned with strides >= kv_heads * head_dim", what);
  PagedRowArgs a{paged_batch(b), PagedCache{c->k, c->v, c->pages, c->kv_heads}, k, v, ldk, ldv, M, 0};
  a.page_sets = (int)(((int64_t)std::min(b->rows_max, M) + 62) / 64 + 1);
  const int64_t wgs = paged_product({b->n_seq, a.page_sets, c->kv_heads});
  if (paged_grid_too_large(wgs, 256)) return set_error(SSD_ERANGE, "%s: too many workgroups", what);
  const dim3 grid((unsigned)wgs), block(256);
  if (write) {
    if (c->head_dim == 64) SSD_LAUNCH((paged_write_kernel<64>), grid, block, 0, stream, a);
    else SSD_LAUNCH((paged_write_kernel<128>), grid, block, 0, stream, a);
  } else {
    if (c->head_dim == 64) SSD_LAUNCH((paged_read_kernel<64>), grid, block, 0, stream, a);
    else SSD_LAUNCH((paged_read_kernel<128>), grid, block, 0, stream, a);
  }
  return check_launch(what);
}

// ------------------------------------------------------------------ eviction
struct EvictArgs {
  PagedBatch b, after;
  PagedCache c;          // layer 0; the others follow
  size_t layer_elems;
  const float* w;        // [layers][n_seq][kv] rows of cap
  int64_t ldw;
  float* w_out;          // the same rows
  int cap, keep, recent, first, layers;
  int* kept;             // [layers][n_seq][kv][keep]
  int* new_len;          // after.lengths
  int dst_pages;
};

// Order-preserving image of a weight: larger ranks higher, -0 equals 0, NaN ranks below every number.
__device__ __forceinline__ uint32_t evict_rank(float f) {
  const uint32_t b = __float_as_uint(f + 0.f);
  return f != f ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

constexpr int EV_T = 1024, EV_BINS = 2048, EV_OWN = 8;  // EV_OWN: ranks that a thread keeps

// Exclusive prefix sum of x over the workgroup's threads, and the total; every thread calls it.
__device__ __forceinline__ int evict_scan(int x, int* wave_sums, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(inc, o);
    if (lane >= o) inc += t;
  }
  __syncthreads();  // the sums of the scan before have been read
  if (lane == 63) wave_sums[w] = inc;
  __syncthreads();
  int base = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < EV_T / 64; ++i) {
    const int v = wave_sums[i];
    base += i < w ? v : 0;
    total += v;
  }
  return base + inc - x;
}

// A workgroup per (layer, sequence, kv head) finds the slots that stay. The least rank that stays is found exactly by three
// histograms of 11, 11 and 10 of its bits; then one pass in slot order writes what ranks above it, and of those that rank with
// it the lowest slots. What bounds it: the dependent passes over a row; 256 rows of up to 4096 weights 11 us (13 with loads
// in every pass).
__global__ __launch_bounds__(EV_T) void evict_select_kernel(EvictArgs a) {
  __shared__ int hist[EV_BINS], wave_sums[EV_T / 64], found[2];
  const int tid = threadIdx.x, row = blockIdx.x, s = row / a.c.kv % a.b.n_seq;
  const int L = min(max(a.b.lengths[s], 0), min(a.cap, a.b.table_cols * PAGE));
  const float* w = a.w + (size_t)row * a.ldw;
  float* w_out = a.w_out + (size_t)row * a.ldw;
  int* kept = a.kept + (size_t)row * a.keep;
  const int m0 = min(a.first, L), m1 = max(L - a.recent, m0);  // the middle, which is ranked
  int need = L <= a.keep ? m1 - m0 : a.keep - a.first - a.recent;
  uint32_t least = 0;  // ranks above it stay, and `need` of those equal to it
  const bool all = need >= m1 - m0;
  if (!all && need > 0) {
    uint32_t mask = 0, own[EV_OWN];  // the first of this thread's ranks, loaded together
#pragma unroll
    for (int i = 0; i < EV_OWN; ++i) own[i] = evict_rank(w[min(m0 + tid + EV_T * i, m1 - 1)]);
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
      hist[tid] = 0, hist[tid + EV_T] = 0;
      __syncthreads();
      auto count = [&](uint32_t u) {
        if ((u & mask) == least) atomicAdd(&hist[(u >> shift) & (bins - 1)], 1);
      };
#pragma unroll
      for (int i = 0; i < EV_OWN; ++i)
        if (m0 + tid + EV_T * i < m1) count(own[i]);
      for (int t = m0 + tid + EV_T * EV_OWN; t < m1; t += EV_T) count(evict_rank(w[t]));
      __syncthreads();
      // bins from the top: thread i holds bins top - 2i and top - 2i - 1
      const int b1 = EV_BINS - 1 - 2 * tid, h1 = hist[b1], h0 = hist[b1 - 1];
      int total;
      const int above = evict_scan(h1 + h0, wave_sums, total);
      if (above < need && need <= above + h1 + h0) {
        const bool high = need <= above + h1;
        found[0] = high ? b1 : b1 - 1;
        found[1] = need - above - (high ? 0 : h1);
      }
      __syncthreads();
      least |= (uint32_t)found[0] << shift;
      need = found[1];
      mask |= (uint32_t)(bins - 1) << shift;
    }
  }
  int out = 0, ties = 0;  // written so far, and of those equal to `least`
  for (int t0 = 0; t0 < L; t0 += 4 * EV_T) {
    const int t = t0 + 4 * tid;
    float x[4];
    bool eq[4], in[4];
    int n_eq = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = t + e < L ? w[t + e] : 0.f;
      const bool mid = t + e >= m0 && t + e < m1;
      const uint32_t u = evict_rank(x[e]);
      in[e] = t + e < L && (!mid || all || (need > 0 && u > least));
      eq[e] = mid && !all && need > 0 && u == least;
      n_eq += eq[e];
    }
    int total, n_in = 0;
    int tie = ties + evict_scan(n_eq, wave_sums, total);
    ties += total;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (eq[e]) in[e] = tie++ < need;
      n_in += in[e];
    }
    int at = out + evict_scan(n_in, wave_sums, total);
    out += total;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (in[e]) {
        kept[at] = t + e;
        w_out[at++] = x[e];
      }
  }
  for (int j = out + tid; j < a.keep; j += EV_T) kept[j] = -1;
  for (int j = out + tid; j < a.cap; j += EV_T) w_out[j] = 0.f;
}

// A workgroup per (layer, sequence, destination page, kv head) gathers the page's rows. Every 16-byte piece of V holds 8 slots of a
// dim, which come from up to 8 places.
// What bounds it: bytes that the layout brings along. Neighbouring slots' pieces share memory's 64 bytes, in K four of them and in V all
// of a piece, so where a third of the slots stays here and there three quarters of the old pages are read: 2 layers, 16 sequences, 8 heads of 128,
// 1024 of 2048 to 4096 slots kept 95 us, 314 MB read and 130 written, 4.7 TB/s (side by side 65). Two bytes a slot of V instead
// of the piece it is in: 8 us more.
template <int HD>
__global__ __launch_bounds__(256) void evict_gather_kernel(EvictArgs a) {
  constexpr int PC = HD / 8;
  __shared__ int src_slot[PAGE], src_page[PAGE];
  __shared__ int counts[4];
  int u = blockIdx.x;
  const int kvh = u % a.c.kv;
  u /= a.c.kv;
  const int p = u % a.dst_pages;
  u /= a.dst_pages;
  const int s = u % a.b.n_seq, layer = u / a.b.n_seq, tid = threadIdx.x;
  const int* kept = a.kept + (((size_t)layer * a.b.n_seq + s) * a.c.kv + kvh) * a.keep;
  if (layer == 0 && p == 0 && kvh == 0) {  // the new length; the select kernel, which reads the old ones, has ended
    int n = 0;
    for (int j = tid; j < a.keep; j += 256) n += kept[j] >= 0;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o);
    if ((tid & 63) == 0) counts[tid >> 6] = n;
    __syncthreads();
    if (tid == 0) a.new_len[s] = counts[0] + counts[1] + counts[2] + counts[3];
  }
  if (p >= a.after.table_cols) return;
  const int page = paged_page(a.after, s, p, a.c.pages);
  if (tid < PAGE) {
    const int j = p * PAGE + tid, t = j < a.keep ? kept[j] : -1;
    src_slot[tid] = t;
    src_page[tid] = t >= 0 ? paged_page(a.b, s, t / PAGE, a.c.pages) : -1;
  }
  __syncthreads();
  if (page < 0 || src_slot[0] < 0) return;
  const bf16_t *K = a.c.k + layer * a.layer_elems, *V = a.c.v + layer * a.layer_elems;
  const size_t at = layer * a.layer_elems + ((size_t)page * a.c.kv + kvh) * PAGE * HD;
  auto from = [&](int o) { return ((size_t)max(src_page[o], 0) * a.c.kv + kvh) * PAGE * HD; };
  // All loads of a thread's pieces are under way before the first is used; places without a source read slot 0 of page 0 and give zeros.
  constexpr int KN = PAGE * PC / 256;
  uint4 kx[KN];
#pragma unroll
  for (int i = 0; i < KN; ++i) {
    const int o = tid % PAGE, d = (tid / PAGE + 4 * i) * 8;
    kx[i] = *(const uint4*)(K + from(o) + k_off(max(src_slot[o], 0) & 63, d, HD));
  }
#pragma unroll
  for (int i = 0; i < KN; ++i) {
    const int o = tid % PAGE, d = (tid / PAGE + 4 * i) * 8;
    if (src_page[o] < 0) kx[i] = make_uint4(0, 0, 0, 0);
    if (src_slot[o] >= 0) *(uint4*)(a.c.k + at + k_off(o, d, HD)) = kx[i];
  }
  // A wave takes 64 dims of eight slots, whose places are the same for all its lanes: whole pieces of V, of which each gives one slot.
#pragma unroll
  for (int i = 0; i < PAGE / 8 * HD / 256; ++i) {
    const int x = 256 * i + tid, d = x % HD, o = __builtin_amdgcn_readfirstlane(x / HD * 8);
    if (src_slot[o] < 0) continue;
    uint4 y[8];
    int t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t[e] = __builtin_amdgcn_readfirstlane(src_page[o + e] < 0 ? -1 : src_slot[o + e]);  // -1: zeros (behind the last kept slot, or no page)
      y[e] = *(const uint4*)(V + from(o + e) + v_off(max(t[e], 0) & 56, d, HD));
    }
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint64_t half = t[e] & 4 ? (uint64_t)y[e].w << 32 | y[e].z : (uint64_t)y[e].y << 32 | y[e].x;
      w[e] = t[e] < 0 ? 0u : (uint32_t)(half >> (16 * (t[e] & 3))) & 0xffffu;
    }
    *(uint4*)(a.c.v + at + v_off(o, d, HD)) = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
  }
}

}  // namespace ssd

using namespace ssd;

SSD_API int ssd_paged_write_bf16(const SsdPagedKv* cache, const SsdPagedBatch* batch, const uint16_t* k, int64_t ldk,
                                 const uint16_t* v, int64_t ldv, int M, hipStream_t stream) {
  return paged_rows_call(cache, batch, const_cast<uint16_t*>(k), ldk, const_cast<uint16_t*>(v), ldv, M, true, stream);
}

SSD_API int ssd_paged_read_bf16(const SsdPagedKv* cache, const SsdPagedBatch* batch, int M, uint16_t* k, int64_t ldk, uint16_t* v,
                                int64_t ldv, hipStream_t stream) {
  return paged_rows_call(cache, batch, k, ldk, v, ldv, M, false, stream);
}

SSD_API int ssd_paged_evict(const SsdPagedKv* cache, int layers, int64_t layer_elems, const SsdPagedBatch* batch,
                            const SsdPagedBatch* after, const float* weights, int64_t ldw, int cap, int keep, int recent, int first,
                            float* out_weights, int32_t* kept, hipStream_t stream) {
  if (int rc = paged_check(cache, batch, "paged_evict")) return rc;
  if (int rc = paged_check(cache, after, "paged_evict")) return rc;
  if (!weights || !out_weights || !kept) return set_error(SSD_EINVAL, "paged_evict: null pointer");
  if (after->n_seq != batch->n_seq) return set_error(SSD_EINVAL, "paged_evict: %d sequences become %d", batch->n_seq, after->n_seq);
  const int64_t one = paged_product({cache->pages, cache->kv_heads, PAGE, cache->head_dim});
  if (layers < 1 || layer_elems < one) return set_error(SSD_EINVAL, "paged_evict: bad layers=%d layer_elems=%lld", layers, (long long)layer_elems);
  if (cap < 1 || ldw < cap) return set_error(SSD_EINVAL, "paged_evict: bad cap=%d ldw=%lld", cap, (long long)ldw);
  if (keep < 1 || recent < 0 || first < 0 || (int64_t)recent + first > keep)
    return set_error(SSD_EINVAL, "paged_evict: keep=%d must hold recent=%d and first=%d", keep, recent, first);
  if ((int64_t)after->table_cols * PAGE < keep)
    return set_error(SSD_EINVAL, "paged_evict: keep=%d > the %d pages a sequence of the new table", keep, after->table_cols);
  if (batch->n_seq == 0) return SSD_OK;
  EvictArgs a{};
  a.b = paged_batch(batch), a.after = paged_batch(after);
  a.c = PagedCache{cache->k, cache->v, cache->pages, cache->kv_heads};
  a.layer_elems = (size_t)layer_elems, a.w = weights, a.ldw = ldw, a.w_out = out_weights, a.cap = cap;
  a.keep = keep, a.recent = recent, a.first = first, a.layers = layers, a.kept = kept, a.new_len = after->lengths;
  a.dst_pages = (keep + PAGE - 1) / PAGE;
  const int64_t rows = paged_product({layers, batch->n_seq, cache->kv_heads});
  if (paged_grid_too_large(rows, EV_T) || paged_grid_too_large(paged_product({rows, a.dst_pages}), 256))
    return set_error(SSD_ERANGE, "paged_evict: too many workgroups");
  const int64_t reach = paged_product({4, paged_product({rows - 1, ldw}) + cap});  // bytes from the first row to the last's end
  if (std::abs((intptr_t)weights - (intptr_t)out_weights) < reach)
    return set_error(SSD_EINVAL, "paged_evict: out_weights must not overlap weights");
  SSD_LAUNCH(evict_select_kernel, dim3((unsigned)rows), dim3(EV_T), 0, stream, a);
  if (int rc = check_launch("paged_evict_select")) return rc;
  const dim3 grid((unsigned)(rows * a.dst_pages));
  if (cache->head_dim == 64) SSD_LAUNCH((evict_gather_kernel<64>), grid, dim3(256), 0, stream, a);
  else SSD_LAUNCH((evict_gather_kernel<128>), grid, dim3(256), 0, stream, a);
  return check_launch("paged_evict_gather");
}
