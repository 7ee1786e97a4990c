// Attention of few new rows a sequence over the paged cache (paged.h), split over the length and joined; with it, on request,
// the weight that each cached slot has received.
//
// The columns of S^T = K Q^T are the (row, q head) pairs of one sequence and kv head, rows outermost, sixteen a tile. A row's keys
// are cut into groups of 4 * span slots: a workgroup folds one group for one tile, its wave w every fourth 64-key block from the
// w-th on, with a running reference m, sum l and output O in fp32; the four waves' states are added in LDS. Several groups leave
// records (m, l, O) that a second launch adds up with weights from their largest m; one group is written out at once.
// So a row's result depends on its own keys, its query and the span, not on the other rows or sequences.
// Probabilities go into the second product as the sum of two bf16 numbers, since the matrix pipe has time for it and one row's few large
// weights are not averaged over many (27000 keys of which few matter: 0.0026 from 64 bits with one, 0.0017 with two, the
// output's own rounding); l sums them as they are.
//
// With weights the second launch, knowing every (row, head)'s final m and l, also adds up 2^(s - m) / l over the rows and heads of
// a kv head. For up to sixteen pairs the first launch leaves it the scores (fp32: 8 bytes a pair and key, written and read, against
// 4 hd bytes of K and V); for more it reads K again and makes them anew, in the same order and so the same.
//
// What bounds it: bytes of K and V, each read once where a kv head's pairs are one tile. A wave has one block's K and V in
// registers and loads the next block's as soon as a product has used the present one's, 32 KB in flight; with 245 registers that
// is two workgroups a CU. 32 heads on 8 kv heads of 128, us of both launches: 32 sequences of one row and up to 8192 keys
// 142 (5.2 TB/s), one row after 131000 keys 97 (5.5); 24 sequences of up to 4000 keys with weights, 15 heads on 5, 38 with K and V in
// the caches (32 + 6), 49 from memory; 6 sequences of 16 rows and 1200 to 4001 keys, four tiles that share K and V through L2, 26 and
// 17 for the join and the weights. One row after 500 keys of the smallest shape 4.8: latency.
// Tried: two tiles a workgroup, whose registers leave one workgroup a CU (6 sequences of 16 rows 29 us against 25, 2 of 60 rows and
// 8000 keys 87 against 76); tiles one after another in a workgroup, K and V on their way for the next while one ends (42 against 41 for
// two, 50 for three: the tiles' chains are better side by side).
#include "paged.h"

#include <algorithm>

namespace ssd {

constexpr int PA_WAVES = 4;
// Most (row, head) pairs of a kv head whose scores are kept for the weights (us of both launches, hd 128, 4 heads a kv head, kept / made
// anew: 24 sequences of one row and 4000 keys 138 / 166, 6 of 4 rows 52 / 54, of 8 rows 58 / 58, of 16 rows and 1200 to 4001 keys
// 63 / 58, 2 of 60 rows and 8000 keys 138 / 107).
constexpr int PA_SCORES = 16;
constexpr int PA_RUN = 8;  // records that a wave loads at once
constexpr int PA_MAX_SPAN = 4096;  // a wave's pages are one table word a lane

struct PagedAttnArgs {
  PagedBatch b;
  PagedCache c;
  const bf16_t* Q;
  int64_t ldq;
  int M, heads, rep, l_cap;  // l_cap: slots from here on are not attended
  int span_blk, n_grps, grp_keys, sets, units;  // grp_keys: keys of a group
  float scale_log2;
  float* ws_o;    // [row][head][group][HD]
  float2* ws_ml;  // [row][head][group]: (m, l)
  float2* ws_t;   // [kv head][group][row][q head of it]: (m, l) once more, as the weights' launch reads them
  float* ws_s;    // [row][head][ld_s]: products q k
  int64_t ld_s;
  bf16_t* out;
  int64_t ldo;
  float* weights;
  int64_t ldw_seq, ldw;
  float decay;
  int weight_wgs, chunks;  // second launch: workgroups that add up weights (the others join), key chunks of a (sequence, kv head)
};

template <int HD>
struct PagedFrags {
  u32x4_t k[4][HD / 32];
  u32x4_t v[HD / 16][2];
};

template <int HD>
struct PagedState {
  float m, l;          // reference (log2 units; -inf: nothing yet), this lane's part of the sum
  f32x4_t o[HD / 16];  // O[column j][16 dt + 4g + e]
};

template <int HD>
__device__ __forceinline__ void paged_load_k(PagedFrags<HD>& f, const bf16_t* K, size_t at, int lane) {
  const bf16_t* p = K + at + lane * 8;
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int ks = 0; ks < HD / 32; ++ks) f.k[kt][ks] = *(const u32x4_t*)(p + (kt * (HD / 32) + ks) * 512);
}
template <int HD>
__device__ __forceinline__ void paged_load_v(PagedFrags<HD>& f, const bf16_t* V, size_t at, int lane) {
  const bf16_t* p = V + at + lane * 8;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt)
#pragma unroll
    for (int c = 0; c < 2; ++c) f.v[dt][c] = *(const u32x4_t*)(p + (dt * 2 + c) * 512);
}

// Folds one block into the state. left: the block's keys below it are attended by this lane's column (64 or more: all); masked
// (uniform): some column does not attend the whole block. The reference follows the maximum only when that has grown by more
// than 2^8: probabilities up to 2^8 are as exact as those up to 1, and after the first blocks nothing is rescaled.
template <int HD, typename TakeOut, typename Scores, typename NextK, typename NextV>
__device__ __forceinline__ void paged_fold(PagedFrags<HD>& f, const u32x4_t (&qf)[HD / 32], int left, bool masked, float scale_log2,
                                           int g, PagedState<HD>& st, TakeOut take_out, Scores scores, NextK next_k, NextV next_v) {
  f32x4_t s[4];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) s[kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < HD / 32; ++ks)
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) s[kt] = mfma16x16x32(bits_bf16x8(f.k[kt][ks]), bits_bf16x8(qf[ks]), s[kt]);
  next_k();
  if (masked) {
    take_out();
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[kt][e] = paged_key(kt, g, e) < left ? s[kt][e] : -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[kt][e]);
  mx = paged_max_lanes(mx) * scale_log2;
  scores(s);
  const float m = mx > st.m + 8.f || st.m == -INFINITY ? mx : st.m;
  const float ms = m == -INFINITY ? 0.f : m;  // nothing attended so far: every p is 0
  if (__any(m != st.m)) {
    const float alpha = __builtin_amdgcn_exp2f(st.m - ms);
    st.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) st.o[dt] *= alpha;
  }
  st.m = m;
  u32x4_t pw[2], rest[2];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[kt][e], scale_log2, -ms));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s[kt][e + 1], scale_log2, -ms));
      st.l += p0 + p1;
      const uint32_t both = pack_bf16x2(p0, p1);
      pw[kt >> 1][(kt & 1) * 2 + e / 2] = both;
      rest[kt >> 1][(kt & 1) * 2 + e / 2] = pack_bf16x2(p0 - __uint_as_float(both << 16), p1 - __uint_as_float(both & 0xffff0000u));
    }
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) {
      st.o[dt] = mfma16x16x32(bits_bf16x8(f.v[dt][c]), bits_bf16x8(rest[c]), st.o[dt]);
      st.o[dt] = mfma16x16x32(bits_bf16x8(f.v[dt][c]), bits_bf16x8(pw[c]), st.o[dt]);
    }
  next_v();
}

__device__ __forceinline__ float paged_weight(float m, float top) {
  return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
}

// The waves' states meet here.
template <int HD>
struct alignas(16) PagedSpans {
  float o[PA_WAVES][16][HD + 4];
  float m[PA_WAVES][16], l[PA_WAVES][16];
  int first_bad[HD];  // paged_take_out's
};

// Workgroup (sequence, group, kv head, tile). The tiles of one (sequence, group, kv head) are ids 8 apart: one XCD, whose L2 they share.
// WK as for the second launch: 1 keeps the scores.
template <int HD, int WK>
__global__ __launch_bounds__(256, 2) void paged_fold_kernel(PagedAttnArgs a) {
  __shared__ PagedSpans<HD> lds;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const int rest = blockIdx.x >> 3, set = rest % a.sets;
  int u = rest / a.sets * 8 + (blockIdx.x & 7);
  if (u >= a.units) return;
  const int kvh = u % a.c.kv;
  u /= a.c.kv;
  const int grp = u % a.n_grps, seq = u / a.n_grps;
  const int b0 = grp * PA_WAVES * a.span_blk, blk = b0 + w + PA_WAVES * lane;
  // lane i has the page of this wave's block i; the table is read before the lengths are known, a chain of loads less
  int mine = lane < a.span_blk && blk * PAGE < a.l_cap ? paged_page(a.b, seq, blk, a.c.pages) : -1;
  const PagedRows r = paged_rows(a.b, seq, a.M);
  const int n_cols = r.n * a.rep, c0 = set * 16;
  if (c0 >= n_cols) return;
  const int last = min(c0 + 15, n_cols - 1);
  const int lim_lo = min(r.first + c0 / a.rep, a.l_cap - 1), lim_hi = min(r.first + last / a.rep, a.l_cap - 1);
  if (a.n_grps > 1 && b0 * PAGE > lim_hi) return;  // no record: the second launch counts them as this does
  const int nb = lim_hi < 0 ? 0 : min(max((lim_hi / PAGE - b0 - w) / PA_WAVES + (lim_hi / PAGE - b0 - w >= 0), 0), a.span_blk);
  const int col = min(c0 + j, n_cols - 1), row = r.r0 + col / a.rep, head = kvh * a.rep + col % a.rep;
  const int lim = min(r.first + col / a.rep, a.l_cap - 1);
  if (threadIdx.x < HD) lds.first_bad[threadIdx.x] = INT32_MAX;
  __syncthreads();
  PagedState<HD> st;
  st.m = -INFINITY, st.l = 0.f;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) st.o[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (nb > 0) {
    auto at = [&](int i) { return ((size_t)max(__builtin_amdgcn_readlane(mine, i), 0) * a.c.kv + kvh) * PAGE * HD; };
    PagedFrags<HD> f;
    paged_load_k<HD>(f, a.c.k, at(0), lane);
    paged_load_v<HD>(f, a.c.v, at(0), lane);
    u32x4_t qf[HD / 32];
#pragma unroll
    for (int ks = 0; ks < HD / 32; ++ks) qf[ks] = *(const u32x4_t*)(a.Q + row * a.ldq + head * HD + ks * 32 + g * 8);
    for (int i = 0; i < nb; ++i) {
      const int key0 = (b0 + w + PA_WAVES * i) * PAGE;
      const bool gone = __builtin_amdgcn_readlane(mine, i) < 0;  // no such page: none of its slots is attended
      const bool masked = gone || key0 + PAGE - 1 > lim_lo;
      const int note = gone ? INT32_MAX - PAGE : key0;
      auto scores = [&](const f32x4_t (&s)[4]) {
        if constexpr (WK == 1) {
          if (c0 + j >= n_cols) return;
          float* dst = a.ws_s + ((int64_t)row * a.heads + head) * a.ld_s + key0;
#pragma unroll
          for (int kt = 0; kt < 4; ++kt) *(f32x4_t*)(dst + paged_key(kt, g, 0)) = s[kt];
        }
      };
      auto next_k = [&] {
        if (i + 1 < nb) paged_load_k<HD>(f, a.c.k, at(i + 1), lane);
      };
      auto next_v = [&] {
        if (i + 1 < nb) paged_load_v<HD>(f, a.c.v, at(i + 1), lane);
      };
      auto take_out = [&] {
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            __builtin_amdgcn_sched_barrier(0);  // one at a time: all at once would spill
            u32x4_t x = f.v[dt][c];
            asm volatile("" : "+v"(x));
            if (__any(paged_not_finite(x[0]) || paged_not_finite(x[1]) || paged_not_finite(x[2]) || paged_not_finite(x[3])))
              f.v[dt][c] = paged_take_out(x, note + c * 32 + g * 8, &lds.first_bad[dt * 16 + j]);
          }
      };
      paged_fold<HD>(f, qf, gone ? 0 : lim - key0 + 1, masked, a.scale_log2, g, st, take_out, scores, next_k, next_v);
    }
  }
  st.l = paged_sum_lanes(st.l);
  lds.m[w][j] = st.m;  // the four lanes of column j write the same values
  lds.l[w][j] = st.l;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) *(f32x4_t*)&lds.o[w][j][dt * 16 + 4 * g] = st.o[dt];
  __syncthreads();
  // column rr, dims 4 dc .. + 4 of every 64
  const int rr = threadIdx.x >> 4, dc = threadIdx.x & 15;
  if (c0 + rr >= n_cols) return;
  float top = -INFINITY, l = 0.f, wgt[PA_WAVES];
#pragma unroll
  for (int i = 0; i < PA_WAVES; ++i) top = fmaxf(top, lds.m[i][rr]);
#pragma unroll
  for (int i = 0; i < PA_WAVES; ++i) {
    wgt[i] = paged_weight(lds.m[i][rr], top);
    l = fmaf(lds.l[i][rr], wgt[i], l);
  }
  const int64_t orow = r.r0 + (c0 + rr) / a.rep;
  const int ohead = kvh * a.rep + (c0 + rr) % a.rep;
  const int olim = min(r.first + (c0 + rr) / a.rep, a.l_cap - 1);
  const int64_t rec = (orow * a.heads + ohead) * a.n_grps + grp;
  const bool direct = a.n_grps == 1;
#pragma unroll
  for (int i = 0; i < HD / 64; ++i) {
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < PA_WAVES; ++v) {
      const f32x4_t x = *(const f32x4_t*)&lds.o[v][rr][i * 64 + dc * 4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], wgt[v], o[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (olim >= lds.first_bad[i * 64 + dc * 4 + e]) o[e] = __uint_as_float(0x7fc00000u);
    if (direct) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = l == 0.f ? 0.f : o[e] / l;  // NaN stays NaN
      *(uint2*)(a.out + orow * a.ldo + ohead * HD + i * 64 + dc * 4) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    } else {
      *(f32x4_t*)(a.ws_o + rec * HD + i * 64 + dc * 4) = o;
    }
  }
  if (dc == 0 && !direct) a.ws_ml[rec] = make_float2(top, l);
  if (WK && dc == 0) a.ws_t[(((int64_t)kvh * a.n_grps + grp) * a.M + r.r0) * a.rep + c0 + rr] = make_float2(top, l);
}

// Largest reference and the sum l of a (row, head)'s records, `step` apart, by the lanes of a power-of-two group of lg lanes.
__device__ __forceinline__ float2 paged_total(const float2* ml, int64_t step, int ng, int part, int lg) {
  float m = -INFINITY, l = 0.f;
  for (int i = part; i < ng; i += 4 * lg) {  // four records on their way at once
    float2 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = ml[min(i + e * lg, ng - 1) * step];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i + e * lg >= ng) break;
      const float top = fmaxf(m, x[e].x);
      l = l * paged_weight(m, top) + x[e].y * paged_weight(x[e].x, top);
      m = top;
    }
  }
  for (int o = 1; o < lg; o <<= 1) {
    const float mo = __shfl_xor(m, o), lo = __shfl_xor(l, o), top = fmaxf(m, mo);
    l = l * paged_weight(m, top) + lo * paged_weight(mo, top);
    m = top;
  }
  return make_float2(m, l);
}

// Second launch. Workgroups that add up the records: WPP waves a (sequence, row, head). PA_RUN groups from each multiple of PA_RUN on are
// added up in order, then these sums in order, by however many waves: the row's bits follow from its own groups. Workgroups that add up
// received weights, of a set of slots of a (sequence, kv head), in a fixed order too: WK = 1 from the kept scores, a lane four slots; WK = 2 from K, a wave a block, sixteen pairs at a time, the lanes' sums last.
template <int HD, int WK, int WPP>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp_keys = a.grp_keys;
  // the workgroups that add up weights, which take longer, come first
  if (WK == 0 || (int)blockIdx.x >= a.weight_wgs) {
    constexpr int V = HD / 64;  // dims a lane
    __shared__ float part[WPP == 4 ? 64 / PA_RUN : 1][HD];  // sums of runs
    int u = blockIdx.x - (WK ? a.weight_wgs : 0);
    if (WPP == 1) u = u * 4 + w;
    const int h = u % a.heads;
    u /= a.heads;
    const int i = u % a.b.rows_max, s = u / a.b.rows_max;
    if (s >= a.b.n_seq) return;
    const PagedRows r = paged_rows(a.b, s, a.M);
    if (i >= r.n) return;
    const int64_t row = r.r0 + i;
    const int lim = min(r.first + i, a.l_cap - 1), ng = lim < 0 ? 0 : lim / grp_keys + 1;
    const float2* ml = a.ws_ml + (row * a.heads + h) * a.n_grps;
    const float* o = a.ws_o + (row * a.heads + h) * a.n_grps * HD + lane * V;
    const float2 all = paged_total(ml, 1, ng, lane, 64);
    float acc[V] = {};
    for (int g0 = 0; g0 < ng; g0 += 64) {
      const float wg = g0 + lane < ng ? paged_weight(ml[g0 + lane].x, all.x) : 0.f;
      const int n = min(64, ng - g0);
      for (int q = WPP == 4 ? PA_RUN * w : 0; q < n; q += PA_RUN * WPP) {
        float x[PA_RUN][V], run[V] = {};
#pragma unroll
        for (int e = 0; e < PA_RUN; ++e)
#pragma unroll
          for (int v = 0; v < V; ++v) x[e][v] = o[(int64_t)(g0 + min(q + e, n - 1)) * HD + v];
#pragma unroll
        for (int e = 0; e < PA_RUN; ++e) {
          const float t = __shfl(wg, min(q + e, 63));
#pragma unroll
          for (int v = 0; v < V; ++v) run[v] = q + e < n ? fmaf(x[e][v], t, run[v]) : run[v];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if constexpr (WPP == 4) part[q / PA_RUN][lane * V + v] = run[v];
          else acc[v] += run[v];
        }
      }
      if constexpr (WPP == 4) {
        __syncthreads();
        for (int q = 0; w == 0 && q < n; q += PA_RUN)
#pragma unroll
          for (int v = 0; v < V; ++v) acc[v] += part[q / PA_RUN][lane * V + v];
        if (g0 + 64 < ng) __syncthreads();  // the runs have been read
      }
    }
    if (WPP == 4 && w) return;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = all.y == 0.f ? 0.f : acc[v] / all.y;
    bf16_t* dst = a.out + row * a.ldo + h * HD + lane * V;
    if constexpr (V == 2) *(uint32_t*)dst = pack_bf16x2(acc[0], acc[1]);
    else *dst = f2bf(acc[0]);
    return;
  }
  if constexpr (WK > 0) {
    int u = blockIdx.x;
    const int ch = u % a.chunks;
    u /= a.chunks;
    const int kvh = u % a.c.kv, s = u / a.c.kv;
    int page = -1;  // of the wave's block, read before the lengths are known, as in the first launch
    if (WK == 2 && (ch * 4 + w) * PAGE < a.l_cap) page = paged_page(a.b, s, ch * 4 + w, a.c.pages);
    const PagedRows r = paged_rows(a.b, s, a.M);
    const int end = min(r.first + r.n, a.l_cap);  // slots in use
    if (r.n == 0 || ch * (WK == 1 ? 1024 : 256) >= end) return;
    const int pairs = r.n * a.rep;
    float* dst = a.weights + s * a.ldw_seq + kvh * a.ldw;
    __shared__ float2 total[256];  // (m, 1 / l) of (row, head) pairs p0 ..
    // a pair whose scores are all -inf gives weights of 0
    auto ready = [](float2 t) { return make_float2(t.x == -INFINITY ? 0.f : t.x, t.y == 0.f ? 0.f : 1.f / t.y); };
    auto limit = [&](int p) { return min(r.first + p / a.rep, a.l_cap - 1); };  // the last slot that pair p attends
    // totals of the np pairs from p0 on, by lg lanes each
    auto totals = [&](int p0, int np) {
      int lg = 16;
      while (lg > 1 && 256 / lg < np) lg >>= 1;
      const int mine = min((int)threadIdx.x / lg, np - 1), lim = limit(p0 + mine);
      const float2 all = paged_total(a.ws_t + ((int64_t)kvh * a.n_grps * a.M + r.r0) * a.rep + p0 + mine, (int64_t)a.M * a.rep,
                                     lim < 0 ? 0 : lim / grp_keys + 1, threadIdx.x % lg, lg);
      if (threadIdx.x % lg == 0 && (int)threadIdx.x / lg < np) total[mine] = ready(all);
      __syncthreads();
    };
    auto share = [&](float x, float2 t) { return __builtin_amdgcn_exp2f(fmaf(x, a.scale_log2, -t.x)); };
    if constexpr (WK == 1) {
      const int key = ch * 1024 + threadIdx.x * 4;
      f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
      totals(0, pairs);
      for (int p = 0; p < pairs; p += 4) {  // four pairs' scores on their way at once; a pair past the last one repeats it and does not count
        f32x4_t x[4];
        int lim[4];
        float2 t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int pc = min(p + e, pairs - 1), i = pc / a.rep;
          lim[e] = p + e < pairs ? limit(pc) : -1;
          t[e] = total[pc];
          // slots that no block holds (behind the bound's last one) read the row's first
          x[e] = *(const f32x4_t*)(a.ws_s + ((int64_t)(r.r0 + i) * a.heads + kvh * a.rep + pc % a.rep) * a.ld_s + (key < a.ld_s ? key : 0));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int q = 0; q < 4; ++q) {  // scores of slots that are not attended may be anything
            const float wgt = share(x[e][q], t[e]) * t[e].y;
            sum[q] += key + q <= lim[e] ? wgt : 0.f;
          }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (key + q < end) dst[key + q] = a.decay == 0.f ? sum[q] : fmaf(a.decay, dst[key + q], sum[q]);
    } else {
      const int j = lane & 15, g = lane >> 4, blk = ch * 4 + w, key0 = blk * PAGE;
      page = key0 < end ? __builtin_amdgcn_readfirstlane(page) : -1;
      PagedFrags<HD> f;
      paged_load_k<HD>(f, a.c.k, ((size_t)max(page, 0) * a.c.kv + kvh) * PAGE * HD, lane);
      auto load_q = [&](int col, u32x4_t (&q)[HD / 32]) {
        const int pc = min(col, pairs - 1);
#pragma unroll
        for (int ks = 0; ks < HD / 32; ++ks)
          q[ks] = *(const u32x4_t*)(a.Q + (r.r0 + pc / a.rep) * a.ldq + (kvh * a.rep + pc % a.rep) * HD + ks * 32 + g * 8);
      };
      u32x4_t qn[HD / 32];
      load_q(j, qn);
      float sum[16] = {};
      for (int p0 = 0; p0 < pairs; p0 += 256) {
        const int np = min(256, pairs - p0);
        if (p0) __syncthreads();
        totals(p0, np);
        if (page < 0) continue;
        for (int c0 = 0; c0 < np; c0 += 16) {
          u32x4_t qf[HD / 32];
#pragma unroll
          for (int ks = 0; ks < HD / 32; ++ks) qf[ks] = qn[ks];
          load_q(p0 + c0 + 16 + j, qn);
          f32x4_t x[4] = {};
#pragma unroll
          for (int ks = 0; ks < HD / 32; ++ks)
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) x[kt] = mfma16x16x32(bits_bf16x8(f.k[kt][ks]), bits_bf16x8(qf[ks]), x[kt]);
          float2 t = total[min(c0 + j, np - 1)];
          if (c0 + j >= np) t.y = 0.f;  // the last pair again
          if (limit(p0 + c0) >= key0 + PAGE - 1) {  // every column attends the whole block
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[i] = fmaf(share(x[i / 4][i % 4], t), t.y, sum[i]);
          } else {  // scores of slots that are not attended may be anything
            const int left = limit(p0 + min(c0 + j, np - 1)) - key0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float wgt = share(x[i / 4][i % 4], t) * t.y;
              sum[i] += paged_key(i / 4, g, i % 4) <= left ? wgt : 0.f;
            }
          }
        }
      }
      float mine = 0.f;  // lane j: the sum over the columns of value j
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float v = sum[i];
        v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xb1, 0xf, 0xf, true));   // lane ^ 1
        v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4e, 0xf, 0xf, true));   // lane ^ 2
        v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xf, 0xf, true));  // the other half of 8
        v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xf, 0xf, true));  // the other half of 16
        mine = i == j ? v : mine;
      }
      const int at = key0 + paged_key(j >> 2, g, j & 3);
      if (at < end) dst[at] = a.decay == 0.f ? mine : fmaf(a.decay, dst[at], mine);
    }
  }
}

// Waves a (row, head): four where few pairs have many records (us of one row of 32 heads with 64 records, one wave / four: 8.9 / 5.5).
template <int HD, int WK>
static int launch_paged_join(PagedAttnArgs& a, hipStream_t stream) {
  const int64_t pairs = a.n_grps > 1 ? (int64_t)a.b.n_seq * a.b.rows_max * a.heads : 0;
  a.chunks = WK == 0 ? 0 : WK == 1 ? (a.l_cap + 1023) / 1024 : (a.l_cap + 255) / 256;
  const bool four = a.n_grps > 8 && pairs <= 2048;
  const int64_t sums = (int64_t)a.b.n_seq * a.c.kv * a.chunks, all = sums + (four ? pairs : (pairs + 3) / 4);
  if (paged_grid_too_large(all, 256)) return set_error(SSD_ERANGE, "paged_attention: too many workgroups");
  a.weight_wgs = (int)sums;
  if (four) SSD_LAUNCH((paged_join_kernel<HD, WK, 4>), dim3((unsigned)all), dim3(256), 0, stream, a);
  else SSD_LAUNCH((paged_join_kernel<HD, WK, 1>), dim3((unsigned)all), dim3(256), 0, stream, a);
  return check_launch("paged_attention_join");
}

static int paged_groups(int64_t l_max, int span) { return (int)((l_max + (int64_t)PA_WAVES * span - 1) / ((int64_t)PA_WAVES * span)); }
static int64_t paged_score_ld(int64_t l_max) { return (l_max + PAGE - 1) / PAGE * PAGE; }

template <int HD, int WK>
static int launch_paged_attn(PagedAttnArgs a, hipStream_t stream) {
  const int tiles = (int)(((int64_t)a.b.rows_max * a.rep + 15) / 16);
  a.sets = tiles;
  const int64_t units = paged_product({a.b.n_seq, a.n_grps, a.c.kv}), grid = paged_product({(units + 7) / 8 * 8, tiles});
  if (units > INT32_MAX || paged_grid_too_large(grid, 256)) return set_error(SSD_ERANGE, "paged_attention: too many workgroups");
  a.units = (int)units;
  // the second launch's size is checked before the first is enqueued
  if (paged_grid_too_large(paged_product({a.b.n_seq, a.b.rows_max * (int64_t)a.heads + (WK ? a.c.kv * (int64_t)(a.l_cap / 256 + 1) : 0)}), 256))
    return set_error(SSD_ERANGE, "paged_attention: too many workgroups");
  SSD_LAUNCH((paged_fold_kernel<HD, WK>), dim3((unsigned)grid), dim3(256), 0, stream, a);
  if (int rc = check_launch("paged_attention_fold")) return rc;
  return WK || a.n_grps > 1 ? launch_paged_join<HD, WK>(a, stream) : SSD_OK;
}

int paged_join(const PagedBatch& b, int M, int heads, int head_dim, int l_cap, int grp_keys, int n_grps, float* ws_o, float2* ws_ml,
               bf16_t* out, int64_t ldo, hipStream_t stream) {
  PagedAttnArgs a{};
  a.b = b, a.M = M, a.heads = heads, a.l_cap = l_cap, a.grp_keys = grp_keys, a.n_grps = n_grps;
  a.b.rows_max = std::min(b.rows_max, M);
  a.ws_o = ws_o, a.ws_ml = ws_ml, a.out = out, a.ldo = ldo;
  return head_dim == 64 ? launch_paged_join<64, 0>(a, stream) : launch_paged_join<128, 0>(a, stream);
}

}  // namespace ssd

using namespace ssd;

SSD_API int64_t ssd_paged_attn_ws_floats(int M, int heads, int head_dim, int64_t l_max, int span, int weights) {
  if (M < 0 || heads < 1 || head_dim < 1 || l_max < 1 || l_max > 1 << 30 || span < 64 || span % 64 || span > PA_MAX_SPAN) return -1;
  const int64_t pairs = (int64_t)M * heads, recs = paged_groups(l_max, span) * (int64_t)(head_dim + (weights ? 4 : 2));
  // scores are kept by a call of few pairs a kv head, which one of fewer rows than M may be
  const int64_t scored = weights == 0 ? 0 : weights <= PA_SCORES ? pairs : (int64_t)std::min(M, PA_SCORES) * heads;
  return std::max(paged_product({pairs, recs}), paged_product({scored, recs + paged_score_ld(l_max)}));
}

SSD_API int ssd_paged_attention_bf16(const SsdPagedKv* cache, const SsdPagedBatch* batch, const uint16_t* q, int64_t ldq, int M,
                                     int heads, int l_max, int span, float scale, float* ws, int64_t ws_floats, float* weights,
                                     int64_t ldw_seq, int64_t ldw, float decay, uint16_t* out, int64_t ldo, hipStream_t stream) {
  if (int rc = paged_check(cache, batch, "paged_attention")) return rc;
  if (M < 0 || heads < 1 || heads % cache->kv_heads)
    return set_error(SSD_EINVAL, "paged_attention: bad M=%d heads=%d kv_heads=%d", M, heads, cache->kv_heads);
  if (l_max < 1 || (int64_t)l_max > (int64_t)batch->table_cols * PAGE)
    return set_error(SSD_EINVAL, "paged_attention: l_max %d outside [1, %lld]", l_max, (long long)batch->table_cols * PAGE);
  if (!(scale > 0.f) || scale > 1e30f) return set_error(SSD_EINVAL, "paged_attention: scale must be positive, got %g", scale);
  if (span < 64 || span % 64 || span > PA_MAX_SPAN)
    return set_error(SSD_EINVAL, "paged_attention: span %d must be a multiple of 64 up to %d", span, PA_MAX_SPAN);
  if (M == 0 || batch->n_seq == 0 || batch->rows_max == 0) return SSD_OK;
  if (!q || !ws || !out) return set_error(SSD_EINVAL, "paged_attention: null pointer");
  const int64_t cols = (int64_t)heads * cache->head_dim;
  if (((uintptr_t)q & 15) || ldq % 8 || ldq < cols || ((uintptr_t)out & 15) || ldo % 8 || ldo < cols)
    return set_error(SSD_EINVAL, "paged_attention: q/out rows must be 16-byte aligned with strides >= heads * head_dim");
  const int rep = heads / cache->kv_heads;
  const int wk = !weights ? 0 : (int64_t)std::min(batch->rows_max, M) * rep <= PA_SCORES ? 1 : 2;
  if (wk == 2 && q == out)  // the second launch reads q while it writes out
    return set_error(SSD_EINVAL, "paged_attention: out must not be q where weights are made from it (more than %d pairs a kv head)", PA_SCORES);
  const int64_t recs = paged_product({M, heads, paged_groups(l_max, span)});
  if (((uintptr_t)ws & 15) || ws_floats < paged_product({recs, cache->head_dim + (wk ? 4 : 2)}) +
                                              (wk == 1 ? paged_product({M, heads, paged_score_ld(l_max)}) : 0))
    return set_error(SSD_EINVAL, "paged_attention: workspace too small or not 16-byte aligned");
  if (weights && (ldw < l_max || ldw_seq < (int64_t)cache->kv_heads * ldw))
    return set_error(SSD_EINVAL, "paged_attention: weights rows of %lld for l_max %d, sequences %lld apart", (long long)ldw, l_max,
                     (long long)ldw_seq);
  if (weights && !(decay >= 0.f && decay <= 1.f)) return set_error(SSD_EINVAL, "paged_attention: decay must be in [0, 1], got %g", decay);
  PagedAttnArgs a{};
  a.b = paged_batch(batch);
  a.b.rows_max = std::min(a.b.rows_max, M);
  a.c = PagedCache{cache->k, cache->v, cache->pages, cache->kv_heads};
  a.Q = q, a.ldq = ldq, a.M = M, a.heads = heads, a.rep = rep, a.l_cap = l_max;
  a.span_blk = span / PAGE, a.n_grps = paged_groups(l_max, span), a.grp_keys = PA_WAVES * span, a.scale_log2 = scale * 1.4426950408889634f;
  a.ws_o = ws, a.ws_ml = (float2*)(ws + recs * cache->head_dim);
  a.ws_t = a.ws_ml + recs, a.ws_s = (float*)(a.ws_t + recs), a.ld_s = paged_score_ld(l_max);
  a.out = out, a.ldo = ldo, a.weights = weights, a.ldw_seq = ldw_seq, a.ldw = ldw, a.decay = decay;
  if (cache->head_dim == 64)
    return wk == 0 ? launch_paged_attn<64, 0>(a, stream) : wk == 1 ? launch_paged_attn<64, 1>(a, stream) : launch_paged_attn<64, 2>(a, stream);
  return wk == 0 ? launch_paged_attn<128, 0>(a, stream) : wk == 1 ? launch_paged_attn<128, 1>(a, stream) : launch_paged_attn<128, 2>(a, stream);
}
