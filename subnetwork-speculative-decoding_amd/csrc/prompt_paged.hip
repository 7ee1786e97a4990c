// Causal attention of whole prompts, or further pieces of them, over the paged cache (paged.h): packed rows of sequences of different
// lengths in one launch.
//
// The columns of S^T = K Q^T are the (row, q head) pairs of one sequence and kv head, rows outermost: whatever the number of
// heads that share a kv head, a workgroup of four waves has 128 columns of one kv head, 32 a wave, and a block's K and V are copied
// into LDS once for all of them (global to LDS, 16 bytes a lane, into two buffers each). Blocks are folded with a running
// reference m, sum l and output O in fp32; the reference follows a column's maximum only when that has grown by more than
// 2^8. Probabilities are rounded to bf16 as the second product's operand; l sums them as rounded, so that what a rounding does to a
// weight that dominates it does to l too.
//
// v_mfma_f32_32x32x16_bf16 rather than 16x16x32: the vector pipe stands still for about 8 cycles with every matrix instruction that another
// wave issues, whatever its size, so half as many of twice the work leave it more (a wave of products beside one of multiply-adds:
// 406 ns against 345 for the same work). While a block's scores become probabilities and meet V, the next block's scores are
// under way; the blocks that some columns attend only part of, one or two a tile, follow without that.
// What bounds it, 32 heads on 8 kv heads of 128 (8b shapes): a prompt of 16384 rows 1.94 ms, 1130 TFLOP/s, where a large library product reaches
// 1280: matrix pipe and vector pipe, each about half of a block's 1.9 us for two workgroups a CU, at the clock that the power leaves.
// Shorter prompts: a tile's beginning and end, about 8 us (rows, pages, first copies; the partly attended blocks; the output), of
// which a second workgroup on the CU hides half, and the last tiles' end: 4096 rows 134 us when a graph repeats the call, 143 among
// passes with their write (960 TFLOP/s), 16 prompts of up to 1500 rows 155 and 164.
// Tried (us of 16 prompts with the write of their K and V, 191 on that card): tiles dealt to resident workgroups, the next one's first
// blocks copied before the output 202; the longest tiles of all sequences first 192. Eight waves a workgroup: a prompt of 4096 rows 138 against 147, of 2048 60 against 50,
// 16 prompts 170 against 160. 64 columns a wave with twice the registers: 4096 rows 269 for 157; two groups of waves that take
// turns at the matrix pipe 155.
#include "paged.h"

#include <algorithm>
#include <type_traits>

namespace ssd {

constexpr int PP_WAVES = 4;

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4;

struct PagedPromptArgs {
  PagedBatch b;
  PagedCache c;
  const bf16_t* Q;
  int64_t ldq;
  int M, heads, rep, l_cap;
  float scale_log2;
  bf16_t* out;
  int64_t ldo;
  int splits, per;  // the length in `splits` parts of `per` blocks
  float* ws_o;      // [row][head][part][HD]: O, for more than one part
  float2* ws_ml;    // [row][head][part]: (m, l)
};

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16_t;

// A wave's 32 columns. v_mfma_f32_32x32x16_bf16 leaves lane (g, n) = 32 g + n column n's rows 8 (r / 4) + 4 g + r % 4 in register r. The
// keys of a half block are assigned to the rows so that registers 8 u .. 8 u + 7 are slots 16 u + 8 g .. + 8 of the half: the second product's
// operand without a move between lanes, against eight consecutive slots of V.
template <int HD>
struct PromptState {
  u32x4_t qf[HD / 16];  // dims 16 q + 8 g .. + 8 of the lane's column
  float m, l;           // reference (log2 units), this lane's part of the sum
  f32x16_t o[HD / 32];  // dims 32 d + 8 (r / 4) + 4 g + r % 4
  int lim;              // the last slot that the column attends
};

__device__ __forceinline__ f32x16_t mfma32x32x16(u32x4_t a, u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(bits_bf16x8(a), bits_bf16x8(b), c, 0, 0, 0);
}

__device__ __forceinline__ int prompt_key(int c, int r, int g) { return 32 * c + 16 * (r >> 3) + 8 * g + (r & 7); }

// Where this lane reads its operands of K and of V in LDS (16-byte pieces; a block lies there as in the page).
struct PromptLanes {
  int k, v;
};
template <int HD>
__device__ __forceinline__ PromptLanes prompt_lanes(int lane) {
  const int g = lane >> 5, h = lane >> 3 & 1, i = (lane >> 4 & 1) * 8 + (lane & 7);
  return PromptLanes{h * (HD / 32) * 64 + g * 16 + i, (lane >> 4 & 1) * 128 + g * 16 + (lane & 15)};
}

// Copies one arena's 64-key block into LDS: wave w, load i takes tile W i + w.
template <int HD>
__device__ __forceinline__ void prompt_copy(const bf16_t* from, int w, int lane, lds_u32x4* to) {
  constexpr int W = PP_WAVES;
  const char* p = (const char*)from + w * 1024;
#pragma unroll
  for (int i = 0; i < HD / 8 / W; ++i)
    __builtin_amdgcn_global_load_lds((const void*)(p + 1024 * W * i + (uint32_t)lane * 16), (lds_void*)(to + 64 * (W * i + w)), 16, 0, 0);
}

template <int HD>
__device__ __forceinline__ void prompt_qk(const PromptState<HD>& st, const PromptLanes& at, const lds_u32x4* __restrict__ ck, f32x16_t (&s)[2]) {
  s[0] = f32x16_t{}, s[1] = f32x16_t{};
#pragma unroll
  for (int q = 0; q < HD / 16; ++q)
#pragma unroll
    for (int c = 0; c < 2; ++c)
      s[c] = mfma32x32x16(ck[at.k + (2 * c * (HD / 32) + q / 2) * 64 + q % 2 * 32], st.qf[q], s[c]);
}

// Takes the reference to the block's maximum where that has outgrown it.
template <int HD>
__device__ __forceinline__ void prompt_reference(PromptState<HD>& st, const f32x16_t (&s)[2], float scale_log2) {
  float mx = -INFINITY;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[c][r]);
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
  mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * scale_log2;
  const bool grow = mx > st.m + 8.f || (st.m == -INFINITY && mx != st.m);
  if (!__any(grow)) return;
  asm volatile("" ::: "memory");  // a branch that is taken now and then, not products with 1 in every block
  const float alpha = grow ? __builtin_amdgcn_exp2f(st.m - mx) : 1.f;
  st.l *= alpha;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d) st.o[d] *= alpha;
  st.m = grow ? mx : st.m;
}

// l plus two bf16 values, in fp32.
__device__ __forceinline__ float prompt_sum2(uint32_t two, float l) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, two), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), l, false);
}

template <int HD>
__device__ __forceinline__ void prompt_exp(PromptState<HD>& st, const f32x16_t (&s)[2], float scale_log2, u32x4_t (&p)[4]) {
  const float ms = st.m == -INFINITY ? 0.f : st.m;  // nothing attended so far: every p is 0
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[c][r], scale_log2, -ms));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s[c][r + 1], scale_log2, -ms));
      const uint32_t both = pack_bf16x2(p0, p1);
      st.l = prompt_sum2(both, st.l);
      p[2 * c + r / 8][r % 8 / 2] = both;
    }
}

template <int HD>
__device__ __forceinline__ void prompt_pv(PromptState<HD>& st, const PromptLanes& at, const lds_u32x4* __restrict__ cv, const u32x4_t (&p)[4]) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) st.o[d] = mfma32x32x16(cv[at.v + (4 * d + t / 2) * 64 + t % 2 * 32], p[t], st.o[d]);
}

// The t-th tile of CW columns: the tiles of all sequences are numbered one behind the other, each sequence's last first. Every wave
// finds it for itself.
struct PromptTile {
  int seq, tile;
  PagedRows rows;
};
template <int CW>
__device__ __forceinline__ PromptTile prompt_tile(const PagedPromptArgs& a, int t, int lane) {
  for (int s0 = 0; s0 < a.b.n_seq; s0 += 64) {
    const PagedRows r = paged_rows(a.b, min(s0 + lane, a.b.n_seq - 1), a.M);
    int inc = s0 + lane < a.b.n_seq ? (r.n * a.rep + CW - 1) / CW : 0;
    for (int o = 1; o < min(a.b.n_seq - s0, 64); o <<= 1) {  // as many steps as there are sequences to add up
      const int x = __shfl_up(inc, o);
      if (lane >= o) inc += x;
    }
    const uint64_t past = __ballot(inc > t);
    if (past) {
      const int l = __builtin_ctzll(past);
      return PromptTile{s0 + l, __builtin_amdgcn_readlane(inc, l) - 1 - t,
                        PagedRows{__builtin_amdgcn_readlane(r.r0, l), __builtin_amdgcn_readlane(r.n, l), __builtin_amdgcn_readlane(r.first, l)}};
    }
    t -= __builtin_amdgcn_readlane(inc, 63);
  }
  return PromptTile{-1, 0, {}};
}

// Workgroup (tile of 32 W columns of some sequence, kv head). The kv head varies fastest: with eight of them an XCD serves one, whose
// blocks its L2 keeps. TURNS: the workgroups of a CU take turns at going first (prompt_turns).
template <int HD, bool TURNS>
__global__ __launch_bounds__(256, 2) void paged_prompt_kernel(PagedPromptArgs a) {
  constexpr int W = PP_WAVES, CW = 32 * W, PIECES = 64 * HD / 8;
  __shared__ int first_bad[HD], any_bad;
  __shared__ __align__(16) u32x4_t kA[PIECES], vA[PIECES], kB[PIECES], vB[PIECES];
  typedef __attribute__((address_space(3))) u32x4_t* lp;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, g = lane >> 5;
  if (TURNS) __builtin_amdgcn_s_setprio(1);
  int u = blockIdx.x;
  const int kvh = u % a.c.kv;
  u /= a.c.kv;
  const int part = u % a.splits;
  const PromptTile pt = prompt_tile<CW>(a, u / a.splits, lane);
  if (pt.seq < 0) return;
  const int seq = pt.seq, c0 = pt.tile * CW, w0 = c0 + w * 32;
  const PagedRows r = pt.rows;
  const int n_cols = r.n * a.rep;
  auto lim_of = [&](int col) { return min(r.first + min(col, n_cols - 1) / a.rep, a.l_cap - 1); };
  const int last = lim_of(c0 + CW - 1), n_blk = min(last < 0 ? 0 : last / PAGE + 1, (part + 1) * a.per);
  const int full = min((lim_of(c0) + 1) / PAGE, n_blk);  // blocks that every column attends whole
  const int hi = w0 < n_cols ? lim_of(w0 + 31) : -1;     // this wave's last key
  int base = part * a.per;
  if (part && base >= n_blk) return;  // no record: the join counts the parts as this does
  int pages = base + lane < n_blk ? paged_page(a.b, seq, base + lane, a.c.pages) : -1;
  const PromptLanes at = prompt_lanes<HD>(lane);
  PromptState<HD> st;
  {
    const int col = min(w0 + n, n_cols - 1), i = col / a.rep;
    st.lim = min(r.first + i, a.l_cap - 1);
    const bf16_t* q = a.Q + (int64_t)(r.r0 + i) * a.ldq + (kvh * a.rep + col % a.rep) * HD;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) st.qf[k] = *(const u32x4_t*)(q + k * 16 + g * 8);
    st.m = -INFINITY, st.l = 0.f;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) st.o[d] = f32x16_t{};
  }
  // the blocks that exist, in order: lane i has the page of block base + i, live those not yet handed out
  struct Block {
    int b;
    size_t at;
  };
  uint64_t live = __ballot(pages >= 0);
  auto next = [&] {
    while (!live && (base += 64) < n_blk) {
      pages = base + lane < n_blk ? paged_page(a.b, seq, base + lane, a.c.pages) : -1;
      live = __ballot(pages >= 0);
    }
    if (!live) return Block{INT32_MAX, 0};
    const int i = __builtin_ctzll(live);
    live &= live - 1;
    return Block{base + i, ((size_t)__builtin_amdgcn_readlane(pages, i) * a.c.kv + kvh) * PAGE * HD};
  };
  auto copy_k = [&](const Block& x, lds_u32x4* to) {
    if (x.b < n_blk) prompt_copy<HD>(a.c.k + x.at, w, lane, to);
  };
  auto copy_v = [&](const Block& x, lds_u32x4* to) {
    if (x.b < n_blk) prompt_copy<HD>(a.c.v + x.at, w, lane, to);
  };
  // What was copied has landed (a barrier does not wait for it), and every wave is done with the other buffers.
  auto landed = [&] {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  for (int i = threadIdx.x; i < HD; i += 64 * W) first_bad[i] = INT32_MAX;
  if (threadIdx.x == 0) any_bad = 0;
  Block cur = next(), nxt = next();  // K and V of the i-th existing block go to buffers A for even i, B for odd
  copy_k(cur, (lp)kA);
  copy_v(cur, (lp)vA);
  copy_k(nxt, (lp)kB);
  landed();
  bool odd = false;
  if (cur.b < full) {
    f32x16_t s0[2], s1[2];
    u32x4_t p[4];
    prompt_qk<HD>(st, at, (lp)kA, s0);
    prompt_reference<HD>(st, s0, a.scale_log2);
    // scores s of the present block; V in cv; the next block's K in nk, its scores into sn; free: ck, nv
    auto step = [&](f32x16_t (&s)[2], f32x16_t (&sn)[2], lds_u32x4* ck, lds_u32x4* cv, lds_u32x4* nk, lds_u32x4* nv) {
      landed();
      const Block then = next();
      copy_k(then, ck);
      copy_v(nxt, nv);
      __builtin_amdgcn_sched_barrier(0);
      prompt_qk<HD>(st, at, nk, sn);
      prompt_exp<HD>(st, s, a.scale_log2, p);
      prompt_pv<HD>(st, at, cv, p);
      prompt_reference<HD>(st, sn, a.scale_log2);
      cur = nxt, nxt = then;
    };
    while (nxt.b < full) {
      if (TURNS) __builtin_amdgcn_s_setprio(2);
      step(s0, s1, (lp)kA, (lp)vA, (lp)kB, (lp)vB);
      odd = true;
      if (!(nxt.b < full)) break;
      if (TURNS) __builtin_amdgcn_s_setprio(0);
      step(s1, s0, (lp)kB, (lp)vB, (lp)kA, (lp)vA);
      odd = false;
    }
    if (TURNS) __builtin_amdgcn_s_setprio(1);
    // the last of them
    landed();
    const Block then = next();
    copy_k(then, odd ? (lp)kB : (lp)kA);
    copy_v(nxt, odd ? (lp)vA : (lp)vB);
    if (odd) {
      prompt_exp<HD>(st, s1, a.scale_log2, p);
      prompt_pv<HD>(st, at, (lp)vB, p);
    } else {
      prompt_exp<HD>(st, s0, a.scale_log2, p);
      prompt_pv<HD>(st, at, (lp)vA, p);
    }
    cur = nxt, nxt = then;
    odd = !odd;
    landed();
  }
  // blocks that some columns attend only part of: K and V of the present one and K of the next one have landed
  for (; cur.b < n_blk; odd = !odd) {
    const lds_u32x4* ck = odd ? (lp)kB : (lp)kA;
    lds_u32x4 *cv = odd ? (lp)vB : (lp)vA, *nv = odd ? (lp)vA : (lp)vB;
    copy_v(nxt, nv);
    // V values that are not finite are taken out
#pragma unroll
    for (int i = 0; i < HD / 8 / W; ++i) {
      const int x = 64 * W * i + (int)threadIdx.x;  // piece x: tile x / 64, lane x % 64
      const u32x4_t y = cv[x];
      if (paged_not_finite(y[0]) || paged_not_finite(y[1]) || paged_not_finite(y[2]) || paged_not_finite(y[3]))
        cv[x] = paged_take_out(y, cur.b * PAGE + (x >> 6 & 1) * 32 + (x >> 4 & 3) * 8, &first_bad[(x >> 7) * 16 + (x & 15)]), any_bad = 1;
    }
    __syncthreads();
    if (cur.b * PAGE <= hi) {
      f32x16_t s[2];
      u32x4_t p[4];
      prompt_qk<HD>(st, at, ck, s);
      const int left = st.lim - cur.b * PAGE + 1;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[c][e] = prompt_key(c, e, g) < left ? s[c][e] : -INFINITY;
      prompt_reference<HD>(st, s, a.scale_log2);
      prompt_exp<HD>(st, s, a.scale_log2, p);
      prompt_pv<HD>(st, at, cv, p);
    }
    __syncthreads();  // this block's K buffer is free
    const Block then = next();
    copy_k(then, odd ? (lp)kB : (lp)kA);
    cur = nxt, nxt = then;
    landed();
  }
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(st.l), __float_as_uint(st.l), false, false);
  const float l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]), inv = a.splits > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;  // NaN stays NaN
#pragma unroll
  for (int d = 0; d < HD / 32; ++d) st.o[d] *= inv;
  if (any_bad) {
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (st.lim >= first_bad[32 * d + e / 4 * 8 + 4 * g + e % 4]) st.o[d][e] = __uint_as_float(0x7fc00000u);
  }
  if (a.splits > 1) {
    const int col = w0 + n;
    if (col >= n_cols) return;
    const int64_t rec = ((int64_t)(r.r0 + col / a.rep) * a.heads + kvh * a.rep + col % a.rep) * a.splits + part;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(f32x4_t*)(a.ws_o + rec * HD + 32 * d + 8 * i + 4 * g) =
            f32x4_t{st.o[d][4 * i], st.o[d][4 * i + 1], st.o[d][4 * i + 2], st.o[d][4 * i + 3]};
    if (g == 0) a.ws_ml[rec] = make_float2(st.m, l);
    return;
  }
  // The wave's columns leave through LDS as whole rows: 16-byte pieces, piece i of column c at i ^ (c & 7) of its row.
  constexpr int PC = HD / 8;
  lds_u32x4* mine = w & 1 ? (w & 2 ? (lp)vB : (lp)vA) : (w & 2 ? (lp)kB : (lp)kA);
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
      const u32x2_t x = {pack_bf16x2(st.o[d][4 * i], st.o[d][4 * i + 1]), pack_bf16x2(st.o[d][4 * i + 2], st.o[d][4 * i + 3])};
      ((__attribute__((address_space(3))) u32x2_t*)(mine + n * PC + ((4 * d + i) ^ (n & 7))))[g] = x;
    }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int i = 0; i < PC / 2; ++i) {
    const int x = 64 * i + lane, c = x / PC, col = w0 + c;
    if (col < n_cols) *(u32x4_t*)(a.out + (int64_t)(r.r0 + col / a.rep) * a.ldo + (kvh * a.rep + col % a.rep) * HD + x % PC * 8) =
        mine[c * PC + (x % PC ^ (c & 7))];
  }
}

// Workgroups of a call with the length in one part, as near as the host can tell: every sequence's tiles are at most those of the
// longest one's rows, exact for rows of one number, and together at most a whole-tile share of the rows and one more each.
static int64_t prompt_tiles(int64_t M, int rep, int n_seq, int rows_max, int kv) {
  constexpr int CW = 32 * PP_WAVES;
  const int64_t most = (std::min<int64_t>(rows_max, M) * rep + CW - 1) / CW;
  return paged_product({std::min(M * rep / CW + n_seq, n_seq * most), kv});
}

// Parts of the length: one while the tiles fill the chip's 256 CUs, else as many as bring two workgroups a CU, of eight blocks or more
// (one / several parts, us: 100 rows of 32 heads after 8000 keys 136 / 37, 500 149 / 87, 40 rows of 15 heads 134 / 22, 16 sequences of 32
// rows of 32 heads after 8000 keys 151 / 120). Two parts pay for their records only over a long length (4 times 100 rows of 64 heads after
// 4000 keys 77 / 83; 700 rows of 32 heads after 6500 126 / 116, 900 after 16000 286 / 262), and not where sequences of one tile read K and V
// once, which is bound by bytes (24 of 32 rows after 8000 168 / 169, 31 192 / 213).
// Where eight blocks a part leave the CUs' second places part empty, one workgroup a CU is better (192 rows after 4000 in 7 / 5 parts 34 / 30,
// 320 after 2000 in 4 / 3 34 / 30, six sequences of 32 rows after 4000 in 7 / 5 34 / 32).
// The fewer rows the longest sequence can have, the fewer tiles and the more parts: rows_max 0 asks for the most.
static int prompt_splits(int64_t M, int rep, int n_seq, int rows_max, int kv, int64_t l_max) {
  const int64_t longest = std::max<int64_t>(rows_max, (M + n_seq - 1) / std::max(n_seq, 1));
  const int64_t wgs = prompt_tiles(M, rep, n_seq, (int)longest, kv), blocks = (l_max + PAGE - 1) / PAGE;
  if (wgs >= 256) return 1;
  int64_t n = std::max<int64_t>(1, std::min(512 / std::max<int64_t>(wgs, 1), blocks / 8));
  const int64_t round = 256 / std::max<int64_t>(wgs, 1);
  if (rows_max && round >= 2 && wgs * n > 256 && wgs * n < 435 && wgs * round >= 205) n = round;
  return n == 2 && (blocks < 96 || (rows_max && longest * rep <= 32 * PP_WAVES)) ? 1 : (int)n;
}

// Of two workgroups on a CU the older one's waves go first, and its tile ends long before the other's (1.7 us a block against 2.4). That is
// as it should be where a last, part round of tiles follows or the longest tiles begin first and all at once. Where all tiles make two
// rounds, or a little more than one behind pasts of different lengths, they had better end together: a wave's priority then goes up and
// down from block to block. us without / with, heads of 128, by workgroups for the 512 places. One prompt: 2048 rows (512) 52 / 54, 3000
// (752) 81 / 84, 3300 (832) 98 / 96, 3600 (904) 115 / 108, 4096 (1024) 143 / 135, 4480 (1120) 166 / 165; of 64 heads 2048 rows (1024) 79 / 74,
// 2240 (1120) 90 / 91. Two prompts of 2048 rows (1024) 80 / 76, but four of 1024 50 / 54. Five pieces of 512 to 1024 rows behind 0 to 4000
// keys (960) 183 / 170; 16 of 256 behind 2000 each (1024) 147 / 148. A little over one round, pieces of 64 heads behind 2500 to 5000 keys
// (528) 150 / 144, (608) 184 / 167; behind 5000 each (528) 231 / 240, (608) 237 / 245: the host cannot tell these apart, and lengths that
// differ are the rule. A whole round behind 5000 each (512) 166 / 164, behind 2500 to 5000 134 / 139. Heads of 64: 2048 rows 35 / 39.
static bool prompt_turns(int64_t wgs, int rows_max, int l_max) {
  return (wgs >= 820 && wgs <= 1126) || (wgs > 512 && wgs <= 614 && rows_max <= l_max / 2);  // 1.6 to 2.2 rounds, 1 to 1.2
}

template <int HD>
static int launch_paged_prompt(const PagedPromptArgs& a, hipStream_t stream) {
  const int64_t wgs = prompt_tiles(a.M, a.rep, a.b.n_seq, a.b.rows_max, a.c.kv) * a.splits;
  if (paged_grid_too_large(wgs, 256)) return set_error(SSD_ERANGE, "paged_prompt: too many workgroups");
  if constexpr (HD == 128) {
    if (prompt_turns(wgs, a.b.rows_max, a.l_cap)) SSD_LAUNCH((paged_prompt_kernel<HD, true>), dim3((unsigned)wgs), dim3(256), 0, stream, a);
    else SSD_LAUNCH((paged_prompt_kernel<HD, false>), dim3((unsigned)wgs), dim3(256), 0, stream, a);
  } else {
    SSD_LAUNCH((paged_prompt_kernel<HD, false>), dim3((unsigned)wgs), dim3(256), 0, stream, a);
  }
  if (int rc = check_launch("paged_prompt")) return rc;
  if (a.splits == 1) return SSD_OK;
  return paged_join(a.b, a.M, a.heads, HD, a.l_cap, a.per * PAGE, a.splits, a.ws_o, a.ws_ml, a.out, a.ldo, stream);
}

}  // namespace ssd

using namespace ssd;

SSD_API int64_t ssd_paged_prompt_ws_floats(int M, int heads, int kv_heads, int head_dim, int n_seq, int64_t l_max) {
  if (M < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || n_seq < 0 || l_max < 1 || l_max > 1 << 30) return -1;
  const int splits = prompt_splits(M, heads / kv_heads, n_seq, 0, kv_heads, l_max);
  return splits == 1 ? 0 : (int64_t)M * heads * splits * (head_dim + 2);
}

SSD_API int ssd_paged_prompt_bf16(const SsdPagedKv* cache, const SsdPagedBatch* batch, const uint16_t* q, int64_t ldq, int M, int heads,
                                  int l_max, float scale, float* ws, int64_t ws_floats, uint16_t* out, int64_t ldo,
                                  hipStream_t stream) {
  if (int rc = paged_check(cache, batch, "paged_prompt")) return rc;
  if (M < 0 || heads < 1 || heads % cache->kv_heads)
    return set_error(SSD_EINVAL, "paged_prompt: bad M=%d heads=%d kv_heads=%d", M, heads, cache->kv_heads);
  if (l_max < 1 || (int64_t)l_max > (int64_t)batch->table_cols * PAGE)
    return set_error(SSD_EINVAL, "paged_prompt: l_max %d outside [1, %lld]", l_max, (long long)batch->table_cols * PAGE);
  if (!(scale > 0.f) || scale > 1e30f) return set_error(SSD_EINVAL, "paged_prompt: scale must be positive, got %g", scale);
  if (M == 0 || batch->n_seq == 0 || batch->rows_max == 0) return SSD_OK;
  if (!q || !out) return set_error(SSD_EINVAL, "paged_prompt: null pointer");
  const int64_t cols = (int64_t)heads * cache->head_dim;
  if (((uintptr_t)q & 15) || ldq % 8 || ldq < cols || ((uintptr_t)out & 15) || ldo % 8 || ldo < cols)
    return set_error(SSD_EINVAL, "paged_prompt: q/out rows must be 16-byte aligned with strides >= heads * head_dim");
  if ((int64_t)M * heads > INT32_MAX / 2) return set_error(SSD_ERANGE, "paged_prompt: %d rows of %d heads", M, heads);
  PagedPromptArgs a{};
  a.b = paged_batch(batch);
  a.c = PagedCache{cache->k, cache->v, cache->pages, cache->kv_heads};
  a.Q = q, a.ldq = ldq, a.M = M, a.heads = heads, a.rep = heads / cache->kv_heads, a.l_cap = l_max;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = out, a.ldo = ldo;
  a.splits = prompt_splits(M, a.rep, batch->n_seq, batch->rows_max, a.c.kv, l_max);
  const int64_t need = a.splits == 1 ? 0 : (int64_t)M * heads * a.splits * (cache->head_dim + 2);
  if (need && (!ws || ((uintptr_t)ws & 15) || ws_floats < need))
    return set_error(SSD_EINVAL, "paged_prompt: workspace too small or not 16-byte aligned");
  a.per = ((l_max + PAGE - 1) / PAGE + a.splits - 1) / a.splits;
  a.ws_o = ws, a.ws_ml = (float2*)(ws + (int64_t)M * heads * a.splits * cache->head_dim);
  return cache->head_dim == 64 ? launch_paged_prompt<64>(a, stream) : launch_paged_prompt<128>(a, stream);
}
