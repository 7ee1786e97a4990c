// Causal attention of whole prompts, or further pieces of them, over the paged cache (paged.h): packed rows of sequences of different
// lengths in one launch.
//
// The columns of S^T = K Q^T are the (row, q head) pairs of one sequence and kv head, rows outermost: whatever the number of
// heads that share a kv head, a workgroup of four waves has 64 NT columns of one kv head, and a block's K and V are copied into
// LDS once for all of them (global to LDS, 16 bytes a lane, one block ahead of their use, in two buffers). Blocks are folded with a
// running reference m, sum l and output O in fp32; the reference follows a column's maximum only when that has grown by more than
// 2^8. Probabilities are rounded to bf16 as the second product's operand; l sums them before that.
#include "paged.h"

#include <algorithm>
#include <type_traits>

namespace ssd {

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
};

template <int HD, int NT>
struct PromptState {
  u32x4_t qf[NT][HD / 32];
  float m[NT], l[NT];  // reference (log2 units), this lane's part of the sum
  f32x4_t o[NT][HD / 16];
  int lim[NT];         // the last slot that this lane's column attends
};

// Copies the 64-key block at element offset `at` of both arenas into LDS: wave w, load i takes pieces 256 i + 64 w + lane.
template <int HD>
__device__ __forceinline__ void prompt_copy(const PagedCache& c, size_t at, int w, int lane, lds_u32x4* k, lds_u32x4* v) {
  const char *ks = (const char*)(c.k + at) + w * 1024, *vs = (const char*)(c.v + at) + w * 1024;
  const uint32_t l16 = lane * 16;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) {
    __builtin_amdgcn_global_load_lds((const void*)(ks + 4096 * i + l16), (lds_void*)(k + 256 * i + 64 * w), 16, 0, 0);
    __builtin_amdgcn_global_load_lds((const void*)(vs + 4096 * i + l16), (lds_void*)(v + 256 * i + 64 * w), 16, 0, 0);
  }
}

// One block from LDS into the wave's columns. MASKED: some column may not attend all of it.
template <int HD, int NT, bool MASKED>
__device__ __forceinline__ void prompt_block(PromptState<HD, NT>& st, int key0, float scale_log2, int lane,
                                             const lds_u32x4* __restrict__ ck, const lds_u32x4* __restrict__ cv) {
  constexpr int KS = HD / 32, DT = HD / 16;
  const int g = lane >> 4;
  f32x4_t s[NT][4];
#pragma unroll
  for (int rt = 0; rt < NT; ++rt)
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) s[rt][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const u32x4_t kf = ck[(kt * KS + ks) * 64 + lane];
#pragma unroll
      for (int rt = 0; rt < NT; ++rt) s[rt][kt] = mfma16x16x32(bits_bf16x8(kf), bits_bf16x8(st.qf[rt][ks]), s[rt][kt]);
    }
  u32x4_t vf[DT][2];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int c = 0; c < 2; ++c) vf[dt][c] = cv[(dt * 2 + c) * 64 + lane];
#pragma unroll
  for (int rt = 0; rt < NT; ++rt) {
    const int left = st.lim[rt] - key0 + 1;
    u32x4_t pw[2];
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (MASKED) s[rt][kt][e] = paged_key(kt, g, e) < left ? s[rt][kt][e] : -INFINITY;
        mx = fmaxf(mx, s[rt][kt][e]);
      }
    mx = paged_max_lanes(mx) * scale_log2;
    const bool grow = mx > st.m[rt] + 8.f || (st.m[rt] == -INFINITY && mx != st.m[rt]);
    const float m = grow ? mx : st.m[rt], ms = m == -INFINITY ? 0.f : m;
    if (__any(grow)) {  // multiplying by 1 changes nothing
      const float alpha = grow ? __builtin_amdgcn_exp2f(st.m[rt] - ms) : 1.f;
      st.l[rt] *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) st.o[rt][dt] *= alpha;
    }
    st.m[rt] = m;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[rt][kt][e], scale_log2, -ms));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[rt][kt][e + 1], scale_log2, -ms));
        st.l[rt] += p0 + p1;
        pw[kt >> 1][(kt & 1) * 2 + e / 2] = pack_bf16x2(p0, p1);
      }
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) st.o[rt][dt] = mfma16x16x32(bits_bf16x8(vf[dt][c]), bits_bf16x8(pw[c]), st.o[rt][dt]);
  }
}

// Workgroup (tile of 64 NT columns of some sequence, kv head); the tiles of all sequences are numbered one behind the other, each
// sequence's last rows, which attend the most, first. The kv head varies fastest: with eight of them an XCD serves one, whose
// blocks its L2 keeps.
template <int HD, int NT>
__global__ __launch_bounds__(256, 2) void paged_prompt_kernel(PagedPromptArgs a) {
  constexpr int KS = HD / 32, DT = HD / 16, CW = 64 * NT, PIECES = 64 * HD / 8;
  __shared__ int first_bad[HD];
  __shared__ __align__(16) u32x4_t kA[PIECES], vA[PIECES], kB[PIECES], vB[PIECES];
  typedef __attribute__((address_space(3))) u32x4_t* lp;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x % a.c.kv;
  // every wave finds the tile's sequence for itself
  int t = blockIdx.x / a.c.kv, seq = -1, tile = 0;
  for (int s0 = 0; s0 < a.b.n_seq; s0 += 64) {
    const int cnt = s0 + lane < a.b.n_seq ? (paged_rows(a.b, s0 + lane, a.M).n * a.rep + CW - 1) / CW : 0;
    int inc = cnt;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(inc, o);
      if (lane >= o) inc += x;
    }
    const uint64_t past = __ballot(inc > t);
    if (past) {
      const int l = __builtin_ctzll(past);
      seq = s0 + l;
      tile = __builtin_amdgcn_readlane(inc, l) - 1 - t;  // the last one first
      break;
    }
    t -= __builtin_amdgcn_readlane(inc, 63);
  }
  if (seq < 0) return;
  seq = __builtin_amdgcn_readfirstlane(seq);
  const PagedRows r = paged_rows(a.b, seq, a.M);
  const int n_cols = r.n * a.rep, c0 = tile * CW, w0 = c0 + w * 16 * NT;
  PromptState<HD, NT> st;
#pragma unroll
  for (int rt = 0; rt < NT; ++rt) {
    const int col = min(w0 + rt * 16 + j, n_cols - 1), i = col / a.rep;
    st.lim[rt] = min(r.first + i, a.l_cap - 1);
    const bf16_t* q = a.Q + (int64_t)(r.r0 + i) * a.ldq + (kvh * a.rep + col % a.rep) * HD;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) st.qf[rt][ks] = *(const u32x4_t*)(q + ks * 32 + g * 8);
    st.m[rt] = -INFINITY, st.l[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) st.o[rt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  auto lim_of = [&](int col) { return min(r.first + min(col, n_cols - 1) / a.rep, a.l_cap - 1); };
  const int last = lim_of(c0 + CW - 1), n_blk = last < 0 ? 0 : last / PAGE + 1;
  const int full = min((lim_of(c0) + 1) / PAGE, n_blk);           // blocks that every column attends whole
  const int hi = w0 < n_cols ? lim_of(w0 + 16 * NT - 1) : -1;  // this wave's last key
  // lane i has the page of block i of the present 64
  int pages = lane < n_blk ? paged_page(a.b, seq, lane, a.c.pages) : -1;
  auto page = [&](int b) { return __builtin_amdgcn_readlane(pages, b & 63); };
  auto place = [&](int pg) { return ((size_t)max(pg, 0) * a.c.kv + kvh) * PAGE * HD; };
  if (threadIdx.x < HD) first_bad[threadIdx.x] = INT32_MAX;  // read behind the first block's barrier
  if (n_blk > 0) prompt_copy<HD>(a.c, place(page(0)), w, lane, (lp)kA, (lp)vA);
  auto step = [&](auto masked, int b, lds_u32x4* ck, lds_u32x4* cv, lds_u32x4* nk, lds_u32x4* nv) {
    // this block's copy has landed (a barrier does not wait for it), and every wave is done with the other buffer
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const bool gone = page(b) < 0;  // nobody attends it
    if (b + 1 < n_blk) {
      if (((b + 1) & 63) == 0) pages = b + 1 + lane < n_blk ? paged_page(a.b, seq, b + 1 + lane, a.c.pages) : -1;
      prompt_copy<HD>(a.c, place(page(b + 1)), w, lane, nk, nv);
    }
    if (gone) return;
    if constexpr (decltype(masked)::value) {
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const int n = 256 * i + (int)threadIdx.x;  // piece n: tile n / 64, lane n % 64
        const u32x4_t x = cv[n];
        if (paged_not_finite(x[0]) || paged_not_finite(x[1]) || paged_not_finite(x[2]) || paged_not_finite(x[3]))
          cv[n] = paged_take_out(x, b * PAGE + (n >> 6 & 1) * 32 + (n >> 4 & 3) * 8, &first_bad[(n >> 7) * 16 + (n & 15)]);
      }
      __syncthreads();
    }
    if (b * PAGE > hi) return;
    prompt_block<HD, NT, decltype(masked)::value>(st, b * PAGE, a.scale_log2, lane, ck, cv);
  };
  using yes_t = std::integral_constant<bool, true>;
  using no_t = std::integral_constant<bool, false>;
  int b = 0;
  for (; b + 1 < full; b += 2) {
    step(no_t{}, b, (lp)kA, (lp)vA, (lp)kB, (lp)vB);
    step(no_t{}, b + 1, (lp)kB, (lp)vB, (lp)kA, (lp)vA);
  }
  for (; b < n_blk; b += 2) {  // at most one block more that every column attends whole, then the others
    step(yes_t{}, b, (lp)kA, (lp)vA, (lp)kB, (lp)vB);
    if (b + 1 < n_blk) step(yes_t{}, b + 1, (lp)kB, (lp)vB, (lp)kA, (lp)vA);
  }
  __syncthreads();  // no block's notes are under way
#pragma unroll
  for (int rt = 0; rt < NT; ++rt) {
    const float l = paged_sum_lanes(st.l[rt]);
    const int col = w0 + rt * 16 + j;
    if (col >= n_cols) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;  // NaN stays NaN
    bf16_t* dst = a.out + (int64_t)(r.r0 + col / a.rep) * a.ldo + (kvh * a.rep + col % a.rep) * HD;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = st.lim[rt] >= first_bad[dt * 16 + 4 * g + e] ? __uint_as_float(0x7fc00000u) : st.o[rt][dt][e] * inv;
      *(uint2*)(dst + dt * 16 + 4 * g) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    }
  }
}

template <int HD, int NT>
static int launch_paged_prompt(const PagedPromptArgs& a, hipStream_t stream) {
  // every sequence's tiles: at most a whole-tile share of the rows and one more each
  const int64_t wgs = ((int64_t)a.M * a.rep / (64 * NT) + a.b.n_seq) * a.c.kv;
  if (paged_grid_too_large(wgs, 256)) return set_error(SSD_ERANGE, "paged_prompt: too many workgroups");
  SSD_LAUNCH((paged_prompt_kernel<HD, NT>), dim3((unsigned)wgs), dim3(256), 0, stream, a);
  return check_launch("paged_prompt");
}

}  // namespace ssd

using namespace ssd;

SSD_API int ssd_paged_prompt_bf16(const SsdPagedKv* cache, const SsdPagedBatch* batch, const uint16_t* q, int64_t ldq, int M, int heads,
                                  int l_max, float scale, uint16_t* out, int64_t ldo, hipStream_t stream) {
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
  const bool small = ((int64_t)M * a.rep / 128 + a.b.n_seq) * a.c.kv <= 256;
  if (cache->head_dim == 64) return small ? launch_paged_prompt<64, 1>(a, stream) : launch_paged_prompt<64, 2>(a, stream);
  return small ? launch_paged_prompt<128, 1>(a, stream) : launch_paged_prompt<128, 2>(a, stream);
}
