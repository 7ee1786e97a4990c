// Tree attention over the 8-bit KV cache for a batch of sequences (layout in kv_q8.h; row model as in attention.hip:
// row t attends cache slots [0, prefix[t]), then its ancestors' slots in depth order).
//
// Arithmetic of a row (the same whatever shares the call): its keys, by logical position, are cut into 64-key
// blocks, spans of whole blocks and groups of four spans. A span is folded block by block with a running
// reference m, sum l and output O (fp32); the spans of a group, then the groups, are added with weights from
// their largest m. First launch: groups that every row of a sequence attends whole are folded for all its rows at
// once, a row's other groups by a workgroup of its own; each (row, head, group) leaves a record (m, l, O).
// Second launch: the groups' sum. Short contexts take one launch that does both.
//
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16: codes become bf16 exactly (v_cvt_scalef32_pk_bf16_fp8,
// with K's exponents as its scale); V's exponents multiply the probabilities before those are rounded to bf16
// (exact), so that rounding -- 2^-8 of a weight at most -- is the only one below fp32. l is summed by the MFMA too, from
// the rounded probabilities (an A operand of 2^-(V exponent)), so the weights O is made of add up to l exactly.
// A product below 2^-126 is 0: at the least V exponent, 2^-100 (a row of zeros, or none above 2^-91), a key whose weight
// is below 2^-26 of its span's reference does not count in l, at most span * 2^-26 of it (2^-17 at spans of up to 512).
//
// What bounds it, 8 kv heads of 128 (us, both launches): one row of 32 sequences at up to 8192 keys 82 for 410 MB, 5.0 TB/s, and
// one row at 131000 keys 47 for 270 MB (41 the fold, 6.5 TB/s): bytes. 25 rows of 64 heads at 16384 keys 32 for 13.4
// GFLOP, 31 of them the fold: of the SIMDs' cycles VALU work (conversion once per two tiles, maximum, exp2, packing) takes 43 %
// and MFMAs 21 %, and a CU has waves 73 % of the time, since 648 workgroups on 512 places take a second turn. 25 rows of 32
// heads at 4096 keys 14 and 12 trees of up to 9 rows at 1900 24: the chains of a workgroup (rows, prefixes, ancestors,
// keys, then one block after the other) at two waves a SIMD, which 248 VGPRs allow, and the second launch. One row at
// 512 keys 5.5: a launch and that chain once.
#include "kv_q8.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace ssd {

constexpr int QA_BLK = 64;
constexpr int QA_MAXD = 32;   // gathered tree slots per row
constexpr int QA_ROWS = 64;   // rows per sequence
constexpr int QA_GRP = 4;     // spans per group

int q8_check(const SsdKvQ8* c, const char* what);

struct AttnQ8Args {
  const bf16_t* Q;
  int64_t ldq;
  const uint8_t *K, *V, *Kx, *Vx;
  int64_t max_len;
  int n_seq, kv, heads, rep, M;
  const int *row_begin, *prefix, *depth, *anc;
  int l_max, span_blk, n_grps;
  int units, sets, tiles_per_set;  // launch geometry of the shared groups
  int own_units, own_rows;         // and of the rows' own
  float scale_log2;
  float* ws_o;    // [row][head][group][HD]: O
  float2* ws_ml;  // [row][head][group]: (m, l)
  bf16_t* out;
  int64_t ldo;
};

template <int HD>
struct Q8Frags {
  u32x4_t k[4][HD / 64];
  u32x4_t v[HD / 16];
  u32x4_t kx;  // K's exponents, the block's layout seen from the key's lane: byte j % 4 of word kt is key 16 kt + j
  u32x4_t vx;  // V's exponents of keys 16 kt + 4g + e: byte e of word kt
};

template <int HD>
struct Q8State {
  float m;              // running maximum (log2 units); -inf: nothing yet
  f32x4_t l;            // sum of weights, the same in all four
  f32x4_t o[HD / 16];   // O[row j][16 dt + 4g + e]
};

// Two words (8 codes) times a power of two -> an MFMA operand.
__device__ __forceinline__ bf16x8_t q8_bf16x8(uint32_t a, uint32_t b, float scale) {
  u32x4_t r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true));
  return bits_bf16x8(r);
}

__device__ __forceinline__ float q8_max16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float q8_max32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Folds one block into the states of T 16-row tiles; every operand is converted once for all of them, right before
// the MFMAs that take it. valid: bit 4 kt + e says whether key 16 kt + 4g + e is attended (masked instance only;
// V codes of the others are 0 and their exponents 127). FIRST: the states are empty. The reference m follows the
// maximum only when that has grown by more than 2^8 (probabilities up to 2^8 are as exact as those up to 1):
// after a span's first block the sums are hardly ever rescaled. Whether a row rescales is the row's own doing; that
// a wave skips the products when none of its rows does changes nothing (they would be by 1).
// next_k / next_v: load the following block's operands into f, called as soon as this block's are used up.
template <int HD, int T, bool MASKED, bool FIRST, typename NextK, typename NextV>
__device__ __forceinline__ void q8_fold(const Q8Frags<HD>& f, const u32x4_t (&qf)[T][HD / 32], uint32_t valid, float scale_log2,
                                        int j, Q8State<HD> (&st)[T], NextK next_k, NextV next_v) {
  // key tiles innermost: consecutive MFMAs go to different accumulators
  f32x4_t s[T][4];
  float ks[4];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) {
    ks[kt] = q8_scale(f.kx[kt] >> (8 * (j & 3)) & 0xffu);
#pragma unroll
    for (int t = 0; t < T; ++t) s[t][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int p = 0; p < HD / 64; ++p)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        const bf16x8_t ka = q8_bf16x8(f.k[kt][p][2 * hf], f.k[kt][p][2 * hf + 1], ks[kt]);
#pragma unroll
        for (int t = 0; t < T; ++t) s[t][kt] = mfma16x16x32(ka, bits_bf16x8(qf[t][2 * p + hf]), s[t][kt]);
      }
  next_k();
  uint32_t pw[T][2][4];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (MASKED) s[t][kt][e] = ((valid >> (kt * 4 + e)) & 1u) ? s[t][kt][e] : -INFINITY;
        mx = fmaxf(mx, s[t][kt][e]);
      }
    mx = q8_max32(q8_max16(mx)) * scale_log2;  // scale_log2 >= 0
    const float m = FIRST || mx > st[t].m + 8.f ? mx : st[t].m;
    const float ms = m == -INFINITY ? 0.f : m;  // nothing attended so far: every p is 0
    if (!FIRST) {
      if (__any(m != st[t].m)) {
        const float alpha = __builtin_amdgcn_exp2f(st[t].m - ms);
        st[t].l *= alpha;
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt) st[t].o[dt] *= alpha;
      }
    }
    st[t].m = m;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[t][kt][e], scale_log2, -ms)) * q8_scale((f.vx[kt] >> (8 * e)) & 0xffu);
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[t][kt][e + 1], scale_log2, -ms)) * q8_scale((f.vx[kt] >> (8 * e + 8)) & 0xffu);
        pw[t][kt >> 1][(kt & 1) * 2 + e / 2] = pack_bf16x2(p0, p1);
      }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    u32x4_t iv;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t x = 0xfefefefeu - f.vx[2 * c + i];  // bytes of 2^-(exponent)
      iv[2 * i] = (x & 0xffu) << 7 | (x & 0xff00u) << 15;
      iv[2 * i + 1] = (x & 0xff0000u) >> 9 | (x & 0xff000000u) >> 1;
    }
    const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const bf16x8_t pb = bits_bf16x8(u32x4_t{pw[t][c][0], pw[t][c][1], pw[t][c][2], pw[t][c][3]});
      st[t].l = mfma16x16x32(bits_bf16x8(iv), pb, FIRST && c == 0 ? zero : st[t].l);
    }
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) {
      const bf16x8_t va = q8_bf16x8(f.v[dt][2 * c], f.v[dt][2 * c + 1], 1.f);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const bf16x8_t pb = bits_bf16x8(u32x4_t{pw[t][c][0], pw[t][c][1], pw[t][c][2], pw[t][c][3]});
        st[t].o[dt] = mfma16x16x32(va, pb, FIRST && c == 0 ? zero : st[t].o[dt]);
      }
    }
  }
  next_v();
}

// Query fragments: operand 2p + hf holds dims 64 p + 16 g + 8 hf .. + 8 of this lane's row.
template <int HD>
__device__ __forceinline__ void q8_load_q(u32x4_t (&qf)[HD / 32], const bf16_t* q, int g) {
#pragma unroll
  for (int p = 0; p < HD / 64; ++p)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) qf[2 * p + hf] = *(const u32x4_t*)(q + 64 * p + 16 * g + 8 * hf);
}

template <int HD>
__device__ __forceinline__ void q8_load_k(Q8Frags<HD>& f, const uint8_t* K, const uint8_t* Kx, int blk, int lane) {
  const uint8_t* kb = K + (size_t)blk * 64 * HD + lane * 16;
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int p = 0; p < HD / 64; ++p) f.k[kt][p] = *(const u32x4_t*)(kb + (kt * (HD / 64) + p) * 1024);
  f.kx = *(const u32x4_t*)(Kx + (size_t)blk * 64 + (lane >> 2 & 3) * 16);
}

template <int HD>
__device__ __forceinline__ void q8_load_v(Q8Frags<HD>& f, const uint8_t* V, const uint8_t* Vx, int blk, int lane) {
  const uint8_t* vb = V + (size_t)blk * 64 * HD + lane * 16;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) f.v[dt] = *(const u32x4_t*)(vb + dt * 1024);
  f.vx = *(const u32x4_t*)(Vx + (size_t)blk * 64 + (lane >> 4) * 16);
}

// Smallest value over the wave's 64 lanes (row exchanges by DPP, then the swaps across rows).
__device__ __forceinline__ int wave_min(int v) {
  v = min(v, __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true));   // lane ^ 1
  v = min(v, __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true));   // lane ^ 2
  v = min(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true));  // the other half of 8
  v = min(v, __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true));  // the other half of 16
  auto r = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = min((int)r[0], (int)r[1]);
  r = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return min((int)r[0], (int)r[1]);
}

// Rows [r0, r1) of a sequence.
__device__ __forceinline__ void q8_rows(const AttnQ8Args& a, int seq, int& r0, int& r1) {
  r0 = min(max(a.row_begin[seq], 0), a.M);
  r1 = min(max(a.row_begin[seq + 1], r0), min(a.M, r0 + QA_ROWS));
}

// The number of blocks that every row of the sequence attends. Called by whole waves.
__device__ __forceinline__ int q8_shared_blocks(const AttnQ8Args& a, int r0, int r1, int lane) {
  const int p = wave_min(lane < r1 - r0 ? a.prefix[r0 + lane] : INT32_MAX);
  return min(max(p, 0), a.l_max) / QA_BLK;
}

__device__ __forceinline__ float q8_weight(float m, float top) {
  return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
}

// The four spans of a group meet in LDS: area for one 16-row tile (rows of a tile are query heads).
template <int HD>
struct alignas(16) Q8Spans {
  float o[QA_GRP][16][HD + 4];
  float m[QA_GRP][16], l[QA_GRP][16];
};

// A wave leaves span s's state for tile rows r0 .. r0 + n, its lanes j < n; one without keys leaves (-inf, 0, 0).
template <int HD>
__device__ __forceinline__ void q8_publish(Q8Spans<HD>& lds, int s, int r0, int n, int j, int g, bool have, const Q8State<HD>& st) {
  if (j >= n) return;
  lds.m[s][r0 + j] = have ? st.m : -INFINITY;  // the four lanes of row j write the same values
  lds.l[s][r0 + j] = have ? st.l[0] : 0.f;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt)
    *(f32x4_t*)&lds.o[s][r0 + j][dt * 16 + 4 * g] = have ? st.o[dt] : f32x4_t{0.f, 0.f, 0.f, 0.f};
}

// Row rr's record, dims 4 dc .. + 4 of every 64: the largest reference first, then the weighted sums in order.
template <int HD>
struct Q8Record {
  float m, l;
  f32x4_t o[HD / 64];
};
template <int HD>
__device__ __forceinline__ Q8Record<HD> q8_merge(const Q8Spans<HD>& lds, int rr, int dc) {
  Q8Record<HD> r;
  r.m = -INFINITY, r.l = 0.f;
#pragma unroll
  for (int i = 0; i < HD / 64; ++i) r.o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < QA_GRP; ++s) r.m = fmaxf(r.m, lds.m[s][rr]);
#pragma unroll
  for (int s = 0; s < QA_GRP; ++s) {
    const float wgt = q8_weight(lds.m[s][rr], r.m);
    r.l = fmaf(lds.l[s][rr], wgt, r.l);
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
      const f32x4_t x = *(const f32x4_t*)&lds.o[s][rr][i * 64 + dc * 4];
#pragma unroll
      for (int e = 0; e < 4; ++e) r.o[i][e] = fmaf(x[e], wgt, r.o[i][e]);
    }
  }
  return r;
}

template <int HD>
__device__ __forceinline__ void q8_store_record(const AttnQ8Args& a, size_t rec, int dc, const Q8Record<HD>& r) {
#pragma unroll
  for (int i = 0; i < HD / 64; ++i) *(f32x4_t*)(a.ws_o + rec * HD + i * 64 + dc * 4) = r.o[i];
  if (dc == 0) a.ws_ml[rec] = make_float2(r.m, r.l);
}

// Shared groups. Workgroup (sequence, group, kv head, set of row tiles): wave w folds span w of the group for T tiles
// of 16 query rows, so that each block's K and V are loaded and converted once for T tiles. The sets of one
// (sequence, group, kv head) are ids 8 apart: one XCD, whose L2 they share.
template <int HD, int T>
__device__ __forceinline__ void q8_shared_group(const AttnQ8Args& a, int id, Q8Spans<HD> (&lds)[T]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const int rest = id >> 3, set = rest % a.sets;
  int u = rest / a.sets * 8 + (id & 7);
  if (u >= a.units) return;
  const int kvh = u % a.kv;
  u /= a.kv;
  const int grp = u % a.n_grps, seq = u / a.n_grps;
  const size_t reg = ((size_t)seq * a.kv + kvh) * a.max_len;
  const uint8_t *K = a.K + reg * HD, *V = a.V + reg * HD, *Kx = a.Kx + reg, *Vx = a.Vx + reg;
  const int b0 = (grp * QA_GRP + w) * a.span_blk, b1 = b0 + a.span_blk;
  Q8Frags<HD> f;
  // One sequence: nearly all its groups are attended, so the first block is loaded before the rows and the
  // prefixes are known (a chain of two loads). Of a batch whole sequences may be shorter than l_max.
  const bool early = a.n_seq == 1 && b1 * QA_BLK <= a.l_max;
  if (early) {
    q8_load_k<HD>(f, K, Kx, b0, lane);
    q8_load_v<HD>(f, V, Vx, b0, lane);
  }
  int r0, r1;
  q8_rows(a, seq, r0, r1);
  const int n_rows = (r1 - r0) * a.rep, tile0 = set * a.tiles_per_set;
  if (r1 <= r0 || tile0 * 16 >= n_rows) return;
  if ((grp + 1) * QA_GRP * a.span_blk > q8_shared_blocks(a, r0, r1, lane)) return;  // the rows' own
  if (!early) {
    q8_load_k<HD>(f, K, Kx, b0, lane);
    q8_load_v<HD>(f, V, Vx, b0, lane);
  }
  u32x4_t qf[T][HD / 32];
  Q8State<HD> st[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {  // rows past the last repeat it
    const int R = min((tile0 + min(t, a.tiles_per_set - 1)) * 16 + j, n_rows - 1);
    q8_load_q<HD>(qf[t], a.Q + (size_t)(r0 + R / a.rep) * a.ldq + (size_t)(kvh * a.rep + R % a.rep) * HD, g);
  }
  int b = b0 + 1;
  auto next_k = [&] {
    if (b < b1) q8_load_k<HD>(f, K, Kx, b, lane);
  };
  auto next_v = [&] {
    if (b < b1) q8_load_v<HD>(f, V, Vx, b, lane);
  };
  q8_fold<HD, T, false, true>(f, qf, 0, a.scale_log2, j, st, next_k, next_v);
  while (b < b1) {
    ++b;
    q8_fold<HD, T, false, false>(f, qf, 0, a.scale_log2, j, st, next_k, next_v);
  }
#pragma unroll
  for (int t = 0; t < T; ++t) q8_publish<HD>(lds[t], w, 0, 16, j, g, true, st[t]);
  __syncthreads();
  const int rr = threadIdx.x >> 4, dc = threadIdx.x & 15;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int R = (tile0 + t) * 16 + rr;
    if (t < a.tiles_per_set && R < n_rows) {
      const size_t head = (size_t)(r0 + R / a.rep) * a.heads + kvh * a.rep + R % a.rep;
      q8_store_record<HD>(a, head * a.n_grps + grp, dc, q8_merge<HD>(lds[t], rr, dc));
    }
  }
}

// A row's ancestors: lane n of each wave that works for the row holds ancestor n's slot (-1: not attended) and V
// exponent, LDS their V codes. The codes are loaded by NT threads in two steps -- begin issues the loads, end
// writes them down -- so that the row's own K and V are on their way at the same time.
template <int HD>
struct alignas(16) Q8Codes {
  uint8_t v[QA_MAXD][HD];
};

template <int HD, int NT>
struct Q8Anc {
  // a thread takes one dim (two with 64 threads for 128 dims) of every STEP-th ancestor; which is the wave's choice
  static constexpr int STEP = NT >= HD ? NT / HD : 1, DIMS = NT >= HD ? 1 : HD / NT;
  static constexpr int BATCH = QA_MAXD / STEP < 8 ? (QA_MAXD + STEP - 1) / STEP : 8;
  int slot, D;
  uint32_t xv;
  uint32_t c[BATCH][DIMS];

  __device__ __forceinline__ uint32_t code(const uint8_t* V, int n, int d) const {
    const int sl = __builtin_amdgcn_readlane(slot, n);
    return sl >= 0 ? V[q8_v_off(sl, d, HD)] : 0;  // uniform
  }
  __device__ __forceinline__ void begin(const AttnQ8Args& a, int raw, int n_anc, const uint8_t* V, const uint8_t* Vx, int tid) {
    const int lane = tid & 63;
    D = n_anc;
    slot = lane < D && raw >= 0 && raw < a.max_len ? raw : -1;
    if (D == 0) return;  // uniform
    const uint32_t x = Vx[q8_x_off(max(slot, 0))];
    xv = slot >= 0 ? x : 127;
    const int n0 = NT >= HD ? __builtin_amdgcn_readfirstlane(tid / HD) : 0, d = tid % HD;
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (n0 + i * STEP < D) {  // uniform
#pragma unroll
        for (int e = 0; e < DIMS; ++e) c[i][e] = code(V, n0 + i * STEP, d + e * NT);
      }
  }
  template <typename Sync>
  __device__ __forceinline__ void end(const uint8_t* V, Q8Codes<HD>& lds, int tid, Sync sync) const {
    if (D == 0) return;
    const int n0 = NT >= HD ? __builtin_amdgcn_readfirstlane(tid / HD) : 0, d = tid % HD;
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (n0 + i * STEP < D) {
#pragma unroll
        for (int e = 0; e < DIMS; ++e) lds.v[n0 + i * STEP][d + e * NT] = (uint8_t)c[i][e];
      }
    for (int n = n0 + BATCH * STEP; n < D; n += STEP)
#pragma unroll
      for (int e = 0; e < DIMS; ++e) lds.v[n][d + e * NT] = (uint8_t)code(V, n, d + e * NT);
    sync();
  }
};

// One block of a row's own keys: positions below P are cache slots, those in [P, L) the ancestors' slots. ready()
// makes the ancestors' codes readable; called once the block's loads are on their way.
template <int HD, int NT, typename Ready>
__device__ __forceinline__ uint32_t q8_load_own(Q8Frags<HD>& f, const uint8_t* K, const uint8_t* V, const uint8_t* Kx,
                                                const uint8_t* Vx, int b, int P, int L, const Q8Anc<HD, NT>& anc,
                                                const Q8Codes<HD>& codes, int lane, Ready ready) {
  const int j = lane & 15, g = lane >> 4, key0 = b * QA_BLK;
  uint32_t valid = 0;
  // K and its exponents: one slot a lane. Loads are unconditional (a key that is not attended reads its own
  // block's first slot, which exists; its score is masked).
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) {
    const int pos = key0 + 16 * kt + j, from = __shfl(anc.slot, (pos - P) & 31);
    const int sl = pos < P ? pos : pos < L && from >= 0 ? from : key0;
    f.kx[kt] = Kx[q8_x_off(sl)] * 0x01010101u;
#pragma unroll
    for (int p = 0; p < HD / 64; ++p) f.k[kt][p] = *(const u32x4_t*)(K + q8_k_off(sl, 64 * p + 16 * g, HD));
  }
  // V and its exponents: the block's own slots, positions from P on cleared, then the ancestors' put in
  f.vx = *(const u32x4_t*)(Vx + key0 + g * 16);
  const uint8_t* vb = V + (size_t)b * 64 * HD + lane * 16;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) f.v[dt] = *(const u32x4_t*)(vb + dt * 1024);
  ready();
  u32x4_t own;
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int pos = key0 + 16 * kt + 4 * g + e;
      if (pos < P) m |= 0xffu << (8 * e), valid |= 1u << (4 * kt + e);
    }
    own[kt] = m;
    f.vx[kt] = (f.vx[kt] & m) | (0x7f7f7f7fu & ~m);
  }
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) f.v[dt] &= own;
  const int a0 = max(P, key0) - P, a1 = min(L, key0 + QA_BLK) - P;
  for (int an = a0; an < a1; ++an) {  // uniform
    const int off = P + an - key0, kt = off >> 4, e = off & 3;
    const bool mine = ((off >> 2) & 3) == g;
    const uint32_t sel = mine ? 0xffu << (8 * e) : 0u, xv = __builtin_amdgcn_readlane(anc.xv, an) * 0x01010101u;
    if (mine && __builtin_amdgcn_readlane(anc.slot, an) >= 0) valid |= 1u << (4 * kt + e);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t m = c == kt ? sel : 0u;
      f.vx[c] = (f.vx[c] & ~m) | (xv & m);
#pragma unroll
      for (int dt = 0; dt < HD / 16; ++dt) f.v[dt][c] = (f.v[dt][c] & ~m) | ((codes.v[an][dt * 16 + j] * 0x01010101u) & m);
    }
  }
  return valid;
}

// A span of keys (positions below P cache slots, those in [P, L) ancestors) for the query at q on each lane j; false:
// no keys.
template <int HD, int NT, typename Ready>
__device__ __forceinline__ bool q8_own_span(const AttnQ8Args& a, size_t reg, const bf16_t* q, int span, int P, int L,
                                            const Q8Anc<HD, NT>& anc, const Q8Codes<HD>& codes, int lane, Q8State<HD> (&st)[1],
                                            Ready ready) {
  const int b0 = span * a.span_blk, b1 = min((L + QA_BLK - 1) / QA_BLK, b0 + a.span_blk), j = lane & 15;
  if (b0 >= b1) return false;
  const uint8_t *K = a.K + reg * HD, *V = a.V + reg * HD, *Kx = a.Kx + reg, *Vx = a.Vx + reg;
  u32x4_t qf[1][HD / 32];
  q8_load_q<HD>(qf[0], q, lane >> 4);
  st[0].m = -INFINITY;
  st[0].l = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) st[0].o[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int b = b0; b < b1; ++b) {
    Q8Frags<HD> f;
    uint32_t valid = 0xffffu;
    if ((b + 1) * QA_BLK <= P) {
      q8_load_k<HD>(f, K, Kx, b, lane);
      q8_load_v<HD>(f, V, Vx, b, lane);
    } else {
      valid = q8_load_own<HD>(f, K, V, Kx, Vx, b, P, L, anc, codes, lane, ready);
    }
    q8_fold<HD, 1, true, false>(f, qf, valid, a.scale_log2, j, st, [] {}, [] {});
  }
  return true;
}

__device__ __forceinline__ void q8_row_keys(const AttnQ8Args& a, int row, int& P, int& L) {
  P = min(max(a.prefix[row], 0), a.l_max);
  L = min(P + min(max(a.depth[row], 0), QA_MAXD), a.l_max);
}

// The groups that rows of a sequence do not attend whole together: from the one the smallest prefix ends in to each
// row's last. One workgroup per (sequence, kv head, up to four rows that fill a tile: 16 / rep); wave w has row w. Spans
// all rows attend whole are folded for the tile (span s by wave 3 - s: with one row wave 0 is free for it), the
// spans after by each row's wave; together they make the rows' records of the group. DIRECT: all keys lie in the first
// group, and its sums are the rows' outputs.
template <int HD, bool DIRECT>
__device__ __forceinline__ void q8_own_groups(const AttnQ8Args& a, int id, Q8Spans<HD>& lds, Q8Codes<HD>& codes) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const int unit = id % a.own_units, kvh = unit % a.kv, seq = unit / a.kv;
  if (seq >= a.n_seq) return;  // units are rounded up to 8: a unit's rows and its shared groups meet on one XCD
  int r0, r1;
  q8_rows(a, seq, r0, r1);
  const int base = r0 + id / a.own_units * a.own_rows, n_rows = min(a.own_rows, r1 - base);
  if (n_rows <= 0) return;
  const int cut = q8_shared_blocks(a, r0, r1, lane) / a.span_blk, per = QA_GRP * a.span_blk * QA_BLK;
  const size_t reg = ((size_t)seq * a.kv + kvh) * a.max_len;
  const int raw = a.anc[(size_t)(base + min(w, n_rows - 1)) * QA_MAXD + (lane & (QA_MAXD - 1))];
  int p_of, l_of;  // of row base + lane (past the last: the last's)
  q8_row_keys(a, base + min(lane, n_rows - 1), p_of, l_of);
  const int n_grp = DIRECT ? 1 : (-wave_min(-l_of) + per - 1) / per;
  const int P = __builtin_amdgcn_readlane(p_of, w), L = __builtin_amdgcn_readlane(l_of, w);
  if (!DIRECT && cut / QA_GRP >= n_grp) return;
  Q8Anc<HD, 64> anc;
  anc.begin(a, raw, w < n_rows ? L - P : 0, a.V + reg * HD, a.Vx + reg, lane);
  bool staged = false;
  auto ready = [&] {
    if (staged) return;  // uniform
    staged = true;
    anc.end(a.V + reg * HD, codes, lane, [] {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // one wave's LDS accesses are in order: keep the compiler's so
      __builtin_amdgcn_wave_barrier();
    });
  };
  for (int grp = DIRECT ? 0 : cut / QA_GRP; grp < n_grp; ++grp)
    for (int t0 = 0; t0 < a.rep; t0 += 16) {  // more than one turn only with one row
      const int nh = min(16, a.rep - t0), h0 = kvh * a.rep + t0;
      __syncthreads();  // the tile before has been merged
      for (int it = -1; it < QA_GRP; ++it) {
        const bool all = it < 0;  // the span for all rows, then the row's own
        const int s = all ? QA_GRP - 1 - w : it, span = grp * QA_GRP + s;
        if (all ? span >= cut : w >= n_rows || span < cut) continue;
        const int r = min(all ? j / nh : w, n_rows - 1), h = h0 + (all ? j % nh : min(j, nh - 1));
        const int keys = all ? (span + 1) * a.span_blk * QA_BLK : 0;
        Q8State<HD> st[1];
        const bool have = q8_own_span<HD>(a, reg, a.Q + (size_t)(base + r) * a.ldq + (size_t)h * HD, span, all ? keys : P,
                                          all ? keys : L, anc, codes, lane, st, ready);
        q8_publish<HD>(lds, s, all ? 0 : w * nh, all ? 16 : nh, j, g, have, st[0]);
      }
      __syncthreads();
      const int rr = threadIdx.x >> 4, dc = threadIdx.x & 15;
      if (rr < n_rows * nh) {
        const int row = base + rr / nh, h = h0 + rr % nh;
        if constexpr (DIRECT) {
          const Q8Record<HD> r = q8_merge<HD>(lds, rr, dc);
          const float wgt = q8_weight(r.m, r.m), l = r.l * wgt;  // the sum over one group, as the other kernels form it
#pragma unroll
          for (int i = 0; i < HD / 64; ++i) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = l == 0.f ? 0.f : fmaf(r.o[i][e], wgt, 0.f) / l;
            *(uint2*)(a.out + (size_t)row * a.ldo + (size_t)h * HD + i * 64 + dc * 4) =
                make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
          }
        } else if (grp * per < __shfl(l_of, rr / nh)) {
          q8_store_record<HD>(a, ((size_t)row * a.heads + h) * a.n_grps + grp, dc, q8_merge<HD>(lds, rr, dc));
        }
      }
    }
}

// Contexts of one group, rows of a sequence that fill a tile a workgroup.
template <int HD>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void q8_short_rows_kernel(AttnQ8Args a) {
  __shared__ Q8Spans<HD> spans;
  __shared__ Q8Codes<HD> codes[4];
  q8_own_groups<HD, true>(a, blockIdx.x, spans, codes[threadIdx.x >> 6]);
}

template <int HD, int T>
union alignas(16) Q8FoldLds {
  Q8Spans<HD> shared[T];
  struct {
    Q8Spans<HD> spans;
    Q8Codes<HD> codes[4];
  } own;
};

// First launch: workgroups of rows (ids first: theirs is the longer chain of loads), then of shared groups.
template <int HD, int T>
__global__ __launch_bounds__(256, 2) void q8_fold_kernel(AttnQ8Args a, int own) {
  __shared__ Q8FoldLds<HD, T> lds;
  if ((int)blockIdx.x < own) q8_own_groups<HD, false>(a, blockIdx.x, lds.own.spans, lds.own.codes[threadIdx.x >> 6]);
  else q8_shared_group<HD, T>(a, blockIdx.x - own, lds.shared);
}

// Sums that stay sums: no multiply-add contraction with the products they are given.
__device__ __forceinline__ float q8_add(float x, float y) {
#pragma clang fp contract(off)
  return x + y;
}

// Second launch: one workgroup of four waves per (row, head). Weights from the groups' largest reference; wave r
// adds groups r, r + 4, ... in order, then the four sums are added in order; l by a fixed exchange between
// lanes, 64 groups at a time.
template <int HD>
__global__ __launch_bounds__(256) void q8_combine_kernel(AttnQ8Args a) {
  constexpr int PER = HD / 64;  // dims a lane
  const int lane = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int row = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const size_t rec0 = ((size_t)row * a.heads + h) * a.n_grps;
  const float* O = a.ws_o + rec0 * HD + lane * PER;
  __shared__ float part[4][HD];
  // the first records before it is known how many there are (the workspace holds n_grps of them)
  float x[4][PER];
  auto load = [&](int g0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < PER; ++d) x[i][d] = O[(size_t)min(g0 + 4 * i, a.n_grps - 1) * HD + d];
  };
  load(r);
  float2 ml = a.ws_ml[rec0 + min(lane, a.n_grps - 1)];
  if (row < a.row_begin[0] || row >= a.row_begin[a.n_seq]) return;  // uniform
  int P, L;
  q8_row_keys(a, row, P, L);
  const int per = QA_GRP * a.span_blk * QA_BLK, n = (L + per - 1) / per;
  if (lane >= n) ml = make_float2(-INFINITY, 0.f);
  float top = ml.x;
  for (int g = lane + 64; g < n; g += 64) top = fmaxf(top, a.ws_ml[rec0 + g].x);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  float l = 0.f, o[PER];
#pragma unroll
  for (int d = 0; d < PER; ++d) o[d] = 0.f;
  for (int g0 = 0; g0 < n; g0 += 64) {
    if (g0) ml = g0 + lane < n ? a.ws_ml[rec0 + g0 + lane] : make_float2(-INFINITY, 0.f);
    const float wgt = q8_weight(ml.x, top);
    float lw = ml.y * wgt;
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) lw = q8_add(lw, __shfl_xor(lw, s));
    l += lw;
    for (int g = g0 + r; g < min(n, g0 + 64); g += 16) {
      if (g != r) load(g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (g + 4 * i >= n) break;  // uniform
        const float wi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wgt), g - g0 + 4 * i));
#pragma unroll
        for (int d = 0; d < PER; ++d) o[d] = fmaf(x[i][d], wi, o[d]);
      }
    }
  }
#pragma unroll
  for (int d = 0; d < PER; ++d) part[r][lane * PER + d] = o[d];
  __syncthreads();
  if (threadIdx.x < HD / 2) {
    const int d = threadIdx.x * 2;
    float y[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float s = ((part[0][d + e] + part[1][d + e]) + part[2][d + e]) + part[3][d + e];
      y[e] = l == 0.f ? 0.f : s / l;  // NaN stays NaN
    }
    *(uint32_t*)(a.out + (size_t)row * a.ldo + (size_t)h * HD + d) = pack_bf16x2(y[0], y[1]);
  }
}

// The same sums for up to G <= 8 groups, HD / 4 lanes a (row, head): every record of a pair is in flight at once.
template <int HD, int G>
__global__ __launch_bounds__(256) void q8_combine_few_kernel(AttnQ8Args a) {
  constexpr int LANES = HD / 4, PAIRS = 256 / LANES;
  const int64_t pair = (int64_t)blockIdx.x * PAIRS + threadIdx.x / LANES;
  const int row = min((int)(pair / a.heads), a.M - 1), h = (int)(pair % a.heads), d = threadIdx.x % LANES * 4;
  const size_t rec0 = ((size_t)row * a.heads + h) * a.n_grps;
  f32x4_t x[G];
  float2 ml[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const size_t rec = rec0 + min(g, a.n_grps - 1);
    x[g] = *(const f32x4_t*)(a.ws_o + rec * HD + d);
    ml[g] = a.ws_ml[rec];
  }
  if (pair >= (int64_t)a.M * a.heads || row < a.row_begin[0] || row >= a.row_begin[a.n_seq]) return;
  int P, L;
  q8_row_keys(a, row, P, L);
  const int per = QA_GRP * a.span_blk * QA_BLK, n = (L + per - 1) / per;
  float top = -INFINITY;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (g >= n) ml[g] = make_float2(-INFINITY, 0.f);
    top = fmaxf(top, ml[g].x);
  }
  float lw[G];
  f32x4_t part[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) part[r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float wgt = q8_weight(ml[g].x, top);
    lw[g] = ml[g].y * wgt;
#pragma unroll
    for (int e = 0; e < 4; ++e) part[g % 4][e] = g < n ? fmaf(x[g][e], wgt, part[g % 4][e]) : part[g % 4][e];
  }
#pragma unroll
  for (int s = G / 2; s >= 1; s >>= 1)
#pragma unroll
    for (int g = 0; g < s; ++g) lw[g] = q8_add(lw[g], lw[g + s]);
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float s = ((part[0][e] + part[1][e]) + part[2][e]) + part[3][e];
    y[e] = lw[0] == 0.f ? 0.f : s / lw[0];  // NaN stays NaN
  }
  *(uint2*)(a.out + (size_t)row * a.ldo + (size_t)h * HD + d) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
}

// Contexts of up to TEAMS <= 4 groups in one launch: a workgroup per (sequence, row, kv head), a team of four waves per
// group. The records stay in LDS and are added as the second launch adds them.
template <int HD, int TEAMS>
struct alignas(16) Q8ShortLds {
  Q8Spans<HD> spans[TEAMS];
  Q8Codes<HD> codes;
};

// Heads of 64 with one team: 128 VGPRs and four workgroups a CU, against two 20 x 9 rows at 200 keys 12.8 -> 11.2 us, 40 x 8
// at 400 22.1 -> 20.4. Heads of 128 spill below 168 and are slower so.
template <int HD, int TEAMS>
__global__ __launch_bounds__(256 * TEAMS, TEAMS == 4 || (TEAMS == 1 && HD == 64) ? 4 : 2) void q8_short_kernel(AttnQ8Args a,
                                                                                                         int rows_max) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6 & 3, team = threadIdx.x >> 8, j = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x % a.kv, seq = blockIdx.x / a.kv / rows_max;
  __shared__ Q8ShortLds<HD, TEAMS> lds;
  __shared__ float rec_m[TEAMS][16], rec_l[TEAMS][16];
  int r0, r1, P, L;
  q8_rows(a, seq, r0, r1);
  const int row = r0 + blockIdx.x / a.kv % rows_max;
  if (row >= r1) return;
  const int raw = a.anc[(size_t)row * QA_MAXD + (lane & (QA_MAXD - 1))];
  q8_row_keys(a, row, P, L);
  const size_t reg = ((size_t)seq * a.kv + kvh) * a.max_len;
  Q8Anc<HD, 256 * TEAMS> anc;
  anc.begin(a, raw, L - P, a.V + reg * HD, a.Vx + reg, threadIdx.x);
  anc.end(a.V + reg * HD, lds.codes, threadIdx.x, [] { __syncthreads(); });
  for (int t0 = 0; t0 < a.rep; t0 += 16) {
    const int nh = min(16, a.rep - t0), h0 = kvh * a.rep + t0;
    Q8State<HD> st[1];
    const bool have = q8_own_span<HD>(a, reg, a.Q + (size_t)row * a.ldq + (size_t)(h0 + min(j, nh - 1)) * HD, team * QA_GRP + w, P,
                                      L, anc, lds.codes, lane, st, [] {});
    if (t0) __syncthreads();  // the heads before have been written out
    q8_publish<HD>(lds.spans[team], w, 0, 16, j, g, have, st[0]);
    __syncthreads();
    const int rr = threadIdx.x >> 4 & 15, dc = threadIdx.x & 15;
    const Q8Record<HD> r = q8_merge<HD>(lds.spans[team], rr, dc);
    float top = r.m;
    if constexpr (TEAMS > 1) {
      __syncthreads();
      if (dc == 0) rec_m[team][rr] = r.m, rec_l[team][rr] = r.l;
#pragma unroll
      for (int i = 0; i < HD / 64; ++i) *(f32x4_t*)&lds.spans[team].o[0][rr][i * 64 + dc * 4] = r.o[i];
      __syncthreads();
      if (team) continue;
#pragma unroll
      for (int t = 1; t < TEAMS; ++t) top = fmaxf(top, rec_m[t][rr]);
    }
    if (rr >= nh) continue;
    // sums of one group each, added in order; l in the order of the second launch's exchange
    float wgt[4], lw[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float m = t == 0 ? r.m : t < TEAMS ? rec_m[t < TEAMS ? t : 0][rr] : -INFINITY;
      wgt[t] = q8_weight(m, top);
      lw[t] = t == 0 ? r.l * wgt[0] : t < TEAMS ? rec_l[t < TEAMS ? t : 0][rr] * wgt[t] : 0.f;
    }
    const float l = q8_add(q8_add(lw[0], lw[2]), q8_add(lw[1], lw[3]));
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float s = fmaf(r.o[i][e], wgt[0], 0.f);
#pragma unroll
        for (int t = 1; t < TEAMS; ++t) s += fmaf(lds.spans[t].o[0][rr][i * 64 + dc * 4 + e], wgt[t], 0.f);
        y[e] = l == 0.f ? 0.f : s / l;
      }
      *(uint2*)(a.out + (size_t)row * a.ldo + (size_t)(h0 + rr) * HD + i * 64 + dc * 4) =
          make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    }
  }
}

static int q8_groups(int64_t l_max, int span) { return (int)((l_max + (int64_t)QA_GRP * span - 1) / ((int64_t)QA_GRP * span)); }

template <int HD>
static int launch_attn_q8(AttnQ8Args a, int rows_max, hipStream_t stream) {
  using std::integral_constant;
  const int64_t rows = (int64_t)a.n_seq * rows_max * a.kv;
  const int tiles = (rows_max * a.rep + 15) / 16;
  const bool single = tiles == 1;
  a.sets = single ? 1 : (tiles + 1) / 2;
  a.tiles_per_set = single ? 1 : (tiles + a.sets - 1) / a.sets;
  const int64_t units = (int64_t)a.n_seq * a.n_grps * a.kv, shared = (units + 7) / 8 * 8 * a.sets;
  // A row a workgroup while all of those are resident at once, each on a CU of its own; then as many rows as fill a
  // tile, since the spans they attend together are folded once. us, one / four rows: 25 rows of one sequence, prefixes
  // 4097, 4060, 4000, 3900: 16.8 / 17.6, 15.8 / 18.0, 14.9 / 16.8, 15.9 / 18.6; 12 trees of 9 rows at 1900 keys 33 / 29, 4 of
  // them 17.8 / 16.3.
  a.own_rows = rows <= 256 ? 1 : std::min(4, std::max(1, 16 / a.rep));
  const int64_t own_units = ((int64_t)a.n_seq * a.kv + 7) / 8 * 8, own = own_units * ((rows_max + a.own_rows - 1) / a.own_rows);
  if (grid_too_large(shared + own, 256) || grid_too_large(rows, 256) || grid_too_large((int64_t)a.M * a.heads, 256))
    return set_error(SSD_ERANGE, "attention_q8: too many workgroups");
  a.units = (int)units, a.own_units = (int)own_units;
  auto one_launch = [&](auto t) {
    SSD_LAUNCH((q8_short_kernel<HD, decltype(t)::value>), dim3((unsigned)rows), dim3(256 * decltype(t)::value), 0, stream, a, rows_max);
    return check_launch("attn_q8_short");
  };
  // One group: four rows a workgroup once a row each would be more than are resident at once. us at 8 kv heads, a row /
  // four: heads of 128, 6 x 9 rows at 98 keys 6.7 / 10.0, 40 x 2 at 60 9.0 / 8.5, 13 x 9 at 98 11.9 / 10.3, 20 x 8 at 60
  // 15.3 / 10.6, 40 x 8 at 60 26 / 18, 12 x 25 at 450 41 / 26; heads of 64, 20 x 9 at 200 11.4 / 9.6, 40 x 25 at 200
  // 49 / 32. With two rows (rep 8), 20 x 9 at 100, it is 17.0 / 17.0.
  if (a.n_grps == 1 && rows > 512 && a.own_rows == 4 && rows_max > 1) {
    SSD_LAUNCH((q8_short_rows_kernel<HD>), dim3((unsigned)own), dim3(256), 0, stream, a);
    return check_launch("attn_q8_short_rows");
  }
  if (a.n_grps == 1) return one_launch(integral_constant<int, 1>());
  // Two to four groups, us in two launches / in one: a row of heads of 128 at 700 keys 9.2 / 7.5, 4 x 9 rows 13.9 / 17.4, 7 x 9
  // 15.9 / 17.4, 8 x 9 17.3 / 25; of heads of 64 at 400 keys 8.1 / 4.9, 4 x 9 11.4 / 9.8, 7 x 9 12.1 / 10.6, 16 x 9 14.5 / 24, at
  // 900 keys 8.2 / 6.9, 3 x 9 10.4 / 8.7, 6 x 9 12.2 / 15.6. (With heads of 128 the border lies below these 512 rows.)
  if (a.n_grps == 2 && rows <= 512) return one_launch(integral_constant<int, 2>());
  if constexpr (HD == 64)
    if (a.n_grps <= 4 && rows <= 256) return one_launch(integral_constant<int, 4>());
  if (single) SSD_LAUNCH((q8_fold_kernel<HD, 1>), dim3((unsigned)(own + shared)), dim3(256), 0, stream, a, (int)own);
  else SSD_LAUNCH((q8_fold_kernel<HD, 2>), dim3((unsigned)(own + shared)), dim3(256), 0, stream, a, (int)own);
  if (int rc = check_launch("attn_q8_fold")) return rc;
  // Up to eight groups: lanes of several (row, head) pairs a workgroup. us of both launches, a workgroup a pair / lanes: 12 trees of
  // 9 rows, 4 groups 32 / 29; 16 of 32 rows, 3 groups 71 / 58; one row, 8 groups 10.0 / 10.0; a tree of 25 rows,
  // 6 groups 15.1 / 14.5. With 9 and 11 groups it would be 16.2 / 16.9 and 18.2 / 19.3.
  const unsigned few = (unsigned)(((int64_t)a.M * a.heads + 1024 / HD - 1) / (1024 / HD));
  if (a.n_grps <= 4) SSD_LAUNCH((q8_combine_few_kernel<HD, 4>), dim3(few), dim3(256), 0, stream, a);
  else if (a.n_grps <= 8) SSD_LAUNCH((q8_combine_few_kernel<HD, 8>), dim3(few), dim3(256), 0, stream, a);
  else SSD_LAUNCH((q8_combine_kernel<HD>), dim3((unsigned)(a.M * a.heads)), dim3(256), 0, stream, a);
  return check_launch("attn_q8_combine");
}

}  // namespace ssd

using namespace ssd;

SSD_API int64_t ssd_attn_q8_ws_floats(int M, int heads, int head_dim, int64_t l_max, int span) {
  if (M < 0 || heads < 1 || head_dim < 1 || l_max < 1 || span < 64 || span % 64 || span > 1 << 20) return -1;
  return (int64_t)M * heads * q8_groups(l_max, span) * (head_dim + 2);
}

SSD_API int ssd_tree_attention_q8(const SsdKvQ8* cache, const uint16_t* q, int64_t ldq, int M, int heads,
                                  const int32_t* row_begin, const int32_t* prefix, const int32_t* depth, const int32_t* anc,
                                  int rows_max, int l_max, int span, float scale, float* ws, int64_t ws_floats,
                                  uint16_t* out, int64_t ldo, hipStream_t stream) {
  if (int rc = q8_check(cache, "attention_q8")) return rc;
  if (!q || !row_begin || !prefix || !depth || !anc || !ws || !out) return set_error(SSD_EINVAL, "attention_q8: null pointer");
  if (M < 0 || heads < 1 || heads % cache->kv_heads)
    return set_error(SSD_EINVAL, "attention_q8: bad M=%d heads=%d kv_heads=%d", M, heads, cache->kv_heads);
  if (rows_max < 1 || rows_max > QA_ROWS)
    return set_error(SSD_ERANGE, "attention_q8: %d rows a sequence (1 to %d)", rows_max, QA_ROWS);
  if (l_max < 1 || l_max > cache->max_len)
    return set_error(SSD_EINVAL, "attention_q8: l_max %d outside [1, max_len %lld]", l_max, (long long)cache->max_len);
  if (!(scale > 0.f) || scale > 1e30f) return set_error(SSD_EINVAL, "attention_q8: scale must be positive, got %g", scale);
  if (span < 64 || span % 64 || span > 1 << 20) return set_error(SSD_EINVAL, "attention_q8: span %d must be a multiple of 64 up to 2^20", span);
  const int64_t cols = (int64_t)heads * cache->head_dim;
  if (((uintptr_t)q & 15) || ldq % 8 || ldq < cols || ((uintptr_t)out & 15) || ldo % 8 || ldo < cols)
    return set_error(SSD_EINVAL, "attention_q8: q/out rows must be 16-byte aligned with strides >= heads * head_dim");
  if (((uintptr_t)ws & 15) || ws_floats < ssd_attn_q8_ws_floats(M, heads, cache->head_dim, l_max, span))
    return set_error(SSD_EINVAL, "attention_q8: workspace too small or not 16-byte aligned");
  if (M == 0) return SSD_OK;
  AttnQ8Args a{};
  a.Q = q, a.ldq = ldq, a.K = cache->k, a.V = cache->v, a.Kx = cache->k_exp, a.Vx = cache->v_exp;
  a.max_len = cache->max_len, a.n_seq = cache->n_seq, a.kv = cache->kv_heads, a.heads = heads, a.rep = heads / a.kv, a.M = M;
  a.row_begin = row_begin, a.prefix = prefix, a.depth = depth, a.anc = anc;
  a.l_max = l_max, a.span_blk = span / 64, a.n_grps = q8_groups(l_max, span);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.ws_o = ws;
  a.ws_ml = (float2*)(ws + (int64_t)M * heads * a.n_grps * cache->head_dim);
  a.out = out, a.ldo = ldo;
  return cache->head_dim == 64 ? launch_attn_q8<64>(a, rows_max, stream) : launch_attn_q8<128>(a, rows_max, stream);
}
