// Tree attention over the 8-bit KV cache for a batch of sequences (layout in kv_q8.h; row model as in attention.hip:
// row t attends cache slots [0, prefix[t]), then its ancestors' slots in depth order).
//
// Arithmetic of a row (the same whatever shares the call): its keys, by logical position, are cut into 64-key
// blocks and spans of whole blocks. A span is folded block by block with a running maximum m, sum l and
// output O (fp32); the spans' records (m, l, O) are folded in order. Keys every row of a sequence attends
// -- whole blocks below the sequence's smallest prefix -- are folded by q8_shared_kernel for all rows at
// once; the rest of a row's keys (its last block or two: committed slots, then ancestors) by q8_tail_kernel,
// one workgroup per (row, kv head), which takes up the span where the shared kernel left it and then folds
// the records. The record holds the fold's own registers, so the cut between the kernels leaves no trace.
//
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16: codes become bf16 exactly (v_cvt_scalef32_pk_bf16_fp8);
// K's exponents multiply the scores, V's the probabilities before they are rounded to bf16 (both exact), so
// that rounding -- relative, 2^-9 -- is the only one below fp32. l is summed by the MFMA too, from the rounded
// probabilities (an A operand of 2^-(V exponent)), so the weights that O is made of add up to l exactly.
#include "kv_q8.h"

#include <math.h>

#include <algorithm>

namespace ssd {

constexpr int QA_BLK = 64;
constexpr int QA_MAXD = 32;   // gathered tree slots per row
constexpr int QA_ROWS = 64;   // rows per sequence

int q8_check(const SsdKvQ8* c, const char* what);

struct AttnQ8Args {
  const bf16_t* Q;
  int64_t ldq;
  const uint8_t *K, *V, *Kx, *Vx;
  int64_t max_len;
  int n_seq, kv, heads, rep, M;
  const int *row_begin, *prefix, *depth, *anc;
  int l_max, span_blk, n_spans, tiles;
  float scale_log2;
  float* ws_o;    // [row][head][span][HD]: O
  float2* ws_ml;  // [row][head][span]: (m, l)
  bf16_t* out;
  int64_t ldo;
};

template <int HD>
struct Q8Frags {
  u32x4_t k[4][HD / 64];
  u32x4_t v[HD / 16];
  u32x4_t kx, vx;  // exponent bytes of keys 16 kt + 4g + e: byte e of word kt
};

template <int HD>
struct Q8State {
  float m;              // running maximum (log2 units); -inf: nothing yet
  f32x4_t l;            // sum of weights, the same in all four
  f32x4_t o[HD / 16];   // O[row j][16 dt + 4g + e]
};

template <int HD>
__device__ __forceinline__ void q8_reset(Q8State<HD>& s) {
  s.m = -INFINITY;
  s.l = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) s.o[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
}

// Two words (8 codes) -> an MFMA operand.
__device__ __forceinline__ bf16x8_t q8_bf16x8(uint32_t a, uint32_t b) {
  u32x4_t r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, true));
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

// Folds one block into the state of a 16-row tile. valid: bit 4 kt + e says whether key 16 kt + 4g + e is
// attended (masked instance only; codes and exponents of the others are 0 and 127).
template <int HD, bool MASKED>
__device__ __forceinline__ void q8_fold(const Q8Frags<HD>& f, const u32x4_t (&qf)[HD / 32], uint32_t valid, float scale_log2,
                                        Q8State<HD>& st) {
  // products and sums stay separate: the masked and unmasked instances must round alike
#pragma clang fp contract(off)
  f32x4_t s[4];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) s[kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int p = 0; p < HD / 64; ++p)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
        s[kt] = mfma16x16x32(q8_bf16x8(f.k[kt][p][2 * hf], f.k[kt][p][2 * hf + 1]), bits_bf16x8(qf[2 * p + hf]), s[kt]);
  float sv[16], mx = -INFINITY;
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = s[kt][e] * (q8_scale((f.kx[kt] >> (8 * e)) & 0xffu) * scale_log2);
      if (MASKED) v = ((valid >> (kt * 4 + e)) & 1u) ? v : -INFINITY;
      sv[kt * 4 + e] = v;
      mx = fmaxf(mx, v);
    }
  mx = q8_max32(q8_max16(mx));
  const float m = fmaxf(st.m, mx);
  const float ms = m == -INFINITY ? 0.f : m;  // nothing attended so far: every p is 0
  const float alpha = __builtin_amdgcn_exp2f(st.m - ms);
  st.m = m;
  uint32_t pw[2][4], iv[2][4];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f(sv[kt * 4 + e] - ms) * q8_scale((f.vx[kt] >> (8 * e)) & 0xffu);
      const float p1 = __builtin_amdgcn_exp2f(sv[kt * 4 + e + 1] - ms) * q8_scale((f.vx[kt] >> (8 * e + 8)) & 0xffu);
      pw[kt >> 1][(kt & 1) * 2 + e / 2] = pack_bf16x2(p0, p1);
    }
    const uint32_t w = 0xfefefefeu - f.vx[kt];  // bytes of 2^-(exponent)
    iv[kt >> 1][(kt & 1) * 2] = (w & 0xffu) << 7 | (w & 0xff00u) << 15;
    iv[kt >> 1][(kt & 1) * 2 + 1] = (w & 0xff0000u) >> 9 | (w & 0xff000000u) >> 1;
  }
  st.l *= alpha;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) st.o[dt] *= alpha;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const bf16x8_t pb = bits_bf16x8(u32x4_t{pw[c][0], pw[c][1], pw[c][2], pw[c][3]});
    st.l = mfma16x16x32(bits_bf16x8(u32x4_t{iv[c][0], iv[c][1], iv[c][2], iv[c][3]}), pb, st.l);
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt)
      st.o[dt] = mfma16x16x32(q8_bf16x8(f.v[dt][2 * c], f.v[dt][2 * c + 1]), pb, st.o[dt]);
  }
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
__device__ __forceinline__ void q8_load_block(Q8Frags<HD>& f, const uint8_t* K, const uint8_t* V, const uint8_t* Kx,
                                              const uint8_t* Vx, int blk, int lane) {
  const uint8_t* kb = K + (size_t)blk * 64 * HD + lane * 16;
  const uint8_t* vb = V + (size_t)blk * 64 * HD + lane * 16;
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int p = 0; p < HD / 64; ++p) f.k[kt][p] = *(const u32x4_t*)(kb + (kt * (HD / 64) + p) * 1024);
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) f.v[dt] = *(const u32x4_t*)(vb + dt * 1024);
  f.kx = *(const u32x4_t*)(Kx + (size_t)blk * 64 + (lane >> 4) * 16);
  f.vx = *(const u32x4_t*)(Vx + (size_t)blk * 64 + (lane >> 4) * 16);
}

template <int HD>
__device__ __forceinline__ void q8_store_state(const AttnQ8Args& a, size_t rec, const Q8State<HD>& st, int g) {
  float* o = a.ws_o + rec * HD + 4 * g;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) *(f32x4_t*)(o + dt * 16) = st.o[dt];
  a.ws_ml[rec] = make_float2(st.m, st.l[0]);
}

template <int HD>
__device__ __forceinline__ void q8_load_state(const AttnQ8Args& a, size_t rec, Q8State<HD>& st, int g) {
  const float* o = a.ws_o + rec * HD + 4 * g;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) st.o[dt] = *(const f32x4_t*)(o + dt * 16);
  const float2 ml = a.ws_ml[rec];
  st.m = ml.x;
  st.l = f32x4_t{ml.y, ml.y, ml.y, ml.y};
}

// Rows [r0, r1) of a sequence and the number of its blocks that every row attends. Called by whole waves.
__device__ __forceinline__ int q8_shared_blocks(const AttnQ8Args& a, int seq, int lane, int& r0, int& r1) {
  r0 = min(max(a.row_begin[seq], 0), a.M);
  r1 = min(max(a.row_begin[seq + 1], r0), min(a.M, r0 + QA_ROWS));
  int p = lane < r1 - r0 ? a.prefix[r0 + lane] : INT32_MAX;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) p = min(p, __shfl_xor(p, o));
  return min(max(p, 0), a.l_max) / QA_BLK;
}

// Shared keys: one wave per (sequence, kv head, span, 16-row tile).
template <int HD>
__global__ __launch_bounds__(64) void q8_shared_kernel(AttnQ8Args a) {
  const int lane = threadIdx.x, j = lane & 15, g = lane >> 4;
  int id = blockIdx.x;
  const int tile = id % a.tiles;
  id /= a.tiles;
  const int kvh = id % a.kv;
  id /= a.kv;
  const int span = id % a.n_spans, seq = id / a.n_spans;
  int r0, r1;
  const int nb = q8_shared_blocks(a, seq, lane, r0, r1);
  const int b0 = span * a.span_blk, b1 = min(nb, b0 + a.span_blk), n_rows = (r1 - r0) * a.rep;
  if (r1 <= r0 || b0 >= b1 || tile * 16 >= n_rows) return;
  const size_t reg = ((size_t)seq * a.kv + kvh) * a.max_len;
  const int R = min(tile * 16 + j, n_rows - 1);  // rows past the last repeat it and store the same record
  const int row = r0 + R / a.rep, h = kvh * a.rep + R % a.rep;
  u32x4_t qf[HD / 32];
  q8_load_q<HD>(qf, a.Q + (size_t)row * a.ldq + (size_t)h * HD, g);
  Q8State<HD> st;
  q8_reset(st);
  for (int b = b0; b < b1; ++b) {
    Q8Frags<HD> f;
    q8_load_block<HD>(f, a.K + reg * HD, a.V + reg * HD, a.Kx + reg, a.Vx + reg, b, lane);
    q8_fold<HD, false>(f, qf, 0, a.scale_log2, st);
  }
  q8_store_state<HD>(a, ((size_t)row * a.heads + h) * a.n_spans + span, st, g);
}

// A row's own keys and the fold of its records: one workgroup per (sequence, row, kv head), 4 waves.
template <int HD>
__global__ __launch_bounds__(256) void q8_tail_kernel(AttnQ8Args a, int rows_max) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x % a.kv, seq = blockIdx.x / a.kv / rows_max, place = blockIdx.x / a.kv % rows_max;
  __shared__ int s_anc[QA_MAXD];
  __shared__ uint8_t s_v[QA_MAXD][HD];          // the ancestors' V codes
  __shared__ uint8_t s_x[2][QA_MAXD];           // and exponents (K, V)
  int r0, r1;
  const int nb = q8_shared_blocks(a, seq, lane, r0, r1);
  const int row = r0 + place;
  if (row >= r1) return;
  const int P = min(max(a.prefix[row], 0), a.l_max);
  const int L = min(P + min(max(a.depth[row], 0), QA_MAXD), a.l_max), D = L - P;
  const size_t reg = ((size_t)seq * a.kv + kvh) * a.max_len;
  const uint8_t *K = a.K + reg * HD, *V = a.V + reg * HD, *Kx = a.Kx + reg, *Vx = a.Vx + reg;
  const int n_blk = (L + QA_BLK - 1) / QA_BLK, n_sp = (n_blk + a.span_blk - 1) / a.span_blk;
  if (threadIdx.x < QA_MAXD) {
    const int sl = threadIdx.x < D ? a.anc[(size_t)row * QA_MAXD + threadIdx.x] : -1;
    const bool ok = sl >= 0 && sl < a.max_len;
    s_anc[threadIdx.x] = ok ? sl : -1;
    s_x[0][threadIdx.x] = ok ? Kx[q8_x_off(sl)] : 127;
    s_x[1][threadIdx.x] = ok ? Vx[q8_x_off(sl)] : 127;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < D * HD; i += 256) {
    const int sl = s_anc[i / HD];
    s_v[i / HD][i % HD] = sl >= 0 ? V[q8_v_off(sl, i % HD, HD)] : 0;
  }
  __syncthreads();
  const int cut = nb / a.span_blk;
  for (int t0 = 0; t0 < a.rep; t0 += 16) {
    const int hr = min(t0 + j, a.rep - 1), h = kvh * a.rep + hr;
    const size_t rec0 = ((size_t)row * a.heads + h) * a.n_spans;
    u32x4_t qf[HD / 32];
    q8_load_q<HD>(qf, a.Q + (size_t)row * a.ldq + (size_t)h * HD, g);
    for (int sp = cut + w; sp < n_sp; sp += 4) {  // spans are independent of each other: one wave each
      const int b0 = max(nb, sp * a.span_blk), b1 = min(n_blk, (sp + 1) * a.span_blk);
      if (b0 >= b1) continue;
      Q8State<HD> st;
      if (b0 > sp * a.span_blk) q8_load_state<HD>(a, rec0 + sp, st, g);
      else q8_reset(st);
      for (int b = b0; b < b1; ++b) {
        const int key0 = b * QA_BLK;
        Q8Frags<HD> f;
        uint32_t valid = 0;
        f.kx = *(const u32x4_t*)(Kx + key0 + g * 16);
        f.vx = *(const u32x4_t*)(Vx + key0 + g * 16);
        // K: one slot a lane. Loads are unconditional (a key that is not attended reads its own block's slot,
        // which exists) and masked after.
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
          const int pos = key0 + 16 * kt + j;
          const int sl = pos < P ? pos : pos < L ? s_anc[pos - P] : -1;
          const uint32_t keep = sl >= 0 ? 0xffffffffu : 0u;
#pragma unroll
          for (int p = 0; p < HD / 64; ++p)
            f.k[kt][p] = *(const u32x4_t*)(K + q8_k_off(sl >= 0 ? sl : key0, 64 * p + 16 * g, HD)) & keep;
        }
        // V and the exponents: the block's own slots, positions from P on cleared, then the ancestors' put in
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
          f.kx[kt] = (f.kx[kt] & m) | (0x7f7f7f7fu & ~m);
          f.vx[kt] = (f.vx[kt] & m) | (0x7f7f7f7fu & ~m);
        }
        const uint8_t* vb = V + (size_t)b * 64 * HD + lane * 16;
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt) f.v[dt] = *(const u32x4_t*)(vb + dt * 1024) & own;
        const int a0 = max(P, key0) - P, a1 = min(L, key0 + QA_BLK) - P;
        for (int an = a0; an < a1; ++an) {  // uniform
          const int off = P + an - key0, kt = off >> 4, e = off & 3;
          const bool mine = ((off >> 2) & 3) == g;
          const uint32_t sel = mine ? 0xffu << (8 * e) : 0u;
          const uint32_t xk = s_x[0][an] * 0x01010101u, xv = s_x[1][an] * 0x01010101u;
          if (mine && s_anc[an] >= 0) valid |= 1u << (4 * kt + e);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t m = c == kt ? sel : 0u;
            f.kx[c] = (f.kx[c] & ~m) | (xk & m);
            f.vx[c] = (f.vx[c] & ~m) | (xv & m);
#pragma unroll
            for (int dt = 0; dt < HD / 16; ++dt)
              f.v[dt][c] = (f.v[dt][c] & ~m) | ((s_v[an][dt * 16 + j] * 0x01010101u) & m);
          }
        }
        q8_fold<HD, true>(f, qf, valid, a.scale_log2, st);
      }
      q8_store_state<HD>(a, rec0 + sp, st, g);
    }
  }
  __syncthreads();  // the records of this workgroup's waves
  // fold the spans in order: maximum first, then the weighted sums
  for (int i = threadIdx.x; i < a.rep * HD; i += 256) {
    const int h = kvh * a.rep + i / HD, d = i % HD;
    const size_t rec0 = ((size_t)row * a.heads + h) * a.n_spans;
    float mx = -INFINITY;
    for (int s = 0; s < n_sp; ++s) mx = fmaxf(mx, a.ws_ml[rec0 + s].x);
    float l = 0.f, o = 0.f;
    for (int s = 0; s < n_sp; ++s) {
      const float2 ml = a.ws_ml[rec0 + s];
      const float wgt = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mx);
      l = fmaf(ml.y, wgt, l);
      o = fmaf(a.ws_o[(rec0 + s) * HD + d], wgt, o);
    }
    a.out[(size_t)row * a.ldo + (size_t)h * HD + d] = f2bf(l == 0.f ? 0.f : o / l);  // NaN stays NaN
  }
}

static int q8_spans(int64_t l_max, int span) { return (int)((l_max + span - 1) / span); }

template <int HD>
static int launch_attn_q8(const AttnQ8Args& a, int rows_max, hipStream_t stream) {
  const int64_t shared = (int64_t)a.n_seq * a.n_spans * a.kv * a.tiles, tail = (int64_t)a.n_seq * rows_max * a.kv;
  if (shared > INT32_MAX || tail > INT32_MAX) return set_error(SSD_ERANGE, "attention_q8: too many workgroups");
  if (a.l_max >= QA_BLK) {
    SSD_LAUNCH((q8_shared_kernel<HD>), dim3((unsigned)shared), dim3(64), 0, stream, a);
    if (int rc = check_launch("attn_q8_shared")) return rc;
  }
  SSD_LAUNCH((q8_tail_kernel<HD>), dim3((unsigned)tail), dim3(256), 0, stream, a, rows_max);
  return check_launch("attn_q8_tail");
}

}  // namespace ssd

using namespace ssd;

SSD_API int64_t ssd_attn_q8_ws_floats(int M, int heads, int head_dim, int64_t l_max, int span) {
  if (M < 0 || heads < 1 || head_dim < 1 || l_max < 1 || span < 64 || span % 64) return -1;
  return (int64_t)M * heads * q8_spans(l_max, span) * (head_dim + 2);
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
  if (span < 64 || span % 64) return set_error(SSD_EINVAL, "attention_q8: span %d must be a multiple of 64", span);
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
  a.l_max = l_max, a.span_blk = span / 64, a.n_spans = q8_spans(l_max, span);
  a.tiles = (rows_max * a.rep + 15) / 16;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.ws_o = ws;
  a.ws_ml = (float2*)(ws + (int64_t)M * heads * a.n_spans * cache->head_dim);
  a.out = out, a.ldo = ldo;
  return cache->head_dim == 64 ? launch_attn_q8<64>(a, rows_max, stream) : launch_attn_q8<128>(a, rows_max, stream);
}
