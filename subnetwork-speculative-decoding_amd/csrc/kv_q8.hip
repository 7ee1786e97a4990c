// Rotary positions, and the 8-bit KV cache's write, read-back and compaction (layout in kv_q8.h).
#include "kv_q8.h"

#include <algorithm>

namespace ssd {

struct RopeArgs {
  const float *cos, *sin;  // [rows][rot / 2], or null: no rotation
  int64_t rows;
  int rot, interleaved;
  const int* pos;
};

struct WriteArgs {
  const bf16_t *q, *k, *v;  // rows of `heads` / `kv` heads each, row strides below
  int64_t ldq, ldk, ldv, ldo;
  bf16_t* q_out;
  int M, heads, kv;
  RopeArgs rope;
  uint8_t *ck, *cv, *cxk, *cxv;
  int n_seq;
  int64_t max_len;
  const int *seq, *slot;
};

template <int E>
struct Chunk {
  float x[E];
};

template <int E>
__device__ __forceinline__ Chunk<E> load_chunk(const bf16_t* p) {
  Chunk<E> c;
  uint32_t w[E / 2];
  if constexpr (E == 8) {
    const uint4 u = *(const uint4*)p;
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else {
    const uint2 u = *(const uint2*)p;
    w[0] = u.x, w[1] = u.y;
  }
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    c.x[2 * i] = __uint_as_float(w[i] << 16);
    c.x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  return c;
}

template <int E>
__device__ __forceinline__ void store_chunk(bf16_t* p, const Chunk<E>& c) {
  uint32_t w[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) w[i] = pack_bf16x2(c.x[2 * i], c.x[2 * i + 1]);
  if constexpr (E == 8) *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
  else *(uint2*)p = make_uint2(w[0], w[1]);
}

enum { ROPE_NONE = 0, ROPE_HALF = 1, ROPE_PAIRS = 2 };  // no rotation; pairs (i, i + rot / 2); pairs (2i, 2i + 1)

// cos and sin of dims d0 .. d0 + E for one token (their pairs' entries for ROPE_PAIRS), and whether they turn.
template <int E, int MODE>
struct Turn {
  static constexpr int N = MODE == ROPE_PAIRS ? E / 2 : E;
  float c[N], s[N];
  bool on;
};

template <int E, int MODE>
__device__ __forceinline__ Turn<E, MODE> load_turn(const RopeArgs& r, int d0, int64_t pos) {
  Turn<E, MODE> t;
  t.on = MODE != ROPE_NONE && d0 < r.rot;
  if (!t.on) return t;
  const int half = r.rot >> 1, e0 = MODE == ROPE_PAIRS ? d0 >> 1 : d0 < half ? d0 : d0 - half;
  const float *ct = r.cos + pos * half + e0, *st = r.sin + pos * half + e0;
#pragma unroll
  for (int i = 0; i < Turn<E, MODE>::N; ++i) t.c[i] = ct[i], t.s[i] = st[i];
  return t;
}

// Dims d0 .. d0 + E of the head at x, rotated. Products and sums are rounded one by one (no multiply-add
// contraction), so the codes a rotated row is quantised to do not depend on the compiler.
template <int E, int MODE>
__device__ __forceinline__ Chunk<E> load_rotated(const bf16_t* x, int d0, const RopeArgs& r, const Turn<E, MODE>& t) {
#pragma clang fp contract(off)
  Chunk<E> c = load_chunk<E>(x + d0);
  if (!t.on) return c;
  if constexpr (MODE == ROPE_PAIRS) {
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float a = c.x[i], b = c.x[i + 1];
      c.x[i] = a * t.c[i / 2] - b * t.s[i / 2];
      c.x[i + 1] = b * t.c[i / 2] + a * t.s[i / 2];
    }
  } else if constexpr (MODE == ROPE_HALF) {
    const int half = r.rot >> 1;  // a multiple of 8: a chunk lies in one half
    const bool low = d0 < half;
    const Chunk<E> o = load_chunk<E>(x + (low ? d0 + half : d0 - half));
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float xc = c.x[i] * t.c[i], os = o.x[i] * t.s[i];
      c.x[i] = low ? xc - os : xc + os;
    }
  }
  return c;
}

template <int MODE>
__device__ __forceinline__ int64_t rope_row(const RopeArgs& r, int row) {
  if (MODE == ROPE_NONE) return 0;
  const int64_t p = r.pos[row];
  return p < 0 ? 0 : p < r.rows ? p : r.rows - 1;
}

// Largest value over the 16 lanes of a row of the wave.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));   // lane ^ 1
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));   // lane ^ 2
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true));  // the other half of 8
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true));  // the other half of 16
}

// The row's exponent byte (the same on its 16 lanes) and the chunk's codes. Values that are not finite do
// not count for the exponent and are stored as NaN. All 16 lanes call it together.
template <int E>
__device__ __forceinline__ int quantise(const Chunk<E>& c, uint32_t (&w)[E / 4]) {
  constexpr uint32_t INF = 0x7f800000u;
  uint32_t u[E], top = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    u[i] = __float_as_uint(c.x[i]) & 0x7fffffffu;
    top = max(top, u[i]);
  }
  float y[E];
#pragma unroll
  for (int i = 0; i < E; ++i) y[i] = c.x[i];
  if (__any(top >= INF)) {  // rare: taken by the wave, changes only what is not finite
    top = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      top = max(top, u[i] < INF ? u[i] : 0u);
      y[i] = u[i] < INF ? y[i] : __uint_as_float(0x7fc00000u);
    }
  }
  const int b = q8_exponent(__uint_as_float(max16(top)));
  const float inv = q8_inv_scale(b);
#pragma unroll
  for (int i = 0; i < E; i += 4) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[i] * inv, y[i + 1] * inv, 0, false);
    w[i / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[i + 2] * inv, y[i + 3] * inv, p, true);
  }
  return b;
}

// Bytes i of four words become word i.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t l01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), h01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t l23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), h23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(l23, l01, 0x05040100u), w[1] = __builtin_amdgcn_perm(l23, l01, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(h23, h01, 0x05040100u), w[3] = __builtin_amdgcn_perm(h23, h01, 0x07060302u);
}

// The R rows of a unit: where each goes, and whether they are four consecutive slots of one aligned quad (whose V
// codes of one dim, and whose exponents, are one word).
template <int R>
struct Places {
  int reg[R];  // sequence * kv_heads, -1: outside the cache (or no such row)
  int slot[R];
  bool quad;
};

// Units of R = 4 rows start where row 0's slot quad does, so that a prompt's consecutive rows fall into whole quads.
template <int R>
__device__ __forceinline__ int unit_row(const int* slot, int unit) {
  return R == 1 ? unit : unit * R - (slot[0] & (R - 1));
}

template <int R>
__device__ __forceinline__ Places<R> load_places(const int* seq, const int* slot, int row0, int M, int n_seq, int max_len, int kv) {
  Places<R> p;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + i, r = min(max(row, 0), M - 1), sq = seq[r];
    p.slot[i] = slot[r];
    p.reg[i] = row == r && (uint32_t)sq < (uint32_t)n_seq && (uint32_t)p.slot[i] < (uint32_t)max_len ? sq * kv : -1;
  }
  p.quad = R == 4 && p.reg[0] >= 0 && (p.slot[0] & 3) == 0;
#pragma unroll
  for (int i = 1; i < R; ++i) p.quad = p.quad && p.reg[i] == p.reg[0] && p.slot[i] == p.slot[0] + i;
  return p;
}

// Workgroups [0, kv_wgs) write K and V: sixteen lanes per (R rows, kv head, K or V), E = head_dim / 16 dims a lane.
// The others rotate q: sixteen lanes per (row, H heads), which share the row's cos and sin. R and H are 4 for
// long calls. 4096 rows of 32 + 8 heads of 128 take 22 us for 94 MB (4.3 TB/s, a copy reaches 5.0): 8 us the rotation
// of q, 14 us K and V, of which the stores are 5.5 and the VALU work of rotating and quantising most of the rest.
template <int HD, int R, int H, int MODE>
__global__ __launch_bounds__(256) void kv_q8_write_kernel(WriteArgs a, int kv_wgs, int kv_units, int q_units) {
  constexpr int E = HD / 16;
  const int ln = threadIdx.x & 15, d0 = ln * E;
  if ((int)blockIdx.x >= kv_wgs) {
    const int64_t id = (int64_t)(blockIdx.x - kv_wgs) * 16 + (threadIdx.x >> 4);
    if (id >= (int64_t)a.M * q_units) return;
    const int row = (int)(id / q_units), h0 = (int)(id % q_units) * H;
    const Turn<E, MODE> t = load_turn<E, MODE>(a.rope, d0, rope_row<MODE>(a.rope, row));
    const bf16_t* x = a.q + (size_t)row * a.ldq;
    bf16_t* y = a.q_out + (size_t)row * a.ldo;
    Chunk<E> c[H];
#pragma unroll
    for (int i = 0; i < H; ++i) c[i] = load_rotated<E, MODE>(x + (size_t)min(h0 + i, a.heads - 1) * HD, d0, a.rope, t);
#pragma unroll
    for (int i = 0; i < H; ++i)
      if (h0 + i < a.heads) store_chunk<E>(y + (size_t)(h0 + i) * HD + d0, c[i]);
    return;
  }
  const int id = blockIdx.x * 16 + (threadIdx.x >> 4), unit = id / (2 * a.kv);
  if (unit >= kv_units) return;
  const int u = id % (2 * a.kv), h = u < a.kv ? u : u - a.kv;
  const bool is_v = u >= a.kv;
  const int row0 = unit_row<R>(a.slot, unit);
  const Places<R> at = load_places<R>(a.seq, a.slot, row0, a.M, a.n_seq, (int)a.max_len, a.kv);
  uint32_t w[R][E / 4];
  int b[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = min(max(row0 + i, 0), a.M - 1);
    Chunk<E> c;
    if (is_v) c = load_chunk<E>(a.v + (size_t)row * a.ldv + (size_t)h * HD + d0);
    else c = load_rotated<E, MODE>(a.k + (size_t)row * a.ldk + (size_t)h * HD, d0, a.rope, load_turn<E, MODE>(a.rope, d0, rope_row<MODE>(a.rope, row)));
    b[i] = quantise<E>(c, w[i]);
  }
  uint8_t *codes = is_v ? a.cv : a.ck, *exps = is_v ? a.cxv : a.cxk;
  if constexpr (R == 4)
    if (at.quad) {
      const int64_t reg = at.reg[0] + h;
      if (ln == 0) *(uint32_t*)(exps + reg * a.max_len + q8_x_off(at.slot[0])) = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
      if (is_v) {
        uint8_t* dst = codes + reg * a.max_len * HD + q8_v_off(at.slot[0], d0, HD);
#pragma unroll
        for (int k = 0; k < E / 4; ++k) {
          uint32_t t[4] = {w[0][k], w[1][k], w[2][k], w[3][k]};
          transpose4(t);
#pragma unroll
          for (int i = 0; i < 4; ++i) *(uint32_t*)(dst + (4 * k + i) * 16) = t[i];
        }
        return;
      }
    }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (at.reg[i] < 0) continue;
    const int64_t reg = at.reg[i] + h;
    if (!is_v) {
      uint8_t* dst = codes + reg * a.max_len * HD + q8_k_off(at.slot[i], d0, HD);
      if constexpr (E == 8) *(uint2*)dst = make_uint2(w[i][0], w[i][1]);
      else *(uint32_t*)dst = w[i][0];
    } else {
      uint8_t* dst = codes + reg * a.max_len * HD + q8_v_off(at.slot[i], d0, HD);
#pragma unroll
      for (int e = 0; e < E; ++e) dst[e * 16] = (uint8_t)(w[i][e / 4] >> (8 * (e & 3)));
    }
    if (ln == 0 && !(R == 4 && at.quad)) exps[reg * a.max_len + q8_x_off(at.slot[i])] = (uint8_t)b[i];
  }
}

struct ReadArgs {
  const uint8_t *ck, *cv, *cxk, *cxv;
  int n_seq, kv, M;
  int64_t max_len;
  const int *seq, *slot;
  bf16_t *k, *v;
  int64_t ldk, ldv;
};

// Sixteen lanes per (R rows, kv head, K or V), as they are written.
template <int HD, int R>
__global__ __launch_bounds__(256) void kv_q8_read_kernel(ReadArgs a, int units) {
  constexpr int E = HD / 16;
  const int id = blockIdx.x * 16 + (threadIdx.x >> 4), unit = id / (2 * a.kv), ln = threadIdx.x & 15, d0 = ln * E;
  if (unit >= units) return;
  const int u = id % (2 * a.kv), h = u < a.kv ? u : u - a.kv;
  const bool is_v = u >= a.kv;
  const int row0 = unit_row<R>(a.slot, unit);
  const Places<R> at = load_places<R>(a.seq, a.slot, row0, a.M, a.n_seq, (int)a.max_len, a.kv);
  const uint8_t *codes = is_v ? a.cv : a.ck, *exps = is_v ? a.cxv : a.cxk;
  uint32_t w[R][E / 4], b[R];
  bool done = false;
  if constexpr (R == 4)
    if (at.quad) {
      const int64_t reg = at.reg[0] + h;
      const uint32_t x = *(const uint32_t*)(exps + reg * a.max_len + q8_x_off(at.slot[0]));
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = x >> (8 * i) & 0xffu;
      if (is_v) {
        done = true;
        const uint8_t* src = codes + reg * a.max_len * HD + q8_v_off(at.slot[0], d0, HD);
#pragma unroll
        for (int k = 0; k < E / 4; ++k) {
          uint32_t t[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) t[i] = *(const uint32_t*)(src + (4 * k + i) * 16);
          transpose4(t);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i][k] = t[i];
        }
      }
    }
  if (!done) {
#pragma unroll
    for (int i = 0; i < R; ++i) {  // places outside the cache read the first one's codes, and are cleared below
      const int64_t reg = max(at.reg[i], 0) + h;
      const int sl = at.reg[i] < 0 ? 0 : at.slot[i];
      b[i] = exps[reg * a.max_len + q8_x_off(sl)];
      if (!is_v) {
        const uint8_t* src = codes + reg * a.max_len * HD + q8_k_off(sl, d0, HD);
        if constexpr (E == 8) {
          const uint2 t = *(const uint2*)src;
          w[i][0] = t.x, w[i][1] = t.y;
        } else {
          w[i][0] = *(const uint32_t*)src;
        }
      } else {
        const uint8_t* src = codes + reg * a.max_len * HD + q8_v_off(sl, d0, HD);
#pragma unroll
        for (int e = 0; e < E; e += 4)
          w[i][e / 4] = src[e * 16] | src[e * 16 + 16] << 8 | src[e * 16 + 32] << 16 | (uint32_t)src[e * 16 + 48] << 24;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + i;
    if (row < 0 || row >= a.M) continue;
    const bool in = at.reg[i] >= 0;
    const float sc = q8_scale(b[i]);
    Chunk<E> c;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i][e / 4], false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i][e / 4], true);
      c.x[e] = in ? lo[0] * sc : 0.f, c.x[e + 1] = in ? lo[1] * sc : 0.f;
      c.x[e + 2] = in ? hi[0] * sc : 0.f, c.x[e + 3] = in ? hi[1] * sc : 0.f;
    }
    store_chunk<E>((is_v ? a.v + (size_t)row * a.ldv : a.k + (size_t)row * a.ldk) + (size_t)h * HD + d0, c);
  }
}

// One workgroup per (layer, sequence, kv head): every source row is read into LDS before the first destination is
// written. Bound by its chain of loads: counts and places, then the rows (16 sequences of up to 5 rows, 8 kv heads, 2 layers: 4.3 us).
constexpr int Q8_MAX_MOVE = 64;

struct CompactArgs {
  uint8_t *ck, *cv, *cxk, *cxv;
  int n_seq, kv, n_max;
  int64_t max_len;
  const int *start, *src, *n;
};

template <int HD>
__global__ __launch_bounds__(256) void kv_q8_compact_kernel(CompactArgs a) {
  const int h = blockIdx.x % a.kv, sq = (blockIdx.x / a.kv) % a.n_seq;
  const int n = min(max(a.n[sq], 0), a.n_max);
  if (n == 0) return;
  const size_t reg = blockIdx.x;  // [layer][sequence][kv head]
  uint8_t *ck = a.ck + reg * a.max_len * HD, *cv = a.cv + reg * a.max_len * HD;
  uint8_t *xk = a.cxk + reg * a.max_len, *xv = a.cxv + reg * a.max_len;
  const int64_t start = a.start[sq];
  __shared__ int s_src[Q8_MAX_MOVE];  // -1: this move names a slot outside the cache
  if (threadIdx.x < n) {
    const int s = a.src[(size_t)sq * a.n_max + threadIdx.x];
    const int64_t d = start + threadIdx.x;
    s_src[threadIdx.x] = s >= 0 && s < a.max_len && d >= 0 && d < a.max_len ? s : -1;
  }
  __syncthreads();
  // K in 16-byte pieces, V and the exponents in bytes, four loads of a thread in flight. Loads are unconditional, from
  // slots that exist (a skipped move reads slot 0 and is not stored).
  constexpr int KC = HD / 16;
  __shared__ uint4 s_k[Q8_MAX_MOVE * KC];
  __shared__ uint8_t s_v[Q8_MAX_MOVE * HD];
  auto fetch = [&](int count, auto load, auto keep) {
    for (int i0 = threadIdx.x; i0 < count; i0 += 1024) {
      decltype(load(0)) v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = load(min(i0 + 256 * u, count - 1));
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + 256 * u < count) keep(i0 + 256 * u, v[u]);
    }
  };
  const int xj = min((int)threadIdx.x >> 1, n - 1);
  uint8_t* xp = threadIdx.x & 1 ? xv : xk;
  const uint8_t x = xp[q8_x_off(max(s_src[xj], 0))];
  fetch(n * KC, [&](int i) { return *(const uint4*)(ck + q8_k_off(max(s_src[i / KC], 0), i % KC * 16, HD)); },
        [&](int i, uint4 v) { s_k[i] = v; });
  fetch(n * HD, [&](int i) { return (uint32_t)cv[q8_v_off(max(s_src[i / HD], 0), i % HD, HD)]; },
        [&](int i, uint32_t v) { s_v[i] = (uint8_t)v; });
  __syncthreads();
  for (int i = threadIdx.x; i < n * KC; i += 256)
    if (s_src[i / KC] >= 0) *(uint4*)(ck + q8_k_off((int)start + i / KC, i % KC * 16, HD)) = s_k[i];
  for (int i = threadIdx.x; i < n * HD; i += 256)
    if (s_src[i / HD] >= 0) cv[q8_v_off((int)start + i / HD, i % HD, HD)] = s_v[i];
  if ((int)threadIdx.x < 2 * n && s_src[xj] >= 0) xp[q8_x_off((int)start + xj)] = x;
}

// Checks shared by the entry points that take the cache.
int q8_check(const SsdKvQ8* c, const char* what) {
  if (!c || !c->k || !c->v || !c->k_exp || !c->v_exp) return set_error(SSD_EINVAL, "%s: null cache", what);
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(SSD_EINVAL, "%s: head_dim %d unsupported (64, 128)", what, c->head_dim);
  if ((int64_t)c->n_seq * c->kv_heads > INT32_MAX) return set_error(SSD_ERANGE, "%s: too many sequences", what);
  if (c->n_seq < 1 || c->kv_heads < 1 || c->max_len < 64 || c->max_len % 64 || c->max_len > 1 << 30)
    return set_error(SSD_EINVAL, "%s: bad cache: %d sequences, %d kv heads, max_len %lld (a multiple of 64 up to 2^30)", what,
                     c->n_seq, c->kv_heads, (long long)c->max_len);
  if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_exp | (uintptr_t)c->v_exp) & 15)
    return set_error(SSD_EINVAL, "%s: cache arrays must be 16-byte aligned", what);
  return SSD_OK;
}

static int rope_check(const SsdRope* r, const int32_t* pos, int head_dim, RopeArgs& out, const char* what) {
  out = RopeArgs{};
  if (!r) return SSD_OK;
  if (!r->cos || !r->sin || !pos || r->rows < 1) return set_error(SSD_EINVAL, "%s: null rotary tables or positions", what);
  if (r->rot_dim < 16 || r->rot_dim % 16 || r->rot_dim > head_dim)
    return set_error(SSD_EINVAL, "%s: rot_dim %d must be a multiple of 16 up to head_dim %d", what, r->rot_dim, head_dim);
  out = RopeArgs{r->cos, r->sin, r->rows, r->rot_dim, r->interleaved != 0, pos};
  return SSD_OK;
}

static bool bad_rows(const void* p, int64_t ld, int64_t cols) { return ((uintptr_t)p & 15) || ld % 8 || ld < cols; }

template <typename F>
static int by_head_dim(int hd, F f) {
  if (hd == 64) f(std::integral_constant<int, 64>());
  else f(std::integral_constant<int, 128>());
  return 0;
}

// Units of R rows that cover M rows: with R = 4 the first may begin up to three rows early.
static int64_t row_units(int M, int r) { return r == 1 ? M : ((int64_t)M + 3) / 4 + 1; }
// From this many (row, kv head) pairs on a unit takes four rows: below, more units and less code are worth more than
// wider accesses. us, one row a unit / four, 8 kv heads and 32 q heads of 128: rotated and written, consecutive slots, 512
// rows 6.9 / 6.7, 768 9.2 / 7.7, 1024 11.9 / 8.6, 4096 37 / 22 (scattered slots, 768 rows 10.2 / 12.5, 1024 12.7 / 13.7, 4096 37 / 39:
// a prompt's case decides); read 512 rows 3.7 / 4.2, 1024 4.9 / 5.0, 2048 7.7 / 6.0, 4096 14.6 / 8.5. Rotation alone has no kv
// heads and counts its rows: 32 heads of 128, 1024 rows 5.0 / 4.9, 4096 14.8 / 13.0, 8192 25.0 / 23.0; 4096 rows of one
// head 2.6 / 3.3.
constexpr int64_t Q8_WRITE_QUADS = 6144, Q8_READ_QUADS = 20480;

template <int HD, int MODE>
static int launch_write_as(const WriteArgs& a, hipStream_t stream, const char* what) {
  const bool many = (int64_t)a.M * std::max(a.kv, 1) >= Q8_WRITE_QUADS;
  const int64_t units = a.kv ? row_units(a.M, many ? 4 : 1) : 0, kv_wgs = (units * 2 * a.kv + 15) / 16;
  const int q_units = (a.heads + (many ? 3 : 0)) / (many ? 4 : 1);
  const int64_t wgs = kv_wgs + ((int64_t)a.M * q_units + 15) / 16;
  if (grid_too_large(wgs, 256)) return set_error(SSD_ERANGE, "%s: too many rows", what);
  if (many) SSD_LAUNCH((kv_q8_write_kernel<HD, 4, 4, MODE>), dim3((unsigned)wgs), dim3(256), 0, stream, a, (int)kv_wgs, (int)units, q_units);
  else SSD_LAUNCH((kv_q8_write_kernel<HD, 1, 1, MODE>), dim3((unsigned)wgs), dim3(256), 0, stream, a, (int)kv_wgs, (int)units, q_units);
  return check_launch(what);
}

template <int HD>
static int launch_write_hd(const WriteArgs& a, hipStream_t stream, const char* what) {
  return !a.rope.cos ? launch_write_as<HD, ROPE_NONE>(a, stream, what)
         : a.rope.interleaved ? launch_write_as<HD, ROPE_PAIRS>(a, stream, what)
                              : launch_write_as<HD, ROPE_HALF>(a, stream, what);
}

static int launch_write(const WriteArgs& a, int hd, hipStream_t stream, const char* what) {
  return hd == 64 ? launch_write_hd<64>(a, stream, what) : launch_write_hd<128>(a, stream, what);
}

template <int HD>
static int launch_read(const ReadArgs& a, hipStream_t stream) {
  const bool many = (int64_t)a.M * a.kv >= Q8_READ_QUADS;
  const int64_t units = row_units(a.M, many ? 4 : 1), wgs = (units * 2 * a.kv + 15) / 16;
  if (grid_too_large(wgs, 256)) return set_error(SSD_ERANGE, "kv_q8_read: too many rows");
  if (many) SSD_LAUNCH((kv_q8_read_kernel<HD, 4>), dim3((unsigned)wgs), dim3(256), 0, stream, a, (int)units);
  else SSD_LAUNCH((kv_q8_read_kernel<HD, 1>), dim3((unsigned)wgs), dim3(256), 0, stream, a, (int)units);
  return check_launch("kv_q8_read");
}

}  // namespace ssd

using namespace ssd;

SSD_API int ssd_rope_bf16(const SsdRope* rope, const int32_t* row_pos, const uint16_t* x, int64_t ldx, int M, int heads,
                          int head_dim, uint16_t* y, int64_t ldy, hipStream_t stream) {
  if (!x || !y || !rope) return set_error(SSD_EINVAL, "rope: null pointer");
  if (M < 0 || heads < 1 || (head_dim != 64 && head_dim != 128))
    return set_error(SSD_EINVAL, "rope: bad M=%d heads=%d head_dim=%d (64, 128)", M, heads, head_dim);
  WriteArgs a{};
  if (int rc = rope_check(rope, row_pos, head_dim, a.rope, "rope")) return rc;
  if (bad_rows(x, ldx, (int64_t)heads * head_dim) || bad_rows(y, ldy, (int64_t)heads * head_dim))
    return set_error(SSD_EINVAL, "rope: rows must be 16-byte aligned with strides >= heads * head_dim");
  if (M == 0) return SSD_OK;
  a.q = x, a.ldq = ldx, a.q_out = y, a.ldo = ldy, a.M = M, a.heads = heads;
  return launch_write(a, head_dim, stream, "rope");
}

SSD_API int ssd_kv_q8_write_bf16(const SsdKvQ8* cache, const uint16_t* k, int64_t ldk, const uint16_t* v, int64_t ldv, int M,
                                 const int32_t* row_seq, const int32_t* row_slot, const SsdRope* rope,
                                 const int32_t* row_pos, const uint16_t* q, int64_t ldq, int heads, uint16_t* q_out,
                                 int64_t ldo, hipStream_t stream) {
  if (int rc = q8_check(cache, "kv_q8_write")) return rc;
  const int hd = cache->head_dim;
  const int64_t cols = (int64_t)cache->kv_heads * hd;
  if (!k || !v || !row_seq || !row_slot) return set_error(SSD_EINVAL, "kv_q8_write: null pointer");
  if (M < 0) return set_error(SSD_EINVAL, "kv_q8_write: bad M=%d", M);
  if (bad_rows(k, ldk, cols) || bad_rows(v, ldv, cols))
    return set_error(SSD_EINVAL, "kv_q8_write: k/v rows must be 16-byte aligned with strides >= kv_heads * head_dim");
  WriteArgs a{};
  if (int rc = rope_check(rope, row_pos, hd, a.rope, "kv_q8_write")) return rc;
  if (q) {
    if (!q_out || heads < 1 || bad_rows(q, ldq, (int64_t)heads * hd) || bad_rows(q_out, ldo, (int64_t)heads * hd))
      return set_error(SSD_EINVAL, "kv_q8_write: q/q_out rows must be 16-byte aligned with strides >= heads * head_dim");
    a.q = q, a.ldq = ldq, a.heads = heads, a.q_out = q_out, a.ldo = ldo;
  }
  if (M == 0) return SSD_OK;
  a.k = k, a.ldk = ldk, a.v = v, a.ldv = ldv, a.M = M, a.kv = cache->kv_heads;
  a.ck = cache->k, a.cv = cache->v, a.cxk = cache->k_exp, a.cxv = cache->v_exp;
  a.n_seq = cache->n_seq, a.max_len = cache->max_len, a.seq = row_seq, a.slot = row_slot;
  return launch_write(a, hd, stream, "kv_q8_write");
}

SSD_API int ssd_kv_q8_read_bf16(const SsdKvQ8* cache, int M, const int32_t* row_seq, const int32_t* row_slot, uint16_t* k,
                                int64_t ldk, uint16_t* v, int64_t ldv, hipStream_t stream) {
  if (int rc = q8_check(cache, "kv_q8_read")) return rc;
  const int64_t cols = (int64_t)cache->kv_heads * cache->head_dim;
  if (!k || !v || !row_seq || !row_slot) return set_error(SSD_EINVAL, "kv_q8_read: null pointer");
  if (M < 0) return set_error(SSD_EINVAL, "kv_q8_read: bad M=%d", M);
  if (bad_rows(k, ldk, cols) || bad_rows(v, ldv, cols))
    return set_error(SSD_EINVAL, "kv_q8_read: k/v rows must be 16-byte aligned with strides >= kv_heads * head_dim");
  if (M == 0) return SSD_OK;
  const ReadArgs a{cache->k, cache->v, cache->k_exp, cache->v_exp, cache->n_seq, cache->kv_heads, M, cache->max_len,
                   row_seq, row_slot, k, v, ldk, ldv};
  return cache->head_dim == 64 ? launch_read<64>(a, stream) : launch_read<128>(a, stream);
}

SSD_API int ssd_kv_q8_compact(const SsdKvQ8* cache, int layers, const int32_t* start, const int32_t* src, const int32_t* n,
                              int n_max, hipStream_t stream) {
  if (int rc = q8_check(cache, "kv_q8_compact")) return rc;
  if (!start || !src || !n) return set_error(SSD_EINVAL, "kv_q8_compact: null pointer");
  if (layers < 1 || n_max < 0) return set_error(SSD_EINVAL, "kv_q8_compact: bad layers=%d n_max=%d", layers, n_max);
  if (n_max > Q8_MAX_MOVE) return set_error(SSD_ERANGE, "kv_q8_compact: n_max %d > %d", n_max, Q8_MAX_MOVE);
  const int64_t wgs = (int64_t)layers * cache->n_seq * cache->kv_heads;
  if (grid_too_large(wgs, 256)) return set_error(SSD_ERANGE, "kv_q8_compact: cache too large");
  if (n_max == 0) return SSD_OK;
  const CompactArgs a{cache->k, cache->v, cache->k_exp, cache->v_exp, cache->n_seq, cache->kv_heads, n_max,
                      cache->max_len, start, src, n};
  by_head_dim(cache->head_dim, [&](auto c) {
    SSD_LAUNCH((kv_q8_compact_kernel<decltype(c)::value>), dim3((unsigned)wgs), dim3(256), 0, stream, a);
  });
  return check_launch("kv_q8_compact");
}
