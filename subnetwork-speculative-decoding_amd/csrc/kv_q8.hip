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

// Dims d0 .. d0 + E of a head at x, rotated for one token. Products and sums are rounded one by one (no
// multiply-add contraction), so the codes a rotated row is quantised to do not depend on the compiler.
template <int E>
__device__ __forceinline__ Chunk<E> load_rotated(const bf16_t* x, int d0, const RopeArgs& r, int64_t pos) {
#pragma clang fp contract(off)
  Chunk<E> c = load_chunk<E>(x + d0);
  if (!r.cos || d0 >= r.rot) return c;
  const int half = r.rot >> 1;
  const float *ct = r.cos + pos * half, *st = r.sin + pos * half;
  if (r.interleaved) {
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float cc = ct[(d0 + i) >> 1], ss = st[(d0 + i) >> 1], a = c.x[i], b = c.x[i + 1];
      c.x[i] = a * cc - b * ss;
      c.x[i + 1] = b * cc + a * ss;
    }
  } else {
    const bool low = d0 < half;  // half is a multiple of 8: a chunk lies in one half
    const Chunk<E> o = load_chunk<E>(x + (low ? d0 + half : d0 - half));
    const int t0 = low ? d0 : d0 - half;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float cc = ct[t0 + i], ss = st[t0 + i];
      const float xc = c.x[i] * cc, os = o.x[i] * ss;
      c.x[i] = low ? xc - os : xc + os;
    }
  }
  return c;
}

__device__ __forceinline__ int64_t rope_row(const RopeArgs& r, int row) {
  if (!r.cos) return 0;
  const int64_t p = r.pos[row];
  return p < 0 ? 0 : p < r.rows ? p : r.rows - 1;
}

// The row's exponent byte (the same on its 16 lanes) and the chunk's codes. Values that are not finite do
// not count for the exponent and are stored as NaN.
template <int E>
__device__ __forceinline__ int quantise(const Chunk<E>& c, uint32_t (&w)[E / 4]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const uint32_t u = __float_as_uint(c.x[i]) & 0x7fffffffu;
    top = max(top, u < 0x7f800000u ? u : 0u);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  const int b = q8_exponent(__uint_as_float(top));
  const float inv = q8_inv_scale(b);
  float y[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const uint32_t u = __float_as_uint(c.x[i]) & 0x7fffffffu;
    y[i] = u < 0x7f800000u ? c.x[i] * inv : __uint_as_float(0x7fc00000u);
  }
#pragma unroll
  for (int i = 0; i < E; i += 4) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[i], y[i + 1], 0, false);
    w[i / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[i + 2], y[i + 3], p, true);
  }
  return b;
}

// Sixteen lanes per (token, head), E = head_dim / 16 dims a lane.
template <int HD>
__global__ __launch_bounds__(256) void kv_q8_write_kernel(WriteArgs a) {
  constexpr int E = HD / 16;
  const int units = a.heads + 2 * a.kv;
  const int64_t id = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (id >= (int64_t)a.M * units) return;
  const int row = (int)(id / units), u = (int)(id % units), ln = threadIdx.x & 15, d0 = ln * E;
  if (u < a.heads) {
    const Chunk<E> c = load_rotated<E>(a.q + (size_t)row * a.ldq + (size_t)u * HD, d0, a.rope, rope_row(a.rope, row));
    store_chunk<E>(a.q_out + (size_t)row * a.ldo + (size_t)u * HD + d0, c);
    return;
  }
  const int sq = a.seq[row], sl = a.slot[row];
  if (sq < 0 || sq >= a.n_seq || sl < 0 || sl >= a.max_len) return;
  const bool is_v = u >= a.heads + a.kv;
  const int h = u - a.heads - (is_v ? a.kv : 0);
  const size_t reg = (size_t)sq * a.kv + h;
  uint32_t w[E / 4];
  if (!is_v) {
    const Chunk<E> c = load_rotated<E>(a.k + (size_t)row * a.ldk + (size_t)h * HD, d0, a.rope, rope_row(a.rope, row));
    const int b = quantise<E>(c, w);
    uint8_t* dst = a.ck + reg * a.max_len * HD + q8_k_off(sl, d0, HD);
    if constexpr (E == 8) *(uint2*)dst = make_uint2(w[0], w[1]);
    else *(uint32_t*)dst = w[0];
    if (ln == 0) a.cxk[reg * a.max_len + q8_x_off(sl)] = (uint8_t)b;
  } else {
    const Chunk<E> c = load_chunk<E>(a.v + (size_t)row * a.ldv + (size_t)h * HD + d0);
    const int b = quantise<E>(c, w);
    uint8_t* dst = a.cv + reg * a.max_len * HD + q8_v_off(sl, d0, HD);
#pragma unroll
    for (int i = 0; i < E; ++i) dst[i * 16] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
    if (ln == 0) a.cxv[reg * a.max_len + q8_x_off(sl)] = (uint8_t)b;
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

template <int HD>
__global__ __launch_bounds__(256) void kv_q8_read_kernel(ReadArgs a) {
  constexpr int E = HD / 16;
  const int64_t id = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (id >= (int64_t)a.M * 2 * a.kv) return;
  const int row = (int)(id / (2 * a.kv)), u = (int)(id % (2 * a.kv)), ln = threadIdx.x & 15, d0 = ln * E;
  const int sq = a.seq[row], sl = a.slot[row];
  const bool is_v = u >= a.kv;
  const int h = is_v ? u - a.kv : u;
  bf16_t* dst = (is_v ? a.v + (size_t)row * a.ldv : a.k + (size_t)row * a.ldk) + (size_t)h * HD + d0;
  if (sq < 0 || sq >= a.n_seq || sl < 0 || sl >= a.max_len) {
    store_chunk<E>(dst, Chunk<E>{});
    return;
  }
  const size_t reg = (size_t)sq * a.kv + h;
  uint32_t w[E / 4];
  if (!is_v) {
    const uint8_t* src = a.ck + reg * a.max_len * HD + q8_k_off(sl, d0, HD);
    if constexpr (E == 8) {
      const uint2 t = *(const uint2*)src;
      w[0] = t.x, w[1] = t.y;
    } else {
      w[0] = *(const uint32_t*)src;
    }
  } else {
    const uint8_t* src = a.cv + reg * a.max_len * HD + q8_v_off(sl, d0, HD);
#pragma unroll
    for (int i = 0; i < E; i += 4)
      w[i / 4] = src[i * 16] | src[i * 16 + 16] << 8 | src[i * 16 + 32] << 16 | (uint32_t)src[i * 16 + 48] << 24;
  }
  const float sc = q8_scale((is_v ? a.cxv : a.cxk)[reg * a.max_len + q8_x_off(sl)]);
  Chunk<E> c;
#pragma unroll
  for (int i = 0; i < E; i += 4) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i / 4], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i / 4], true);
    c.x[i] = lo[0] * sc, c.x[i + 1] = lo[1] * sc, c.x[i + 2] = hi[0] * sc, c.x[i + 3] = hi[1] * sc;
  }
  store_chunk<E>(dst, c);
}

// One workgroup per (layer, sequence, kv head): every source row is read (K and V as 16-byte pieces of
// dims, through registers) before the first destination is written.
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
  constexpr int KC = HD / 16;                             // 16-byte pieces of a K row
  constexpr int KI = Q8_MAX_MOVE * KC / 256, VI = Q8_MAX_MOVE * HD / 256;
  uint4 kr[KI];
  uint8_t vr[VI];
  uint8_t x = 0;
#pragma unroll
  for (int it = 0; it < KI; ++it) {
    const int j = (threadIdx.x + it * 256) / KC, d = (threadIdx.x + it * 256) % KC * 16;
    if (j < n && s_src[j] >= 0) kr[it] = *(const uint4*)(ck + q8_k_off(s_src[j], d, HD));
  }
#pragma unroll
  for (int it = 0; it < VI; ++it) {
    const int j = (threadIdx.x + it * 256) / HD, d = (threadIdx.x + it * 256) % HD;
    if (j < n && s_src[j] >= 0) vr[it] = cv[q8_v_off(s_src[j], d, HD)];
  }
  const int xj = threadIdx.x >> 1;
  uint8_t* xp = threadIdx.x & 1 ? xv : xk;
  if (xj < n && s_src[xj] >= 0) x = xp[q8_x_off(s_src[xj])];
  __syncthreads();
#pragma unroll
  for (int it = 0; it < KI; ++it) {
    const int j = (threadIdx.x + it * 256) / KC, d = (threadIdx.x + it * 256) % KC * 16;
    if (j < n && s_src[j] >= 0) *(uint4*)(ck + q8_k_off((int)start + j, d, HD)) = kr[it];
  }
#pragma unroll
  for (int it = 0; it < VI; ++it) {
    const int j = (threadIdx.x + it * 256) / HD, d = (threadIdx.x + it * 256) % HD;
    if (j < n && s_src[j] >= 0) cv[q8_v_off((int)start + j, d, HD)] = vr[it];
  }
  if (xj < n && s_src[xj] >= 0) xp[q8_x_off((int)start + xj)] = x;
}

// Checks shared by the entry points that take the cache.
int q8_check(const SsdKvQ8* c, const char* what) {
  if (!c || !c->k || !c->v || !c->k_exp || !c->v_exp) return set_error(SSD_EINVAL, "%s: null cache", what);
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(SSD_EINVAL, "%s: head_dim %d unsupported (64, 128)", what, c->head_dim);
  if (c->n_seq < 1 || c->kv_heads < 1 || c->max_len < 64 || c->max_len % 64 || c->max_len > INT32_MAX - 63)
    return set_error(SSD_EINVAL, "%s: bad cache: %d sequences, %d kv heads, max_len %lld (a multiple of 64)", what,
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

static int launch_write(const WriteArgs& a, int hd, hipStream_t stream, const char* what) {
  const int64_t wgs = ((int64_t)a.M * (a.heads + 2 * a.kv) + 15) / 16;
  if (wgs > INT32_MAX) return set_error(SSD_ERANGE, "%s: too many rows", what);
  by_head_dim(hd, [&](auto c) {
    SSD_LAUNCH((kv_q8_write_kernel<decltype(c)::value>), dim3((unsigned)wgs), dim3(256), 0, stream, a);
  });
  return check_launch(what);
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
  const int64_t wgs = ((int64_t)M * 2 * cache->kv_heads + 15) / 16;
  if (wgs > INT32_MAX) return set_error(SSD_ERANGE, "kv_q8_read: too many rows");
  if (M == 0) return SSD_OK;
  const ReadArgs a{cache->k, cache->v, cache->k_exp, cache->v_exp, cache->n_seq, cache->kv_heads, M, cache->max_len,
                   row_seq, row_slot, k, v, ldk, ldv};
  by_head_dim(cache->head_dim, [&](auto c) {
    SSD_LAUNCH((kv_q8_read_kernel<decltype(c)::value>), dim3((unsigned)wgs), dim3(256), 0, stream, a);
  });
  return check_launch("kv_q8_read");
}

SSD_API int ssd_kv_q8_compact(const SsdKvQ8* cache, int layers, const int32_t* start, const int32_t* src, const int32_t* n,
                              int n_max, hipStream_t stream) {
  if (int rc = q8_check(cache, "kv_q8_compact")) return rc;
  if (!start || !src || !n) return set_error(SSD_EINVAL, "kv_q8_compact: null pointer");
  if (layers < 1 || n_max < 0) return set_error(SSD_EINVAL, "kv_q8_compact: bad layers=%d n_max=%d", layers, n_max);
  if (n_max > Q8_MAX_MOVE) return set_error(SSD_ERANGE, "kv_q8_compact: n_max %d > %d", n_max, Q8_MAX_MOVE);
  const int64_t wgs = (int64_t)layers * cache->n_seq * cache->kv_heads;
  if (wgs > INT32_MAX) return set_error(SSD_ERANGE, "kv_q8_compact: cache too large");
  if (n_max == 0) return SSD_OK;
  const CompactArgs a{cache->k, cache->v, cache->k_exp, cache->v_exp, cache->n_seq, cache->kv_heads, n_max,
                      cache->max_len, start, src, n};
  by_head_dim(cache->head_dim, [&](auto c) {
    SSD_LAUNCH((kv_q8_compact_kernel<decltype(c)::value>), dim3((unsigned)wgs), dim3(256), 0, stream, a);
  });
  return check_launch("kv_q8_compact");
}
