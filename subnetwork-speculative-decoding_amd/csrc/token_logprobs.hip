// Log probabilities of given tokens, the rows' entropy, the tokens' rank and the most likely alternatives, in one pass over the logits.
//
// With m = max x, z = sum e^(x - m) and t = sum e^(x - m) (x - m): log p(c) = x_c - m - ln z, entropy = ln z - t / z. A thread keeps
// (m, z, t) of the columns it has seen and rescales them when its maximum grows; threads, then chunks of a row, are added with
// weights from their largest m.
// The k alternatives: the maxima of 64 groups of threads are values of the row, so its k-th largest value is at least the k-th
// largest of them; only the few threads whose maximum reaches that bound look at their columns again (from registers, or a wave
// together), what reaches it is collected, and a value's place is the number of those above it. Equal values rank by column, lowest
// first. More candidates than the list holds (rows of equal logits) take a pass over the chunk for each place.
// What bounds it: bytes and the vector pipe (about 14 operations a column): 1800 rows of 50257 fp32 columns 68 us, 5.3 TB/s; 1400
// of 128256 bf16 columns 77 without alternatives, 4.7 TB/s, and 87 with 5. For few rows the latency of two launches and their
// steps: 25 rows of 128256 bf16 columns 6.7 us without alternatives, 13.3 with 5.
#include "topk.h"

#include <algorithm>
#include <type_traits>

namespace ssd {

constexpr int LP_TOP = 32;       // alternatives
constexpr int LP_LIST = 1024;    // collected candidates
constexpr int LP_CHUNKS = 64;    // chunks of a row
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;

struct LogprobArgs {
  const void* x;
  int64_t ld;
  int M, V, chunks, vecs;  // vecs: 16-byte vectors of a chunk
  const void* tok;
  int tok64, top;
  char* ws;  // [row][chunk] records
  float *logprob, *entropy;
  int* rank;
  int* top_ids;
  float* top_lp;
};

struct LpSum {
  float m, z, t;  // t in log2 units
};

// A record of a chunk: its sums, the number of its columns that rank before the token, the token's logit, then `top` keys, best first (0: no more columns).
struct LpRecord {
  LpSum sum;
  int ahead;
  float xt, unused[3];  // the token's logit
};
__host__ __device__ inline int64_t lp_record_bytes(int top) { return (int64_t)sizeof(LpRecord) + 8 * top; }

// The larger, NaN if either is.
__device__ __forceinline__ float lp_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ LpSum lp_rescale(const LpSum& a, float m) {  // m >= a.m, or NaN
  if (a.m == -INFINITY) return LpSum{m, 0.f, 0.f};
  const float d = (a.m - m) * LP_LOG2E, w = __builtin_amdgcn_exp2f(d);
  return LpSum{m, a.z * w, a.m == m ? a.t : w == 0.f ? 0.f : w * fmaf(a.z, d, a.t)};
}
__device__ __forceinline__ LpSum lp_add(const LpSum& a, const LpSum& b) {
  const float m = lp_max(a.m, b.m);
  const LpSum x = lp_rescale(a, m), y = lp_rescale(b, m);
  return LpSum{m, x.z + y.z, x.t + y.t};
}

// f over a wave's lanes, the same on all: DPP exchanges within 16 lanes, then the swaps across them.
template <typename F>
__device__ __forceinline__ uint32_t lp_wave(uint32_t v, F f) {
  v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));   // lane ^ 1
  v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));   // lane ^ 2
  v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true));  // the other half of 8
  v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true));  // the other half of 16
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = f(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return f(r[0], r[1]);
}
__device__ __forceinline__ float lp_wave_sum(float v) {
  return __uint_as_float(lp_wave(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
__device__ __forceinline__ int lp_wave_sum(int v) {
  return (int)lp_wave((uint32_t)v, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ LpSum lp_wave_add(const LpSum& s) {
  const float m = __uint_as_float(
      lp_wave(__float_as_uint(s.m), [](uint32_t a, uint32_t b) { return __float_as_uint(lp_max(__uint_as_float(a), __uint_as_float(b))); }));
  const LpSum x = lp_rescale(s, m);
  return LpSum{m, lp_wave_sum(x.z), lp_wave_sum(x.t)};
}

template <typename T, int E>
__device__ __forceinline__ void lp_unpack(const uint4& u, float (&x)[E]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
    else if constexpr (std::is_same<T, _Float16>::value) x[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i / 2] >> (16 * (i & 1))));
    else x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
}
template <typename T>
__device__ __forceinline__ float lp_one(const T* p) {
  if constexpr (sizeof(T) == 4 || std::is_same<T, _Float16>::value) return (float)*p;
  else return bf2f(*p);
}

// A row's columns: `head` ones before the first 16-byte boundary, whole vectors, `tail` ones behind them. Chunk 0 takes head and
// tail, one column a thread.
template <typename T>
struct LpRow {
  static constexpr int E = 16 / sizeof(T);
  const T* p;
  int head, vecs, extra;
  __device__ __forceinline__ LpRow(const LogprobArgs& a, int row) {
    p = (const T*)a.x + row * a.ld;
    head = min((int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T), a.V);
    vecs = (a.V - head) / E;
    extra = a.V - vecs * E;
  }
  __device__ __forceinline__ int column(int v) const { return head + v * E; }
  __device__ __forceinline__ int extra_column(int i) const { return i < head ? i : i + vecs * E; }
  __device__ __forceinline__ uint4 load(int v) const { return *(const uint4*)(p + column(v)); }
};

__device__ __forceinline__ int lp_token(const LogprobArgs& a, int row) {
  const int64_t t = a.tok64 ? ((const int64_t*)a.tok)[row] : ((const int*)a.tok)[row];
  return t >= 0 && t < a.V ? (int)t : -1;
}

// Places of the n keys in list (all different, none 0): the k largest into best, in order.
__device__ __forceinline__ void lp_places(const uint64_t* list, int n, int k, uint64_t* best) {
  for (int i = threadIdx.x; i < n; i += 256) {
    const uint64_t mine = list[i];
    int above = 0;
#pragma unroll 4
    for (int q = 0; q < n; ++q) above += list[q] > mine;
    if (above < k) best[above] = mine;
  }
}

// Results of a row, by thread 0 and the first `top` threads.
__device__ __forceinline__ void lp_write(const LogprobArgs& a, int row, const LpSum& s, int ahead, float xt, int tok, const uint64_t* best) {
  const float lnz = logf(s.z);
  const bool nan = s.m != s.m;
  if (threadIdx.x == 0) {
    a.logprob[row] = tok < 0 ? 0.f : nan ? s.m : (xt - s.m) - lnz;
    a.entropy[row] = nan ? s.m : lnz - LP_LN2 * (s.t / s.z);
    a.rank[row] = tok < 0 || nan ? -1 : ahead;
  }
  if ((int)threadIdx.x < a.top) {
    const uint64_t key = best[threadIdx.x];
    a.top_ids[(int64_t)row * a.top + threadIdx.x] = key_col(key);
    a.top_lp[(int64_t)row * a.top + threadIdx.x] = nan ? s.m : (key_value(key) - s.m) - lnz;
  }
}

struct LpShared {
  LpSum part[4];
  int ahead[4];
  alignas(16) float group[64];
  uint64_t best[LP_TOP], wave[4];
  int n;
  uint64_t list[LP_LIST];
};

template <typename T, bool TOP>
__global__ __launch_bounds__(256) void lp_chunk_kernel(LogprobArgs a) {
  constexpr int E = 16 / sizeof(T), U = 32 / E;  // 32 columns a thread at a time
  __shared__ LpShared sh;
  const int row = blockIdx.x / a.chunks, ch = blockIdx.x % a.chunks, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const LpRow<T> r(a, row);
  const int v0 = ch * a.vecs, v1 = min(v0 + a.vecs, r.vecs);
  // a batch's absent vectors are all -inf; the first batch is on its way before the token's chain of two loads
  constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, _Float16>::value ? 0xfc00fc00u : 0xff80ff80u;
  uint4 u[U];
  auto load = [&](int v) {
#pragma unroll
    for (int i = 0; i < U; ++i) u[i] = v + 256 * i < v1 ? r.load(v + 256 * i) : make_uint4(NONE, NONE, NONE, NONE);
  };
  load(v0 + tid);
  const int tok = lp_token(a, row);
  const float xt = tok >= 0 ? lp_one(r.p + tok) : 0.f;
  LpSum s{-INFINITY, 0.f, 0.f};
  int ahead = 0;
  auto fold = [&](const float (&x)[32]) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = lp_max(top, x[i]);
    const float m = lp_max(s.m, top);
    if (__any(m != s.m)) s = lp_rescale(s, m);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      // The difference first: products with log2 e are rounded by the logits' size, which lp_write's x_c - m would not take back, and
      // overflow at a type's lowest and largest values. -inf: a weight of 0, and 0 times it.
      const float y = fmaxf((x[i] - ref) * LP_LOG2E, -1e4f);
      const float e = __builtin_amdgcn_exp2f(y);
      s.z += e;
      s.t = fmaf(e, y, s.t);
    }
  };
  // Columns before the token rank before it from its value on, those behind it above its value: not (x <= the next smaller float) and
  // not (x <= it). The token's own vector counts as behind; its columns before the token are looked at one by one.
  const uint32_t xb = __float_as_uint(xt + 0.f);
  const float under = xt == -INFINITY ? __uint_as_float(0x7fc00000u) : __uint_as_float(xb == 0 ? 0x80000001u : (xb >> 31) ? xb + 1 : xb - 1);
  {
    const int tv = tok >= r.head ? (tok - r.head) / E : -1, c = r.column(tv) + tid;
    if (tv >= v0 && tv < v1 && c < tok) ahead += lp_one(r.p + c) == xt;
  }
  for (int v = v0 + tid; v < v1; v += 256 * U) {
    if (v != v0 + tid) load(v);
    float x[32];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float y[E];
      lp_unpack<T, E>(u[i], y);
#pragma unroll
      for (int e = 0; e < E; ++e) x[i * E + e] = y[e];
    }
    fold(x);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int vi = v + 256 * i;
      const float over = vi >= v1 ? INFINITY : r.column(vi) + E <= tok ? under : xt;
#pragma unroll
      for (int e = 0; e < E; ++e) ahead += !(x[i * E + e] <= over);
    }
  }
  const bool has = ch == 0 && tid < r.extra;  // one column of head or tail
  const int xcol = has ? r.extra_column(tid) : 0;
  float xone = -INFINITY;
  if (has) {
    xone = lp_one(r.p + xcol);
    s = lp_add(s, LpSum{xone, xone == -INFINITY ? 0.f : 1.f, 0.f});
    ahead += xone > xt || (xone == xt && xcol < tok);
  }
  const float own = s.m;  // the largest of this thread's columns
  s = lp_wave_add(s);
  ahead = lp_wave_sum(ahead);
  if (lane == 0) sh.part[w] = s, sh.ahead[w] = ahead;
  if (TOP) {
    float gm = lp_max(own, __shfl_xor(own, 1));
    gm = lp_max(gm, __shfl_xor(gm, 2));
    if ((lane & 3) == 0) sh.group[tid >> 2] = gm;
    if (tid == 0) sh.n = 0;
    if (tid < LP_TOP) sh.best[tid] = 0;
  }
  __syncthreads();
  s = lp_add(lp_add(sh.part[0], sh.part[1]), lp_add(sh.part[2], sh.part[3]));
  ahead = sh.ahead[0] + sh.ahead[1] + sh.ahead[2] + sh.ahead[3];
  if constexpr (TOP) {
    bool slow = s.m != s.m;  // a NaN hides its thread's other columns
    if (!slow) {
      const float mine = sh.group[lane];
      int above = 0;
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        const f32x4_t x = *(const f32x4_t*)&sh.group[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) above += x[e] > mine || (x[e] == mine && i + e < lane);
      }
      const float bound = __shfl(mine, __builtin_ctzll(__ballot(above == a.top - 1)));
      auto collect = [&](float y, int col) {
        if (y >= bound) {
          const int at = atomicAdd(&sh.n, 1);
          if (at < LP_LIST) sh.list[at] = rank_key(y + 0.f, col);  // -0 ranks as 0
        }
      };
      // the columns of a vector that reach the bound, one after the other
      auto pick = [&](const uint4& w4, int col) {
        float y[E];
        lp_unpack<T, E>(w4, y);
        uint32_t hit = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) hit |= (y[e] >= bound ? 1u : 0u) << e;
        for (; hit; hit &= hit - 1) {
          const int c = col + __builtin_ctz(hit);
          collect(lp_one(r.p + c), c);
        }
      };
      if (v1 - v0 <= 256 * U) {  // one batch, still in registers
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (v0 + tid + 256 * i < v1) pick(u[i], r.column(v0 + tid + 256 * i));
      } else {
        for (uint64_t who = __ballot(own >= bound); who; who &= who - 1) {
          const int l = __builtin_ctzll(who);
          for (int q = v0 + 64 * w + l + 256 * lane; q < v1; q += 256 * 64) pick(r.load(q), r.column(q));
        }
      }
      if (has) collect(xone, xcol);
      __syncthreads();
      slow = sh.n > LP_LIST;
      if (!slow) lp_places(sh.list, sh.n, a.top, sh.best);
    }
    if (slow) {  // a pass over the chunk for every place
      uint64_t below = ~0ull;
      for (int k = 0; k < a.top; ++k) {
        uint64_t most = 0;
        auto look = [&](float y, int col) {
          const uint64_t key = rank_key(y + 0.f, col);
          if (key < below && key > most) most = key;
        };
        for (int c = r.column(v0) + tid; c < r.column(v1); c += 256) look(lp_one(r.p + c), c);
        if (has) look(xone, xcol);
        most = wave_max_u64(most);
        __syncthreads();
        if (lane == 0) sh.wave[w] = most;
        __syncthreads();
        below = max(max(sh.wave[0], sh.wave[1]), max(sh.wave[2], sh.wave[3]));
        if (tid == 0) sh.best[k] = below;
        if (below == 0) break;  // no more columns
      }
    }
    __syncthreads();
  }
  if (a.chunks == 1) {
    lp_write(a, row, s, ahead, xt, tok, sh.best);
    return;
  }
  char* rec = a.ws + (int64_t)blockIdx.x * lp_record_bytes(a.top);
  if (tid == 0) *(LpRecord*)rec = LpRecord{s, ahead, xt, {}};
  if (TOP && tid < a.top) ((uint64_t*)(rec + sizeof(LpRecord)))[tid] = sh.best[tid];
}

// Adds up a row's chunks; their keys' places are found among those that reach the k-th best of the chunks' first ones.
__global__ __launch_bounds__(256) void lp_merge_kernel(LogprobArgs a) {
  __shared__ uint64_t all[LP_CHUNKS * LP_TOP], list[LP_CHUNKS * LP_TOP], best[LP_TOP];
  __shared__ int n;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, keys = a.chunks * a.top;
  const int64_t size = lp_record_bytes(a.top);
  const char* rec = a.ws + (int64_t)row * a.chunks * size;
  const int tok = lp_token(a, row);
  for (int i = tid; i < keys; i += 256) all[i] = ((const uint64_t*)(rec + i / a.top * size + sizeof(LpRecord)))[i % a.top];
  const LpRecord x = *(const LpRecord*)(rec + min(lane, a.chunks - 1) * size);
  const LpSum s = lp_wave_add(lane < a.chunks ? x.sum : LpSum{-INFINITY, 0.f, 0.f});
  const int ahead = lp_wave_sum(lane < a.chunks ? x.ahead : 0);
  if (a.top) {
    if (tid == 0) n = 0;
    if (tid < LP_TOP) best[tid] = 0;
    __syncthreads();
    // the chunks' first keys, as many of each as make `top` or more; 0 for no column
    const int firsts = a.chunks * ((a.top + a.chunks - 1) / a.chunks);  // fewer than 64, or a.chunks
    const uint64_t mine = lane < firsts ? all[lane % a.chunks * a.top + lane / a.chunks] : 0;
    int above = 0;
    for (int i = 0; i < firsts; ++i) {
      const uint64_t y = (uint64_t)__builtin_amdgcn_readlane((uint32_t)(mine >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)mine, i);
      above += y > mine || (y == mine && i < lane);
    }
    const int l = __builtin_ctzll(__ballot(above == a.top - 1));
    const uint64_t bound = max((uint64_t)1, (uint64_t)__builtin_amdgcn_readlane((uint32_t)(mine >> 32), l) << 32 |
                                                (uint32_t)__builtin_amdgcn_readlane((uint32_t)mine, l));
    for (int i = tid; i < keys; i += 256)
      if (all[i] >= bound) list[atomicAdd(&n, 1)] = all[i];
    __syncthreads();
    lp_places(list, n, a.top, best);
    __syncthreads();
  }
  lp_write(a, row, s, ahead, x.xt, tok, best);
}

// Chunks of a row. A workgroup takes about 6 us and 0.7 to 1.1 for each batch of 32 columns a thread (whatever their type), the second
// launch 4 to 6, so short rows, and those of many rows, are one chunk; else as many as bring 1024 workgroups, or of one batch each where
// those are at most 1.4 times as many (us as many / one batch each: 64 rows of 200000 fp32 columns 23 / 26, of 128256 in 13 chunks 21.5 / 18.7,
// 300 of 65000 30 / 33). us with 5 alternatives, 1 / 4 / 16 chunks: 128256 bf16 columns, 1 row 22 / 15 / 12, 64 27 / 18 / 17, 300
// 37 / 34 / 50, 399 39 / 41 / 63; fp32 25 / 15 / 12, 30 / 20 / 19, 42 / 44 / 54, 48 / 54 / 68. 50257 columns, 1 / 7 chunks: 25 rows
// bf16 15 / 12, fp32 16 / 12, 64 15 / 13, 17 / 15, 150 17 / 21, 19 / 22, 300 21 / 29, 23 / 30; 32000 columns, 1 / 4: 25 rows 12 / 12, 12.5 / 12.3.
constexpr int LP_BATCH = 256 * 32;
static int lp_chunks(int M, int V) {
  const int64_t batches = (V + LP_BATCH - 1) / LP_BATCH;
  if (M >= 400 || batches < (M > 100 ? 8 : 6)) return 1;
  const int64_t want = (1024 + M - 1) / std::max(M, 1);
  return (int)std::min<int64_t>(7 * want >= 5 * batches ? batches : want, LP_CHUNKS);
}

}  // namespace ssd

using namespace ssd;

SSD_API int64_t ssd_token_logprobs_ws_bytes(int M, int V, int dtype, int top) {
  if (M < 0 || V < 1 || V > 1 << 24 || dtype < 0 || dtype > 2 || top < 0 || top > LP_TOP) return -1;
  const int chunks = lp_chunks(M, V);
  return chunks == 1 ? 0 : (int64_t)M * chunks * lp_record_bytes(top);
}

SSD_API int ssd_token_logprobs(const void* logits, int dtype, int64_t ld, int M, int V, const void* tokens, int tokens64, int top, void* ws,
                               int64_t ws_bytes, float* logprobs, float* entropy, int32_t* rank, int32_t* top_ids,
                               float* top_logprobs, hipStream_t stream) {
  if (M < 0 || V < 1) return set_error(SSD_EINVAL, "token_logprobs: bad M=%d V=%d", M, V);
  if (V > 1 << 24) return set_error(SSD_ERANGE, "token_logprobs: %d columns > 2^24", V);
  if (dtype < 0 || dtype > 2) return set_error(SSD_EINVAL, "token_logprobs: dtype %d (0 bf16, 1 fp16, 2 fp32)", dtype);
  if (top < 0 || top > V) return set_error(SSD_EINVAL, "token_logprobs: %d alternatives of %d columns", top, V);
  if (top > LP_TOP) return set_error(SSD_ERANGE, "token_logprobs: %d alternatives > %d", top, LP_TOP);
  if (M == 0) return SSD_OK;
  if (!logits || !tokens || !logprobs || !entropy || !rank || (top && (!top_ids || !top_logprobs)))
    return set_error(SSD_EINVAL, "token_logprobs: null pointer");
  const int elem = dtype == 2 ? 4 : 2;
  if (ld < V && M > 1) return set_error(SSD_EINVAL, "token_logprobs: row stride %lld < V", (long long)ld);
  if ((uintptr_t)logits % elem) return set_error(SSD_EINVAL, "token_logprobs: logits not aligned to their type");
  LogprobArgs a{};
  a.x = logits, a.ld = ld, a.M = M, a.V = V, a.chunks = lp_chunks(M, V);
  a.vecs = (int)((((int64_t)V * elem + 15) / 16 + a.chunks - 1) / a.chunks);
  a.tok = tokens, a.tok64 = (tokens64 ? 1 : 0), a.top = top, a.ws = (char*)ws;
  a.logprob = logprobs, a.entropy = entropy, a.rank = rank, a.top_ids = top_ids, a.top_lp = top_logprobs;
  const int64_t need = ssd_token_logprobs_ws_bytes(M, V, dtype, top);
  if (need && (!ws || ((uintptr_t)ws & 15) || ws_bytes < need))
    return set_error(SSD_EINVAL, "token_logprobs: workspace too small or not 16-byte aligned");
  if ((int64_t)M * a.chunks * 256 > (int64_t)UINT32_MAX) return set_error(SSD_ERANGE, "token_logprobs: too many rows");
  const dim3 grid((unsigned)(M * a.chunks)), block(256);
#define LP_LAUNCH(T)                                                             \
  if (top) SSD_LAUNCH((lp_chunk_kernel<T, true>), grid, block, 0, stream, a);    \
  else SSD_LAUNCH((lp_chunk_kernel<T, false>), grid, block, 0, stream, a)
  if (dtype == 0) { LP_LAUNCH(uint16_t); }
  else if (dtype == 1) { LP_LAUNCH(_Float16); }
  else { LP_LAUNCH(float); }
#undef LP_LAUNCH
  if (int rc = check_launch("token_logprobs")) return rc;
  if (a.chunks == 1) return SSD_OK;
  SSD_LAUNCH(lp_merge_kernel, dim3((unsigned)M), dim3(256), 0, stream, a);
  return check_launch("token_logprobs_merge");
}
