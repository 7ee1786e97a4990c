// Log probabilities of given tokens, the rows' entropy, the tokens' rank and the most likely alternatives, in one pass over the logits.
//
// With m = max x, z = sum e^(x - m) and t = sum e^(x - m) (x - m): log p(c) = x_c - m - ln z, entropy = ln z - t / z. A thread keeps
// (m, z, t) of the columns it has seen and rescales them when its maximum grows; threads, then chunks of a row, are added with
// weights from their largest m.
// The k alternatives: the maxima of 64 groups of threads are values of the row, so its k-th largest value is at least the k-th
// largest of them; only the few threads whose maximum reaches that bound look at their columns again (a wave together), what
// reaches it is collected, and a value's place is the number of those above it. Equal values rank by column, lowest first.
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
  float group[64];
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
  const int tok = lp_token(a, row);
  const float xt = tok >= 0 ? lp_one(r.p + tok) : 0.f;
  LpSum s{-INFINITY, 0.f, 0.f};
  int ahead = 0;
  auto fold = [&](const float (&x)[32], int n) {  // n: of them there, whole vectors
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) top = lp_max(top, x[i]);
    const float m = lp_max(s.m, top);
    if (__any(m != s.m)) s = lp_rescale(s, m);
    const float ref = m == -INFINITY ? 0.f : m * LP_LOG2E;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) {
        const float y = fmaxf(fmaf(x[i], LP_LOG2E, -ref), -1e4f);  // -inf: a weight of 0, and 0 times it
        const float e = __builtin_amdgcn_exp2f(y);
        s.z += e;
        s.t = fmaf(e, y, s.t);
      }
  };
  auto count = [&](const float* x, int col) {  // a vector
    if (col + E <= tok) {
#pragma unroll
      for (int i = 0; i < E; ++i) ahead += x[i] >= xt;
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) ahead += x[i] > xt || (x[i] == xt && col + i < tok);
    }
  };
  int v = v0 + tid;
  for (; v + 256 * (U - 1) < v1; v += 256 * U) {
    uint4 u[U];
#pragma unroll
    for (int i = 0; i < U; ++i) u[i] = r.load(v + 256 * i);
    float x[32];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float y[E];
      lp_unpack<T, E>(u[i], y);
#pragma unroll
      for (int e = 0; e < E; ++e) x[i * E + e] = y[e];
    }
    fold(x, 32);
#pragma unroll
    for (int i = 0; i < U; ++i) count(x + i * E, r.column(v + 256 * i));
  }
  for (; v < v1; v += 256) {
    float y[E], x[32];
    lp_unpack<T, E>(r.load(v), y);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = y[e];
    fold(x, E);
    count(x, r.column(v));
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
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const LpSum q{__shfl_xor(s.m, o), __shfl_xor(s.z, o), __shfl_xor(s.t, o)};
    s = lp_add(s, q);
    ahead += __shfl_xor(ahead, o);
  }
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
      for (int i = 0; i < 64; ++i) above += sh.group[i] > mine || (sh.group[i] == mine && i < lane);
      const float bound = __shfl(mine, __builtin_ctzll(__ballot(above == a.top - 1)));
      auto collect = [&](float y, int col) {
        if (y >= bound) {
          const int at = atomicAdd(&sh.n, 1);
          if (at < LP_LIST) sh.list[at] = rank_key(y + 0.f, col);  // -0 ranks as 0
        }
      };
      for (uint64_t who = __ballot(own >= bound); who; who &= who - 1) {
        const int l = __builtin_ctzll(who);
        for (int q = v0 + 64 * w + l + 256 * lane; q < v1; q += 256 * 64) {
          float y[E];
          lp_unpack<T, E>(r.load(q), y);
#pragma unroll
          for (int e = 0; e < E; ++e) collect(y[e], r.column(q) + e);
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
        for (int q = v0 + tid; q < v1; q += 256) {
          float y[E];
          lp_unpack<T, E>(r.load(q), y);
#pragma unroll
          for (int e = 0; e < E; ++e) look(y[e], r.column(q) + e);
        }
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

// Adds up a row's chunks, in order of the lanes; their keys' places are found among those that reach the k-th best first key.
__global__ __launch_bounds__(256) void lp_merge_kernel(LogprobArgs a) {
  __shared__ uint64_t list[LP_CHUNKS * LP_TOP], first[LP_CHUNKS], best[LP_TOP];
  __shared__ int n;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int64_t size = lp_record_bytes(a.top);
  const char* rec = a.ws + (int64_t)row * a.chunks * size;
  const int tok = lp_token(a, row);
  LpSum s{-INFINITY, 0.f, 0.f};
  int ahead = 0;
  if (lane < a.chunks) {
    const LpRecord x = *(const LpRecord*)(rec + lane * size);
    s = x.sum, ahead = x.ahead;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const LpSum q{__shfl_xor(s.m, o), __shfl_xor(s.z, o), __shfl_xor(s.t, o)};
    s = lp_add(s, q);
    ahead += __shfl_xor(ahead, o);
  }
  if (a.top) {
    auto key = [&](int c, int k) { return ((const uint64_t*)(rec + c * size + sizeof(LpRecord)))[k]; };
    if (tid < a.chunks) first[tid] = key(tid, 0);
    if (tid == 0) n = 0;
    if (tid < LP_TOP) best[tid] = 0;
    __syncthreads();
    uint64_t bound = 1;
    if (a.chunks >= a.top) {
      const uint64_t mine = lane < a.chunks ? first[lane] : 0;
      int above = 0;
      for (int i = 0; i < a.chunks; ++i) above += first[i] > mine || (first[i] == mine && i < lane);
      const int l = __builtin_ctzll(__ballot(above == a.top - 1));
      bound = max(bound, (uint64_t)__shfl((uint32_t)(mine >> 32), l) << 32 | __shfl((uint32_t)mine, l));
    }
    for (int i = tid; i < a.chunks * a.top; i += 256) {
      const uint64_t x = key(i / a.top, i % a.top);
      if (x >= bound) list[atomicAdd(&n, 1)] = x;
    }
    __syncthreads();
    lp_places(list, n, a.top, best);
    __syncthreads();
  }
  lp_write(a, row, s, ahead, ((const LpRecord*)rec)->xt, tok, best);
}

// Chunks of a row: one where the rows fill the chip (four workgroups a CU and more), else as many as bring 1024 workgroups, of 1024
// vectors at least.
static int lp_chunks(int M, int V, int elem) {
  const int64_t vecs = ((int64_t)V * elem + 15) / 16;
  const int64_t want = (1024 + M - 1) / std::max(M, 1), most = (vecs + 1023) / 1024;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, LP_CHUNKS}));
}

}  // namespace ssd

using namespace ssd;

SSD_API int64_t ssd_token_logprobs_ws_bytes(int M, int V, int dtype, int top) {
  if (M < 0 || V < 1 || V > 1 << 24 || dtype < 0 || dtype > 2 || top < 0 || top > LP_TOP) return -1;
  const int chunks = lp_chunks(M, V, dtype == 2 ? 4 : 2);
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
  a.x = logits, a.ld = ld, a.M = M, a.V = V, a.chunks = lp_chunks(M, V, elem);
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
