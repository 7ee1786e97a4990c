// Verification of drafted chains from given random numbers, a batch of sequences in two launches.
//
// chain_sum: workgroup (sequence, chunk of 4096 columns). Every workgroup of a sequence resolves the acceptance
// tests itself (one wave, one gather per drafted token), which tells it the row to draw from, and adds up its
// chunk's mass of max(P_n - Q_n, 0) and of P_n in 64 bits. chain_draw: one workgroup per sequence finds the
// chunk that holds u_next * total, then the column in it.
// What bounds it: two rows of V fp32 a sequence.
#include "common.h"

namespace ssd {

constexpr int CHAIN_CHUNK = 4096, CHAIN_MAX = 64;

struct ChainArgs {
  const float *P, *Q;
  int64_t ldp_seq, ldp, ldq_seq, ldq;
  int V, k_max, chunks;
  const int *draft, *n_draft;
  const float *u, *u_next;
  double* ws;  // [n_seq][chunks] pairs: residual mass, target mass
  int *out_tok, *out_n;
};

// Number of accepted tokens of sequence s, by one whole wave: lane i tests token i, the first refusal ends
// the chain. u * q has at most 48 significant bits, so the test is exact in doubles.
__device__ __forceinline__ int chain_accepted(const ChainArgs& a, int s, int lane, int& todo) {
  todo = a.n_draft ? min(max(a.n_draft[s], 0), a.k_max) : a.k_max;
  bool ok = false;
  if (lane < todo) {
    const int x = a.draft[(size_t)s * a.k_max + lane];
    if (x >= 0 && x < a.V) {
      const float p = a.P[s * a.ldp_seq + lane * a.ldp + x], q = a.Q[s * a.ldq_seq + lane * a.ldq + x];
      ok = (double)a.u[(size_t)s * a.k_max + lane] * (double)q < (double)p;
    }
  }
  const uint64_t refused = ~__ballot(ok);
  return refused ? __builtin_ctzll(refused) : CHAIN_MAX;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Columns c .. c + 4 of row x (fewer at the row's end; absent ones are 0).
__device__ __forceinline__ float4 load4(const float* x, int c, int V, bool wide) {
  if (wide && c + 4 <= V) return *(const float4*)(x + c);
  float4 r;
  r.x = c < V ? x[c] : 0.f;
  r.y = c + 1 < V ? x[c + 1] : 0.f;
  r.z = c + 2 < V ? x[c + 2] : 0.f;
  r.w = c + 3 < V ? x[c + 3] : 0.f;
  return r;
}

__device__ __forceinline__ double residual(float p, float q) {
  const double d = (double)p - (double)q;
  return d > 0. ? d : 0.;
}

__global__ __launch_bounds__(256) void chain_sum_kernel(ChainArgs a) {
  const int s = blockIdx.x / a.chunks, ch = blockIdx.x % a.chunks, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int todo;
  const int n = chain_accepted(a, s, lane, todo);  // every wave: no barrier before the rows' loads
  const float* p = a.P + s * a.ldp_seq + n * a.ldp;
  const float* q = n < todo ? a.Q + s * a.ldq_seq + n * a.ldq : nullptr;
  const bool wp = !((uintptr_t)p & 15), wq = !((uintptr_t)q & 15);
  double rs = 0., ps = 0.;
#pragma unroll
  for (int it = 0; it < CHAIN_CHUNK / 1024; ++it) {
    const int c = ch * CHAIN_CHUNK + it * 1024 + threadIdx.x * 4;
    const float4 x = load4(p, c, a.V, wp);
    const float4 y = q ? load4(q, c, a.V, wq) : make_float4(0.f, 0.f, 0.f, 0.f);
    rs += residual(x.x, y.x) + residual(x.y, y.y) + residual(x.z, y.z) + residual(x.w, y.w);
    ps += residual(x.x, 0.f) + residual(x.y, 0.f) + residual(x.z, 0.f) + residual(x.w, 0.f);
  }
  __shared__ double part[4][2];
  rs = wave_sum(rs), ps = wave_sum(ps);
  if (lane == 0) part[w][0] = rs, part[w][1] = ps;
  __syncthreads();
  if (threadIdx.x < 2)
    a.ws[((size_t)s * a.chunks + ch) * 2 + threadIdx.x] =
        part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
}

// Exclusive prefix of v over the workgroup's 256 threads, and the total.
__device__ __forceinline__ double block_prefix(double v, double* s_w, double& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  double inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double t = __shfl_up(inc, o);
    if (lane >= o) inc += t;
  }
  __syncthreads();  // s_w may still be read from an earlier call
  if (lane == 63) s_w[w] = inc;
  __syncthreads();
  double base = 0.;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < w) base += s_w[i];
  total = s_w[0] + s_w[1] + s_w[2] + s_w[3];
  return base + inc - v;
}

__global__ __launch_bounds__(256) void chain_draw_kernel(ChainArgs a) {
  const int s = blockIdx.x, lane = threadIdx.x & 63;
  __shared__ double s_w[4];
  __shared__ int s_best, s_last;
  int todo;
  const int n = chain_accepted(a, s, lane, todo);
  const double* ws = a.ws + (size_t)s * a.chunks * 2;
  // total residual mass; without any, draw from the target row
  double rs = 0., ps = 0.;
  for (int c = threadIdx.x; c < a.chunks; c += 256) rs += ws[2 * c], ps += ws[2 * c + 1];
  double rt, pt;
  block_prefix(rs, s_w, rt);
  block_prefix(ps, s_w, pt);
  const bool res = rt > 0.;
  const double total = res ? rt : pt, want = (double)a.u_next[s] * total;
  // the chunk: the first whose end passes `want`, else the last with mass
  if (threadIdx.x == 0) s_best = INT32_MAX, s_last = -1;
  double base = 0., before = 0.;  // mass before this window of 256 chunks; before the chosen chunk
  int chunk = -1;
  double chunk_before = 0.;
  for (int c0 = 0; c0 < a.chunks; c0 += 256) {
    const int c = c0 + threadIdx.x;
    const double m = c < a.chunks ? ws[2 * c + (res ? 0 : 1)] : 0.;
    double tot;
    before = base + block_prefix(m, s_w, tot);
    if (m > 0.) {
      atomicMax(&s_last, c);
      if (before + m > want) atomicMin(&s_best, c);
    }
    __syncthreads();
    const int pick = s_best != INT32_MAX ? s_best : s_last;
    if (c == pick) chunk_before = before, chunk = c;
    base += tot;
    __syncthreads();
  }
  __shared__ double s_before;
  __shared__ int s_chunk;
  const int pick = s_best != INT32_MAX ? s_best : s_last;
  if (threadIdx.x == 0) s_chunk = pick;
  if (chunk == pick && chunk >= 0) s_before = chunk_before;
  __syncthreads();
  int tok = -1;
  if (s_chunk >= 0) {
    const float* p = a.P + s * a.ldp_seq + n * a.ldp;
    const float* q = res && n < todo ? a.Q + s * a.ldq_seq + n * a.ldq : nullptr;
    const int c0 = s_chunk * CHAIN_CHUNK + threadIdx.x * 16;
    double m[16], sum = 0.;
    const bool wp = !((uintptr_t)p & 15), wq = !((uintptr_t)q & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 x = load4(p, c0 + 4 * i, a.V, wp);
      const float4 y = q ? load4(q, c0 + 4 * i, a.V, wq) : make_float4(0.f, 0.f, 0.f, 0.f);
      m[4 * i] = residual(x.x, y.x), m[4 * i + 1] = residual(x.y, y.y);
      m[4 * i + 2] = residual(x.z, y.z), m[4 * i + 3] = residual(x.w, y.w);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += m[i];
    double tot;
    double cum = s_before + block_prefix(sum, s_w, tot);
    if (threadIdx.x == 0) s_best = INT32_MAX, s_last = -1;
    __syncthreads();
    int first = INT32_MAX, last = -1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      cum += m[i];
      if (m[i] > 0.) {
        last = c0 + i;
        if (cum > want && first == INT32_MAX) first = c0 + i;
      }
    }
    if (first != INT32_MAX) atomicMin(&s_best, first);
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    tok = s_best != INT32_MAX ? s_best : s_last;
  }
  int* out = a.out_tok + (size_t)s * (a.k_max + 1);
  for (int i = threadIdx.x; i <= a.k_max; i += 256) out[i] = i < n ? a.draft[(size_t)s * a.k_max + i] : i == n ? tok : -1;
  if (threadIdx.x == 0) a.out_n[s] = n;
}

}  // namespace ssd

using namespace ssd;

SSD_API int64_t ssd_verify_chain_ws_bytes(int n_seq, int V) {
  if (n_seq < 0 || V < 1) return -1;
  return (int64_t)n_seq * ((V + CHAIN_CHUNK - 1) / CHAIN_CHUNK) * 2 * (int64_t)sizeof(double);
}

SSD_API int ssd_verify_chain(const float* P, int64_t ldp_seq, int64_t ldp, const float* Q, int64_t ldq_seq, int64_t ldq, int V,
                             int n_seq, int k_max, const int32_t* draft, const int32_t* n_draft, const float* u,
                             const float* u_next, void* ws, int64_t ws_bytes, int32_t* out_tok, int32_t* out_n,
                             hipStream_t stream) {
  if (n_seq < 0 || k_max < 0 || V < 1) return set_error(SSD_EINVAL, "verify_chain: bad n_seq=%d k_max=%d V=%d", n_seq, k_max, V);
  if (k_max > CHAIN_MAX) return set_error(SSD_ERANGE, "verify_chain: %d drafted tokens > %d", k_max, CHAIN_MAX);
  if (V > 1 << 24) return set_error(SSD_ERANGE, "verify_chain: %d columns > 2^24", V);
  if (!P || !u_next || !ws || !out_tok || !out_n || (k_max && (!Q || !draft || !u)))
    return set_error(SSD_EINVAL, "verify_chain: null pointer");
  if (ldp < V || (k_max && ldq < V)) return set_error(SSD_EINVAL, "verify_chain: row strides below V");
  if ((uintptr_t)ws & 7) return set_error(SSD_EINVAL, "verify_chain: workspace must be 8-byte aligned");
  if (ws_bytes < ssd_verify_chain_ws_bytes(n_seq, V)) return set_error(SSD_EINVAL, "verify_chain: workspace too small");
  const int chunks = (V + CHAIN_CHUNK - 1) / CHAIN_CHUNK;
  if ((int64_t)n_seq * chunks > INT32_MAX) return set_error(SSD_ERANGE, "verify_chain: too many sequences");
  if (n_seq == 0) return SSD_OK;
  const ChainArgs a{P, Q, ldp_seq, ldp, ldq_seq, ldq, V, k_max, chunks, draft, n_draft, u, u_next, (double*)ws, out_tok, out_n};
  SSD_LAUNCH(chain_sum_kernel, dim3((unsigned)(n_seq * chunks)), dim3(256), 0, stream, a);
  if (int rc = check_launch("chain_sum")) return rc;
  SSD_LAUNCH(chain_draw_kernel, dim3((unsigned)n_seq), dim3(256), 0, stream, a);
  return check_launch("chain_draw");
}
