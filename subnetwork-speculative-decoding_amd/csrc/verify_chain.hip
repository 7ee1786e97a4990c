// Verification of drafted chains from given random numbers, a batch of sequences in two launches.
//
// chain_sum: workgroup (sequence, chunk of columns; at most 64 chunks of whole 4096-column pieces a row). Each resolves
// the sequence's acceptance tests itself (a gather per drafted token, one wave), which tells it the row to draw
// from, and adds up its chunk's mass of max(P_n - Q_n, 0) and of P_n in 64 bits. chain_draw: one workgroup per sequence
// finds the chunk that holds u_next * total (a lane a chunk), then the column in it.
// What bounds it: two rows of V fp32 a sequence for a batch (48 of V = 128256: 49 MB, 10.2 us in chain_sum, 4.8 TB/s, and
// 4.8 in chain_draw), the latency of two launches for a few sequences (one: 4.2 + 3.8).
#include "common.h"

namespace ssd {

constexpr int CHAIN_PIECE = 4096, CHAIN_MAX = 64, CHAIN_CHUNKS = 64;

struct ChainArgs {
  const float *P, *Q;
  int64_t ldp_seq, ldp, ldq_seq, ldq;
  int V, k_max, chunks, pieces;  // pieces of 4096 columns in a chunk
  const int *draft, *n_draft;
  const float *u, *u_next;
  double2* ws;  // [n_seq][chunks + 1]: (residual mass, target mass) of each chunk, then (accepted, draws from the residual)
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

// Sixteen columns of a row pair from column c on: the residual's mass, or the target's where q is null.
__device__ __forceinline__ void load_mass(const float* p, const float* q, int c, int V, double (&m)[16]) {
  const bool wp = !((uintptr_t)p & 15), wq = !((uintptr_t)q & 15);
  float4 x[4], y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = load4(p, c + 4 * i, V, wp);
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = q ? load4(q, c + 4 * i, V, wq) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[4 * i] = residual(x[i].x, y[i].x), m[4 * i + 1] = residual(x[i].y, y[i].y);
    m[4 * i + 2] = residual(x[i].z, y[i].z), m[4 * i + 3] = residual(x[i].w, y[i].w);
  }
}

__global__ __launch_bounds__(256) void chain_sum_kernel(ChainArgs a) {
  const int s = blockIdx.x / a.chunks, ch = blockIdx.x % a.chunks, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int todo;
  const int n = chain_accepted(a, s, lane, todo);  // every wave: no barrier before the rows' loads
  const float* p = a.P + s * a.ldp_seq + n * a.ldp;
  const float* q = n < todo ? a.Q + s * a.ldq_seq + n * a.ldq : nullptr;
  const bool wp = !((uintptr_t)p & 15), wq = !((uintptr_t)q & 15);
  double rs = 0., ps = 0.;
  for (int pc = 0; pc < a.pieces; ++pc) {
#pragma unroll
    for (int it = 0; it < CHAIN_PIECE / 1024; ++it) {
      const int c = (ch * a.pieces + pc) * CHAIN_PIECE + it * 1024 + threadIdx.x * 4;
      const float4 x = load4(p, c, a.V, wp);
      const float4 y = q ? load4(q, c, a.V, wq) : make_float4(0.f, 0.f, 0.f, 0.f);
      rs += residual(x.x, y.x) + residual(x.y, y.y) + residual(x.z, y.z) + residual(x.w, y.w);
      ps += residual(x.x, 0.f) + residual(x.y, 0.f) + residual(x.z, 0.f) + residual(x.w, 0.f);
    }
  }
  __shared__ double part[4][2];
  rs = wave_sum(rs), ps = wave_sum(ps);
  if (lane == 0) part[w][0] = rs, part[w][1] = ps;
  __syncthreads();
  double2* out = a.ws + (size_t)s * (a.chunks + 1);
  if (threadIdx.x == 0)
    out[ch] = make_double2(part[0][0] + part[1][0] + part[2][0] + part[3][0], part[0][1] + part[1][1] + part[2][1] + part[3][1]);
  if (threadIdx.x == 64 && ch == 0) out[a.chunks] = make_double2(n, q ? 1. : 0.);
}

__device__ __forceinline__ double wave_scan(double v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double t = __shfl_up(v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// The least element whose cumulative mass exceeds `want`, else the last that has any; -1: none has.
__device__ __forceinline__ int pick(uint64_t past, uint64_t any) {
  return past ? __builtin_ctzll(past) : any ? 63 - __builtin_clzll(any) : -1;
}

__global__ __launch_bounds__(256) void chain_draw_kernel(ChainArgs a) {
  const int s = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const double2* ws = a.ws + (size_t)s * (a.chunks + 1);
  const double2 own = lane < a.chunks ? ws[lane] : make_double2(0., 0.), head = ws[a.chunks];
  const float u = a.u_next[s];
  const int n = (int)head.x;
  // every wave finds the chunk: the residual's mass, or the target's without any
  const double rc = wave_scan(own.x, lane), pc = wave_scan(own.y, lane);
  const bool res = head.y != 0. && __shfl(rc, 63) > 0.;
  const double m = res ? own.x : own.y, cum = res ? rc : pc, want = (double)u * __shfl(cum, 63);
  const int ch = pick(__ballot(m > 0. && cum > want), __ballot(m > 0.));
  const float* p = a.P + s * a.ldp_seq + n * a.ldp;
  const float* q = res ? a.Q + s * a.ldq_seq + n * a.ldq : nullptr;
  double base = __shfl(cum, max(ch - 1, 0));
  if (ch <= 0) base = 0.;
  __shared__ double sum[4];
  __shared__ int first[4], last[4];
  int tok = -1;
  for (int pc2 = 0; ch >= 0 && pc2 < a.pieces; ++pc2) {  // uniform
    const int c0 = (ch * a.pieces + pc2) * CHAIN_PIECE + threadIdx.x * 16;
    double x[16], mine = 0.;
    load_mass(p, q, c0, a.V, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) mine += x[i];
    const double inc = wave_scan(mine, lane);
    __syncthreads();  // the piece before has been read
    if (lane == 63) sum[w] = inc;
    __syncthreads();
    double at = base;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < w) at += sum[i];
      base += sum[i];
    }
    const double below = __shfl_up(inc, 1);
    at += lane ? below : 0.;
    int f = -1, l = -1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      at += x[i];
      if (x[i] > 0.) {
        l = c0 + i;
        if (at > want && f < 0) f = c0 + i;
      }
    }
    const uint64_t past = __ballot(f >= 0), any = __ballot(l >= 0);
    const int fw = __shfl(f, past ? __builtin_ctzll(past) : 0), lw = __shfl(l, any ? 63 - __builtin_clzll(any) : 0);
    if (lane == 0) first[w] = past ? fw : -1, last[w] = any ? lw : -1;
    __syncthreads();
    int found = -1;
#pragma unroll
    for (int i = 3; i >= 0; --i) found = first[i] >= 0 ? first[i] : found;
#pragma unroll
    for (int i = 0; i < 4; ++i) tok = last[i] >= 0 ? last[i] : tok;
    if (found >= 0) {
      tok = found;
      break;
    }
  }
  int* out = a.out_tok + (size_t)s * (a.k_max + 1);
  if ((int)threadIdx.x <= a.k_max) {
    const int i = threadIdx.x;
    out[i] = i < n ? a.draft[(size_t)s * a.k_max + i] : i == n ? tok : -1;
  }
  if (threadIdx.x == 0) a.out_n[s] = n;
}

// Pieces a chunk so that a row has at most 64 chunks.
static int chain_pieces(int V) { return (V + CHAIN_PIECE * CHAIN_CHUNKS - 1) / (CHAIN_PIECE * CHAIN_CHUNKS); }
static int chain_chunks(int V) {
  const int w = CHAIN_PIECE * chain_pieces(V);
  return (V + w - 1) / w;
}

}  // namespace ssd

using namespace ssd;

SSD_API int64_t ssd_verify_chain_ws_bytes(int n_seq, int V) {
  if (n_seq < 0 || V < 1 || V > 1 << 24) return -1;
  return (int64_t)n_seq * (chain_chunks(V) + 1) * (int64_t)sizeof(double2);
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
  if ((uintptr_t)ws & 15) return set_error(SSD_EINVAL, "verify_chain: workspace must be 16-byte aligned");
  if (ws_bytes < ssd_verify_chain_ws_bytes(n_seq, V)) return set_error(SSD_EINVAL, "verify_chain: workspace too small");
  const int chunks = chain_chunks(V);
  if ((int64_t)n_seq * chunks * 256 > (int64_t)UINT32_MAX) return set_error(SSD_ERANGE, "verify_chain: too many sequences");
  if (n_seq == 0) return SSD_OK;
  const ChainArgs a{P, Q, ldp_seq, ldp, ldq_seq, ldq, V, k_max, chunks, chain_pieces(V), draft, n_draft, u, u_next, (double2*)ws,
                    out_tok, out_n};
  SSD_LAUNCH(chain_sum_kernel, dim3((unsigned)(n_seq * chunks)), dim3(256), 0, stream, a);
  if (int rc = check_launch("chain_sum")) return rc;
  SSD_LAUNCH(chain_draw_kernel, dim3((unsigned)n_seq), dim3(256), 0, stream, a);
  return check_launch("chain_draw");
}
