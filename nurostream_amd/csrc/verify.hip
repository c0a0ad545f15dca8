// Verification of drafted tokens against the target model's logits (gfx950).
//
// A sequence has n nodes: node 0 is its last known token, every other node a drafted token under its parent. Row i of
// the logits is the target's distribution behind node i, p_i = softmax(logits_i / temperature). The walk starts at node
// 0 and tries the current node's children in order, x a child's token and u its random number in [0, 1):
//   drafts without probabilities: accepted when u * left < p(x), left being what p's refused children leave of 1 (a
//     token refused here before has nothing left); after the last refusal the following token is drawn from p without
//     the refused tokens;
//   drafts drawn from q (a chain): accepted when u * q(x) < p(x); after a refusal the following token is drawn from
//     max(p - q, 0).
// Either way the tokens are distributed as if each had been drawn from p. A draw takes the first token, in index order,
// at which the running sum of the weights exceeds node 0's random number times their total. Temperature 0: p is one
// at the largest logit, the lowest index of equals.
//
// Exponentials, sums and comparisons in 64 bits: a vocabulary's running sum is compared with a random number. A NaN
// logit counts as -infinity; of +infinity in a row, its tokens share the row's whole weight; a row without any weight
// gives the token -1. Sequences with no nodes (length 0) give count 0 and token -1.
#include "nsx_common.h"

#include <algorithm>
#include <math.h>

namespace {

constexpr int VF_CHUNK = 4096;  // logits per workgroup of the row passes
constexpr int VF_THREADS = 256;
constexpr int VF_PER = VF_CHUNK / VF_THREADS;
constexpr int VF_MAX_CHUNKS = 1024;  // chunks of a row that one workgroup's threads hold four each

// A chunk's largest logit, its (lowest) index and the weights' sum relative to it.
struct Part {
  float m;
  int32_t at;
  double s;
};

struct VerifyArgs {
  const void* logits;
  int dtype;
  int64_t row_stride;  // elements
  int B, n;
  int64_t V;
  const int32_t *tokens, *parents, *lengths;
  int64_t parents_stride;  // 0: one tree for all sequences
  const float *u, *q;
  double inv_temp;  // 0: greedy
  int32_t *count, *path, *token;
  int nchunk;
  Part* part;      // [B * n][nchunk]
  double* resid;   // q: [B][nchunk], the sums of max(p - q, 0) at the last node
  int32_t* state;  // q: [B], the last node reached where a child was refused there, else -1
};

__device__ __forceinline__ float vf_logit(const VerifyArgs& a, int64_t row, int64_t i) {
  const float x = nsx_load_act(a.logits, a.dtype, row * a.row_stride + i);
  return x == x ? x : -INFINITY;
}

// The weight of logit x beside the largest, M > -infinity.
__device__ __forceinline__ double vf_weight(float x, float M, double inv_temp) {
  return x == M ? 1.0 : exp(((double)x - (double)M) * inv_temp);  // (equals first: their difference may be of infinities)
}

template <typename T, typename Op>
__device__ __forceinline__ T vf_block_reduce(T v, T* red, Op op) {  // over 256 threads, the same order in each
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return op(op(red[0], red[1]), op(red[2], red[3]));
}

// Elements of chunk c of a row: element c * VF_CHUNK + 256 u + thread.
__global__ __launch_bounds__(VF_THREADS) void verify_stats_kernel(VerifyArgs a) {
  __shared__ float redf[4];
  __shared__ int redi[4];
  __shared__ double redd[4];
  const int64_t row = blockIdx.y;
  const int c = blockIdx.x;
  const int64_t i0 = (int64_t)c * VF_CHUNK;
  float x[VF_PER], m = -INFINITY;
#pragma unroll
  for (int u = 0; u < VF_PER; ++u) {
    const int64_t i = i0 + VF_THREADS * u + threadIdx.x;
    x[u] = i < a.V ? vf_logit(a, row, i) : -INFINITY;
    m = fmaxf(m, x[u]);
  }
  m = vf_block_reduce(m, redf, [](float p, float q) { return fmaxf(p, q); });
  int at = 0x7fffffff;
  double s = 0.0;
#pragma unroll
  for (int u = VF_PER - 1; u >= 0; --u) {
    const int64_t i = i0 + VF_THREADS * u + threadIdx.x;
    if (x[u] == m && i < a.V) at = (int)i;
    if (a.inv_temp != 0.0 && m > -INFINITY) s += vf_weight(x[u], m, a.inv_temp);
  }
  at = vf_block_reduce(at, redi, [](int p, int q) { return min(p, q); });
  s = vf_block_reduce(s, redd, [](double p, double q) { return p + q; });
  if (threadIdx.x == 0) a.part[row * a.nchunk + c] = Part{m, at, s};
}

// The row's largest logit, its index and the weights' sum, from its chunks: one wave.
__device__ __forceinline__ Part vf_row(const VerifyArgs& a, int64_t row, int lane) {
  const Part* p = a.part + row * a.nchunk;
  float M = -INFINITY;
  int at = 0x7fffffff;
  for (int c = lane; c < a.nchunk; c += 64)
    if (p[c].m > M || at == 0x7fffffff) M = p[c].m, at = p[c].at;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(M, o, 64);
    const int a2 = __shfl_xor(at, o, 64);
    if (m2 > M || (m2 == M && a2 < at)) M = m2, at = a2;
  }
  double s = 0.0;
  if (a.inv_temp != 0.0 && M > -INFINITY)
    for (int c = lane; c < a.nchunk; c += 64)
      if (p[c].m > -INFINITY) s += p[c].s * vf_weight(p[c].m, M, a.inv_temp);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  return Part{M, at, s};
}

// What the draw needs of the last node.
struct Last {
  int node;
  float M;
  double Z;
  bool refused;
};

// The weight of token i at the last node; refused: the refused tokens (drafts without probabilities).
__device__ __forceinline__ double vf_left(const VerifyArgs& a, int b, const Last& z, const int* refused, int nref,
                                          int64_t i) {
  double w = vf_weight(vf_logit(a, (int64_t)b * a.n + z.node, i), z.M, a.inv_temp);
  if (a.q && z.refused) return fmax(w / z.Z - (double)a.q[((int64_t)b * (a.n - 1) + z.node) * a.V + i], 0.0);
  for (int r = 0; r < nref; ++r) w = refused[r] == i ? 0.0 : w;
  return w;
}

// The first token whose running sum exceeds u times the total, from the chunks' sums (in LDS): 256 threads.
__device__ int vf_pick(const VerifyArgs& a, int b, const Last& z, const int* refused, int nref, double u,
                       const double* sums, double* red) {
  __shared__ int s_chunk;
  __shared__ double s_before, s_target;
  __shared__ int s_at, s_last;
  const int t = threadIdx.x;
  if (t == 0) {
    double total = 0.0;
    for (int c = 0; c < a.nchunk; ++c) total += sums[c];
    const double target = u * total;
    double run = 0.0, before = 0.0;
    int pick = -1;
    for (int c = 0; c < a.nchunk; ++c) {
      if (!(sums[c] > 0.0)) continue;
      if (pick >= 0 && !(run <= target)) break;
      pick = c;  // (rounding may leave the target past the last weight: then the last chunk)
      before = run;
      run += sums[c];
    }
    s_chunk = pick;
    s_before = before;
    s_target = target;
    s_at = 0x7fffffff;
    s_last = -1;
  }
  __syncthreads();
  const int c = s_chunk;
  if (c < 0) return -1;
  // thread t: VF_PER elements in a row
  const int64_t i0 = (int64_t)c * VF_CHUNK + t * VF_PER;
  double w[VF_PER], mine = 0.0;
  for (int k = 0; k < VF_PER; ++k) {
    w[k] = i0 + k < a.V ? vf_left(a, b, z, refused, nref, i0 + k) : 0.0;
    mine += w[k];
  }
  red[t] = mine;
  __syncthreads();
  double run = s_before;
  for (int k = 0; k < t; ++k) run += red[k];
  const double end = run + mine;  // the next thread's start, to the bit
  int found = -1, last = -1;
  for (int k = 0; k < VF_PER; ++k) {
    run += w[k];
    if (w[k] > 0.0) last = (int)(i0 + k);
    if (found < 0 && w[k] > 0.0 && run > s_target) found = last;
  }
  if (found < 0 && end > s_target) found = last;
  if (found >= 0) atomicMin(&s_at, found);
  if (last >= 0) atomicMax(&s_last, last);  // (rounding may leave the target past the chunk's last weight)
  __syncthreads();
  return s_at != 0x7fffffff ? s_at : s_last;
}

// One workgroup per sequence: the rows' statistics, the walk and, unless a q is to be taken off, the draw.
__global__ __launch_bounds__(VF_THREADS) void verify_walk_kernel(VerifyArgs a) {
  __shared__ float sM[64];
  __shared__ int sat[64], sref[64];
  __shared__ double sZ[64];
  __shared__ double sums[VF_MAX_CHUNKS], red[VF_THREADS];
  __shared__ int s_node, s_nref;
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, n = a.n;
  const int len = a.lengths ? min(a.lengths[b], n) : n;
  for (int r = wave; r < n; r += 4) {
    const Part p = vf_row(a, (int64_t)b * n + r, lane);
    if (lane == 0) sM[r] = p.m, sat[r] = p.at, sZ[r] = p.s;
  }
  __syncthreads();
  if (len <= 0) {
    if (t < n) a.path[(int64_t)b * n + t] = -1;
    if (t == 0) a.count[b] = 0, a.token[b] = -1;
    if (t == 0 && a.state) a.state[b] = -1;
    return;
  }
  if (wave == 0) {
    const bool live = lane < len;
    int par = -1, tok = -1;
    if (live) {
      tok = a.tokens[(int64_t)b * n + lane];
      par = a.parents ? a.parents[(int64_t)b * a.parents_stride + lane] : lane - 1;
      if (par < 0 || par >= lane) par = -1;
    }
    const bool can = live && par >= 0 && tok >= 0 && tok < a.V;
    double p = 0.0, q = 1.0, u = 0.0;
    if (can) {
      if (a.inv_temp == 0.0) {
        p = sM[par] > -INFINITY && sat[par] == tok ? 1.0 : 0.0;
      } else {
        if (sM[par] > -INFINITY) p = vf_weight(vf_logit(a, (int64_t)b * n + par, tok), sM[par], a.inv_temp) / sZ[par];
        u = a.u[(int64_t)b * n + lane];
        if (a.q) q = a.q[((int64_t)b * (n - 1) + par) * a.V + tok];
      }
    }
    int cur = 0, last = 0, got = 1;
    double left = 1.0;
    uint64_t refused = 0, taken = 1;
    while (true) {
      const uint64_t cand = __ballot(live && par == cur && lane > last);
      if (!cand) break;
      const int i = __ffsll((unsigned long long)cand) - 1;
      const int ti = __shfl(tok, i, 64);
      const bool again = __ballot((refused >> lane & 1) && tok == ti) != 0;
      const double pi = again ? 0.0 : __shfl(p, i, 64), ui = __shfl(u, i, 64);
      const bool ok = a.q && a.inv_temp != 0.0 ? ui * __shfl(q, i, 64) < pi : ui * left < pi;
      last = i;
      if (ok) {
        cur = i;
        taken |= 1ull << i;
        ++got;
        refused = 0;
        left = 1.0;
      } else {
        refused |= 1ull << i;
        left -= pi;
      }
    }
    const int slot = __popcll(taken & ((1ull << lane) - 1));
    if (lane < n && (taken >> lane & 1)) a.path[(int64_t)b * n + slot] = lane;
    if (lane < n && lane >= got) a.path[(int64_t)b * n + lane] = -1;
    if (refused >> lane & 1) sref[__popcll(refused & ((1ull << lane) - 1))] = tok;
    if (lane == 0) {
      a.count[b] = got;
      s_node = cur;
      s_nref = __popcll(refused);
      if (a.state) a.state[b] = refused ? cur : -1;
    }
  }
  __syncthreads();
  const Last z{s_node, sM[s_node], sZ[s_node], s_nref > 0};
  if (!(z.M > -INFINITY)) {
    if (t == 0) a.token[b] = -1;
    if (t == 0 && a.state) a.state[b] = -1;
    return;
  }
  if (a.inv_temp == 0.0) {
    if (t == 0) a.token[b] = sat[z.node];
    return;
  }
  if (a.q && z.refused) return;
  // the chunks' sums, without the refused tokens
  const Part* pr = a.part + ((int64_t)b * n + z.node) * a.nchunk;
  for (int c = t; c < a.nchunk; c += VF_THREADS) {
    double s = pr[c].m > -INFINITY ? pr[c].s * vf_weight(pr[c].m, z.M, a.inv_temp) : 0.0;
    for (int r = 0; r < s_nref; ++r) {
      bool dup = sref[r] < 0 || sref[r] >= a.V || sref[r] / VF_CHUNK != c;
      for (int k = 0; k < r; ++k) dup = dup || sref[k] == sref[r];
      if (!dup) s -= vf_weight(vf_logit(a, (int64_t)b * n + z.node, sref[r]), z.M, a.inv_temp);
    }
    sums[c] = fmax(s, 0.0);
  }
  __syncthreads();
  const int tok = vf_pick(a, b, z, sref, s_nref, (double)a.u[(int64_t)b * n], sums, red);
  if (t == 0) a.token[b] = tok;
}

// q: chunk sums of max(p - q, 0) at the last node, where a child was refused.
__global__ __launch_bounds__(VF_THREADS) void verify_resid_kernel(VerifyArgs a) {
  __shared__ double redd[4];
  __shared__ float sM;
  __shared__ double sZ;
  const int b = blockIdx.y, c = blockIdx.x, node = a.state[b];
  if (node < 0) return;
  if (threadIdx.x < 64) {
    const Part p = vf_row(a, (int64_t)b * a.n + node, threadIdx.x);
    if (threadIdx.x == 0) sM = p.m, sZ = p.s;
  }
  __syncthreads();
  const Last z{node, sM, sZ, true};
  double s = 0.0;
  for (int k = 0; k < VF_PER; ++k) {
    const int64_t i = (int64_t)c * VF_CHUNK + VF_THREADS * k + threadIdx.x;
    if (i < a.V) s += vf_left(a, b, z, nullptr, 0, i);
  }
  s = vf_block_reduce(s, redd, [](double p, double q) { return p + q; });
  if (threadIdx.x == 0) a.resid[(int64_t)b * a.nchunk + c] = s;
}

__global__ __launch_bounds__(VF_THREADS) void verify_draw_kernel(VerifyArgs a) {
  __shared__ double sums[VF_MAX_CHUNKS], red[VF_THREADS];
  __shared__ float sM;
  __shared__ double sZ;
  const int b = blockIdx.x, node = a.state[b];
  if (node < 0) return;
  if (threadIdx.x < 64) {
    const Part p = vf_row(a, (int64_t)b * a.n + node, threadIdx.x);
    if (threadIdx.x == 0) sM = p.m, sZ = p.s;
  }
  double any = 0.0;
  for (int c = threadIdx.x; c < a.nchunk; c += VF_THREADS) any += sums[c] = a.resid[(int64_t)b * a.nchunk + c];
  any = vf_block_reduce(any, red, [](double p, double q) { return p + q; });
  __syncthreads();
  Last z{node, sM, sZ, true};
  if (!(any > 0.0)) {  // p nowhere above q (to rounding): drawn from p
    z.refused = false;
    const Part* pr = a.part + ((int64_t)b * a.n + node) * a.nchunk;
    for (int c = threadIdx.x; c < a.nchunk; c += VF_THREADS)
      sums[c] = pr[c].m > -INFINITY ? pr[c].s * vf_weight(pr[c].m, z.M, a.inv_temp) : 0.0;
    __syncthreads();
  }
  const int tok = vf_pick(a, b, z, nullptr, 0, (double)a.u[(int64_t)b * a.n], sums, red);
  if (threadIdx.x == 0) a.token[b] = tok;
}

int64_t up16(int64_t v) { return (v + 15) & ~15ll; }

}  // namespace

extern "C" int64_t nsx_verify_workspace_bytes(int64_t batch, int n_nodes, int64_t vocab) {
  if (batch <= 0 || n_nodes <= 0 || vocab <= 0) return -1;
  const int64_t nchunk = nsx_cdiv(vocab, VF_CHUNK);
  return batch * n_nodes * nchunk * (int64_t)sizeof(Part) + up16(batch * nchunk * 8) + up16(batch * 4);
}

extern "C" int nsx_verify(const void* logits, int logits_dtype, int64_t row_stride, int64_t batch, int n_nodes,
                          int64_t vocab, const int32_t* tokens, const int32_t* parents, int64_t parents_stride,
                          const int32_t* lengths, const float* uniforms, const float* draft_probs, double temperature,
                          int32_t* count, int32_t* path, int32_t* token, void* workspace, int64_t workspace_bytes,
                          void* stream) {
  NSX_REQUIRE(logits_dtype == NSX_DT_F32 || logits_dtype == NSX_DT_F16 || logits_dtype == NSX_DT_BF16, NSX_ETYPE,
              "logits element type %d", logits_dtype);
  NSX_REQUIRE(n_nodes > 0 && n_nodes <= NSX_TREE_MAX_NODES, NSX_EINVAL, "%d nodes (1 to %d)", n_nodes,
              NSX_TREE_MAX_NODES);
  NSX_REQUIRE(batch >= 0 && batch * n_nodes < 65536, NSX_EINVAL, "%lld sequences of %d nodes: fewer than 65536 rows",
              (long long)batch, n_nodes);
  NSX_REQUIRE(vocab > 0 && vocab <= (int64_t)VF_CHUNK * VF_MAX_CHUNKS, NSX_EINVAL, "vocabulary of %lld (1 to %lld)",
              (long long)vocab, (long long)VF_CHUNK * VF_MAX_CHUNKS);
  NSX_REQUIRE(row_stride >= vocab, NSX_EINVAL, "rows %lld elements apart for %lld logits", (long long)row_stride,
              (long long)vocab);
  NSX_REQUIRE(temperature == 0.0 || (temperature >= 1e-30 && temperature <= 1e30), NSX_EINVAL, "temperature %g (0, or 1e-30 to 1e30)",
              temperature);
  NSX_REQUIRE(parents_stride == 0 || parents_stride >= n_nodes, NSX_EINVAL, "parents_stride=%lld",
              (long long)parents_stride);
  NSX_REQUIRE(!(draft_probs && parents), NSX_EINVAL, "draft probabilities go with chains (no parents)");
  if (batch == 0) return NSX_OK;
  NSX_REQUIRE(logits && tokens && count && path && token && workspace, NSX_EINVAL, "null buffer");
  NSX_REQUIRE(temperature == 0.0 || uniforms, NSX_EINVAL, "a temperature above 0 needs uniforms");
  const int64_t need = nsx_verify_workspace_bytes(batch, n_nodes, vocab);
  NSX_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0, NSX_EINVAL,
              "workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)workspace_bytes, (long long)need);
  const int nchunk = (int)nsx_cdiv(vocab, VF_CHUNK);
  const bool residual = draft_probs && temperature > 0.0 && n_nodes > 1;
  uint8_t* w = (uint8_t*)workspace;
  Part* part = (Part*)w;
  w += batch * n_nodes * nchunk * (int64_t)sizeof(Part);
  double* resid = (double*)w;
  w += up16(batch * nchunk * 8);
  VerifyArgs a{logits, logits_dtype, row_stride, (int)batch, n_nodes, vocab, tokens, parents, lengths, parents_stride,
               uniforms, residual ? draft_probs : nullptr, temperature > 0.0 ? 1.0 / temperature : 0.0, count, path,
               token, nchunk, part, resid, residual ? (int32_t*)w : nullptr};
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(verify_stats_kernel, dim3(nchunk, (unsigned)(batch * n_nodes)), dim3(VF_THREADS), 0, st, a);
  NSX_LAUNCHED();
  hipLaunchKernelGGL(verify_walk_kernel, dim3((unsigned)batch), dim3(VF_THREADS), 0, st, a);
  NSX_LAUNCHED();
  if (residual) {
    hipLaunchKernelGGL(verify_resid_kernel, dim3(nchunk, (unsigned)batch), dim3(VF_THREADS), 0, st, a);
    NSX_LAUNCHED();
    hipLaunchKernelGGL(verify_draw_kernel, dim3((unsigned)batch), dim3(VF_THREADS), 0, st, a);
    NSX_LAUNCHED();
  }
  return NSX_OK;
}
