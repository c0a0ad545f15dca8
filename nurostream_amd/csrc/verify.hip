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
// Weights, sums and comparisons in 64 bits: a vocabulary's running sum is compared with a random number, and with 32-bit
// weights the answer would be another one in about one draw of a million; and what refused tokens leave of a row is a
// difference, which a weight's error outgrows where they had nearly all of it. A NaN logit counts as -infinity; of
// +infinity in a row, its tokens share the row's whole weight; a row without any weight gives the token -1. Sequences with
// no nodes (length 0) give count 0 and token -1, and rows behind a length are not read.
//
// Two launches. The rows' chunk sums read all logits once: 32 rows of 201088 fp32 logits 11.7 us, of which the bytes (2.2
// TB/s with the launch; 8 us without weights) and then some 18 64-bit operations per logit; 120 rows of 151936 in bf16 14.
// The walk with the draw is five dependent round trips to memory: 10 us, 3.1 where nothing is drawn (temperature 0).
#include "nsx_common.h"

#include <algorithm>
#include <type_traits>
#include <math.h>

namespace {

constexpr int VF_CHUNK = 4096;       // logits per workgroup of the row passes
constexpr int VF_THREADS = 256;      // of the row passes
constexpr int VF_WALK = 1024;        // of the walk and the draw
constexpr int VF_WALK_Q = 512;       // of the same, a workgroup per chunk
constexpr int VF_MAX_CHUNKS = 1024;
constexpr int VF_VEC = 8;            // chunks begin where the row's address is a multiple of this many elements

// A chunk's largest logit, its (lowest) index and the weights' sum relative to it.
struct Part {
  float m;
  int32_t at;
  double s;
};

struct VerifyArgs {
  const void* logits;
  int64_t row_stride;  // elements
  int B, n;
  int64_t V;
  const int32_t *tokens, *parents, *lengths;
  int64_t parents_stride;  // 0: one tree for all sequences
  const float *u, *q;
  double scale2;  // log2(e) / temperature; 0: greedy
  double least;   // -1000 / scale2
  int32_t *count, *path, *token;
  int nchunk;
  Part* part;     // [B * n][nchunk]
  double* resid;    // q: [B][nchunk], the sums of max(p - q, 0) at the last node
  uint32_t* ticket;  // q: [B], how many of a sequence's workgroups have written theirs
};

template <typename LT>  // float, _Float16, or uint16_t for bf16
struct Row {
  const LT* p;
  int off;  // elements that the row's start lies behind a multiple of VF_VEC
  __device__ __forceinline__ Row(const VerifyArgs& a, int64_t row)
      : p((const LT*)a.logits + row * a.row_stride), off((int)((uintptr_t)p / sizeof(LT) % VF_VEC)) {}
  static __device__ __forceinline__ float value(LT x) {
    float f;
    if constexpr (sizeof(LT) == 4) f = x;
    else if constexpr (std::is_same_v<LT, _Float16>) f = (float)x;
    else f = nsx_bf2f(x);
    return f == f ? f : -INFINITY;
  }
  __device__ __forceinline__ float at(int64_t i) const { return value(p[i]); }
  // The N elements from place v (a multiple of N) of the row's chunks on; -infinity where the row has none.
  template <int N>
  __device__ __forceinline__ void run(int64_t v, int64_t V, float (&x)[N]) const {
    const int64_t i = v - off;
    if (i >= 0 && i + N <= V) {
      struct alignas(N * sizeof(LT)) Vec {
        LT e[N];
      };
      const Vec w = *(const Vec*)(p + i);
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = value(w.e[k]);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = i + k >= 0 && i + k < V ? at(i + k) : -INFINITY;
    }
  }
};

// 2^(j / 32) in LDS: 32 entries, one on each pair of the 64 banks.
struct Pow2 {
  double t[32];
  __device__ __forceinline__ void fill() {
    if (threadIdx.x < 32) t[threadIdx.x] = exp2((double)threadIdx.x / 32);
  }
};

// The weight 2^(scale2 (x - M)) of logit x beside the largest, M > -infinity. The exponent is n + j / 32 + r with
// |r| <= 1 / 64 by adding 1.5 * 2^47; 2^r - 1 = r (ln2 + ..) to the sixth power of r leaves out 2^-58: with the roundings
// 2^-51 of the weight (to the fourth power 2^-39), beside what the product with scale2 loses, as any exp(x / T) does. No
// weight is below 2^-1000, `least` being the least difference: beside the largest one's 1 that is nothing.
__device__ __forceinline__ double vf_weight_finite(float x, float M, const VerifyArgs& a, const Pow2& tab) {
  const double d = fmax((double)x - (double)M, a.least);
  const double t = fma(d, a.scale2, 0x1.8p47);
  const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, t);
  const double r = fma(d, a.scale2, -(t - 0x1.8p47));
  double h = 0.00015403530393381609;  // ln2^6 / 720, ln2^5 / 120, ..
  h = fma(r, h, 0.0013333558146428443);
  h = fma(r, h, 0.0096181291076284772);
  h = fma(r, h, 0.055504108664821580);
  h = fma(r, h, 0.24022650695910071);
  h = fma(r, h, 0.69314718055994531);
  const double c = tab.t[k & 31], w = fma(r * h, c, c);
  const uint64_t bits = __builtin_bit_cast(uint64_t, w);
  const uint32_t high = (uint32_t)(bits >> 32) + ((k & ~31u) << 15);  // 2^n into the exponent
  return __builtin_bit_cast(double, (uint64_t)high << 32 | (uint32_t)bits);
}
// With zero for what is below 2^-1000, and for M = +infinity.
__device__ __forceinline__ double vf_weight(float x, float M, const VerifyArgs& a, const Pow2& tab) {
  if (M == INFINITY) return x == M ? 1.0 : 0.0;
  const double w = vf_weight_finite(x, M, a, tab);
  return (double)x - (double)M < a.least ? 0.0 : w;
}

// Wave-wide operations on DPP moves and readlanes: no trip through LDS.
template <int CTRL>
__device__ __forceinline__ double vf_dpp(double v) {  // lanes without a source get 0
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float vf_lane(float v, int i) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i));
}
__device__ __forceinline__ double vf_lane(double v, int i) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), i) << 32 |
                                        (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, i));
}
__device__ __forceinline__ float vf_wave_max(float v) {
  v = nsx_row_fmax(v);
  return fmaxf(fmaxf(vf_lane(v, 0), vf_lane(v, 16)), fmaxf(vf_lane(v, 32), vf_lane(v, 48)));
}
__device__ __forceinline__ double vf_wave_sum(double v) {
  v += vf_dpp<NSX_DPP_ROR(8)>(v);
  v += vf_dpp<NSX_DPP_ROR(4)>(v);
  v += vf_dpp<NSX_DPP_ROR(2)>(v);
  v += vf_dpp<NSX_DPP_ROR(1)>(v);
  return (vf_lane(v, 0) + vf_lane(v, 16)) + (vf_lane(v, 32) + vf_lane(v, 48));
}
__device__ __forceinline__ double vf_wave_scan(double v) {  // inclusive: rows of 16 by shifts, then the rows before
  v += vf_dpp<0x111>(v);
  v += vf_dpp<0x112>(v);
  v += vf_dpp<0x114>(v);
  v += vf_dpp<0x118>(v);
  const int row = (threadIdx.x & 63) >> 4;
  const double r0 = vf_lane(v, 15), r1 = r0 + vf_lane(v, 31), r2 = r1 + vf_lane(v, 47);
  return row == 0 ? v : (row == 1 ? r0 : row == 2 ? r1 : r2) + v;
}
// Over 256 threads, the same order in every one.
__device__ __forceinline__ float vf_block_max(float v, float* red) {
  v = vf_wave_max(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
__device__ __forceinline__ int vf_block_min(int v, int* red) {  // of values >= 0
  v = (int)nsx_wave_min_u32((uint32_t)v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return min(min(red[0], red[1]), min(red[2], red[3]));
}
template <int NW = 4>
__device__ __forceinline__ double vf_block_sum(double v, double* red) {
  v = vf_wave_sum(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int k = 1; k < NW; ++k) v += red[k];
  return v;
}

template <typename LT, bool GREEDY>
__global__ __launch_bounds__(VF_THREADS) void verify_stats_kernel(VerifyArgs a) {
  constexpr int W = 16 / sizeof(LT), RUNS = VF_CHUNK / VF_THREADS / W;  // elements of a 16-byte load, loads
  __shared__ float redf[4];
  __shared__ int redi[4];
  __shared__ double redd[4];
  __shared__ Pow2 tab;
  const int c = blockIdx.x, i = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  if (a.ticket && i == 0 && c == 0 && t == 0) a.ticket[b] = 0;
  if (a.lengths && i >= a.lengths[b]) return;
  const int64_t row = (int64_t)b * a.n + i;
  const Row<LT> r(a, row);
  float x[RUNS][W], m = -INFINITY;
#pragma unroll
  for (int u = 0; u < RUNS; ++u) r.run((int64_t)c * VF_CHUNK + (u * VF_THREADS + t) * W, a.V, x[u]);
  if (!GREEDY) tab.fill();
#pragma unroll
  for (int u = 0; u < RUNS; ++u)
#pragma unroll
    for (int k = 0; k < W; ++k) m = fmaxf(m, x[u][k]);
  m = vf_block_max(m, redf);
  int at = 0x7fffffff;
  double s = 0.0;
  if constexpr (GREEDY) {
#pragma unroll
    for (int u = RUNS - 1; u >= 0; --u)
#pragma unroll
      for (int k = W - 1; k >= 0; --k)
        if (x[u][k] == m) at = max(0, (int)((int64_t)c * VF_CHUNK + (u * VF_THREADS + t) * W + k - r.off));
    at = vf_block_min(at, redi);
  } else {
    if (m == INFINITY) {
#pragma unroll
      for (int u = 0; u < RUNS; ++u)
#pragma unroll
        for (int k = 0; k < W; ++k) s += x[u][k] == m ? 1.0 : 0.0;
    } else if (m > -INFINITY) {
#pragma unroll
      for (int u = 0; u < RUNS; ++u)
#pragma unroll
        for (int k = 0; k < W; ++k) s += vf_weight_finite(x[u][k], m, a, tab);
    }
    s = vf_block_sum(s, redd);
  }
  if (t == 0) a.part[row * a.nchunk + c] = Part{m, at, s};
}

// A lane's first chunk of a row (with most vocabularies its only one).
__device__ __forceinline__ Part vf_part(const VerifyArgs& a, int64_t row, int lane) {
  return lane < a.nchunk ? a.part[row * a.nchunk + lane] : Part{-INFINITY, 0x7fffffff, 0.0};
}
// The row's largest logit, its index and the weights' sum, from its chunks: one wave.
__device__ __forceinline__ Part vf_row(const VerifyArgs& a, int64_t row, int lane, const Part& p0, const Pow2& tab) {
  const Part* p = a.part + row * a.nchunk;
  float mx = p0.m;
  int at = p0.at;
  for (int c = lane + 64; c < a.nchunk; c += 64)
    if (p[c].m > mx) mx = p[c].m, at = p[c].at;
  const float M = vf_wave_max(mx);
  if (a.scale2 == 0.0) return Part{M, (int)nsx_wave_min_u32(mx == M ? (uint32_t)at : 0x7fffffffu), 0.0};
  double s = 0.0;
  if (M > -INFINITY) {
    if (p0.m > -INFINITY) s = p0.s * vf_weight(p0.m, M, a, tab);
    for (int c = lane + 64; c < a.nchunk; c += 64)
      if (p[c].m > -INFINITY) s += p[c].s * vf_weight(p[c].m, M, a, tab);
  }
  return Part{M, 0, vf_wave_sum(s)};
}

template <int T>
struct PickLds {
  double sums[VF_MAX_CHUNKS + 1];  // the chunks' sums
  double wave[T / 64];
  double before, target;
  int chunk, at, last;
};

// The first token whose running sum exceeds u times the total, from the chunks' sums; weight(i, load(i)): token i's. -1:
// no sum is above zero. (A sum that is only rounding, all its chunk's tokens refused, is struck out and the draw made again.)
template <int T, typename L, typename F>
__device__ int vf_pick(const VerifyArgs& a, PickLds<T>& s, double u, int off, L load, F weight) {
  constexpr int PER = VF_CHUNK / T;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  for (;;) {
    __syncthreads();
    if (wv == 0) {
      double total = 0.0;
      for (int c0 = 0; c0 < a.nchunk; c0 += 64)
        total += vf_lane(vf_wave_scan(c0 + lane < a.nchunk ? s.sums[c0 + lane] : 0.0), 63);
      const double target = u * total;
      double run = 0.0, before = 0.0;
      int pick = -1;
      for (int c0 = 0; c0 < a.nchunk; c0 += 64) {
        const double v = c0 + lane < a.nchunk ? s.sums[c0 + lane] : 0.0;
        const double up = vf_wave_scan(v), prev = __shfl_up(up, 1, 64);
        const uint64_t some = __ballot(v > 0.0), hit = __ballot(v > 0.0 && run + up > target);
        if (some) {  // (rounding may leave the target past the last weight: then the last chunk that has one)
          const int at = hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll((long long)some);
          const double pr = vf_lane(prev, at);
          pick = c0 + at;
          before = at ? run + pr : run;
        }
        if (hit) break;
        run += vf_lane(up, 63);
      }
      if (lane == 0) {
        s.chunk = pick;
        s.before = before;
        s.target = target;
        s.at = 0x7fffffff;
        s.last = -1;
      }
    }
    __syncthreads();
    const int c = s.chunk;
    if (c < 0) return -1;
    const int64_t i0 = (int64_t)c * VF_CHUNK + t * PER - off;
    decltype(load(0)) raw[PER];  // all loads on their way, then the weights
    double w[PER], mine = 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k) raw[k] = load(min(max(i0 + k, (int64_t)0), a.V - 1));
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      w[k] = weight(i0 + k, raw[k]);
      w[k] = i0 + k >= 0 && i0 + k < a.V ? w[k] : 0.0;
      mine += w[k];
    }
    const double up = vf_wave_scan(mine), prev = __shfl_up(up, 1, 64);
    if (lane == 63) s.wave[wv] = up;
    __syncthreads();
    double base = s.before;
    for (int k = 0; k < wv; ++k) base += s.wave[k];
    const double end = base + up;  // the next thread's start, to the bit
    double run = lane ? base + prev : base;
    int found = -1, last = -1;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      run += w[k];
      if (w[k] > 0.0) last = (int)(i0 + k);
      if (found < 0 && w[k] > 0.0 && run > s.target) found = last;
    }
    if (found < 0 && end > s.target) found = last;
    if (found >= 0) atomicMin(&s.at, found);
    if (last >= 0) atomicMax(&s.last, last);  // (rounding may leave the target past the chunk's last weight)
    __syncthreads();
    const int got = s.at != 0x7fffffff ? s.at : s.last;
    if (got >= 0) return got;
    if (t == 0) s.sums[c] = 0.0;
  }
}

// max(p - q, 0) at the last node.
template <typename LT>
struct Resid {
  const VerifyArgs& a;
  const Row<LT> row;
  const float* q;
  const float M;
  const double inv_z;
  struct Raw {
    float x, q;
  };
  __device__ __forceinline__ Resid(const VerifyArgs& a, int b, int node, float M, double Z)
      : a(a), row(a, (int64_t)b * a.n + node), q(a.q + ((int64_t)b * (a.n - 1) + node) * a.V), M(M), inv_z(1.0 / Z) {}
  __device__ __forceinline__ Raw load(int64_t i) const { return Raw{row.at(i), q[i]}; }
  __device__ __forceinline__ double weight(const Raw& r, const Pow2& tab) const {
    return fmax(vf_weight(r.x, M, a, tab) * inv_z - (double)r.q, 0.0);
  }
};

// The rows' statistics, the walk and the draw: one workgroup per sequence. With q there is one per chunk and sequence, as
// a draw from max(p - q, 0) needs all of that row's sums: each makes the same walk, the first alone writes it, and each
// sums its chunk, the last to do so drawing. (The walks are made side by side, where a launch each for the residual's sums
// and their draw came one after the other: 24 sequences of 5 rows of 151936 bf16 logits 42 us in four launches, 28 in two.
// 512 threads: with 1024 31 us, and a workgroup of 256 spills.)
template <typename LT, bool Q, int T>
__global__ __launch_bounds__(T) void verify_walk_kernel(VerifyArgs a) {
  __shared__ float sM[64];
  __shared__ int sat[64], sref[64];
  __shared__ double sZ[64], swref[64];
  __shared__ PickLds<T> pick;
  __shared__ Pow2 tab;
  __shared__ int s_node, s_nref, s_last;
  const int c = Q ? blockIdx.x : 0, b = Q ? blockIdx.y : blockIdx.x;
  const bool first = c == 0;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, n = a.n;
  const int len = a.lengths ? min(a.lengths[b], n) : n;
  const double u0 = a.u ? a.u[(int64_t)b * n] : 0.f;
  // the nodes' own loads ahead of the rows' sums
  int par = -1, tok = -1;
  float u = 0.f, x = -INFINITY, q = 1.f;
  if (wave == 0 && lane < len) {
    tok = a.tokens[(int64_t)b * n + lane];
    par = a.parents ? a.parents[(int64_t)b * a.parents_stride + lane] : lane - 1;
    if (par >= lane) par = -1;
    if (par >= 0 && tok >= 0 && tok < a.V && a.scale2 != 0.0) {
      u = a.u[(int64_t)b * n + lane];
      x = Row<LT>(a, (int64_t)b * n + par).at(tok);
      if (Q) q = a.q[((int64_t)b * (n - 1) + par) * a.V + tok];
    }
  }
  constexpr int AHEAD = 4, NW = T / 64;  // the rows' chunks too, of a wave's first rows
  Part ahead[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (wave + k * NW < len) ahead[k] = vf_part(a, (int64_t)b * n + wave + k * NW, lane);
  tab.fill();
  nsx_lds_barrier();
  auto row_of = [&](int r, const Part& p0) {
    const Part p = vf_row(a, (int64_t)b * n + r, lane, p0, tab);
    if (lane == 0) sM[r] = p.m, sat[r] = p.at, sZ[r] = p.s;
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (wave + k * NW < len) row_of(wave + k * NW, ahead[k]);
  for (int r = wave + AHEAD * NW; r < len; r += NW) row_of(r, vf_part(a, (int64_t)b * n + r, lane));
  __syncthreads();
  if (len <= 0) {
    if (first && t < n) a.path[(int64_t)b * n + t] = -1;
    if (first && t == 0) {
      a.count[b] = 0;
      a.token[b] = -1;
    }
    return;
  }
  if (wave == 0) {
    double w = 0.0, p = 0.0;
    if (par >= 0 && tok >= 0 && tok < a.V && sM[par] > -INFINITY) {
      if (a.scale2 == 0.0) {
        p = sat[par] == tok ? 1.0 : 0.0;
      } else {
        w = vf_weight(x, sM[par], a, tab);
        p = w / sZ[par];
      }
    }
    int cur = 0, last = 0, got = 1;
    double left = 1.0;
    uint64_t refused = 0, taken = 1, again = 0;
    while (true) {
      const uint64_t cand = __ballot(lane < len && par == cur && lane > last);
      if (!cand) break;
      const int i = __ffsll((unsigned long long)cand) - 1;
      const int ti = __builtin_amdgcn_readlane(tok, i);
      const bool dup = __ballot((refused >> lane & 1) && tok == ti) != 0;
      const double pi = dup ? 0.0 : vf_lane(p, i), ui = vf_lane(u, i);
      const bool ok = a.q ? ui * (double)vf_lane(q, i) < pi : ui * left < pi;
      last = i;
      if (ok) {
        cur = i;
        taken |= 1ull << i;
        ++got;
        refused = again = 0;
        left = 1.0;
      } else {
        refused |= 1ull << i;
        again |= (uint64_t)dup << i;
        left -= pi;
      }
    }
    const int slot = __popcll(taken & ((1ull << lane) - 1));
    if (first && lane < n && (taken >> lane & 1)) a.path[(int64_t)b * n + slot] = lane;
    if (first && lane < n && lane >= got) a.path[(int64_t)b * n + lane] = -1;
    if (refused >> lane & 1) {
      const int k = __popcll(refused & ((1ull << lane) - 1));
      sref[k] = tok;
      swref[k] = again >> lane & 1 ? 0.0 : w;  // (zero too where the token is no token)
    }
    if (lane == 0) {
      if (first) a.count[b] = got;
      s_node = cur;
      s_nref = __popcll(refused);
    }
  }
  __syncthreads();
  const int node = s_node, nref = s_nref;
  const float M = sM[node];
  if (!(M > -INFINITY) || a.scale2 == 0.0) {
    if (first && t == 0) a.token[b] = M > -INFINITY ? sat[node] : -1;
    return;
  }
  const Part* pr = a.part + ((int64_t)b * n + node) * a.nchunk;
  const bool residual = Q && nref;
  int got = -1;
  if constexpr (Q) {
    if (residual) {
      constexpr int PER = VF_CHUNK / T;
      const Resid<LT> r(a, b, node, M, sZ[node]);
      typename Resid<LT>::Raw raw[PER];
      const int64_t i0 = (int64_t)c * VF_CHUNK + t - r.row.off;
#pragma unroll
      for (int k = 0; k < PER; ++k) raw[k] = r.load(min(max(i0 + T * k, (int64_t)0), a.V - 1));
      double s = 0.0;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int64_t i = i0 + T * k;
        const double w = r.weight(raw[k], tab);
        s += i >= 0 && i < a.V ? w : 0.0;
      }
      s = vf_block_sum<T / 64>(s, pick.wave);
      double* sums = a.resid + (int64_t)b * a.nchunk;
      if (t == 0) {  // the sum first, then the count, as every workgroup on the device sees them
        __hip_atomic_store(sums + c, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = __hip_atomic_fetch_add(a.ticket + b, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == a.nchunk - 1u;
      }
      __syncthreads();
      if (!s_last) return;
      for (int k = t; k < a.nchunk; k += T)
        pick.sums[k] = __hip_atomic_load(sums + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      got = vf_pick(a, pick, u0, r.row.off, [&](int64_t i) { return r.load(i); },
                    [&](int64_t, const typename Resid<LT>::Raw& x) { return r.weight(x, tab); });
    } else if (!first) {
      return;
    }
  }
  if (got < 0) {  // (from the residual: p is nowhere above q, to rounding, and the draw is from p)
    // the chunks' sums, without the refused tokens
    const int out = residual ? 0 : nref;
    const Row<LT> row(a, (int64_t)b * n + node);
    for (int k = t; k < a.nchunk; k += T) {
      double s = pr[k].m > -INFINITY ? pr[k].s * vf_weight(pr[k].m, M, a, tab) : 0.0;
      for (int r = 0; r < out; ++r)
        if (swref[r] > 0.0 && (sref[r] + row.off) / VF_CHUNK == k) s -= swref[r];
      pick.sums[k] = fmax(s, 0.0);
    }
    got = vf_pick(a, pick, u0, row.off, [&](int64_t i) { return row.at(i); }, [&](int64_t i, float x) {
      double w = vf_weight(x, M, a, tab);
      for (int r = 0; r < out; ++r) w = sref[r] == i ? 0.0 : w;
      return w;
    });
  }
  if (t == 0) a.token[b] = got;
}

int64_t up16(int64_t v) { return (v + 15) & ~15ll; }
int64_t chunks(int64_t vocab) { return nsx_cdiv(vocab + VF_VEC - 1, VF_CHUNK); }

template <typename LT>
int verify_launch(const VerifyArgs& a, hipStream_t st) {
  const dim3 rows(a.nchunk, a.n, a.B), seqs(a.nchunk, a.B);
  if (a.scale2 == 0.0) hipLaunchKernelGGL((verify_stats_kernel<LT, true>), rows, dim3(VF_THREADS), 0, st, a);
  else hipLaunchKernelGGL((verify_stats_kernel<LT, false>), rows, dim3(VF_THREADS), 0, st, a);
  NSX_LAUNCHED();
  if (a.q) hipLaunchKernelGGL((verify_walk_kernel<LT, true, VF_WALK_Q>), seqs, dim3(VF_WALK_Q), 0, st, a);
  else hipLaunchKernelGGL((verify_walk_kernel<LT, false, VF_WALK>), dim3(a.B), dim3(VF_WALK), 0, st, a);
  NSX_LAUNCHED();
  return NSX_OK;
}

}  // namespace

extern "C" int64_t nsx_verify_workspace_bytes(int64_t batch, int n_nodes, int64_t vocab) {
  if (batch <= 0 || n_nodes <= 0 || vocab <= 0) return -1;
  return batch * n_nodes * chunks(vocab) * (int64_t)sizeof(Part) + up16(batch * chunks(vocab) * 8) +
         batch * (int64_t)sizeof(uint32_t);
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
              (long long)vocab, (long long)VF_CHUNK * VF_MAX_CHUNKS);  // (then at most VF_MAX_CHUNKS + 1 chunks)
  NSX_REQUIRE(row_stride >= vocab, NSX_EINVAL, "rows %lld elements apart for %lld logits", (long long)row_stride,
              (long long)vocab);
  NSX_REQUIRE(temperature == 0.0 || (temperature >= 1e-30 && temperature <= 1e30), NSX_EINVAL,
              "temperature %g (0, or 1e-30 to 1e30)", temperature);
  NSX_REQUIRE(parents_stride == 0 || parents_stride >= n_nodes, NSX_EINVAL, "parents_stride=%lld",
              (long long)parents_stride);
  NSX_REQUIRE(!(draft_probs && parents), NSX_EINVAL, "draft probabilities go with chains (no parents)");
  if (batch == 0) return NSX_OK;
  NSX_REQUIRE(logits && tokens && count && path && token && workspace, NSX_EINVAL, "null buffer");
  NSX_REQUIRE(temperature == 0.0 || uniforms, NSX_EINVAL, "a temperature above 0 needs uniforms");
  const int64_t need = nsx_verify_workspace_bytes(batch, n_nodes, vocab);
  NSX_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0, NSX_EINVAL,
              "workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)workspace_bytes, (long long)need);
  const bool residual = draft_probs && temperature > 0.0 && n_nodes > 1;
  const int nchunk = (int)chunks(vocab);
  uint8_t* w = (uint8_t*)workspace;
  Part* part = (Part*)w;
  w += batch * n_nodes * nchunk * (int64_t)sizeof(Part);
  double* resid = (double*)w;
  w += up16(batch * nchunk * 8);
  const double scale2 = temperature > 0.0 ? 1.44269504088896340736 / temperature : 0.0;
  const VerifyArgs a{logits, row_stride, (int)batch, n_nodes, vocab, tokens, parents, lengths, parents_stride, uniforms,
                     residual ? draft_probs : nullptr, scale2, scale2 > 0.0 ? -1000.0 / scale2 : 0.0,
                     count, path, token, nchunk, part, resid, residual ? (uint32_t*)w : nullptr};
  hipStream_t st = (hipStream_t)stream;
  if (logits_dtype == NSX_DT_F32) return verify_launch<float>(a, st);
  if (logits_dtype == NSX_DT_F16) return verify_launch<_Float16>(a, st);
  return verify_launch<uint16_t>(a, st);
}
