// A token for each row of logits by temperature, top-k, top-p and min-p from given random numbers (gfx950).
//
// A token's weight is 2^(log2(e) (x - M) / T), M the row's largest logit, computed in 64 bits and rounded to a whole multiple of
// 2^-bits: sums of weights are sums of whole numbers, the same in any order, so that the row may be split over workgroups and
// added up by atomics, and no launch or grid changes a token. A token's order is its logit's bits, made to order as numbers
// do, over its index's complement: every token has another one, larger for larger logits and among equals for lower indices; a
// filter keeps the tokens from some order on, and nothing is sorted.
//
// Four launches, each over all rows:
//  1. the largest order of each workgroup's parts (the row's is known behind it); the row's histogram is cleared;
//  2. the histogram: weight and number of the tokens in each 16th of an octave below M;
//  3. every part reads the histogram: the bin in which top-k ends, the bins in which top-p may (it counts from what top-k
//     leaves of its last bin); the weight of its tokens above those, and the list of the tokens in them;
//  4. a workgroup per row: where the filters end among the listed tokens; the parts' sums with what is kept of those; the part
//     in which the random number falls, and in that part the token.
// Where all rows are greedy the second and third are left out, without top-k and top-p the second; of few rows, the last of a
// row's workgroups in the third does the fourth's work.
//
// Bytes bind nothing here: 48 rows of 151936 bf16 logits are 2.9 us of a copy's time. The launches take 2.9, 4.8 and 13 us for
// one row of 201088 with top-k 50 and top-p 0.95, each a chain of a few loads and barriers (the token's some 20 000 cycles on one
// CU), and 6, 11, 15 and 16 us for 48 rows of settings of their own, where the second and third are bound by the weights: some 30
// vector instructions of a logit, most of 64 bits.
#include "nsx_common.h"
#include "pow2.h"

#include <algorithm>
#include <type_traits>
#include <math.h>

namespace {

constexpr int THREADS = 512;
constexpr int VEC = 8;                  // logits of a thread, consecutive
constexpr int PART = THREADS * VEC;     // logits of a part
constexpr int INDEX = 22;               // bits of an index
constexpr uint32_t LAST_INDEX = (1u << INDEX) - 1;
constexpr int MAX_PARTS = 1 + (1 << INDEX) / PART;
constexpr int BINS = 1024;              // 64 octaves of 16: no weight lies lower
// Listed tokens. A row with more in its last bins is read again instead, by its one workgroup of the last step, for every digit
// and sum: one row of 201088 at temperature 0.1 with top-k 50, where fewer than 50 tokens lie within 64 octaves and all others
// share the last bin, 399 us, with top-p 0.95 as well 683; of logits of deviation 0.1 with top-p 0.95 627; 48 rows of 151936 the
// same (temperature 0.8: 22 and 39).
constexpr int LIST = 8192;
constexpr int HELD = 4;                 // listed tokens that a thread holds in registers
constexpr int FEW = HELD * THREADS / 2;  // a top-k up to which all tokens that it may keep are listed (see few())
// Listed tokens up to which each is compared with each, all threads at once, in place of digit after digit: the last step
// takes 9.3 us so for 52 tokens, 11.6 by digits.
constexpr int RANK = THREADS / 4;
// Workgroups of a pass over all rows, four on each of 256 CUs: rows differ in work, and smaller shares of them level that
// (48 rows of settings of their own 59 us in all with 512 and with 768, 55 with 1024, 57 with all parts apart).
constexpr int GRID = 1024;
// Workgroups up to which the last of a row's goes on to its token, a launch less (its registers leave two workgroups a CU):
// rows of 151936 bf16 logits with top-p 0.9, so / by a launch of its own: 1 row 23.6 / 26.3 us, 4 25.7 / 27.2, 8 32.5 / 30.7,
// 48 66 / 52; without filters 13.1 / 14.7, 15.4 / 14.9, 18.6 / 16.7, 38 / 31.
constexpr int FUSED = 160;

struct SampleArgs {
  const void* logits;
  int64_t row_stride, V;
  const float* u;
  double temperature, top_p, min_p;
  int64_t top_k;
  const float *temperatures, *top_ps, *min_ps;
  const int32_t* top_ks;
  int32_t* token;
  int bits;  // of a weight behind the point
  int parts;
  int groups;           // workgroups of a row in the passes over all rows
  uint64_t* best;       // [batch][groups]
  uint64_t* sums;       // [batch][parts]
  uint64_t* mass;       // [batch][BINS]
  uint32_t* many;       // [batch][BINS]
  uint32_t* listed;     // [batch]
  uint32_t* ended;      // [batch]: workgroups of a row that are through its parts
  uint32_t* list;       // [batch][LIST]
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ double uniform(double x) {  // (the same in all lanes: out of the vector registers)
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)uniform((int)(u >> 32)) << 32 | (uint32_t)uniform((int)(uint32_t)u));
}

// A row's logits and settings.
template <typename LT>  // float, _Float16, or uint16_t for bf16
struct Row {
  const LT* p;
  int64_t V;
  int off;  // elements that the row's start lies behind a multiple of VEC
  double T, top_p, min_p, scale2, least, unit;
  int64_t top_k;
  float M = 0.f, scale32 = 0.f;
  bool infinite = false;  // the largest logit is: its equals count as 0 from then on, the others as -infinity
  __device__ __forceinline__ Row(const SampleArgs& a, int64_t row)
      : p((const LT*)a.logits + row * a.row_stride), V(a.V), off((int)((uintptr_t)p / sizeof(LT) % VEC)) {
    T = a.temperatures ? (double)a.temperatures[row] : a.temperature;
    top_p = a.top_ps ? (double)a.top_ps[row] : a.top_p;
    if (T > 0.0) T = fmin(fmax(T, 1e-30), 1e30);  // (a row's own is not looked at before)
    min_p = a.min_ps ? (double)a.min_ps[row] : a.min_p;
    min_p = min_p > 0.0 ? fmin(min_p, 1.0) : 0.0;
    top_k = a.top_ks ? a.top_ks[row] : a.top_k;
    if (top_k <= 0 || top_k >= V) top_k = 0;
    min_p = uniform(min_p);
    scale2 = uniform(1.44269504088896340736 / T);
    least = uniform(-1000.0 / scale2);
    unit = __builtin_bit_cast(double, (uint64_t)(1023 + a.bits) << 52);
  }
  // What top-p's tokens, of `whole` in all, are the first to reach: each of them has less than that before it.
  __device__ __forceinline__ uint64_t target(uint64_t whole) const {
    const uint64_t t = (uint64_t)ceil(fmax(top_p, 0.0) * (double)whole);
    return t < 1 ? 1 : t < whole || whole < 1 ? t : whole;
  }
  __device__ __forceinline__ bool drawn() const { return T > 0.0 && M > -INFINITY; }  // not the largest, not none
  __device__ __forceinline__ bool cut() const { return top_k || top_p < 1.0; }
  // Few tokens of the highest are wanted: counting finds their last bin, and all of them are listed, so that no other token's
  // weight is computed.
  __device__ __forceinline__ bool few() const { return top_k && top_k <= FEW; }
  __device__ __forceinline__ void largest(uint64_t order) {
    const uint32_t u = (uint32_t)(order >> INDEX) << SAME;
    const uint32_t bits = (u ^ ((int32_t)u < 0 ? 0x80000000u : 0xffffffffu)) & (0xffffffffu << SAME);
    M = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(bits));
    infinite = M == INFINITY;
    if (infinite) M = 0.f;
    // (times a difference of zero: zero)
    scale32 = __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, (float)fmin(16.0 * scale2, 3e38))));
  }
  static __device__ __forceinline__ float value(LT x) {
    float f;
    if constexpr (std::is_same_v<LT, uint16_t>) f = nsx_bf2f(x);
    else f = (float)x;
    return fmaxf(f + 0.f, -INFINITY);  // (no -0, no NaN)
  }
  __device__ __forceinline__ float seen(float x) const { return !infinite ? x : x == INFINITY ? 0.f : -INFINITY; }
  __device__ __forceinline__ float at(int64_t i) const { return seen(value(p[i])); }
  // The elements from place v (a multiple of VEC) of the row's parts on, element k being token v - off + k; -infinity where
  // there is none. Loaded as they lie, a vector, or one by one at the row's ends.
  struct alignas(16) Raw {
    LT e[VEC];
  };
  __device__ __forceinline__ Raw load(int64_t v) const {
    const int64_t i = v - off;
    Raw w;
    if (i >= 0 && i + VEC <= V) {
      w = *(const Raw*)(p + i);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) w.e[k] = i + k >= 0 && i + k < V ? p[i + k] : LT(0);
    }
    return w;
  }
  __device__ __forceinline__ void values(int64_t v, const Raw& w, float (&x)[VEC]) const {
    const int64_t i = v - off;
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = value(w.e[k]);
    if (i < 0 || i + VEC > V) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = i + k >= 0 && i + k < V ? x[k] : -INFINITY;
    }
    if (infinite) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = seen(x[k]);
    }
  }
  __device__ __forceinline__ void run(int64_t v, float (&x)[VEC]) const { values(v, load(v), x); }
  // (without the bits that are the same in all: few digits tell two orders apart)
  static constexpr int SAME = std::is_same_v<LT, float> ? 0 : std::is_same_v<LT, uint16_t> ? 16 : 13;
  static __device__ __forceinline__ uint64_t order(float x, int64_t i) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return (uint64_t)((u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u)) >> SAME) << INDEX | (~(uint32_t)i & LAST_INDEX);
  }
  __device__ __forceinline__ double real(float x, const Pow2& tab) const {  // (2^-1000 for -infinity)
    return nsx_pow2(fmax((double)x - (double)M, least), scale2, tab);
  }
  __device__ __forceinline__ uint64_t whole(double w) const {  // in units, to the nearest: the last bits of a sum with 2^52
    return __builtin_bit_cast(uint64_t, fma(w, unit, 0x1p52)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ uint64_t weight(float x, const Pow2& tab) const { return whole(real(x, tab)); }
  // How many 16ths of an octave below M a logit lies: 32-bit operations that never fall as x does; and the bin that it is in.
  __device__ __forceinline__ float depth(float x) const {
    return (M - x) * scale32;
  }
  static __device__ __forceinline__ int bin_at(float depth) { return depth < BINS - 1 ? (int)depth : BINS - 1; }
  __device__ __forceinline__ int bin(float x) const { return bin_at(depth(x)); }
};

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
// Wave-wide operations on DPP moves and readlanes: no trip through LDS.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {  // lanes without a source, or outside ROWS, get 0
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {  // of the lanes up to this one
  v += dpp64<0x111, 0xf>(v);  // row_shr
  v += dpp64<0x112, 0xf>(v);
  v += dpp64<0x114, 0xf>(v);
  v += dpp64<0x118, 0xf>(v);
  v += dpp64<0x142, 0xa>(v);  // row_bcast:15 into the odd rows
  v += dpp64<0x143, 0xc>(v);  // row_bcast:31 into the upper half
  return v;
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int i) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), i) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, i);
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) { return lane64(wave_scan(v), 63); }
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
  const uint32_t hi = nsx_wave_max_u32((uint32_t)(v >> 32));
  return (uint64_t)hi << 32 | nsx_wave_max_u32((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0);
}
constexpr int NW = THREADS / 64;
// The workgroup's largest v / the sum of the threads before this one with the whole sum; s: NW words of LDS, free again behind
// the call.
__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* s) {
  v = wave_max64(v);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) v = max64(v, s[i]);
  __syncthreads();
  return v;
}
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* s, uint64_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t x = wave_scan(v);
  if (lane == 63) s[wave] = x;
  __syncthreads();
  uint64_t before = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    before += i < wave ? s[i] : 0;
    all += s[i];
  }
  __syncthreads();
  return before + x - v;
}

// What a workgroup reads of the passes before, all of it on its way before the first of it is waited for: the row's largest
// orders, one per workgroup, and the histogram.
struct Known {
  static constexpr int PER = BINS / THREADS;
  uint64_t best = 0, mass[PER];
  uint32_t many[PER];
  __device__ __forceinline__ Known(const SampleArgs& a, int64_t row, bool cut) {
    for (int i = threadIdx.x; i < a.groups; i += THREADS) best = max64(best, a.best[row * a.groups + i]);
    if (cut) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        mass[i] = a.mass[row * BINS + threadIdx.x * PER + i];
        many[i] = a.many[row * BINS + threadIdx.x * PER + i];
      }
    }
  }
};

// f(part, index of the first, logits) for the workgroup's share of a row's parts, a thread VEC logits of each, the next part's
// on their way meanwhile.
template <typename LT, typename F>
__device__ __forceinline__ void each_part(const SampleArgs& a, const Row<LT>& r, F f) {
  typename Row<LT>::Raw next = r.load((int64_t)blockIdx.x * PART + threadIdx.x * VEC);
  for (int part = blockIdx.x; part < a.parts; part += gridDim.x) {
    const int64_t v = (int64_t)part * PART + threadIdx.x * VEC;
    const typename Row<LT>::Raw now = next;
    if (part + (int)gridDim.x < a.parts) next = r.load(v + (int64_t)gridDim.x * PART);
    float x[VEC];
    r.values(v, now, x);
    f(part, v - r.off, x);
  }
}

template <typename LT>
__global__ __launch_bounds__(THREADS) void best_kernel(SampleArgs a) {
  __shared__ uint64_t s[NW];
  const int64_t row = blockIdx.y;
  const Row<LT> r(a, row);
  if (a.mass)
    for (int i = blockIdx.x * THREADS + threadIdx.x; i < BINS; i += gridDim.x * THREADS) {
      a.mass[row * BINS + i] = 0;
      a.many[row * BINS + i] = 0;
      if (i == 0) a.listed[row] = 0;
    }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.ended[row] = 0;
  // (a thread keeps the eight logits among which its largest is, and looks for that one's place behind the last)
  typename Row<LT>::Raw next = r.load((int64_t)blockIdx.x * PART + threadIdx.x * VEC), held = next;
  float most = -INFINITY;
  int64_t from = 0;
  for (int part = blockIdx.x; part < a.parts; part += gridDim.x) {
    const int64_t v = (int64_t)part * PART + threadIdx.x * VEC;
    const typename Row<LT>::Raw now = next;
    if (part + (int)gridDim.x < a.parts) next = r.load(v + (int64_t)gridDim.x * PART);
    float x[VEC], top = most;
    r.values(v, now, x);
#pragma unroll
    for (int k = 0; k < VEC; ++k) top = fmaxf(top, x[k]);
    if (top > most) most = top, from = v, held = now;
  }
  uint64_t best = 0;
  if (most > -INFINITY) {
    float x[VEC];
    r.values(from, held, x);
    int at = 0;
#pragma unroll
    for (int k = 1; k < VEC; ++k) at = x[k] > x[0] ? (x[0] = x[k], k) : at;
    best = Row<LT>::order(most, from - r.off + at);
  }
  best = block_max(best, s);
  if (threadIdx.x == 0) a.best[row * a.groups + blockIdx.x] = best;
}

template <typename LT>
__global__ __launch_bounds__(THREADS) void bins_kernel(SampleArgs a) {
  __shared__ uint64_t s[NW], mass[BINS];
  __shared__ uint32_t many[BINS];
  __shared__ Pow2 tab;
  const int64_t row = blockIdx.y;
  Row<LT> r(a, row);
  if (!r.cut()) return;
  const Known known(a, row, false);
  tab.fill();
  for (int i = threadIdx.x; i < BINS; i += THREADS) mass[i] = 0, many[i] = 0;
  r.largest(block_max(known.best, s));  // (its barriers order the clearing as well)
  if (!r.drawn()) return;
  const bool few = r.few();
  each_part(a, r, [&](int, int64_t, const float (&x)[VEC]) {
    if (few) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (x[k] > -INFINITY) atomicAdd(&many[r.bin(x[k])], 1u);
      return;
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const uint64_t w = r.weight(x[k], tab);
      if (w) {
        const int b = r.bin(x[k]);
        atomicAdd((unsigned long long*)&mass[b], (unsigned long long)w);
        if (r.top_k) atomicAdd(&many[b], 1u);
      }
    }
  });
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS) {
    if (mass[i]) atomicAdd((unsigned long long*)&a.mass[row * BINS + i], (unsigned long long)mass[i]);
    if (many[i]) atomicAdd(&a.many[row * BINS + i], many[i]);
  }
}

// Where a row's filters end, as far as its histogram tells.
struct Ends {
  int kbin, plo, phi;         // top-k's last bin; the bins that top-p's may be; BINS: no such filter
  uint64_t above_k, above_p;  // the weight above kbin, above plo
  uint32_t before_k;          // the number of tokens above kbin
  uint64_t all;               // the whole weight
  template <typename LT>
  __device__ __forceinline__ void find(const Row<LT>& r, const Known& known, uint64_t* s, Ends* shared) {
    constexpr int PER = Known::PER;
    if (threadIdx.x == 0) *shared = Ends{BINS, BINS, BINS, 0, 0, 0, 0};
    uint64_t am = 0, cm = 0, bm = 0;
    if (!r.few()) {
      uint64_t sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += known.mass[i];
      cm = bm = block_scan(sum, s, am);
    }
    if (r.top_k) {
      uint64_t sum = 0, all;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += known.many[i];
      uint64_t cn = block_scan(sum, s, all);
#pragma unroll
      for (int i = 0; i < PER; ++i) {  // (one thread finds it, if any)
        const uint64_t m = r.few() ? 0 : known.mass[i];
        if (cn < (uint64_t)r.top_k && cn + known.many[i] >= (uint64_t)r.top_k) {
          shared->kbin = threadIdx.x * PER + i;
          shared->above_k = cm;
          shared->before_k = (uint32_t)cn;
          shared->all = cm + m;
        }
        cm += m, cn += known.many[i];
      }
    }
    __syncthreads();
    Ends e = *shared;
    if (r.few()) {  // (no weights are known: every token down to kbin is open)
      const int kbin = e.kbin < BINS ? e.kbin : BINS - 1;
      *this = Ends{uniform(kbin), 0, uniform(kbin), 0, 0, 0, 0};
      return;
    }
    __syncthreads();
    if (e.kbin == BINS) e.above_k = e.all = am;
    if (r.top_p < 1.0) {
      // (what top-k leaves lies between above_k and all)
      const uint64_t lo = r.target(e.kbin == BINS ? e.all : e.above_k), hi = r.target(e.all);
      cm = bm;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint64_t m = known.mass[i];
        if (cm < lo && cm + m >= lo) shared->plo = threadIdx.x * PER + i, shared->above_p = cm;
        if (cm < hi && cm + m >= hi) shared->phi = threadIdx.x * PER + i;
        cm += m;
      }
      __syncthreads();
      e.plo = shared->plo, e.phi = shared->phi, e.above_p = shared->above_p;
    }
    e.all = e.kbin == BINS ? am : 0;
    *this = e;
    kbin = uniform(kbin), plo = uniform(plo), phi = uniform(phi);
  }
  __device__ __forceinline__ int last() const { return kbin < BINS ? kbin : phi; }  // bin that is sure or open
  __device__ __forceinline__ bool sure(int bin) const { return bin < kbin && bin < plo; }
  __device__ __forceinline__ bool open(int bin) const { return bin == kbin || (bin >= plo && bin <= phi && bin <= kbin); }
};

// Among tokens, the order of the one with which their sum from the highest on reaches `want`; 0 where all of them do not.
// each(f): f(order, weight) for every token, by whichever threads. By digits of 10 bits of what an order lies above the lowest,
// from the highest bit that one has, until the digits are all or few tokens are left.
constexpr int DIGIT = 10;
struct Pick {
  uint64_t s[NW], t[NW], mass[1 << DIGIT], above, order[64], weight[64];
  uint32_t many[1 << DIGIT], n;
  int digit;
};
struct Rank {
  uint64_t order[RANK], k_order[RANK], weight[RANK], before[RANK];
  uint32_t many[RANK];
};
template <typename Each>
__device__ __forceinline__ uint64_t pick_order(Pick& p, uint64_t want, Each each) {
  uint64_t above = 0, lo = 0, hi = 0;  // lo: the largest complement
  each([&](uint64_t o, uint64_t) { hi = max64(hi, o), lo = max64(lo, ~o); });
  hi = wave_max64(hi), lo = wave_max64(lo);
  if ((threadIdx.x & 63) == 0) p.s[threadIdx.x >> 6] = hi, p.t[threadIdx.x >> 6] = lo;
  for (int i = threadIdx.x; i < 1 << DIGIT; i += THREADS) p.mass[i] = 0, p.many[i] = 0;
  if (threadIdx.x == 0) p.digit = -1, p.n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) hi = max64(hi, p.s[i]), lo = max64(lo, p.t[i]);
  lo = ~lo;
  if (hi == lo) {
    __syncthreads();
    return hi;
  }
  int shift = hi < lo ? 0 : 64 - __clzll((long long)(hi - lo)), bits = 0;  // digits of orders in [lo, lo + 2^shift) (2^64: all)
  while (true) {
    const int width = shift < DIGIT ? shift : DIGIT;
    shift -= width;
    bits = width;
    each([&](uint64_t o, uint64_t w) {
      const uint64_t d = (o - lo) >> shift;
      if (o < lo || d >> bits) return;
      atomicAdd((unsigned long long*)&p.mass[d], (unsigned long long)w);
      atomicAdd(&p.many[d], 1u);
    });
    __syncthreads();
    // from the largest digit down: the first at which the running sum reaches what is wanted
    constexpr int PER = (1 << DIGIT) / THREADS;
    uint64_t m[PER], sum = 0, all;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += m[i] = p.mass[(1 << DIGIT) - 1 - threadIdx.x * PER - i];
    uint64_t run = above + block_scan(sum, p.s, all);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (run < want && run + m[i] >= want) {
        p.digit = (1 << DIGIT) - 1 - threadIdx.x * PER - i;
        p.above = run;
      }
      run += m[i];
    }
    __syncthreads();
    const int d = p.digit;
    if (d < 0) return 0;
    above = p.above;
    const uint32_t n = p.many[d];
    lo += (uint64_t)d << shift;
    if (n <= 64) {  // few: each with each, a lane one token, the same in all waves
      each([&](uint64_t o, uint64_t w) {
        if (o < lo || (o - lo) >> shift) return;
        const uint32_t i = atomicAdd(&p.n, 1u);
        p.order[i] = o, p.weight[i] = w;
      });
      __syncthreads();
      const uint32_t lane = threadIdx.x & 63;
      const uint64_t o = lane < n ? p.order[lane] : 0, w = lane < n ? p.weight[lane] : 0;
      uint64_t run = above;
      for (uint32_t j = 0; j < n; ++j) run += p.order[j] > o ? p.weight[j] : 0;
      return lane64(o, __builtin_amdgcn_readfirstlane(__ffsll(__ballot(w && run < want && run + w >= want)) - 1));
    }
    if (shift == 0) return lo;
    __syncthreads();
    for (int i = threadIdx.x; i < 1 << DIGIT; i += THREADS) p.mass[i] = 0, p.many[i] = 0;
    if (threadIdx.x == 0) p.digit = -1;
    __syncthreads();
  }
}

// What a row's last step holds in LDS.
struct Draw {
  Pick p;
  Rank rank;
  uint64_t sums[MAX_PARTS];
  int found;
};
// What other workgroups of the same launch (SAME) or of the one before wrote.
template <bool SAME, typename T>
__device__ __forceinline__ T fetch(const T* p) {
  return SAME ? __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *p;
}
// A row's token, by one workgroup, from what its parts' workgroups found: their sums, in d.sums, and the n listed tokens, of which
// `first` are this thread's.
template <typename LT, bool SAME>
__device__ __forceinline__ void draw(const SampleArgs& a, int64_t row, const Row<LT>& r, const Ends& e, bool cut, const Pow2& tab,
                                     Draw& d, uint32_t n, const uint32_t (&first)[HELD]) {
  Pick& p = d.p;
  Rank& rank = d.rank;
  uint64_t* sums = d.sums;
  const uint32_t* list = a.list + row * LIST;
  uint64_t last = 0;  // the order of the last token that the filters keep
  if (cut) {
    // f(order, weight, bin, whether min-p keeps it) for the listed tokens: held in registers; or where they are more, taken
    // from the list, or from all of the row's in those bins
    uint64_t ho[HELD] = {}, hw[HELD] = {};
    int hb[HELD];
    bool hk[HELD];
    auto look = [&](uint32_t t, uint64_t& o, uint64_t& w, int& b, bool& keep) {
      const float x = r.at(t);
      const double y = r.real(x, tab);
      o = Row<LT>::order(x, t), w = r.whole(y), b = r.bin(x), keep = !(y < r.min_p);
    };
    if (n <= HELD * THREADS) {
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (threadIdx.x + i * THREADS < n) look(first[i], ho[i], hw[i], hb[i], hk[i]);
    }
    auto tokens = [&](auto f) {
      if (n <= HELD * THREADS) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
          if (hw[i]) f(ho[i], hw[i], hb[i], hk[i]);
      } else {
        const int64_t end = n <= LIST ? n : a.V;
#pragma unroll 1
        for (int64_t i = threadIdx.x; i < end; i += THREADS) {
          uint64_t o, w;
          int b;
          bool keep;
          look(n <= LIST ? fetch<SAME>(list + i) : (uint32_t)i, o, w, b, keep);
          if (w && e.open(b)) f(o, w, b, keep);
        }
      }
    };
    uint64_t whole = e.all;
    // (of the few all are listed, of others those of the last bin)
    const int from = r.few() ? 0 : e.kbin;
    if (n <= RANK) {
      const int i = threadIdx.x % RANK;
      const bool mine = threadIdx.x < RANK && hw[0];
      const bool in_k = mine && e.kbin < BINS && hb[0] >= from && hb[0] <= e.kbin;
      const bool in_p = mine && hb[0] >= e.plo && hb[0] <= e.phi;
      if (threadIdx.x < RANK) {
        rank.order[i] = ho[0];
        rank.k_order[i] = in_k ? ho[0] : 0;
        rank.weight[i] = in_p ? hw[0] : 0;
        rank.before[i] = 0;
        rank.many[i] = 0;
      }
      __syncthreads();
      const uint64_t o = rank.order[i];
      uint64_t before = 0;
      uint32_t more = 0;
      if (o) {
        constexpr int SHARE = RANK * RANK / THREADS;
        const int from_j = threadIdx.x / RANK * SHARE;
#pragma unroll 8
        for (int j = from_j; j < from_j + SHARE; ++j) {  // (behind the last: order 0)
          more += rank.k_order[j] > o;
          before += rank.order[j] > o ? rank.weight[j] : 0;
        }
        if (more) atomicAdd(&rank.many[i], more);
        if (before) atomicAdd((unsigned long long*)&rank.before[i], (unsigned long long)before);
      }
      __syncthreads();
      more = rank.many[i], before = rank.before[i];
      bool kept = mine && (!in_k || e.before_k + more < r.top_k);
      if (e.kbin < BINS) {
        block_scan(in_k && kept ? hw[0] : 0, p.s, whole);
        whole += e.above_k;
      }
      // (what is open past phi, of top-k's last bin, lies behind top-p's end)
      if (r.top_p < 1.0) kept = kept && in_p && e.above_p + before < r.target(whole);
      last = block_max(kept ? ~ho[0] : 0, p.s);
      last = last ? ~last : 0;
      if (kept && hk[0])
        atomicAdd((unsigned long long*)&sums[((~(uint32_t)ho[0] & LAST_INDEX) + r.off) / PART], (unsigned long long)hw[0]);
      __syncthreads();
    } else {
      if (e.kbin < BINS) {
        last = pick_order(p, (uint64_t)r.top_k - e.before_k, [&](auto f) {
          tokens([&](uint64_t o, uint64_t, int b, bool) {
            if (b >= from && b <= e.kbin) f(o, 1);
          });
        });
        uint64_t in = 0;
        tokens([&](uint64_t o, uint64_t w, int b, bool) {
          if (b >= from && b <= e.kbin && o >= last) in += w;
        });
        block_scan(in, p.s, whole);
        whole += e.above_k;
      }
      if (r.top_p < 1.0) {
        last = max64(last, pick_order(p, r.target(whole) - e.above_p, [&](auto f) {
          tokens([&](uint64_t o, uint64_t w, int b, bool) {
            if (b >= e.plo && b <= e.phi && o >= last) f(o, w);
          });
        }));
      }
      tokens([&](uint64_t o, uint64_t w, int, bool keep) {
        if (o >= last && keep)
          atomicAdd((unsigned long long*)&sums[((~(uint32_t)o & LAST_INDEX) + r.off) / PART], (unsigned long long)w);
      });
      __syncthreads();
    }
  }
  // the part in which the random number falls
  constexpr int PER = (MAX_PARTS + THREADS - 1) / THREADS;
  uint64_t sum = 0, total;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum += threadIdx.x * PER + i < a.parts ? sums[threadIdx.x * PER + i] : 0;
  uint64_t run = block_scan(sum, p.s, total);
  const double want = fmin(fmax((double)a.u[row] * (double)total, 0.0), (double)total);
  const uint64_t target = (uint64_t)want < total ? (uint64_t)want : total - 1;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int part = threadIdx.x * PER + i;
    const uint64_t m = part < a.parts ? sums[part] : 0;
    if (run <= target && run + m > target) {
      d.found = part;
      p.above = run;
    }
    run += m;
  }
  __syncthreads();
  const int part = d.found;
  if (part >= a.parts) return;  // (no weight is a number: does not happen)
  // and the token in it
  const int64_t v = (int64_t)part * PART + threadIdx.x * VEC;
  float x[VEC];
  r.run(v, x);
  uint64_t w[VEC];
  sum = 0;
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    w[k] = 0;
    if (Row<LT>::order(x[k], v - r.off + k) >= last) {  // (of a row cut short, few waves have one)
      const double y = r.real(x[k], tab);
      w[k] = y < r.min_p ? 0 : r.whole(y);
    }
    sum += w[k];
  }
  run = p.above;
  run += block_scan(sum, p.s, total);
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    if (run <= target && run + w[k] > target) a.token[row] = (int32_t)(v - r.off + k);
    run += w[k];
  }
}

// LAST: the last workgroup of a row goes on to its token. What it needs of the others they store past their caches, then count
// themselves.
template <typename LT, bool LAST>
__global__ __launch_bounds__(THREADS) void sums_kernel(SampleArgs a) {
  constexpr int OPEN = 2048;  // listed tokens of a workgroup; where they are more, the row is read again
  __shared__ uint64_t s[NW], sums[MAX_PARTS];
  __shared__ uint32_t list[OPEN], n, base;
  __shared__ Ends shared;
  __shared__ Pow2 tab;
  const int64_t row = blockIdx.y;
  Row<LT> r(a, row);
  const bool cut = a.mass && r.cut();
  const Known known(a, row, cut);
  tab.fill();
  if (threadIdx.x == 0) n = 0;
  for (int i = threadIdx.x; i < (a.parts - 1) / a.groups + 1; i += THREADS) sums[i] = 0;
  const uint64_t best = block_max(known.best, s);
  r.largest(best);
  if (!r.drawn()) {
    if (LAST && blockIdx.x == 0 && threadIdx.x == 0)
      a.token[row] = r.M > -INFINITY ? (int32_t)(~(uint32_t)best & LAST_INDEX) : -1;
    return;
  }
  Ends e{BINS, BINS, BINS, 0, 0, 0, 0};
  if (cut) e.find(r, known, s, &shared);
  const float deepest = e.last() < BINS - 1 ? (float)(e.last() + 1) : INFINITY;  // (one look tells most tokens from those kept)
  each_part(a, r, [&](int part, int64_t i, const float (&x)[VEC]) {
    uint64_t sum = 0;
    bool sure[VEC], any = false;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const float depth = r.depth(x[k]);
      const int b = Row<LT>::bin_at(depth);
      sure[k] = depth < deepest && e.sure(b);
      any |= sure[k];
      if (depth < deepest && e.open(b)) {
        const uint32_t at = atomicAdd(&n, 1u);
        if (at < OPEN) list[at] = (uint32_t)(i + k);
      }
    }
    if (__any(any)) {
#pragma unroll 4
      for (int k = 0; k < VEC; ++k) {
        const double w = r.real(x[k], tab);
        sum += sure[k] && !(w < r.min_p) ? r.whole(w) : 0;
      }
    }
    if (__any(sum != 0)) {
      sum = wave_sum64(sum);
      if ((threadIdx.x & 63) == 0) atomicAdd((unsigned long long*)&sums[part / a.groups], (unsigned long long)sum);
    }
  });
  __syncthreads();
  const uint32_t mine = n;
  if (mine && threadIdx.x == 0) base = atomicAdd(&a.listed[row], mine <= OPEN ? mine : LIST + 1);
  auto put = [](auto* p, auto v) {
    if constexpr (LAST) __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else *p = v;
  };
  for (int part = blockIdx.x + threadIdx.x * a.groups; part < a.parts; part += THREADS * a.groups)
    put(a.sums + row * a.parts + part, sums[part / a.groups]);
  if (mine) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < mine && i < OPEN; i += THREADS)
      if (base + i < LIST) put(a.list + row * LIST + base + i, list[i]);
  }
  if constexpr (LAST) {
    __shared__ Draw d;
    __shared__ bool last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (stored where every part of the chip sees it)
    __syncthreads();
    if (threadIdx.x == 0) {
      last = __hip_atomic_fetch_add(a.ended + row, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == a.groups - 1u;
      d.found = 0x7fffffff;
    }
    __syncthreads();
    if (!last) return;
    uint32_t first[HELD], count = 0;
    if (cut) {
      count = fetch<true>(a.listed + row);
#pragma unroll
      for (int i = 0; i < HELD; ++i) first[i] = fetch<true>(a.list + row * LIST + threadIdx.x + i * THREADS);
    }
    for (int i = threadIdx.x; i < a.parts; i += THREADS) d.sums[i] = fetch<true>(a.sums + row * a.parts + i);
    __syncthreads();
    draw<LT, true>(a, row, r, e, cut, tab, d, count, first);
  }
}

template <typename LT>
__global__ __launch_bounds__(THREADS) void draw_kernel(SampleArgs a) {
  __shared__ Draw d;
  __shared__ Ends shared;
  __shared__ Pow2 tab;
  const int64_t row = blockIdx.x;
  Row<LT> r(a, row);
  const bool cut = a.mass && r.cut();
  const Known known(a, row, cut);
  const uint32_t* list = a.list + row * LIST;
  uint32_t first[HELD], n = 0;
  if (cut) {
    n = a.listed[row];
#pragma unroll
    for (int i = 0; i < HELD; ++i) first[i] = list[threadIdx.x + i * THREADS];  // (as many as there are count)
  }
  tab.fill();
  for (int i = threadIdx.x; i < a.parts; i += THREADS) d.sums[i] = a.sums[row * a.parts + i];  // (of a drawn row)
  if (threadIdx.x == 0) d.found = 0x7fffffff;
  const uint64_t best = block_max(known.best, d.p.s);
  r.largest(best);
  if (!r.drawn()) {
    if (threadIdx.x == 0) a.token[row] = r.M > -INFINITY ? (int32_t)(~(uint32_t)best & LAST_INDEX) : -1;
    return;
  }
  Ends e{BINS, BINS, BINS, 0, 0, 0, 0};
  if (cut) e.find(r, known, d.p.s, &shared);
  draw<LT, false>(a, row, r, e, cut, tab, d, n, first);
}

int parts_of(int64_t vocab) { return (int)nsx_cdiv(vocab + VEC - 1, PART); }
int64_t up16(int64_t v) { return (v + 15) & ~15ll; }

template <typename LT>
int sample_launch(const SampleArgs& a, int64_t batch, bool cut, bool greedy, hipStream_t st) {
  const dim3 grid(a.groups, (unsigned)batch);
  if (const int rc = nsx_launch(best_kernel<LT>, grid, dim3(THREADS), 0, st, a)) return rc;
  if (cut)
    if (const int rc = nsx_launch(bins_kernel<LT>, grid, dim3(THREADS), 0, st, a)) return rc;
  if (!greedy && a.groups * batch <= FUSED) return nsx_launch(sums_kernel<LT, true>, grid, dim3(THREADS), 0, st, a);
  if (!greedy)
    if (const int rc = nsx_launch(sums_kernel<LT, false>, grid, dim3(THREADS), 0, st, a)) return rc;
  return nsx_launch(draw_kernel<LT>, dim3((unsigned)batch), dim3(THREADS), 0, st, a);
}

}  // namespace

extern "C" int64_t nsx_sample_workspace_bytes(int64_t batch, int64_t vocab) {
  if (batch <= 0 || vocab <= 0 || vocab > (1 << INDEX)) return -1;
  return batch * ((int64_t)parts_of(vocab) * 16 + BINS * 12 + LIST * 4) + up16(batch * 8);
}

extern "C" int nsx_sample(const void* logits, int logits_dtype, int64_t row_stride, int64_t batch, int64_t vocab,
                          const float* uniforms, const nsx_sampling* settings, int32_t* token, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  NSX_REQUIRE(logits_dtype == NSX_DT_F32 || logits_dtype == NSX_DT_F16 || logits_dtype == NSX_DT_BF16, NSX_ETYPE,
              "logits element type %d", logits_dtype);
  NSX_REQUIRE(batch >= 0 && batch < 65536 && vocab > 0 && vocab <= (1 << INDEX), NSX_EINVAL,
              "%lld rows of %lld logits (fewer than 65536, 1 to 4194304)", (long long)batch, (long long)vocab);
  NSX_REQUIRE(row_stride >= vocab, NSX_EINVAL, "rows %lld elements apart for %lld logits", (long long)row_stride,
              (long long)vocab);
  NSX_REQUIRE(settings, NSX_EINVAL, "null settings");
  const nsx_sampling& s = *settings;
  NSX_REQUIRE(s.temperatures || s.temperature == 0.0 || (s.temperature >= 1e-30 && s.temperature <= 1e30), NSX_EINVAL,
              "temperature %g (0, or 1e-30 to 1e30)", s.temperature);
  NSX_REQUIRE(s.top_ps || (s.top_p > 0.0 && s.top_p <= 1.0), NSX_EINVAL, "top_p %g (above 0, up to 1)", s.top_p);
  NSX_REQUIRE(s.min_ps || (s.min_p >= 0.0 && s.min_p <= 1.0), NSX_EINVAL, "min_p %g (0 to 1)", s.min_p);
  NSX_REQUIRE(s.top_ks || s.top_k >= 0, NSX_EINVAL, "top_k %lld", (long long)s.top_k);
  if (batch == 0) return NSX_OK;
  NSX_REQUIRE(logits && token && workspace, NSX_EINVAL, "null buffer");
  NSX_REQUIRE(uniforms || (!s.temperatures && s.temperature == 0.0), NSX_EINVAL, "a temperature above 0 needs uniforms");
  const int64_t need = nsx_sample_workspace_bytes(batch, vocab);
  NSX_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0, NSX_EINVAL,
              "workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)workspace_bytes, (long long)need);
  int bits = 62;  // (sums below 2^63; a weight below 2^52)
  while (bits > 0 && (1ll << (62 - bits)) < vocab) --bits;
  bits = std::min(bits, 51);
  const bool cut = s.top_ks || s.top_ps || s.top_k > 0 || s.top_p < 1.0, greedy = !s.temperatures && s.temperature == 0.0;
  const int parts = parts_of(vocab), groups = (int)std::min<int64_t>(parts, nsx_cdiv(GRID, batch));
  uint64_t *best = (uint64_t*)workspace, *sums = best + batch * parts, *mass = sums + batch * parts;
  uint32_t *many = (uint32_t*)(mass + batch * BINS), *list = many + batch * BINS, *listed = list + batch * LIST;
  const SampleArgs a{logits, row_stride, vocab, uniforms, s.temperature, s.top_p, s.min_p, s.top_k, s.temperatures,
                     s.top_ps, s.min_ps, s.top_ks, token, bits, parts, groups, best, sums, cut && !greedy ? mass : nullptr,
                     many, listed, listed + batch, list};
  hipStream_t st = (hipStream_t)stream;
  if (logits_dtype == NSX_DT_F32) return sample_launch<float>(a, batch, cut && !greedy, greedy, st);
  if (logits_dtype == NSX_DT_F16) return sample_launch<_Float16>(a, batch, cut && !greedy, greedy, st);
  return sample_launch<uint16_t>(a, batch, cut && !greedy, greedy, st);
}
