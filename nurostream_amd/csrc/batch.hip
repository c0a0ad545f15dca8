// Several sequences at once (gfx950): the new tokens' rows into a cache of 16 or 8 bits, finished rows into it and back, and
// attention over a prefix that all sequences share and the rows of their own.
//
// A cache row of 8 bits is codes c with one fp32 scale: x ~ c s, s the row's largest magnitude over the type's (127 for int8,
// 448 for e4m3). Codes of either type, and bf16 rows, are bf16 numbers exactly, so attention multiplies the codes themselves
// on the matrix cores and puts a key's scale to its score, a value row's to its weight.
//
// Times below are kernels' own, of replayed graphs or traces, on one MI355X; a large copy reaches 5.08 TB/s there (read and
// written), a large bf16 product 1375 TFLOP/s.
#include "nsx_common.h"

#include <algorithm>
#include <type_traits>
#include <math.h>

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LOWEST = -3.4028235e38f;  // a running maximum's start, finite: rows that see nothing weigh e^-infinity = 0

struct KvRows {
  void *k, *v;
  float *ks, *vs;
  const int32_t* pos;
  int64_t n_seq, ctx_max;
};

// --- element types ---------------------------------------------------------

struct Half {
  static constexpr int CODE = NSX_DT_F16;
  uint16_t bits;
};
struct Bf16 {
  static constexpr int CODE = NSX_DT_BF16;
  uint16_t bits;
};

// N consecutive elements (a vector access of N * sizeof(T) bytes) as fp32, and back
template <typename T, int N>
struct alignas(N * sizeof(T)) Vec {
  T e[N];
};
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(Half x) { return nsx_h2f(x.bits); }
__device__ __forceinline__ float to_f(Bf16 x) { return nsx_bf2f(x.bits); }
__device__ __forceinline__ void from_f(float& y, float x) { y = x; }
__device__ __forceinline__ void from_f(Half& y, float x) {
  asm("" : "+v"(x));  // the fp32 value, rounded: not one instruction with what made it, rounding once
  y.bits = (uint16_t)nsx_f2h(x);
}
__device__ __forceinline__ void from_f(Bf16& y, float x) { y.bits = (uint16_t)nsx_f2bf(x); }
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&x)[4]) {
  const Vec<T, 4> v = *(const Vec<T, 4>*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = to_f(v.e[i]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&x)[4]) {
  Vec<T, 4> v;
#pragma unroll
  for (int i = 0; i < 4; ++i) from_f(v.e[i], x[i]);
  *(Vec<T, 4>*)p = v;
}

// A row of D elements lies in D / 8 lanes, lane l's elements 4 l .. and D / 2 + 4 l .. (the partners of a rotation are one
// lane's). Reductions over those lanes by DPP moves.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int LANES, typename Op>
__device__ __forceinline__ uint32_t row_all(uint32_t v, Op op) {
  v = op(v, dpp_u<0xB1>(v));   // quad_perm: lane ^ 1
  v = op(v, dpp_u<0x4E>(v));   // lane ^ 2
  v = op(v, dpp_u<0x141>(v));  // row_half_mirror: the other quad of 8
  if constexpr (LANES == 16) v = op(v, dpp_u<0x140>(v));  // row_mirror: the other half of 16
  return v;
}
template <int LANES>
__device__ __forceinline__ float row_sum(float x) {
  return __builtin_bit_cast(float, row_all<LANES>(__builtin_bit_cast(uint32_t, x), [](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
  }));
}
template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  return row_all<LANES>(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

__device__ __forceinline__ uint32_t near2(float lo, float hi) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{lo, hi}), b2));
}
// The codes of a lane's 8 elements of a row, and the row's scale. The largest is taken of the elements' bits, which order NaN
// above infinity above every number. A code is the quotient by the scale, to fp32's nearest, then to the code's: the product with
// the scale's reciprocal (the nearest as well) and one correction by what it leaves, exact in a fused multiply-add, so that
// an element that is half of a step lies where a division puts it. Scales below 2^-60, beside which what a product leaves
// may end below the least number, are divided by.
template <int KV, int D>
__device__ __forceinline__ void codes8(const float (&x)[8], uint32_t (&c)[2], float& scale) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu;
    m = u > m ? u : m;
  }
  m = row_max<D / 8>(m);
  constexpr float TOP = KV == NSX_KV_INT8 ? 127.f : 448.f;
  const bool finite = m < 0x7f800000u;
  const float s = __builtin_bit_cast(float, m) / TOP, r = 1.f / s;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float z = x[i] * r;
    y[i] = fmaf(fmaf(-z, s, x[i]), r, z);
  }
  if (!(s >= 0x1p-60f) || !finite) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = finite && s > 0.f ? fminf(fmaxf(x[i] / s, -TOP), TOP) : 0.f;
      asm volatile("" : "+v"(y[i]));  // (a branch: few rows take it)
    }
  }
  scale = finite ? s : __builtin_nanf("");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (KV == NSX_KV_INT8) {
      uint32_t z[4];  // 1.5 * 2^23 more: the nearest whole number's low byte in the lowest one
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = __builtin_bit_cast(uint32_t, y[4 * h + i] + 12582912.f);
      c[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(z[3], z[2], 0x0c0c0400u),
                                   __builtin_amdgcn_perm(z[1], z[0], 0x0c0c0400u), 0x05040100u);
    } else {
      const int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
      c[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], w, true);
    }
  }
}
// A row's 8 elements per lane (4 l .., D / 2 + 4 l ..) into a cache: rounded to bf16, or as codes with the row's scale.
template <int KV, int D>
__device__ __forceinline__ void put_row(void* rows, float* scales, int64_t row, int l, const float (&x)[8]) {
  if constexpr (KV == NSX_DT_BF16) {
    uint16_t* p = (uint16_t*)rows + row * D + 4 * l;
    *(v2u*)p = v2u{near2(x[0], x[1]), near2(x[2], x[3])};
    *(v2u*)(p + D / 2) = v2u{near2(x[4], x[5]), near2(x[6], x[7])};
  } else {
    uint32_t c[2];
    float s;
    codes8<KV, D>(x, c, s);
    uint8_t* p = (uint8_t*)rows + row * D + 4 * l;
    *(uint32_t*)p = c[0];
    *(uint32_t*)(p + D / 2) = c[1];
    if (l == 0) scales[row] = s;
  }
}
// The values of 4 codes, without the scale.
template <int KV>
__device__ __forceinline__ void codes4(uint32_t w, float (&x)[4]) {
  if constexpr (KV == NSX_KV_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  } else {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  }
}
// Row `row` of a cache, elements 4 l .. and D / 2 + 4 l ..
template <int KV, int D>
__device__ __forceinline__ void get_row(const void* rows, const float* scales, int64_t row, int l, float (&x)[8]) {
  float a[4], b[4], s = 1.f;
  if constexpr (KV == NSX_DT_BF16) {
    const Bf16* p = (const Bf16*)rows + row * D + 4 * l;
    load4(p, a);
    load4(p + D / 2, b);
  } else {
    const uint8_t* p = (const uint8_t*)rows + row * D + 4 * l;
    const uint32_t w0 = *(const uint32_t*)p, w1 = *(const uint32_t*)(p + D / 2);
    s = scales[row];
    codes4<KV>(w0, a);
    codes4<KV>(w1, b);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i] * s, x[4 + i] = b[i] * s;
}

// --- rows into the cache and back ------------------------------------------

struct AppendArgs {
  const void* qkv;
  const float *qb, *kb, *vb, *qn, *kn, *inv;
  float eps, amp;
  int H, G, passes;
  int64_t n;
  const int32_t *counts, *prefix;
  KvRows kv;
  void* q;
};

// x + bias; of a query or key head, with norm weights w, x <- x w / sqrt(mean(x^2) + eps); then (a, b) <- (a cos - b sin, b cos
// + a sin) of partners d / 2 apart, at position * inv_freq; queries out in the input's type, rows into the cache. All of a row
// lies in one row of lanes' registers from the first load to the stores, in fp32: everything is read and written once.
//
// A workgroup takes a token and 256 / (D / 8) of its heads at a time, so that its angles are computed once: the sine of a
// position's 64-bit angle costs what some hundred fp32 operations do. `passes` of such heads follow each other in a workgroup
// where tokens alone fill the chip: bf16 tokens of 80 heads of 64 into int8, one pass / all of them in a workgroup: 64 tokens
// 3.0 / 4.0 us, 512 4.6 / 4.7, 4001 16.7 / 14.9. Few tokens are bound by the launch (one: 2.6 us), many by memory: 4001 fp32
// tokens 25.7 us, where a copy of their 152 MB takes 29.9 (part of them stays in the caches).
template <typename XT, int KV, int D>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES;
  __shared__ float2 turn[D / 2];
  const int64_t tok = blockIdx.x, b = tok / a.n, j = tok - b * a.n;
  const bool live = !a.counts || j < a.counts[b];
  const int64_t row = (int64_t)a.kv.pos[b] + j, at = row + (a.prefix ? *a.prefix : 0);
  if (threadIdx.x < D / 2) {
    // the angle in 64 bits, less its whole turns: far positions are many of them
    double t = (double)at * (double)a.inv[threadIdx.x];
    t -= rint(t * 0.15915494309189533577) * 6.2831853071795864769;
    float s, c;
    sincosf((float)t, &s, &c);
    turn[threadIdx.x] = float2{c * a.amp, s * a.amp};
  }
  __syncthreads();
  const int l = threadIdx.x % LANES, heads = a.H + 2 * a.G;
  for (int i = 0; i < a.passes; ++i) {
    const int h = (blockIdx.y * a.passes + i) * ROWS + threadIdx.x / LANES;
    if (h >= heads) return;
    const XT* src = (const XT*)a.qkv + (tok * heads + h) * D + 4 * l;
    float lo[4], hi[4];
    load4(src, lo);
    load4(src + D / 2, hi);
    const bool isq = h < a.H, isv = h >= a.H + a.G;
    const float* bias = isq ? a.qb : isv ? a.vb : a.kb;
    const int g = isq ? h : isv ? h - a.H - a.G : h - a.H;
    if (bias) {
      float x[4];
      load4(bias + g * D + 4 * l, x);
#pragma unroll
      for (int k = 0; k < 4; ++k) lo[k] += x[k];
      load4(bias + g * D + D / 2 + 4 * l, x);
#pragma unroll
      for (int k = 0; k < 4; ++k) hi[k] += x[k];
    }
    if (!isv) {
      const float* norm = isq ? a.qn : a.kn;
      if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) ss = fmaf(lo[k], lo[k], fmaf(hi[k], hi[k], ss));
        const float r = 1.f / sqrtf(row_sum<LANES>(ss) / D + a.eps);
        float w[4];
        load4(norm + 4 * l, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) lo[k] = lo[k] * r * w[k];
        load4(norm + D / 2 + 4 * l, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) hi[k] = hi[k] * r * w[k];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 t = turn[4 * l + k];
        const float z = fmaf(lo[k], t.x, -(hi[k] * t.y));
        hi[k] = fmaf(hi[k], t.x, lo[k] * t.y);
        lo[k] = z;
      }
    }
    if (isq) {
#pragma unroll
      for (int k = 0; k < 4; ++k) lo[k] = live ? lo[k] : 0.f, hi[k] = live ? hi[k] : 0.f;
      XT* q = (XT*)a.q + (tok * a.H + h) * D + 4 * l;
      store4(q, lo);
      store4(q + D / 2, hi);
    } else if (live && row >= 0 && row < a.kv.ctx_max) {
      const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      put_row<KV, D>(isv ? a.kv.v : a.kv.k, isv ? a.kv.vs : a.kv.ks, (b * a.G + g) * a.kv.ctx_max + row, l, x);
    }
  }
}

struct RowsArgs {
  void *k, *v;  // [n_seq][G][n][D]
  KvRows kv;
  const int32_t* start;
  int64_t start0, n, rows;
  int G;
};

// 8 consecutive elements as they lie
template <typename T>
struct alignas(16) Eight {
  T e[8];
};
// A lane takes 8 consecutive elements of a row, D / 8 lanes a row, a thread RPT rows: all of their loads at once. Bound by
// memory: 4 x 16000 rows of 8 heads of 64, k and v: bf16 into int8 38.9 us and back 33.4, of 32.7 that a copy of the same 166
// MB takes (with a row a thread 53). 37 rows are launches: 2.5 and 2.7 us.
template <typename XT, int KV, int D, bool STORE, int RPT>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES;
  const int l = threadIdx.x % LANES;
  const bool v = blockIdx.y;
  XT* x = (XT*)(v ? a.v : a.k);
  uint8_t* cache = (uint8_t*)(v ? a.kv.v : a.kv.k);
  float* scales = v ? a.kv.vs : a.kv.ks;
  const uint32_t n = (uint32_t)a.n, first = blockIdx.x * (ROWS * RPT) + threadIdx.x / LANES, rows = (uint32_t)a.rows;
  using Code = std::conditional_t<KV == NSX_DT_BF16, v4u, v2u>;
  Eight<XT> in[RPT] = {};
  Code code[RPT] = {};
  float scale[RPT];
  int64_t at[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const uint32_t r = min(first + ROWS * i, rows - 1), bg = r / n, b = bg / (uint32_t)a.G;
    const int64_t row = (a.start ? (int64_t)a.start[b] : a.start0) + (r - bg * n);
    at[i] = first + ROWS * i < rows && row >= 0 && row < a.kv.ctx_max ? (int64_t)bg * a.kv.ctx_max + row : -1;
    if constexpr (STORE) {
      in[i] = *(const Eight<XT>*)(x + (int64_t)r * D + 8 * l);
    } else if (at[i] >= 0) {
      code[i] = *(const Code*)(cache + (at[i] * D + 8 * l) * (int)(sizeof(Code) / 8));
      scale[i] = KV == NSX_DT_BF16 ? 1.f : scales[at[i]];
    }
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    float y[8];
    if constexpr (STORE) {
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = to_f(in[i].e[k]);
      if constexpr (KV == NSX_DT_BF16) {
        const v4u w{near2(y[0], y[1]), near2(y[2], y[3]), near2(y[4], y[5]), near2(y[6], y[7])};
        if (at[i] >= 0) *(Code*)(cache + (at[i] * D + 8 * l) * 2) = w;
      } else {
        uint32_t c[2];
        float s;
        codes8<KV, D>(y, c, s);  // (every lane of a row has the same `at`)
        if (at[i] >= 0) {
          *(Code*)(cache + at[i] * D + 8 * l) = v2u{c[0], c[1]};
          if (l == 0) scales[at[i]] = s;
        }
      }
    } else if (first + ROWS * i < rows) {
      float lo[4], hi[4];
      if constexpr (KV == NSX_DT_BF16) {
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = nsx_bf2f(code[i][k >> 1] >> (16 * (k & 1)) & 0xffffu);
      } else {
        codes4<KV>(code[i][0], lo);
        codes4<KV>(code[i][1], hi);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = lo[k] * scale[i], y[4 + k] = hi[k] * scale[i];
      }
      Eight<XT> out;
#pragma unroll
      for (int k = 0; k < 8; ++k) from_f(out.e[k], at[i] >= 0 ? y[k] : 0.f);
      *(Eight<XT>*)(x + ((int64_t)first + ROWS * i) * D + 8 * l) = out;
    }
  }
}

// --- attention ---------------------------------------------------------------
//
// out = sum_t 2^(s_t - m) v_t / (sum_t 2^(s_t - m) + 2^(sink - m)), s_t = q . k_t scale log2(e), in one pass over the keys with
// a running reference m and sum, all in fp32.
//
// The heads of a kv head, times the tokens, times (for the shared prefix) the sequences are the rows of one product: 64
// sequences of 8 heads each make 512 rows, for which a prefix's keys are read once. Operations bind where rows are many (64
// tokens behind 32768 rows: 34.7 GFLOP, 25 us of the matrix cores' time against 12 us of the bytes'), launches and latency
// where they are few.
//
// A wave takes 32 rows, on v_mfma_f32_32x32x16_bf16. S = K Q^T, not Q K^T: the 16 scores that a lane then holds are of one row,
// so that maxima and sums need one exchange between lane halves, and the weights are at once the second operand of V^T W^T,
// without a trip through LDS. K's and V's rows lie in LDS as bf16, V's read transposed on the way (ds_read_b64_tr_b16).
//
// Queries and weights are NT bf16 terms: bf16 queries are themselves and their weights are rounded to bf16 (2^-8 of one at
// most, as the output is); fp16's 11 bits are two terms of 8 exactly, weights 16 bits of theirs; fp32's 24 bits are three,
// exactly. More terms are more products, not more reads.
//
// What it runs at: 64 bf16 tokens of 64 heads of 64 behind 32768 e4m3 rows 64 us (540 TFLOP/s): of the CUs' busy cycles the
// vector units work in 77 % (per score a scale, half a maximum, an exponential of 4 issue slots, a sum, a scale, half a
// rounding), the matrix cores in 32 %: the two overlap in part only, with 3 waves a SIMD. 4 x 512 tokens of 32 heads of 128
// behind 2000 bf16 rows 75 us (760 TFLOP/s): 48 % and 42 % of busy cycles, each wave's chain of products, exponentials and
// products bound by itself: sharing the rows of ragged sequences out evenly over the workgroups made no difference. (A card that
// has been at work for some time; from rest the first calls of these two take 69 and 96 us, calls that are waited for 66 and 86.)
// fp32 queries, three products for one: 256 tokens of 64 heads of 64 behind 32000 bf16 rows 335 us, of the 294 that the
// matrix cores take for 404 GFLOP; 64 tokens behind 32768 108 us of 76, where splits, the join and the exponentials show.

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
#define LDS_AS __attribute__((address_space(3)))

constexpr int AT_ROWS = 32;   // rows (tokens x heads of a kv head) of a wave
constexpr int AT_NW = 4;      // waves of a workgroup
constexpr int AT_MAX_SPLIT = 64;

struct AttnArgs {
  const void* q;
  KvRows kv, pre;  // pre.n_seq 0: none
  const int32_t* counts;
  const float* sinks;
  int H, G, rep, window;
  int64_t n;
  float scale2;  // scale * log2(e): the softmax is taken in powers of two
  float* part;   // [token][head][splits][D], then [token][head][splits] of (maximum, sum)
  void* out;
  // what rows are cut into: tiles of so many rows, splits of their keys
  struct Cut {
    int rows, tiles, splits;
  } pcut, ocut;
  int pblocks, splits;  // workgroups that take the prefix's keys alone; splits of all of a row's keys
};

// A cache row's elements as bf16, which holds all of their bits, 16 bytes of the row at a time.
template <int KV>
struct Codes {
  static constexpr int BYTES = KV == NSX_DT_BF16 ? 2 : 1, PER = 16 / BYTES;  // of an element; elements of 16 bytes
  static __device__ __forceinline__ void put(uint8_t* lds, v4u x) {
    if constexpr (KV == NSX_DT_BF16) {
      *(v4u*)lds = x;
    } else {
      v4u y[2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a, b;
        if constexpr (KV == NSX_KV_E4M3) {
          a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], 1.f, false));
          b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], 1.f, true));
        } else {
          float f[4];
          codes4<KV>(x[i], f);
          a = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[1]), __builtin_bit_cast(uint32_t, f[0]), 0x07060302u);
          b = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[3]), __builtin_bit_cast(uint32_t, f[2]), 0x07060302u);
        }
        y[i >> 1][2 * (i & 1)] = a;
        y[i >> 1][2 * (i & 1) + 1] = b;
      }
      *(v4u*)lds = y[0];
      *(v4u*)(lds + 16) = y[1];
    }
  }
};

// Two bf16 from the upper halves of two fp32; what they leave.
__device__ __forceinline__ uint32_t top2(float lo, float hi) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
}
__device__ __forceinline__ float below(float x) {
  return x - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u);
}
// 8 fp32 as NT bf16 terms: the first ones 8 bits each toward zero, the last one to the nearest (of three: exact).
template <int NT>
__device__ __forceinline__ void terms8(const float (&x)[8], v4u (&t)[NT]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      if (k + 1 < NT) {
        t[k][i] = top2(a, b);
        a = below(a), b = below(b);
      } else {
        t[k][i] = near2(a, b);
      }
    }
  }
}
__device__ __forceinline__ f16v dot(const v4u& a, const v4u& b, const f16v& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float other_half_max(float x) {  // the larger of lane and lane ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float other_half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// Rows that a workgroup's keys come from: the prefix's, or a sequence's own, of a kv head.
struct Source {
  const uint8_t *k, *v;
  const float *ks, *vs;
};
// Where a workgroup stands: rows r0 .. of a kv head's rows (all sequences' or, with `own`, sequence b's), which see keys of the
// prefix (source 0), of their sequence (1), or both, one after the other; its split of those keys.
struct Place {
  Source src[2];
  bool own, with[2];
  int g, split, splits, slot;  // kv head; split of so many; which of the splits of all of a row's keys
  int b, r0, rows;
  int P;  // the prefix's length
};
// Row r of a place (the last one's in place of those behind it): its token and head, and the keys [lo, hi) that it sees of
// each source.
struct Row {
  int tok, h, lo[2], hi[2];
  bool live;
  __device__ __forceinline__ Row(const AttnArgs& a, const Place& p, int r) {
    const uint32_t x = (uint32_t)min(r, p.rows - 1), t = x / (uint32_t)a.rep;
    tok = p.own ? p.b * (int)a.n + (int)t : (int)t;
    h = p.g * a.rep + (int)(x - t * (uint32_t)a.rep);
    const uint32_t b = p.own ? p.b : a.n == 1 ? t : t / (uint32_t)a.n, j = p.own ? t : a.n == 1 ? 0 : t - b * (uint32_t)a.n;
    const int64_t row = (int64_t)a.kv.pos[b] + j;
    live = !a.counts || (int)j < a.counts[b];
    const int64_t first = a.window > 0 ? p.P + row + 1 - a.window : 0;
    const int64_t end = row + 1 < 0 ? 0 : row + 1 < a.kv.ctx_max ? row + 1 : a.kv.ctx_max;
    hi[0] = p.with[0] ? p.P : 0;
    hi[1] = p.with[1] ? (int)end : 0;
    lo[0] = (int)(first < 0 ? 0 : first < hi[0] ? first : hi[0]);
    lo[1] = (int)(first < p.P ? 0 : first - p.P < hi[1] ? first - p.P : hi[1]);
  }
};

struct At {
  int tok, h;
  bool live;
};

// A row's (or split's) end: its maximum (of scores in powers of two), sum and D values over the sum's weights.
template <typename XT, int D>
struct End {
  const AttnArgs& a;
  const Place& p;
  __device__ __forceinline__ float* part(const At& r) const {
    return a.part + ((int64_t)(r.tok * a.H + r.h) * a.splits + p.slot) * D;
  }
  // The factor that values are stored with: 1 for a part, what divides by the whole sum for the answer. `any` false: zeros, of
  // a token that is not there or sees nothing, whatever the values are.
  struct Factor {
    float f;
    bool any;
  };
  __device__ __forceinline__ Factor factor(const At& r, float m, float l, bool first) const {
    if (a.splits > 1) {
      if (first) {
        float2* ml = (float2*)(a.part + (int64_t)(a.kv.n_seq * a.n * a.H) * a.splits * D);
        ml[(int64_t)(r.tok * a.H + r.h) * a.splits + p.slot] = float2{m, l};
      }
      return {1.f, true};
    }
    float f = 1.f;
    if (a.sinks) {
      const float sink = a.sinks[r.h] * LOG2E, M = fmaxf(m, sink);
      f = __builtin_amdgcn_exp2f(m - M);
      l = fmaf(l, f, __builtin_amdgcn_exp2f(sink - M));
    }
    return {f / l, r.live && l != 0.f};
  }
  // Values d .. d + 3
  __device__ __forceinline__ void store(const At& r, int d, const Factor& f, const float (&x)[4]) const {
    if (a.splits > 1) {
      *(v4f*)(part(r) + d) = v4f{x[0], x[1], x[2], x[3]};
    } else {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = f.any ? x[i] * f.f : 0.f;
      store4((XT*)a.out + (int64_t)(r.tok * a.H + r.h) * D + d, y);
    }
  }
};

// The keys of a workgroup: of each source's rows [from, to), those that any of its rows sees, in tiles, the tiles from `first`
// to `end` of both.
struct Range {
  int from[2], to[2], tiles[2], first, end;
  template <int KEYS>
  __device__ __forceinline__ void split(const Place& p, int round) {
#pragma unroll
    for (int i = 0; i < 2; ++i) tiles[i] = to[i] > from[i] ? (to[i] - from[i] + KEYS - 1) / KEYS : 0;
    const int all = tiles[0] + tiles[1], per = ((all + p.splits - 1) / p.splits + round - 1) / round * round;
    first = min(p.split * per, all);
    end = min(first + per, all);
  }
};

// A row once more, key by key and none that it does not see: for rows whose sums are not finite, as an infinity or a NaN
// beside a weight of zero makes them in a product of matrices. A wave's work.
template <typename XT, int KV, int D, int KEYS>
__device__ __forceinline__ void row_alone(const AttnArgs& a, const Place& p, const Range& w, int r) {
  const int lane = threadIdx.x & 63;
  const Row row(a, p, r);
  const XT* q = (const XT*)a.q + (int64_t)(row.tok * a.H + row.h) * D;
  float m = LOWEST, l = 0.f, acc[D / 64] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const Source src = p.src[i];
    const int t0 = i ? max(w.first - w.tiles[0], 0) : min(w.first, w.tiles[0]);
    const int t1 = i ? max(w.end - w.tiles[0], 0) : min(w.end, w.tiles[0]);
    const int lo = max(row.lo[i], w.from[i] + t0 * KEYS), hi = t1 > t0 ? min(row.hi[i], w.from[i] + t1 * KEYS) : 0;
#pragma unroll 1
    for (int t = lo; t < hi; t += 64) {
      const int key = t + lane;
      float s = -INFINITY;
      if (key < hi) {
        s = 0.f;
#pragma unroll 1
        for (int c = 0; c < D / 8; ++c) {
          float x[8], lo4[4], hi4[4];
          get_row<KV, D>(src.k, src.ks, key, c, x);
          load4(q + 4 * c, lo4);
          load4(q + D / 2 + 4 * c, hi4);
#pragma unroll
          for (int k = 0; k < 4; ++k) s = fmaf(lo4[k], x[k], fmaf(hi4[k], x[4 + k], s));
        }
        s *= a.scale2;
      }
      float M = s;
#pragma unroll
      for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
      M = fmaxf(M, m);
      const float e = key < hi ? __builtin_amdgcn_exp2f(s - M) : 0.f, f = __builtin_amdgcn_exp2f(m - M);
      l = l * f + nsx_wave_sum(e);
      m = M;
#pragma unroll
      for (int k = 0; k < D / 64; ++k) acc[k] *= f;
#pragma unroll 1
      for (int u = 0; u < min(64, hi - t); ++u) {
        const float eu = __shfl(e, u, 64);
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
          const int64_t at = (int64_t)(t + u) * D + lane + 64 * k;
          float x;
          if constexpr (KV == NSX_DT_BF16) {
            x = to_f(((const Bf16*)src.v)[at]);
          } else {
            float c[4];
            codes4<KV>(src.v[at], c);
            x = c[0] * src.vs[t + u];
          }
          acc[k] = fmaf(eu, x, acc[k]);
        }
      }
    }
  }
  const End<XT, D> end{a, p};
  const At at{row.tok, row.h, row.live};
  const auto f = end.factor(at, m, l, lane == 0);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    if (a.splits > 1) end.part(at)[lane + 64 * i] = acc[i];
    else from_f(((XT*)a.out + (int64_t)(row.tok * a.H + row.h) * D)[lane + 64 * i], f.any ? acc[i] * f.f : 0.f);
  }
}

// A stage of KEYS key rows and as many value rows in LDS, as bf16. Keys are read 16 bytes of each of 8 rows at once, values
// (transposed) 64 bytes of each of 4: pitches of 4 and of 16 (or 48) of the 64 banks past a multiple of them keep those apart.
template <int D>
struct Pitch {
  static constexpr int K = 2 * D + 16, V = D == 64 ? 192 : 320;
  static constexpr int stage(int keys) { return keys * (K + V); }
};

// A wave's 32 rows over its keys. Scores are K Q^T, so that a lane holds 16 of 32 keys' scores of one row (lane % 32; the
// other lane of the row holds the others), and its weights are at once the second operand of V^T W^T, of which it holds D / 2
// values of the same row. The operand's order of keys is the scores' own, and V's rows are read from LDS in it, transposed.
template <int KV, int D, int NT, int NB, bool FIRST>
struct Wave {
  v4u q[NT][D / 16];
  f16v acc[D / 32];
  float m, l;

  template <typename XT>
  __device__ __forceinline__ void start(const XT* row) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      if constexpr (NT == 1) {
        q[0][ks] = *(const v4u*)(row + 16 * ks + 8 * h);
      } else {
        float a[4], b[4];
        load4(row + 16 * ks + 8 * h, a);
        load4(row + 16 * ks + 8 * h + 4, b);
        const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        v4u t[NT];
        terms8<NT>(x, t);
#pragma unroll
        for (int k = 0; k < NT; ++k) q[k][ks] = t[k];
      }
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = f16v{};
    m = LOWEST;
    l = 0.f;
  }

  // NB blocks of 32 keys in LDS, the first of them key `key0` of its source; the lane's row sees [lo, hi) (`all`: these keys at
  // least).
  __device__ __forceinline__ void step(const uint8_t* kl, const uint8_t* vl, const float* sk, const float* sv, float c, bool all,
                                       int key0, int lo, int hi) {
    const int lane = threadIdx.x & 63, i32 = lane & 31, h = lane >> 5;
    f16v s[NB];
    v4u k[D / 16];
    // what codes' scores are taken from at once: the reference, or 0 where there is none yet
    const float from = KV == NSX_DT_BF16 || m == LOWEST ? 0.f : m;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) k[ks] = *(const v4u*)(kl + i32 * Pitch<D>::K + 32 * ks + 16 * h);
    if constexpr (D == 64) __builtin_amdgcn_sched_barrier(0);  // (all of them on their way before the first is waited for)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      s[nb] = f16v{};
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int t = NT - 1; t >= 0; --t) s[nb] = dot(k[ks], q[t][ks], s[nb]);
        if (nb + 1 < NB) k[ks] = *(const v4u*)(kl + (32 * (nb + 1) + i32) * Pitch<D>::K + 32 * ks + 16 * h);
      }
      if constexpr (KV != NSX_DT_BF16) {  // (a score's factor is its key's scale, which has the one of all in it)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const v4f f = *(const v4f*)(sk + 32 * nb + 2 * e + 4 * h);
#pragma unroll
          for (int x = 0; x < 4; ++x) s[nb][e + x] = fmaf(s[nb][e + x], f[x], -from);
        }
      }
    }
    if (!all) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = key0 + 32 * nb + 8 * (e >> 2) + 4 * h + (e & 3);
          float x = key >= lo && key < hi ? s[nb][e] : -INFINITY;
          asm volatile("" : "+v"(x));  // (a branch, not selects: few tiles take it)
          s[nb][e] = x;
        }
    }
    // The reference is an earlier maximum, moved only when a score is 8 above it: weights stay below 2^8, and the sums are
    // seldom rescaled (one look a stage: 68 us became 66 for 64 tokens behind 32768 e4m3 rows, 87 81 for prompts of 512).
    float most = s[0][0];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 16; e += 2) most = fmaxf(fmaxf(most, s[nb][e]), s[nb][e + 1]);
    most = other_half_max(most);
    most = KV == NSX_DT_BF16 ? most * c : most + from;
    if (__any(most > m + 8.f)) {
      const float to = fmaxf(most, m), by = __builtin_amdgcn_exp2f(m - to);
      if constexpr (KV != NSX_DT_BF16) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[nb][e] -= to - from;
      }
      m = to;
      l *= by;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] *= by;
    }
    // 16 keys at a time: their products stand beside the next ones' exponentials. FIRST: a SIMD's other waves wait for these. 4 x
    // 512 tokens of heads of 128 behind 2000 bf16 rows 81 us, so 75, over int8 92 and 88; 2 x 300 of heads of 64 behind 20000 in
    // bf16 290 and 273, in fp32 734 and 612, over int8 870 and 775; 64 tokens in fp32 behind 32000 int8 rows 115 and 113; but 64
    // of heads of 128 behind 32000 e4m3 rows 56.6 and 57.8, 1000 of one sequence 39.8 and 41.3. Not where waves share no keys (16
    // tokens in fp32 behind 32000 int8 rows 42.7 and 43.5) or a SIMD has one (4 x 512 in fp32, heads of 128, 222 and 226).
    v4u v[D / 32], w[NT];
    auto load = [&](int u, v4u (&to)[D / 32]) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        // values of dimension 32 i + lane % 32, keys 16 u + 4 h .. + 3 and 8 behind them
        const uint8_t* at = vl + (16 * u + 4 * h + ((lane & 15) >> 2)) * Pitch<D>::V +
                            2 * (32 * i + 16 * ((lane >> 4) & 1) + 4 * (lane & 3));
        const v2u a = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s4*)at));
        const v2u b = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s4*)(at + 8 * Pitch<D>::V)));
        to[i] = v4u{a[0], a[1], b[0], b[1]};
      }
    };
    auto weigh = [&](int u, v4u (&to)[NT]) {
      v4f g[2];  // the values' scales
      if constexpr (KV != NSX_DT_BF16) {
#pragma unroll
        for (int e = 0; e < 2; ++e) g[e] = *(const v4f*)(sv + 16 * u + 8 * e + 4 * h);
      }
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = s[u >> 1][8 * (u & 1) + e];
        x[e] = __builtin_amdgcn_exp2f(KV == NSX_DT_BF16 ? fmaf(y, c, -m) : y);
        l += x[e];
        if constexpr (KV != NSX_DT_BF16) x[e] *= g[e >> 2][e & 3];
      }
      terms8<NT>(x, to);
    };
    load(0, v);
    weigh(0, w);
    if constexpr (FIRST) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int u = 0; u < 2 * NB; ++u) {
      v4u vn[D / 32], wn[NT];
      if constexpr (D == 64) __builtin_amdgcn_sched_barrier(0);
      if (u + 1 < 2 * NB) load(u + 1, vn);
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int t = NT - 1; t >= 0; --t) acc[i] = dot(v[i], w[t], acc[i]);
      if (u + 1 < 2 * NB) {
        weigh(u + 1, wn);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) v[i] = vn[i];
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t] = wn[t];
      }
    }
    if constexpr (FIRST) __builtin_amdgcn_s_setprio(0);
  }
  __device__ __forceinline__ bool finite() const {
    float z = l * 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) z = fmaf(acc[i][e], 0.f, z);
    return z == 0.f;
  }
};

// 16-byte pieces of KEYS rows of k and v (and their scales) by THREADS threads: from memory to registers, then to LDS as bf16.
template <int KV, int D, int KEYS, int THREADS>
struct Stage {
  static constexpr int PIECES = D / Codes<KV>::PER, N = KEYS * PIECES / THREADS;
  v4u k[N], v[N];
  float s;
  __device__ __forceinline__ void load(const Source& p, int t0, int last, int t) {  // rows t0 .., none past `last`
    const uint8_t *kp = p.k + (int64_t)t0 * (D * Codes<KV>::BYTES), *vp = p.v + (int64_t)t0 * (D * Codes<KV>::BYTES);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = t + THREADS * i, at = min(x / PIECES, last - t0) * (D * Codes<KV>::BYTES) + x % PIECES * 16;
      k[i] = *(const v4u*)(kp + at);
      v[i] = *(const v4u*)(vp + at);
    }
    if constexpr (KV != NSX_DT_BF16) {
      static_assert(THREADS >= 2 * KEYS, "a thread per scale");
      if (t < 2 * KEYS) s = (t < KEYS ? p.ks : p.vs)[t0 + min(t % KEYS, last - t0)];
    }
  }
  __device__ __forceinline__ void store(uint8_t* kl, uint8_t* vl, float* sc, float c, int t) const {  // sc: KEYS of k, KEYS of v
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = t + THREADS * i, row = x / PIECES, at = x % PIECES * (2 * Codes<KV>::PER);
      Codes<KV>::put(kl + row * Pitch<D>::K + at, k[i]);
      Codes<KV>::put(vl + row * Pitch<D>::V + at, v[i]);
    }
    if constexpr (KV != NSX_DT_BF16) {
      if (t < 2 * KEYS) sc[t] = t < KEYS ? s * c : s;
    }
  }
};

template <int D>
constexpr int attn_lds() {
  return 2 * Pitch<D>::stage(64) + 2048;  // two stages of 64 keys (or four waves' of 32), scales; then sums to be joined
}
// A workgroup's rows over its keys. SHARED: its four waves take 32 rows each and share every stage of 64 keys, the next on its
// way from memory meanwhile, the one behind it in the other half of LDS: a barrier a stage. Else all of them take the same 32
// rows, each every fourth stage of 32 keys, without a barrier, and their sums are joined in LDS: more waves for few rows (64
// tokens behind 8000 int8 rows 32 us so, SHARED 38; behind 32768 e4m3 rows 86 and 68).
template <typename XT, int KV, int D, int NT, bool SHARED>
__device__ __forceinline__ void attend(const AttnArgs& a, const Place& p, uint8_t* lds) {
  constexpr int KEYS = SHARED ? 64 : 32, THREADS = SHARED ? 256 : 64;
  constexpr int STAGE = Pitch<D>::stage(KEYS), SUMS = 2 * Pitch<D>::stage(64);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i32 = lane & 31, h = lane >> 5;
  const int r = p.r0 + (SHARED ? AT_ROWS * wave : 0) + i32;
  Wave<KV, D, NT, KEYS / 32, SHARED && !(NT == 3 && D == 128)> w;
  Stage<KV, D, KEYS, THREADS> st;
  // of each source, the keys that any live row of the workgroup sees, and those that all of the wave's do
  Range range;
  const Row row(a, p, r);
  const At at{row.tok, row.h, row.live};
  w.start((const XT*)a.q + (int64_t)(row.tok * a.H + row.h) * D);
  int all0[2], all1[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    range.from[i] = 0, range.to[i] = 0, all0[i] = 0, all1[i] = 0;
    if (p.with[i]) {
      const uint32_t lo = (uint32_t)row.lo[i], hi = (uint32_t)row.hi[i];
      range.from[i] = (int)min(nsx_wave_min_u32(row.live ? lo : ~0u), 0x7fffffffu);
      range.to[i] = (int)nsx_wave_max_u32(row.live ? hi : 0);
      all0[i] = (int)nsx_wave_max_u32(row.live ? lo : 0);
      all1[i] = (int)min(nsx_wave_min_u32(row.live ? hi : ~0u), 0x7fffffffu);
    }
  }
  if constexpr (SHARED) {
    int4* each = (int4*)lds;
    if (lane == 0) each[wave] = int4{range.from[0], range.to[0], range.from[1], range.to[1]};
    __syncthreads();
#pragma unroll
    for (int i = 0; i < AT_NW; ++i) {
      const int4 x = each[i];
      range.from[0] = min(range.from[0], __builtin_amdgcn_readfirstlane(x.x));
      range.to[0] = max(range.to[0], __builtin_amdgcn_readfirstlane(x.y));
      range.from[1] = min(range.from[1], __builtin_amdgcn_readfirstlane(x.z));
      range.to[1] = max(range.to[1], __builtin_amdgcn_readfirstlane(x.w));
    }
    __syncthreads();
  }
  range.split<KEYS>(p, SHARED ? 1 : AT_NW);

  uint8_t* tile = lds + (SHARED ? 0 : STAGE * wave);
  float* scales = (float*)(lds + SUMS) + (SHARED ? 0 : 2 * KEYS * wave);
  const int t = SHARED ? threadIdx.x : lane, step = SHARED ? 1 : AT_NW;
  const int w0 = __builtin_amdgcn_readfirstlane(wave);
  auto first_key = [&](int i) {  // of tile i, in its source
    return i >= range.tiles[0] ? range.from[1] + (i - range.tiles[0]) * KEYS : range.from[0] + i * KEYS;
  };
  auto load = [&](int i) {
    const bool o = i >= range.tiles[0];
    const Source src{o ? p.src[1].k : p.src[0].k, o ? p.src[1].v : p.src[0].v, o ? p.src[1].ks : p.src[0].ks,
                     o ? p.src[1].vs : p.src[0].vs};
    st.load(src, first_key(i), (o ? range.to[1] : range.to[0]) - 1, t);
  };
  int i = range.first + (SHARED ? 0 : w0), buf = 0;
  if (i < range.end) load(i);
  for (; i < range.end; i += step) {
    uint8_t *kl = tile + (SHARED ? buf * STAGE : 0), *vl = kl + KEYS * Pitch<D>::K;
    float* sc = scales + (SHARED ? buf * 2 * KEYS : 0);
    st.store(kl, vl, sc, a.scale2, t);
    if (i + step < range.end) load(i + step);
    if constexpr (SHARED) nsx_lds_barrier();
    else __builtin_amdgcn_wave_barrier();
    const bool o = i >= range.tiles[0];
    const int key0 = first_key(i);
    const bool all = key0 >= (o ? all0[1] : all0[0]) && key0 + KEYS <= (o ? all1[1] : all1[0]);
    w.step(kl, vl, sc, sc + KEYS, a.scale2, all, key0, o ? row.lo[1] : row.lo[0], o ? row.hi[1] : row.hi[0]);
    buf ^= 1;
    if constexpr (!SHARED) __builtin_amdgcn_wave_barrier();
  }
  const End<XT, D> fin{a, p};
  const bool mine = r < p.rows;
  const uint64_t odd = __ballot(!w.finite() && mine && row.live);
  uint32_t bad = (uint32_t)odd | (uint32_t)(odd >> 32);
  w.l = other_half_sum(w.l);
  if constexpr (SHARED) {
    if (mine && !(bad >> i32 & 1)) {
      const auto f = fin.factor(at, w.m, w.l, h == 0);
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float x[4] = {w.acc[i][e], w.acc[i][e + 1], w.acc[i][e + 2], w.acc[i][e + 3]};
          fin.store(at, 32 * i + 2 * e + 4 * h, f, x);
        }
    }
    for (; bad; bad &= bad - 1) row_alone<XT, KV, D, KEYS>(a, p, range, p.r0 + AT_ROWS * wave + __builtin_ctz(bad));
  } else {
    // the waves' sums, on the largest of their references
    constexpr int OP = D + 4;
    float* sums = (float*)lds;                         // [wave][row][OP]
    float2* ml = (float2*)(lds + SUMS);             // [wave][row]
    uint32_t* odds = (uint32_t*)(ml + AT_NW * AT_ROWS);
    static_assert(AT_NW * AT_ROWS * OP * 4 <= SUMS && AT_NW * (AT_ROWS * 8 + 4) <= 2048, "LDS");
    __syncthreads();
    if (h == 0) ml[wave * AT_ROWS + i32] = float2{w.m, w.l};
    if (lane == 0) odds[wave] = bad;
    __syncthreads();
    bad = odds[0] | odds[1] | odds[2] | odds[3];
    float M = LOWEST, L = 0.f;
#pragma unroll
    for (int k = 0; k < AT_NW; ++k) M = fmaxf(M, ml[k * AT_ROWS + i32].x);
#pragma unroll
    for (int k = 0; k < AT_NW; ++k) {
      const float2 x = ml[k * AT_ROWS + i32];
      L = fmaf(x.y, __builtin_amdgcn_exp2f(x.x - M), L);
    }
    const float f = __builtin_amdgcn_exp2f(w.m - M);
#pragma unroll
    for (int blk = 0; blk < D / 32; ++blk)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f16v& y = w.acc[blk];
        *(v4f*)(sums + (wave * AT_ROWS + i32) * OP + 32 * blk + 2 * e + 4 * h) =
            v4f{y[e] * f, y[e + 1] * f, y[e + 2] * f, y[e + 3] * f};
      }
    __syncthreads();
    // a wave a quarter of the dimensions of every row, two lanes a row
    if (mine && !(bad >> i32 & 1)) {
      const auto y = fin.factor(at, M, L, threadIdx.x < 32);
#pragma unroll
      for (int e = 0; e < D / 8; e += 4) {
        const int d = D / 4 * wave + D / 8 * h + e;
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          x[k] = (sums[i32 * OP + d + k] + sums[(AT_ROWS + i32) * OP + d + k]) +
                 (sums[(2 * AT_ROWS + i32) * OP + d + k] + sums[(3 * AT_ROWS + i32) * OP + d + k]);
        fin.store(at, d, y, x);
      }
    }
    for (int k = 0; bad; bad &= bad - 1, ++k)
      if (k % AT_NW == wave) row_alone<XT, KV, D, KEYS>(a, p, range, p.r0 + __builtin_ctz(bad));
  }
}

template <typename XT>
constexpr int attn_terms() {
  // bf16 terms of a query (and of the weights beside it) that hold all of its 8, 11 or 24 bits
  return std::is_same_v<XT, float> ? 3 : std::is_same_v<XT, Half> ? 2 : 1;
}
template <typename XT, int KV, int D>
__global__ __launch_bounds__(256, (attn_terms<XT>() == 3 && D == 128 ? 1 : 2)) void attn_kernel(AttnArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  constexpr int NT = attn_terms<XT>();
  Place p;
  p.own = (int)blockIdx.x >= a.pblocks;
  const AttnArgs::Cut cut = p.own ? a.ocut : a.pcut;
  // Workgroups go to the chip's eight parts (a cache each) in turn: those of one run of keys to the same one.
  const int id = p.own ? blockIdx.x - a.pblocks : blockIdx.x;
  const int units = (p.own ? (int)a.kv.n_seq : 1) * a.G * cut.splits;
  const int eight = id / (8 * cut.tiles), left = min(8, units - 8 * eight), in = id - eight * 8 * cut.tiles;
  const int unit = 8 * eight + (int)((uint32_t)in % (uint32_t)left), tile = (int)((uint32_t)in / (uint32_t)left);
  p.split = unit % cut.splits;
  p.splits = cut.splits;
  p.slot = p.split + (p.own ? a.pcut.splits : 0);
  p.g = unit / cut.splits % a.G;
  p.b = unit / cut.splits / a.G;
  p.rows = (int)(p.own ? a.n : a.kv.n_seq * a.n) * a.rep;
  p.r0 = tile * cut.rows;
  p.P = a.pre.n_seq ? (int)min((int64_t)max(*a.pre.pos, 0), a.pre.ctx_max) : 0;
  p.with[0] = !p.own || a.pblocks == 0;
  p.with[1] = p.own;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const KvRows& kv = i ? a.kv : a.pre;
    const int64_t base = (int64_t)(i ? p.b * a.G + p.g : p.g) * kv.ctx_max;
    p.src[i].k = (const uint8_t*)kv.k + base * (D * Codes<KV>::BYTES);
    p.src[i].v = (const uint8_t*)kv.v + base * (D * Codes<KV>::BYTES);
    p.src[i].ks = kv.ks + (KV == NSX_DT_BF16 ? 0 : base);
    p.src[i].vs = kv.vs + (KV == NSX_DT_BF16 ? 0 : base);
  }
  if (cut.rows == AT_ROWS) attend<XT, KV, D, NT, false>(a, p, lds);
  else attend<XT, KV, D, NT, true>(a, p, lds);
}

// out = (sum_s 2^(m_s - M) y_s) / (sum_s 2^(m_s - M) l_s + 2^(sink - M)) over a (token, head)'s splits s: a wave each, D / 4
// lanes a split, the splits in the same order in every call. The first rounds of y are loaded before the weights are known: 1
// token of 64 heads over 30000 rows 10.7 us in all, so 8.8. Bound by latency: 4 us for 16 tokens of 64 heads, 6.4 for 64.
template <typename XT, int D>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
  constexpr int LPR = D / 4, AT_ONCE = 64 / LPR;
  const int lane = threadIdx.x & 63;
  const int64_t rows = a.kv.n_seq * a.n * a.H, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int64_t tok = row / a.H, b = tok / a.n;
  const int h = (int)(row - tok * a.H);
  const bool live = !a.counts || tok - b * a.n < a.counts[b];
  const float2* ml = (const float2*)(a.part + rows * a.splits * D) + row * a.splits;
  float m = LOWEST, l = 0.f;
  if (lane < a.splits) {
    const float2 x = ml[lane];
    m = x.x;
    l = x.y;
  }
  const float* part = a.part + row * a.splits * D + 4 * (lane % LPR);
  constexpr int AHEAD = 4;  // rounds of loads in one go, before the weights are known
  v4f y[AHEAD];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) y[i] = *(const v4f*)(part + (int64_t)min(s0 + AT_ONCE * i + lane / LPR, a.splits - 1) * D);
  };
  load(0);
  const float sink = a.sinks ? a.sinks[h] * LOG2E : LOWEST;
  float M = nsx_row_fmax(fmaxf(m, sink));
  M = fmaxf(M, __shfl_xor(M, 16, 64));
  M = other_half_max(M);
  // (a split without a key is 0 times 0; a sum or a value that is no number stays none beside any weight)
  const float w = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - M);
  const float Z = nsx_wave_sum(w * l) + (a.sinks ? __builtin_amdgcn_exp2f(sink - M) : 0.f);
  float x[4] = {};
  for (int s0 = 0; s0 < a.splits; s0 += AHEAD * AT_ONCE) {
    if (s0) load(s0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int s = s0 + AT_ONCE * i + lane / LPR;
      const float ws = __shfl(w, min(s, 63), 64);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = s < a.splits ? fmaf(ws, y[i][k], x[k]) : x[k];
    }
  }
#pragma unroll
  for (int o = LPR; o < 64; o *= 2)
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] += __shfl_xor(x[k], o, 64);
  const bool any = live && Z != 0.f;
  const float f = 1.f / Z;
  if (lane < LPR) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = any ? x[k] * f : 0.f;
    store4((XT*)a.out + row * D + 4 * lane, x);
  }
}

// How a call's rows and keys are cut into workgroups: by the caches' sizes, not their lengths, so that a captured call serves
// every length. Both sides of each rule in us, attention and join together:
//  - sequences of up to 64 rows each (a step of decoding) meet the prefix together, in workgroups of its own, joined with their
//    own keys; where all keys are 512 at most, or rows more, a sequence's workgroups meet the prefix ahead of their own keys,
//    with no join for it (2 sequences behind 200 rows 6.7, apart 8.9; 32 sequences with a window of 128 7.5 and 11.2; but 64
//    behind 1000 21.2, apart 12.4, 16 in fp32 14.8 and 11.6);
//  - SHARED workgroups where a wave of 2048 has more than 20 pieces of 32 rows by 32 keys to do and there are more than 64 rows
//    (19 pieces: 64 tokens behind 8000 int8 rows 38, else 32; 16: 16 in fp32 behind 32000 47 and 45; 37: 64 behind 16000 42 and
//    53 to 64);
//  - as many workgroups as the chip holds at once, but 3 pieces a wave in a split at least (16 sequences behind 1000 rows: 2
//    10.9, 3 11.5, 4 12.9; 64: 4 best), of which a sequence's own keys take their share, a quarter at least, and the prefix
//    what they leave, half at least; or, beyond 10 pieces a wave, all of them once more (64 behind 8000: 32, else 41; 64 behind
//    16000 of 128 44 and 48; but 64 in fp32 behind 3000 31, else 27).
struct Plan {
  AttnArgs::Cut pre, own;
  int64_t pblocks, oblocks;
  int splits;
};
Plan attn_plan(int G, int rep, int64_t B, int64_t n, int64_t ctx_max, int64_t prefix_max, int window, int occ) {
  Plan p{};
  const int64_t prows = B * n * rep, orows = n * rep;
  const int64_t pk = window > 0 ? std::min<int64_t>(prefix_max, window + n) : prefix_max;
  const int64_t ok = window > 0 ? std::min<int64_t>(ctx_max, window + n) : ctx_max;
  // pieces of 32 rows x 32 keys, and how many of them a wave takes where the chip's share them
  const int64_t pw = G * nsx_cdiv(prows, AT_ROWS) * nsx_cdiv(pk, 32), ow = B * G * nsx_cdiv(orows, AT_ROWS) * nsx_cdiv(ok, 32);
  const int64_t each = nsx_cdiv(pw + ow, 2048);
  const bool many = each > 20;
  const int64_t slots = 256 * (many ? occ : std::min(occ, 2));
  auto cut = [&](int64_t rows, int64_t keys, int64_t units, int64_t room) {
    AttnArgs::Cut c;
    const int waves = rows > 2 * AT_ROWS && many ? 1 : AT_NW;  // that share a row's keys
    c.rows = waves > 1 ? AT_ROWS : AT_NW * AT_ROWS;
    c.tiles = (int)nsx_cdiv(rows, c.rows);
    const int64_t most = nsx_cdiv(nsx_cdiv(keys, 32), 3 * waves);
    c.splits = (int)std::max<int64_t>(1, std::min<int64_t>({AT_MAX_SPLIT / 2, most, room / (units * c.tiles)}));
    return c;
  };
  const bool apart = prefix_max && orows <= 2 * AT_ROWS && pk + ok > 512;
  if (apart) {
    p.own = cut(orows, ok, B * G, std::max<int64_t>(slots / 4, slots * ow / (pw + ow)));
    const int64_t left = slots - B * G * p.own.tiles * p.own.splits;
    p.pre = cut(prows, pk, G, each > 10 ? slots : std::max<int64_t>(slots / 2, left));
  } else {
    p.own = cut(orows, ok + pk, B * G, slots);
  }
  p.pblocks = (int64_t)G * p.pre.tiles * p.pre.splits;
  p.oblocks = B * G * p.own.tiles * p.own.splits;
  p.splits = p.pre.splits + p.own.splits;
  return p;
}
// Workgroups of a kernel that a CU is taken to hold, by its registers: up to 512, 256 or 168 a lane. (fp16 with heads of 64 needs
// 168 as well, and three would fit; it is planned for two.)
int attn_occ(int x_dtype, int head_dim) {
  return x_dtype == NSX_DT_F32 && head_dim == 128 ? 1 : x_dtype == NSX_DT_BF16 && head_dim == 64 ? 3 : 2;
}

// ---------------------------------------------------------------------------

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int64_t x_size(int dt) { return dt == NSX_DT_F32 ? 4 : 2; }

int batch_types(int x_dtype, int kv_type) {
  NSX_REQUIRE(x_dtype == NSX_DT_F32 || x_dtype == NSX_DT_F16 || x_dtype == NSX_DT_BF16, NSX_ETYPE, "element type %d",
              x_dtype);
  NSX_REQUIRE(kv_type == NSX_DT_BF16 || kv_type == NSX_KV_INT8 || kv_type == NSX_KV_E4M3, NSX_ETYPE, "cache row type %d",
              kv_type);
  return NSX_OK;
}
int batch_heads(int n_head, int n_kv, int head_dim) {
  NSX_REQUIRE(head_dim == 64 || head_dim == 128, NSX_ENOTIMPL, "head_dim %d (the kernels are written for 64 and 128)",
              head_dim);
  NSX_REQUIRE(n_kv > 0 && n_kv <= 1024 && n_head > 0 && n_head <= 4096 && n_head % n_kv == 0, NSX_EINVAL,
              "n_head=%d, n_kv=%d: n_head (up to 4096) must be a multiple of n_kv (up to 1024)", n_head, n_kv);
  return NSX_OK;
}
// A cache as the kernels take it: its rows' numbers fit 64 bits, a position's 32.
int batch_cache(const nsx_kv_rows* kv, int kv_type, int n_kv, const char* name) {
  NSX_REQUIRE(kv && kv->k && kv->v, NSX_EINVAL, "%s: null buffer", name);
  NSX_REQUIRE(kv->n_seq > 0 && kv->n_seq < 65536 && kv->ctx_max > 0 && kv->ctx_max < (1ll << 30), NSX_EINVAL,
              "%s: %lld sequences of %lld rows (below 65536, below 2^30)", name, (long long)kv->n_seq,
              (long long)kv->ctx_max);
  NSX_REQUIRE(kv_type == NSX_DT_BF16 || (kv->k_scale && kv->v_scale), NSX_EINVAL, "%s: rows of 8 bits need scales", name);
  NSX_REQUIRE(aligned16(kv->k) && aligned16(kv->v) && ((uintptr_t)kv->k_scale & 3) == 0 && ((uintptr_t)kv->v_scale & 3) == 0,
              NSX_EINVAL, "%s: rows must be 16-byte aligned, scales 4-byte", name);
  return NSX_OK;
}
KvRows kv_rows(const nsx_kv_rows* kv) { return KvRows{kv->k, kv->v, kv->k_scale, kv->v_scale, kv->pos, kv->n_seq, kv->ctx_max}; }
bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

// f(std::integral_constant row type, head_dim) for an element type
template <typename F>
int with_types(int x_dtype, int kv_type, int head_dim, F f) {
  auto kv = [&](auto x) {
    auto d = [&](auto t) {
      return head_dim == 64 ? f(x, t, std::integral_constant<int, 64>{}) : f(x, t, std::integral_constant<int, 128>{});
    };
    if (kv_type == NSX_DT_BF16) return d(std::integral_constant<int, NSX_DT_BF16>{});
    if (kv_type == NSX_KV_INT8) return d(std::integral_constant<int, NSX_KV_INT8>{});
    return d(std::integral_constant<int, NSX_KV_E4M3>{});
  };
  if (x_dtype == NSX_DT_F32) return kv(float{});
  if (x_dtype == NSX_DT_F16) return kv(Half{});
  return kv(Bf16{});
}

}  // namespace

extern "C" int nsx_append_qkv(const void* qkv, int x_dtype, const float* q_bias, const float* k_bias,
                              const float* v_bias, const float* q_norm, const float* k_norm, float eps,
                              const float* inv_freq, float amplitude, int n_head, int n_kv, int head_dim, int64_t n,
                              const int32_t* counts, const nsx_kv_rows* kv, int kv_type, const int32_t* prefix_pos,
                              void* q_out, void* stream) {
  if (const int rc = batch_types(x_dtype, kv_type)) return rc;
  if (const int rc = batch_heads(n_head, n_kv, head_dim)) return rc;
  if (const int rc = batch_cache(kv, kv_type, n_kv, "kv")) return rc;
  NSX_REQUIRE(n >= 0 && n < (1ll << 24) && kv->n_seq * n < (1ll << 24), NSX_EINVAL,
              "%lld tokens of %lld sequences: fewer than 2^24", (long long)n, (long long)kv->n_seq);
  NSX_REQUIRE(eps >= 0.f, NSX_EINVAL, "eps %g", eps);
  if (n == 0) return NSX_OK;
  NSX_REQUIRE(qkv && q_out && inv_freq && kv->pos, NSX_EINVAL, "null buffer");
  for (const void* p : {qkv, (const void*)q_out, (const void*)q_bias, (const void*)k_bias, (const void*)v_bias,
                        (const void*)q_norm, (const void*)k_norm})
    NSX_REQUIRE(aligned16(p), NSX_EINVAL, "qkv, q_out, biases and norm weights must be 16-byte aligned");
  const int heads = n_head + 2 * n_kv;
  const int64_t tokens = kv->n_seq * n, e = x_size(x_dtype) * head_dim;
  NSX_REQUIRE(!overlap(qkv, tokens * heads * e, q_out, tokens * n_head * e), NSX_EINVAL, "q_out overlaps qkv");
  const int rows = 256 / (head_dim / 8), all = (int)nsx_cdiv(heads, rows);
  const int passes = tokens >= 512 ? all : 1;  // (both sides at append_kernel)
  const AppendArgs a{qkv, q_bias, k_bias, v_bias, q_norm, k_norm, inv_freq, eps, amplitude, n_head, n_kv, passes, n, counts,
                     prefix_pos, kv_rows(kv), q_out};
  return with_types(x_dtype, kv_type, head_dim, [&](auto x, auto t, auto d) {
    return nsx_launch(append_kernel<decltype(x), t(), d()>, dim3((unsigned)tokens, (unsigned)nsx_cdiv(all, passes)), dim3(256), 0,
                      (hipStream_t)stream, a);
  });
}

template <bool STORE>
static int move_rows(void* k, void* v, int x_dtype, int64_t n, const int32_t* start, int64_t start0, int n_kv,
                     int head_dim, const nsx_kv_rows* kv, int kv_type, void* stream) {
  if (const int rc = batch_types(x_dtype, kv_type)) return rc;
  if (const int rc = batch_heads(n_kv, n_kv, head_dim)) return rc;
  if (const int rc = batch_cache(kv, kv_type, n_kv, "kv")) return rc;
  NSX_REQUIRE(n >= 0 && n < (1ll << 31) && start0 > -(1ll << 31) && start0 < (1ll << 31), NSX_EINVAL, "n=%lld start=%lld",
              (long long)n, (long long)start0);
  if (n == 0) return NSX_OK;
  NSX_REQUIRE(k && v && aligned16(k) && aligned16(v), NSX_EINVAL, "k and v must be 16-byte aligned buffers");
  const int64_t rows = kv->n_seq * n_kv * n;
  NSX_REQUIRE(rows < (1ll << 28), NSX_EINVAL, "%lld rows: fewer than 2^28", (long long)rows);
  const int64_t bytes = rows * head_dim * x_size(x_dtype);
  NSX_REQUIRE(STORE || !overlap(k, bytes, v, bytes), NSX_EINVAL, "k overlaps v");
  const RowsArgs a{k, v, kv_rows(kv), start, start0, n, rows, n_kv};
  return with_types(x_dtype, kv_type, head_dim, [&](auto x, auto t, auto d) {
    // four rows a thread where that leaves workgroups for every CU (4 x 16000 rows of 8 heads into int8: 38 us, with one 53;
    // 2 rows back: 3.2 us, with one 2.2)
    constexpr int ROWS = 256 / (d() / 8);
    const bool four = rows >= 4 * ROWS * 512;
    auto* kernel = four ? rows_kernel<decltype(x), t(), d(), STORE, 4> : rows_kernel<decltype(x), t(), d(), STORE, 1>;
    return nsx_launch(kernel, dim3((unsigned)nsx_cdiv(rows, (four ? 4 : 1) * ROWS), 2), dim3(256), 0, (hipStream_t)stream, a);
  });
}
extern "C" int nsx_store_rows(const void* k, const void* v, int x_dtype, int64_t n, const int32_t* start, int64_t start0,
                              int n_kv, int head_dim, const nsx_kv_rows* kv, int kv_type, void* stream) {
  return move_rows<true>((void*)k, (void*)v, x_dtype, n, start, start0, n_kv, head_dim, kv, kv_type, stream);
}
extern "C" int nsx_load_rows(const nsx_kv_rows* kv, int kv_type, int n_kv, int head_dim, const int32_t* start,
                             int64_t start0, int64_t n, void* k, void* v, int x_dtype, void* stream) {
  return move_rows<false>(k, v, x_dtype, n, start, start0, n_kv, head_dim, kv, kv_type, stream);
}

extern "C" int64_t nsx_batch_attn_workspace_bytes(int n_head, int n_kv, int head_dim, int64_t n_seq, int64_t n,
                                                  int64_t ctx_max, int64_t prefix_max, int window) {
  if (batch_heads(n_head, n_kv, head_dim) != NSX_OK || n_seq <= 0 || n_seq >= 65536 || n <= 0 || n >= (1ll << 24) ||
      n_seq * n >= (1ll << 24) || ctx_max <= 0 || ctx_max >= (1ll << 30) || prefix_max < 0 || prefix_max >= (1ll << 30) ||
      window < 0)
    return -1;
  int splits = 1;  // (whatever the type)
  for (const int dt : {NSX_DT_F32, NSX_DT_F16, NSX_DT_BF16})
    splits = std::max(splits, attn_plan(n_kv, n_head / n_kv, n_seq, n, ctx_max, prefix_max, window, attn_occ(dt, head_dim)).splits);
  return splits > 1 ? n_seq * n * n_head * splits * (head_dim + 2) * 4 : 0;
}

extern "C" int nsx_batch_attn(const void* q, int x_dtype, const nsx_kv_rows* kv, const nsx_kv_rows* prefix, int kv_type,
                              int n_head, int n_kv, int head_dim, int64_t n, const int32_t* counts, const float* sinks,
                              int window, float scale, void* workspace, int64_t workspace_bytes, void* out,
                              void* stream) {
  if (const int rc = batch_types(x_dtype, kv_type)) return rc;
  if (const int rc = batch_heads(n_head, n_kv, head_dim)) return rc;
  if (const int rc = batch_cache(kv, kv_type, n_kv, "kv")) return rc;
  if (prefix) {
    if (const int rc = batch_cache(prefix, kv_type, n_kv, "prefix")) return rc;
    NSX_REQUIRE(prefix->n_seq == 1 && prefix->pos, NSX_EINVAL, "the prefix is one sequence's rows (got %lld) with a length",
                (long long)prefix->n_seq);
  }
  NSX_REQUIRE(scale > 0.f && scale < INFINITY, NSX_EINVAL, "scale %g", scale);
  NSX_REQUIRE(n >= 0 && n < (1ll << 24) && window >= 0 && kv->n_seq * n < (1ll << 24), NSX_EINVAL,
              "n=%lld window=%d: fewer than 2^24 tokens", (long long)n, window);
  if (n == 0) return NSX_OK;
  NSX_REQUIRE(q && out && kv->pos && aligned16(q) && aligned16(out), NSX_EINVAL, "q and out must be 16-byte aligned buffers");
  const int64_t need = nsx_batch_attn_workspace_bytes(n_head, n_kv, head_dim, kv->n_seq, n, kv->ctx_max,
                                                      prefix ? prefix->ctx_max : 0, window);
  NSX_REQUIRE((workspace || !need) && aligned16(workspace) && workspace_bytes >= need, NSX_EINVAL,
              "workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)workspace_bytes, (long long)need);
  const int64_t bytes = kv->n_seq * n * n_head * head_dim * x_size(x_dtype);
  NSX_REQUIRE(!overlap(q, bytes, out, bytes), NSX_EINVAL, "out overlaps q");
  const Plan plan = attn_plan(n_kv, n_head / n_kv, kv->n_seq, n, kv->ctx_max, prefix ? prefix->ctx_max : 0, window,
                              attn_occ(x_dtype, head_dim));
  NSX_REQUIRE(plan.pblocks + plan.oblocks < (1ll << 24) && kv->n_seq * n * n_head <= (1ll << 26) - 4, NSX_EINVAL,
              "%lld tokens of %d heads: too many for one call", (long long)(kv->n_seq * n), n_head);
  const AttnArgs a{q, kv_rows(kv), prefix ? kv_rows(prefix) : KvRows{}, counts, sinks, n_head, n_kv, n_head / n_kv, window, n,
                   scale * LOG2E, (float*)workspace, out, plan.pre, plan.own, (int)plan.pblocks, plan.splits};
  return with_types(x_dtype, kv_type, head_dim, [&](auto x, auto t, auto d) {
    using XT = decltype(x);
    constexpr int LDS = attn_lds<d()>();
    auto* kernel = attn_kernel<XT, t(), d()>;
    if (const int rc = nsx_allow_lds((const void*)kernel, LDS)) return rc;
    const dim3 grid((unsigned)(plan.pblocks + plan.oblocks));
    if (const int rc = nsx_launch(kernel, grid, dim3(256), LDS, (hipStream_t)stream, a)) return rc;
    if (plan.splits == 1) return (int)NSX_OK;
    const dim3 join((unsigned)nsx_cdiv(kv->n_seq * n * n_head, 4));
    return nsx_launch(join_kernel<XT, d()>, join, dim3(256), 0, (hipStream_t)stream, a);
  });
}
