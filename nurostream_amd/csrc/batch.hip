// Several sequences at once (gfx950): the new tokens' rows into a cache of 16 or 8 bits, and attention over a prefix that
// all sequences share and the rows of their own.
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

// A row's 8 elements per lane into a cache: rounded to bf16, or as codes with the row's scale. The largest is taken of the
// elements' bits, which order NaN above infinity above every number.
template <int KV, int D>
__device__ __forceinline__ void put_row(void* rows, float* scales, int64_t row, int l, const float (&x)[8]) {
  const float a[4] = {x[0], x[1], x[2], x[3]}, b[4] = {x[4], x[5], x[6], x[7]};
  if constexpr (KV == NSX_DT_BF16) {
    Bf16* p = (Bf16*)rows + row * D + 4 * l;
    store4(p, a);
    store4(p + D / 2, b);
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu;
      m = u > m ? u : m;
    }
    m = row_max<D / 8>(m);
    const bool finite = m < 0x7f800000u;
    const float s = __builtin_bit_cast(float, m) / (KV == NSX_KV_INT8 ? 127.f : 448.f);
    uint32_t c[2] = {0, 0};
    if (finite && s > 0.f) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i] / s;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (KV == NSX_KV_INT8) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            c[h] |= ((uint32_t)(int)rintf(fminf(fmaxf(y[4 * h + i], -127.f), 127.f)) & 0xffu) << (8 * i);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[4 * h + i] = fminf(fmaxf(y[4 * h + i], -448.f), 448.f);
          int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
          c[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], w, true);
        }
      }
    }
    uint8_t* p = (uint8_t*)rows + row * D + 4 * l;
    *(uint32_t*)p = c[0];
    *(uint32_t*)(p + D / 2) = c[1];
    if (l == 0) scales[row] = finite ? s : __builtin_nanf("");
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

// A workgroup per token and 256 / (D / 8) x passes of its heads.
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

template <typename XT, int KV, int D, bool STORE>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES;
  const int l = threadIdx.x % LANES;
  const int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (r >= a.rows) return;
  const int64_t bg = r / a.n, b = bg / a.G, at = (a.start ? a.start[b] : a.start0) + (r - bg * a.n);
  const bool in = at >= 0 && at < a.kv.ctx_max;
  const int64_t row = bg * a.kv.ctx_max + at;
  const bool v = blockIdx.y;
  XT* p = (XT*)(v ? a.v : a.k) + r * D + 4 * l;
  void* cache = v ? a.kv.v : a.kv.k;
  float* scale = v ? a.kv.vs : a.kv.ks;
  if constexpr (STORE) {
    if (!in) return;
    float lo[4], hi[4];
    load4(p, lo);
    load4(p + D / 2, hi);
    const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    put_row<KV, D>(cache, scale, row, l, x);
  } else {
    float x[8] = {};
    if (in) get_row<KV, D>(cache, scale, row, l, x);
    const float lo[4] = {x[0], x[1], x[2], x[3]}, hi[4] = {x[4], x[5], x[6], x[7]};
    store4(p, lo);
    store4(p + D / 2, hi);
  }
}

// --- attention ---------------------------------------------------------------

struct AttnArgs {
  const void* q;
  KvRows kv, pre;  // pre.n_seq 0: none
  const int32_t* counts;
  const float* sinks;
  int H, G, rep, window;
  int64_t n;
  float scale;
  float* part;
  void* out;
};

// A wave per (token, head).
template <typename XT, int KV, int D>
__global__ __launch_bounds__(64) void attn_kernel(AttnArgs a) {
  const int64_t tok = blockIdx.x, b = tok / a.n, j = tok - b * a.n;
  const int h = blockIdx.y, g = h / a.rep, lane = threadIdx.x;
  __shared__ float qs[D];
  __shared__ float ps[64];
  XT* out = (XT*)a.out + (tok * a.H + h) * D;
  const bool live = !a.counts || j < a.counts[b];
  const int64_t P = a.pre.n_seq ? min((int64_t)max(*a.pre.pos, 0), a.pre.ctx_max) : 0;
  const int64_t L = live ? min((int64_t)a.kv.pos[b] + j + 1, a.kv.ctx_max) : 0;
  float acc[D / 64] = {};
  float m = LOWEST, l = 0.f;
  if (live) {
    const XT* q = (const XT*)a.q + (tok * a.H + h) * D;
    for (int i = lane; i < D; i += 64) qs[i] = to_f(q[i]);
    __syncthreads();
    const int64_t at = P + a.kv.pos[b] + j, first = a.window > 0 ? max((int64_t)0, at + 1 - a.window) : 0;
    for (int seg = 0; seg < 2; ++seg) {
      const KvRows& kv = seg ? a.kv : a.pre;
      const int64_t lo = seg ? max((int64_t)0, first - P) : first, hi = seg ? L : P;
      const int64_t base = (seg ? b * a.G + g : g) * kv.ctx_max;
      for (int64_t t0 = lo; t0 < hi; t0 += 64) {
        float s = -INFINITY;
        if (t0 + lane < hi) {
          s = 0.f;
          for (int c = 0; c < D / 8; ++c) {
            float x[8];
            get_row<KV, D>(kv.k, kv.ks, base + t0 + lane, c, x);
            for (int i = 0; i < 4; ++i) s += qs[4 * c + i] * x[i] + qs[D / 2 + 4 * c + i] * x[4 + i];
          }
          s *= a.scale * LOG2E;
        }
        float mx = s;
        for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        mx = fmaxf(mx, m);
        const float p = t0 + lane < hi ? exp2f(s - mx) : 0.f, f = exp2f(m - mx);
        float z = p;
        for (int o = 32; o; o >>= 1) z += __shfl_xor(z, o, 64);
        l = l * f + z;
        m = mx;
        ps[lane] = p;
        __syncthreads();
        for (int i = 0; i < D / 64; ++i) acc[i] *= f;
        for (int64_t t = t0; t < min(hi, t0 + 64); ++t)
          for (int i = 0; i < D / 64; ++i) {
            const int64_t e = (base + t) * D + lane + 64 * i;
            float x;
            if constexpr (KV == NSX_DT_BF16) x = to_f(((const Bf16*)kv.v)[e]);
            else {
              float c[4];
              codes4<KV>(((const uint8_t*)kv.v)[e], c);
              x = c[0] * kv.vs[base + t];
            }
            acc[i] = fmaf(ps[t - t0], x, acc[i]);
          }
        __syncthreads();
      }
    }
    if (a.sinks) {
      const float sink = a.sinks[h] * LOG2E, mx = fmaxf(m, sink), f = exp2f(m - mx);
      l = l * f + exp2f(sink - mx);
      for (int i = 0; i < D / 64; ++i) acc[i] *= f;
    }
  }
  for (int i = 0; i < D / 64; ++i) from_f(out[lane + 64 * i], l == 0.f ? 0.f : acc[i] / l);
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
  NSX_REQUIRE(n >= 0 && n < (1ll << 24) && kv->n_seq * n < (1ll << 24), NSX_EINVAL, "%lld tokens of %lld sequences: fewer than 2^24",
              (long long)n, (long long)kv->n_seq);
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
  const int passes = tokens >= 512 ? all : 1;
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
  const int64_t groups = nsx_cdiv(rows, 256 / (head_dim / 8));
  NSX_REQUIRE(groups < (1ll << 24), NSX_EINVAL, "%lld rows", (long long)rows);
  const RowsArgs a{k, v, kv_rows(kv), start, start0, n, rows, n_kv};
  return with_types(x_dtype, kv_type, head_dim, [&](auto x, auto t, auto d) {
    return nsx_launch(rows_kernel<decltype(x), t(), d(), STORE>, dim3((unsigned)groups, 2), dim3(256), 0,
                      (hipStream_t)stream, a);
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
  return 16;
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
  NSX_REQUIRE(n >= 0 && n < (1ll << 24) && window >= 0 && kv->n_seq * n < (1ll << 24), NSX_EINVAL, "n=%lld window=%d: fewer than 2^24 tokens",
              (long long)n, window);
  if (n == 0) return NSX_OK;
  NSX_REQUIRE(q && out && kv->pos && aligned16(q) && aligned16(out), NSX_EINVAL, "q and out must be 16-byte aligned buffers");
  const int64_t need = nsx_batch_attn_workspace_bytes(n_head, n_kv, head_dim, kv->n_seq, n, kv->ctx_max,
                                                      prefix ? prefix->ctx_max : 0, window);
  NSX_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, NSX_EINVAL,
              "workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)workspace_bytes, (long long)need);
  const AttnArgs a{q, kv_rows(kv), prefix ? kv_rows(prefix) : KvRows{}, counts, sinks, n_head, n_kv, n_head / n_kv, window, n,
                   scale, (float*)workspace, out};
  return with_types(x_dtype, kv_type, head_dim, [&](auto x, auto t, auto d) {
    return nsx_launch(attn_kernel<decltype(x), t(), d()>, dim3((unsigned)(kv->n_seq * n), n_head), dim3(64), 0,
                      (hipStream_t)stream, a);
  });
}
