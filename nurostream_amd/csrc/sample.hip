// A token for each row of logits by temperature, top-k, top-p and min-p from given random numbers (gfx950).
#include "nsx_common.h"

#include <type_traits>
#include <math.h>

namespace {

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
};

constexpr int THREADS = 1024;

template <typename LT>  // float, _Float16, or uint16_t for bf16
__device__ __forceinline__ float logit(const LT* p, int64_t i) {
  float f;
  if constexpr (std::is_same_v<LT, uint16_t>) f = nsx_bf2f(p[i]);
  else f = (float)p[i];
  return f == f ? f + 0.f : -INFINITY;  // (no -0)
}
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}

template <typename LT>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a) {
  __shared__ uint64_t mass[256];
  __shared__ uint32_t many[256];
  __shared__ uint64_t s64[THREADS];
  __shared__ uint32_t s32[THREADS];
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const LT* p = (const LT*)a.logits + row * a.row_stride;
  const double T = a.temperatures ? (double)a.temperatures[row] : a.temperature;
  const double top_p = a.top_ps ? (double)a.top_ps[row] : a.top_p, min_p = fmin(a.min_ps ? (double)a.min_ps[row] : a.min_p, 1.0);
  const int64_t top_k = a.top_ks ? a.top_ks[row] : a.top_k;
  // the largest and its lowest index
  uint64_t best = 0;
  for (int64_t i = t; i < a.V; i += THREADS) {
    const uint64_t v = (uint64_t)order_of(logit(p, i)) << 32 | (uint32_t)~(uint32_t)i;
    best = v > best ? v : best;
  }
  s64[t] = best;
  __syncthreads();
  for (int o = THREADS / 2; o; o >>= 1) {
    if (t < o) s64[t] = s64[t + o] > s64[t] ? s64[t + o] : s64[t];
    __syncthreads();
  }
  best = s64[0];
  __syncthreads();
  const int32_t at = (int32_t)~(uint32_t)best;
  const float M = logit(p, at);
  if (!(M > -INFINITY) || !(T > 0.0)) {
    if (t == 0) a.token[row] = M > -INFINITY ? at : -1;
    return;
  }
  auto real = [&](float x) { return M == INFINITY ? (x == M ? 1.0 : 0.0) : exp(((double)x - (double)M) / T); };
  auto weight = [&](float x) { return (uint64_t)rint(ldexp(real(x), a.bits)); };
  // the border: tokens above key are kept, and `ties` of those at it, by their index
  uint32_t key = 0, ties = 0xffffffffu;
  uint64_t whole = 0;
  for (int mode = 0; mode < 2; ++mode) {  // 0: by their number, 1: by their weight
    if (mode == 0 ? !(top_k > 0 && top_k < a.V) : !(top_p < 1.0)) continue;
    if (mode == 1) {
      // the whole weight of what top_k left
      uint64_t s = 0;
      for (int64_t i = t; i < a.V; i += THREADS) {
        const float x = logit(p, i);
        if (order_of(x) > key) s += weight(x);
        else if (order_of(x) == key && ties == 0xffffffffu) s += weight(x);
      }
      s64[t] = s;
      __syncthreads();
      for (int o = THREADS / 2; o; o >>= 1) {
        if (t < o) s64[t] += s64[t + o];
        __syncthreads();
      }
      whole = s64[0];
      __syncthreads();
      if (ties != 0xffffffffu) {
        const uint32_t u = key ^ ((int32_t)key < 0 ? 0x80000000u : 0xffffffffu);
        whole += ties * weight(__builtin_bit_cast(float, u));
      }
    }
    const uint64_t want = mode == 0 ? (uint64_t)top_k : (uint64_t)ceil(fmax(top_p, 0.0) * (double)whole);
    uint64_t above = 0;
    uint32_t found = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = t; i < 256; i += THREADS) mass[i] = 0, many[i] = 0;
      __syncthreads();
      for (int64_t i = t; i < a.V; i += THREADS) {
        const float x = logit(p, i);
        const uint32_t o = order_of(x);
        if (shift == 24 || (o >> (shift + 8)) == (found >> (shift + 8))) {
          atomicAdd(&many[o >> shift & 255], 1u);
          if (mode) atomicAdd((unsigned long long*)&mass[o >> shift & 255], (unsigned long long)weight(x));
        }
      }
      __syncthreads();
      if (t == 0) {
        int d = 255;
        uint64_t sum = above;
        for (;; --d) {
          const uint64_t m = mode ? mass[d] : many[d];
          if (sum + m >= want && many[d]) break;
          if (d == 0) break;
          sum += m;
        }
        s64[0] = sum;
        s32[0] = d;
      }
      __syncthreads();
      above = s64[0];
      found |= s32[0] << shift;
      __syncthreads();
    }
    const uint32_t u = found ^ ((int32_t)found < 0 ? 0x80000000u : 0xffffffffu);
    const uint64_t w = mode ? weight(__builtin_bit_cast(float, u)) : 1;
    uint64_t r = want > above ? (w ? (want - above + w - 1) / w : 0xffffffffu) : 0;
    if (mode && found == order_of(M) && r == 0) r = 1;  // (the likeliest token stays)
    if (found > key) key = found, ties = (uint32_t)(r < 0xffffffffu ? r : 0xffffffffu);
    else if (found == key) ties = (uint32_t)(r < ties ? r : ties);
  }
  // the draw: passes over the row in index order, a thread a run of tokens
  const int64_t per = (a.V + THREADS - 1) / THREADS, i0 = t * per, i1 = i0 + per < a.V ? i0 + per : a.V;
  uint32_t mine = 0;
  for (int64_t i = i0; i < i1; ++i) mine += order_of(logit(p, i)) == key;
  s32[t] = mine;
  __syncthreads();
  if (t == 0) {
    uint32_t s = 0;
    for (int i = 0; i < THREADS; ++i) {
      const uint32_t v = s32[i];
      s32[i] = s;
      s += v;
    }
  }
  __syncthreads();
  const uint32_t before = s32[t];
  auto kept = [&](float x, uint32_t& tie) -> uint64_t {
    const uint32_t o = order_of(x);
    if (o < key) return 0;
    if (o == key && tie++ >= ties) return 0;
    return real(x) < min_p ? 0 : weight(x);
  };
  uint64_t sum = 0;
  uint32_t tie = before;
  for (int64_t i = i0; i < i1; ++i) sum += kept(logit(p, i), tie);
  s64[t] = sum;
  __syncthreads();
  if (t == 0) {
    uint64_t s = 0;
    for (int i = 0; i < THREADS; ++i) {
      const uint64_t v = s64[i];
      s64[i] = s;
      s += v;
    }
    mass[0] = s;
  }
  __syncthreads();
  const uint64_t total = mass[0];
  const double x = fmin(fmax((double)a.u[row] * (double)total, 0.0), (double)total);
  const uint64_t target = (uint64_t)x < total ? (uint64_t)x : total - 1;
  uint64_t run = s64[t];
  if (run <= target && run + sum > target) {
    tie = before;
    for (int64_t i = i0; i < i1; ++i) {
      run += kept(logit(p, i), tie);
      if (run > target) {
        a.token[row] = (int32_t)i;
        break;
      }
    }
  }
}

}  // namespace

extern "C" int64_t nsx_sample_workspace_bytes(int64_t batch, int64_t vocab) {
  if (batch <= 0 || vocab <= 0) return -1;
  return 16;
}

extern "C" int nsx_sample(const void* logits, int logits_dtype, int64_t row_stride, int64_t batch, int64_t vocab,
                          const float* uniforms, const nsx_sampling* settings, int32_t* token, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  NSX_REQUIRE(logits_dtype == NSX_DT_F32 || logits_dtype == NSX_DT_F16 || logits_dtype == NSX_DT_BF16, NSX_ETYPE,
              "logits element type %d", logits_dtype);
  NSX_REQUIRE(batch >= 0 && batch < 65536 && vocab > 0 && vocab <= (1 << 22), NSX_EINVAL,
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
  int bits = 62;
  while (bits > 0 && (1ll << (62 - bits)) < vocab) --bits;
  const SampleArgs a{logits, row_stride, vocab, uniforms, s.temperature, s.top_p, s.min_p, s.top_k, s.temperatures,
                     s.top_ps, s.min_ps, s.top_ks, token, bits};
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)batch);
  if (logits_dtype == NSX_DT_F32) return nsx_launch(sample_kernel<float>, grid, dim3(THREADS), 0, st, a);
  if (logits_dtype == NSX_DT_F16) return nsx_launch(sample_kernel<_Float16>, grid, dim3(THREADS), 0, st, a);
  return nsx_launch(sample_kernel<uint16_t>, grid, dim3(THREADS), 0, st, a);
}
