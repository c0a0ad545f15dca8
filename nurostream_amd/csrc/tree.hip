// Attention of drafted tokens over a KV cache and over one another (gfx950).
//
// N drafted tokens (nodes) hang off the cache's last row as a tree: parents[i] < i is node i's parent, anything else
// makes it a first node. Node i stands at position pos + depth(i). It sees the cache's rows 0 .. pos - 1 and, of the
// nodes, its ancestors and itself -- the last `window` positions of those when window > 0 -- and the softmax has a
// sink, as the one-token attention (attn.hip):
//   out_i = sum_j e^(s_ij - m) v_j / (sum_j e^(s_ij - m) + e^(sink - m)),  s_ij = scale q_i . k_j,  m the largest.
// The nodes' key and value rows live beside the cache ([n_kv][max_nodes][64], the cache's type), so that refused
// drafts never touch it; tree_commit_kernel moves the accepted ones in.
//
// Cache and node rows: fp32, fp16 or bf16; queries, sums and outputs fp32. A call is one launch where a kv head's keys are
// one split, with the merge of the splits two.
#include "nsx_common.h"
#include "rope.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int TREE_KEYS = 32;       // keys per wave and step
constexpr int TREE_NW = 4;          // waves of a workgroup, 8 where it takes all keys
constexpr int TREE_MAX_SPLIT = 128;  // splits of a kv head's keys: the combine kernel's lanes hold two each
constexpr int TREE_GRID = 512;      // workgroups to fill the chip with: two on each of 256 CUs
constexpr float LOG2E = 1.44269504088896340736f;

struct TreeArgs {
  const float* q;  // [nodes][n_head][64], rotated
  const void *kc, *vc, *dk, *dv;
  const int32_t *parents, *pos;
  int64_t ctx_max;
  int window, n_rep, n_kv, n_head, nodes, max_nodes;
  int nsplit, ncb;   // splits of the keys, blocks of columns
  int keys, round;   // keys of a tile; a split is a multiple of so many tiles
  float scale2;  // scale * log2(e): the softmax is taken in powers of two
  float* part;
  const float* sinks;
  float* out;
  // from raw projections: q is [nodes][n_head + 2 n_kv][64], and the nodes' rows are written to wk, wv (dk, dv)
  const float *bq, *bk, *bv, *inv_freq;
  float amp;
  void *wk, *wv;
};

// Which tiles a split takes: the cache's rows from the first that any node sees, then the nodes' own rows.
struct Tiles {
  int lo, cache, all, per;  // first row; tiles of the cache's rows; with the nodes'; of a split
  __device__ __forceinline__ Tiles(const TreeArgs& a, int P, int keys, int round) {
    lo = a.window > 0 ? max(0, P + 1 - a.window) : 0;
    cache = (P - lo + keys - 1) / keys;
    all = cache + (a.nodes + keys - 1) / keys;
    per = ((all + a.nsplit - 1) / a.nsplit + round - 1) / round * round;
  }
};

// Lane i's node: its ancestors and itself as bits, from the nodes' parents (-1 in lanes past the last node, which hold only
// their own bit), each round doubling the path's length. Every lane of the wave takes part.
__device__ __forceinline__ int tree_parent(const int32_t* __restrict__ parents, int nodes, int lane) {
  return lane >= nodes ? -1 : parents ? parents[lane] : lane - 1;
}
__device__ __forceinline__ uint64_t tree_lineage(int up, int lane) {
  up = up < 0 || up >= lane ? -1 : up;
  uint64_t bits = 1ull << lane;
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    const int from = up < 0 ? lane : up;
    const uint32_t lo = __shfl((uint32_t)bits, from, 64), hi = __shfl((uint32_t)(bits >> 32), from, 64);
    const int next = __shfl(up, from, 64);
    if (up >= 0) {
      bits |= (uint64_t)hi << 32 | lo;
      up = next;
    }
  }
  return bits;
}

template <typename KT>
__device__ __forceinline__ void store_kv(void* p, int64_t i, float v) {
  if constexpr (std::is_same_v<KT, float>) ((float*)p)[i] = v;
  else if constexpr (std::is_same_v<KT, _Float16>) {
    asm("" : "+v"(v));  // the fp32 value, rounded: not one instruction with what made it, rounding once
    ((_Float16*)p)[i] = (_Float16)v;
  }
  else ((uint16_t*)p)[i] = (uint16_t)nsx_f2bf(v);
}
struct Bf16 {
  uint16_t bits;
};

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ b8 as_b8(v4u x) { return __builtin_bit_cast(b8, x); }

// Two bf16 from the upper halves of two fp32.
__device__ __forceinline__ uint32_t top2(float lo, float hi) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
}
__device__ __forceinline__ float below(float x) {  // what the upper half leaves of x
  return x - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u);
}
// The first NT bf16 terms of 8 fp32: each takes 8 bits toward zero, so three hold all 24, and a product of two values
// overflows, if at all, with one sign in all of its terms.
template <int NT>
__device__ __forceinline__ void split8(const float (&x)[8], v4u (&t)[NT]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      t[k][i] = top2(a, b);
      if (k + 1 < NT) a = below(a), b = below(b);
    }
  }
}

// Two fp16 terms of 8 fp32, each rounded to nearest. They miss an element of at least 2^-2 by up to 2^-23 of
// itself (2^-24 at 2^-1 .. 1), a smaller one by up to 2^-25 whatever its size: half of fp16's least number.
__device__ __forceinline__ void halves8(const float (&x)[8], v4u (&t)[2]) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const h2 a = __builtin_convertvector((f2{x[2 * i], x[2 * i + 1]}), h2);
    t[0][i] = __builtin_bit_cast(uint32_t, a);
    asm("" : "+v"(t[0][i]));  // (both halves from here, not from conversions of their own)
    const h2 c = __builtin_bit_cast(h2, (uint32_t)t[0][i]);
    t[1][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x[2 * i] - (float)c[0], x[2 * i + 1] - (float)c[1]}), h2));
  }
}

// How queries meet keys of a type. fp32 and bf16 keys: three bf16 terms of a query, all its 24 bits. fp16 keys, one fp16 term
// as they are: two fp16 terms of the queries, scaled by a power of two so that a column's largest lies in 2^13 .. 2^14 (its
// scores scaled back). Elements down to 2^-16 of the largest keep 23 bits, smaller ones lose some. What a column loses that
// way may change a score by no more than 2^-18 over any fp16 keys, by 2^-20 over keys below 2^14 (`query_lost`); where it
// could, the scores are fp32 products of the queries as they are, a workgroup's (the wide kernel: a wave's) columns at a time.
// A column whose scaled largest is below 32 (a query of 177) does not lose as much by one small element, and one of 27000
// normal elements is that small. All columns so: 7 nodes over 131000 rows 59 us for 53, 64 over 32000 243 for 116. (With 2^-20
// over any keys queries of 71 made the latter 200.)
template <typename KT>
struct Meets {
  static constexpr int QT = 3;
  static constexpr bool SCALED = false;
  static __device__ __forceinline__ void split(const float (&x)[8], v4u (&t)[QT]) {
    split8(x, t);
#pragma unroll
    for (int e = 0; e < 8; ++e)  // an infinite query: one infinite term, not infinity - infinity beside it
#pragma unroll
      for (int k = 1; k < QT; ++k) t[k][e >> 1] &= fabsf(x[e]) == INFINITY ? (e & 1 ? 0xffffu : 0xffff0000u) : ~0u;
  }
  static __device__ __forceinline__ v4f dot(const v4u& a, const v4u& b, const v4f& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(a), as_b8(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float term(const v4u& x, int e) {
    return __builtin_bit_cast(float, e & 1 ? x[e >> 1] & 0xffff0000u : x[e >> 1] << 16);
  }
};
template <>
struct Meets<_Float16> {
  static constexpr int QT = 2;
  static constexpr bool SCALED = true;
  static __device__ __forceinline__ void split(const float (&x)[8], v4u (&t)[QT]) { halves8(x, t); }
  static __device__ __forceinline__ v4f dot(const v4u& a, const v4u& b, const v4f& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float term(const v4u& x, int e) { return nsx_h2f(e & 1 ? x[e >> 1] >> 16 : x[e >> 1] & 0xffffu); }
};
// The exponent that brings `most`, a column's largest |query|, into 2^13 .. 2^14.
__device__ __forceinline__ int query_shift(float most) {
  return most > 0.f && most < INFINITY ? 14 - max(__builtin_amdgcn_frexp_expf(most), -100) : 0;
}
// What two fp16 terms miss of 8 scaled queries beyond 2^-23 of each (infinite and NaN ones: NaN).
__device__ __forceinline__ float query_lost(const float (&x)[8], const v4u (&t)[2]) {
  float lost = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float r = fabsf((x[e] - Meets<_Float16>::term(t[0], e)) - Meets<_Float16>::term(t[1], e));
    lost += r <= 0x1p-23f * fabsf(x[e]) ? 0.f : r;
  }
  return lost;
}
// Whether a column's queries, having lost so much when scaled by 2^up, need fp32 products: over keys up to 65504 < 2^16 a
// score is off by up to 2^16 times that, of which 2^-18 is let pass.
__device__ __forceinline__ bool query_spread(float lost, int up) { return !(ldexpf(lost, -up) <= 0x1p-34f); }

// How a wave holds 32 rows of a type: K8, 8 dimensions of a key row; V4, 4 dimensions of a value row; NT, the terms that a
// key's element takes exactly (`Meets`); VT, the bf16 terms that a value's does.
//
// Weights are three bf16 terms over every type, as a light key's must keep its bits beside a heavy key whose value is zero.
// (Two fp16 terms, for fp16 values as they are, end at 2^-25: 300 keys of 2^-20 the largest weight erred by 1.6e-4 of what
// they left with the largest at 2^7, and a larger one moves that by 8 bits at most.)
template <typename KT>
struct Rows;
template <>
struct Rows<float> {
  static constexpr int NT = 3, VT = 3, BYTES = 4 * ATTN_D;
  // The 8 dimensions that lane group g of a product holds of dimensions 32 j ..: 4 g .. + 3 and the same 16 further on, so
  // that a load instruction takes 64 contiguous bytes of each row.
  static __device__ __forceinline__ int dim(int j, int g, int e) { return 32 * j + 16 * (e >> 2) + 4 * g + (e & 3); }
  struct K8 {
    v4u a, b;
  };
  using V4 = v4u;
  static __device__ __forceinline__ K8 k8(__amdgpu_buffer_rsrc_t r, int row, int j, int g) {
    const int o = row * BYTES + 128 * j + 16 * g;
    return K8{__builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(r, o, 0, 0)),
              __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(r, o + 64, 0, 0))};
  }
  static __device__ __forceinline__ V4 v4(__amdgpu_buffer_rsrc_t r, int row, int i) {
    return __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(r, row * BYTES + 16 * i, 0, 0));
  }
  static __device__ __forceinline__ K8 k8(const uint8_t* row, int j, int g) {
    return K8{*(const v4u*)(row + 128 * j + 16 * g), *(const v4u*)(row + 128 * j + 16 * g + 64)};
  }
  static __device__ __forceinline__ V4 v4(const uint8_t* row, int i) { return *(const v4u*)(row + 16 * i); }
  static __device__ __forceinline__ float k(const K8& x, int e) {
    return __builtin_bit_cast(float, e < 4 ? x.a[e & 3] : x.b[e & 3]);
  }
  static __device__ __forceinline__ float v(const V4& x, int d) { return __builtin_bit_cast(float, (uint32_t)x[d]); }
};
template <typename KT>
struct Rows16 {  // dimensions 32 j + 8 g .. + 7
  static constexpr int NT = 1, VT = std::is_same_v<KT, Bf16> ? 1 : 2, BYTES = 2 * ATTN_D;
  static __device__ __forceinline__ int dim(int j, int g, int e) { return 32 * j + 8 * g + e; }
  using K8 = v4u;
  using V4 = v2u;
  static __device__ __forceinline__ K8 k8(__amdgpu_buffer_rsrc_t r, int row, int j, int g) {
    return __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(r, row * BYTES + 64 * j + 16 * g, 0, 0));
  }
  static __device__ __forceinline__ V4 v4(__amdgpu_buffer_rsrc_t r, int row, int i) {
    return __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(r, row * BYTES + 8 * i, 0, 0));
  }
  static __device__ __forceinline__ K8 k8(const uint8_t* row, int j, int g) { return *(const v4u*)(row + 64 * j + 16 * g); }
  static __device__ __forceinline__ V4 v4(const uint8_t* row, int i) { return *(const v2u*)(row + 8 * i); }
  static __device__ __forceinline__ float one(uint32_t w, int hi) {
    if constexpr (std::is_same_v<KT, Bf16>) return __builtin_bit_cast(float, hi ? w & 0xffff0000u : w << 16);
    else return nsx_h2f(hi ? w >> 16 : w & 0xffffu);
  }
  static __device__ __forceinline__ float k(const K8& x, int e) { return one(x[e >> 1], e & 1); }
  static __device__ __forceinline__ float v(const V4& x, int d) { return one(x[d >> 1], d & 1); }
};
template <>
struct Rows<_Float16> : Rows16<_Float16> {};
template <>
struct Rows<Bf16> : Rows16<Bf16> {};

template <typename KT>
__device__ __forceinline__ void key_terms(const typename Rows<KT>::K8& x, v4u (&t)[Rows<KT>::NT]) {
  if constexpr (Rows<KT>::NT == 1) {
    t[0] = x;
  } else {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = Rows<KT>::k(x, e);
    split8(f, t);
  }
}
__device__ __forceinline__ v4f dot_bf16(const v4u& a, const v4u& b, const v4f& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(a), as_b8(b), c, 0, 0, 0);
}
// Dimension d of a lane's 8 value rows.
template <typename KT>
__device__ __forceinline__ void value_terms(const typename Rows<KT>::V4 (&x)[8], int d, v4u (&t)[Rows<KT>::VT]) {
  if constexpr (Rows<KT>::VT == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      t[0][i] = __builtin_amdgcn_perm(x[2 * i + 1][d >> 1], x[2 * i][d >> 1], d & 1 ? 0x07060302u : 0x05040100u);
  } else {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = Rows<KT>::v(x[e], d);
    split8(f, t);
  }
}

// The sines and cosines of nodes na .. nb - 1, times the amplitude: turn[node][pair of dimensions], by NT threads, a
// thread keeping its dimension, whose frequency is `freq`.
template <int NT>
__device__ __forceinline__ void tree_turns(float freq, float amp, int P, const int* depth, int na, int nb, float2* turn) {
  constexpr int HALF = ATTN_D / 2;
  for (int i = na * HALF + threadIdx.x; i < nb * HALF; i += NT) {
    float s, co;
    sincosf((float)(P + depth[i / HALF]) * freq, &s, &co);
    turn[i] = float2{co * amp, s * amp};
  }
}
// The key and value rows of nodes r0 .. r0 + rows - 1 of kv head g from the raw projections, by NT threads, a thread taking
// dimensions d and d + 32 of every NT / 32'th row: all loads at once, ahead of the sines.
template <typename KT, int NT>
struct NodeRows {
  static constexpr int HALF = ATTN_D / 2, N = NSX_TREE_MAX_NODES * HALF / NT;
  float k[N][2], v[N][2];
  __device__ __forceinline__ NodeRows(const TreeArgs& a, int g, int r0, int rows) {
    const int d = threadIdx.x % HALF, first = threadIdx.x / HALF;
    const float* x = a.q + ((int64_t)r0 * (a.n_head + 2 * a.n_kv) + a.n_head + g) * ATTN_D + d;
    float b[4];
    if (a.bk) b[0] = a.bk[g * ATTN_D + d], b[1] = a.bk[g * ATTN_D + d + HALF];
    if (a.bv) b[2] = a.bv[g * ATTN_D + d], b[3] = a.bv[g * ATTN_D + d + HALF];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int row = min(first + n * (NT / HALF), max(rows, 1) - 1);
      const float *kp = x + (int64_t)row * (a.n_head + 2 * a.n_kv) * ATTN_D, *vp = kp + (int64_t)a.n_kv * ATTN_D;
      k[n][0] = kp[0], k[n][1] = kp[HALF], v[n][0] = vp[0], v[n][1] = vp[HALF];
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (a.bk) k[n][0] += b[0], k[n][1] += b[1];
      if (a.bv) v[n][0] += b[2], v[n][1] += b[3];
    }
  }
  // f(row, d, key's two elements, value's), rotated by turn (of the node)
  template <typename F>
  __device__ __forceinline__ void each(int r0, int rows, const float2* turn, F f) const {
    const int d = threadIdx.x % HALF, first = threadIdx.x / HALF;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int row = first + n * (NT / HALF);
      if (row < rows) {
        const float2 w = turn[(r0 + row) * HALF + d];
        const float z0 = fmaf(k[n][0], w.x, -(k[n][1] * w.y)), z1 = fmaf(k[n][1], w.x, k[n][0] * w.y);  // (as rope_elem)
        f(row, d, z0, z1, v[n][0], v[n][1]);
      }
    }
  }
};
template <typename KT>
__device__ __forceinline__ void store_row(void* k, void* v, int64_t row, int d, float k0, float k1, float v0, float v1) {
  const int64_t at = row * ATTN_D + d;
  store_kv<KT>(k, at, k0), store_kv<KT>(k, at + ATTN_D / 2, k1);
  store_kv<KT>(v, at, v0), store_kv<KT>(v, at + ATTN_D / 2, v1);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.4028235e38f; }

// Workgroup (kv head g, block cb of 16 NC query columns, split c of the keys). A column is a (node, query head of the
// kv head) pair, node-major. The keys are the cache's rows from the first that any node sees, in tiles of 32, then the
// nodes' own rows in tiles of their own; a split is a run of tiles and wave w takes every NW'th of them. Splits
// past the present length return at once: the grid goes by ctx_max, so that it does not depend on the position.
//
// A tile: scores by v_mfma_f32_16x16x32_bf16 (_f16), A = 16 keys x 32 dimensions, B = 32 dimensions x 16 columns, an element
// being the sum of its terms (`Meets`, `Rows`; three bf16 terms of an fp32 value, exactly). Left out are the products of two
// terms from 2^-22 of the whole product on: the terms being cut toward zero, a product is short by 2^-21 of itself at the most,
// 2^-24 in the mean, whatever its sign. Lane l's results are column l % 16 and keys 4 (l / 16) .. + 3 of each 16: the B operand
// of the second product as they stand, when A's lane l holds of each value row the keys of its group and dimensions
// 4 (l % 16) ..; D then has column l % 16, dimensions 16 (l / 16) + 4 r + dt. So every row is read once by one wave, in
// pieces of 8 or 16 bytes, and turned into terms once for the wave's 16 NC columns, whose own terms lie in LDS.
//
// The softmax's reference m only moves (and the sums are only rescaled) when a tile has a score beyond 2^8 times it:
// weights stay below 2^8, a sum of 2^31 of them below 2^39. So a tile mostly needs no exchange between lanes.
//
// A key with weight zero takes no part whatever its value row holds (0 * NaN would be NaN): a wave whose sums are not
// finite at the end goes through its tiles again, with products in fp32 and values added one key at a time under their
// weights. (That is also what infinite keys and values take: of their terms the second is NaN. Infinite queries keep one
// term; where it meets a key's zero term, the second way has the score.)
//
// ROPE: q is the nodes' raw projections. A workgroup forms the sines and cosines of its columns' nodes (of all nodes where
// its split has some of theirs) once, as a table in LDS, and rotates its queries by it; a split with node tiles also
// makes those tiles' rows, for its own use in LDS and, the first block of columns, for the cache's keeper in wk and wv. What
// does not depend on the position is loaded ahead of it, and the first tiles ahead of the sines (a launch of its own for the
// rows, and their loads where they were used, took 23 nodes 17.7 us and 13.2; ahead 11.4, with eight waves 10.7).
//
// Bounds: few keys, the chain of dependent loads (position, parents, rows) and the launch -- one node over 203 bf16 rows 5.6
// us; many keys and few columns, their bytes -- 7 nodes over 131000 fp16 rows, 268 MB, 52 us, 5.2 TB/s; many
// columns, the terms' VALU work beside the products, which the wide kernel below shares among four waves.
template <typename KT, int NC, int NW, bool ROPE>
__global__ __launch_bounds__(64 * NW, 2) void tree_attn_kernel(TreeArgs a) {
  using R = Rows<KT>;
  using Q = Meets<KT>;
  constexpr int NT = 64 * NW, COLS = 16 * NC, KTN = R::NT, VT = R::VT, QT = Q::QT, PT = 3;
  constexpr int QROW = 2 * ATTN_D + 16, OROW = ATTN_D + 4;  // bytes of a column's term, floats of a column's sums
  constexpr int QBYTES = QT * COLS * QROW, PBYTES = TREE_KEYS * COLS * 4;
  constexpr int HALF = ATTN_D / 2, NROW = R::BYTES + 16, NBYTES = NSX_TREE_MAX_NODES * NROW;
  constexpr int TABLE = ROPE ? NSX_TREE_MAX_NODES * HALF * (int)sizeof(float2) : 0;
  constexpr int NODES_AT = QBYTES + std::max(NW * PBYTES, TABLE);
  constexpr int LDS = std::max(NODES_AT + (ROPE ? 2 * NBYTES : 0), NW * COLS * OROW * 4);
  // first the columns' query terms [term][column]; behind them the table, then each wave's weights of a tile (the second
  // way); behind those the node tiles' keys and values; in the end each wave's sums
  __shared__ __align__(16) uint8_t lds[LDS];
  __shared__ float sm[NW][COLS], sl[NW][COLS];
  __shared__ float sunit[COLS];  // scaled queries: what a column's scores are in units of
  __shared__ int sspread[NW];    // and whether a wave's columns need fp32 products
  __shared__ uint64_t svis[64];
  __shared__ int sdep[64];
  const int t = threadIdx.x, lane = t & 63, i16 = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int g = blockIdx.x % a.n_kv, cb = blockIdx.x / a.n_kv, c = blockIdx.y;
  // what does not wait for the position: the wave's parents, a thread's frequency, its eight elements of a query and
  // those that they turn with
  const int heads = ROPE ? a.n_head + 2 * a.n_kv : a.n_head;  // rows of a node in q
  const int ncol = a.nodes * a.n_rep, col0 = cb * COLS;
  const int up = wave == 0 ? tree_parent(a.parents, a.nodes, lane) : -1;
  const float freq = ROPE ? a.inv_freq[t % HALF] : 0.f;
  const int qc = t / (ATTN_D / 8), qcol = min(col0 + qc, ncol - 1), qj = t / 4 % 2, qg = t % 4;
  const int qnode = qcol / a.n_rep, qh = g * a.n_rep + qcol % a.n_rep;
  auto eight = [&](const float* p, int j, float (&x)[8]) {
    const v4f x0 = *(const v4f*)(p + R::dim(j, qg, 0)), x1 = *(const v4f*)(p + R::dim(j, qg, 4));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < 4 ? x0[e & 3] : x1[e & 3];
  };
  float qx[8], qy[8], bx[8], by[8];
  static_assert(COLS * (ATTN_D / 8) <= NT);
  if (qc < COLS) {
    const float* p = a.q + ((int64_t)qnode * heads + qh) * ATTN_D;
    eight(p, qj, qx);
    if constexpr (ROPE) {
      eight(p, qj ^ 1, qy);
      if (a.bq) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          bx[e] = a.bq[qh * ATTN_D + R::dim(qj, qg, e)], by[e] = a.bq[qh * ATTN_D + R::dim(qj ^ 1, qg, e)];
      }
    }
  }
  const int P = *a.pos;
  if (P < 0 || P > a.ctx_max) return;
  const Tiles tl(a, P, TREE_KEYS, NW);
  const int lo = tl.lo, pt = tl.cache, t0 = c * tl.per, t1 = min(tl.all, t0 + tl.per);
  if (t0 >= t1) return;
  // ROPE: the node tiles come after the loop, from LDS
  const int first = t0 + wave, end = ROPE ? min(t1, pt) : t1, last = end - 1, nodes0 = max(t0, pt);

  typename R::K8 kr[2][2];
  typename R::V4 vr[8];
  auto rsrc = [&](int tile, bool values) {  // rows past the last read as zero, as does a tile before the split's first
    const bool own = !ROPE && tile >= pt;
    const int r0 = own ? (tile - pt) * TREE_KEYS : lo + tile * TREE_KEYS;
    const int rows = tile < t0 ? 0 : min((own ? a.nodes : P) - r0, TREE_KEYS);
    const char* base = (const char*)(own ? (values ? a.dv : a.dk) : (values ? a.vc : a.kc));
    return nsx_rsrc(base + ((int64_t)g * (own ? a.max_nodes : a.ctx_max) + (tile < t0 ? 0 : r0)) * R::BYTES,
                    (uint32_t)(rows * R::BYTES));
  };
  auto load_k = [&](int tile) {
    const auto r = rsrc(tile, false);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int j = 0; j < 2; ++j) kr[kt][j] = R::k8(r, 16 * kt + i16, j, kq);
  };
  auto load_v = [&](int tile) {
    const auto r = rsrc(tile, true);
#pragma unroll
    for (int e = 0; e < 8; ++e) vr[e] = R::v4(r, 16 * (e >> 2) + 4 * kq + (e & 3), i16);
  };
  // key (or value) row k of a node tile in LDS, the last row for those past it
  auto node_row = [&](int tile, int k, bool values) {
    const int row = min((tile - pt) * TREE_KEYS + k, a.nodes - 1) - (nodes0 - pt) * TREE_KEYS;
    return (const uint8_t*)&lds[NODES_AT + (values ? NBYTES : 0) + row * NROW];
  };
  auto node_k = [&](int tile) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int j = 0; j < 2; ++j) kr[kt][j] = R::k8(node_row(tile, 16 * kt + i16, false), j, kq);
  };
  auto node_v = [&](int tile) {
#pragma unroll
    for (int e = 0; e < 8; ++e) vr[e] = R::v4(node_row(tile, 16 * (e >> 2) + 4 * kq + (e & 3), true), i16);
  };
  load_k(min(first, last));
  load_v(min(first, last));

  if (wave == 0) {
    uint64_t line = tree_lineage(up, lane);
    const int dep = __popcll(line) - 1;
    if (a.window > 0 && a.window < a.nodes) {  // ancestors out of the window
      for (int j = 0; j < a.nodes; ++j)
        if (dep - __shfl(dep, j, 64) >= a.window) line &= ~(1ull << j);
    }
    svis[lane] = line;
    sdep[lane] = dep;
  }
  float2* turn = (float2*)&lds[QBYTES];  // amplitude times (cosine, sine)
  if constexpr (ROPE) {
    const bool makes = t1 > pt;  // this split has nodes' rows: all nodes' sines, as the rows it makes are
    const int na = makes ? 0 : col0 / a.n_rep, nb = makes ? a.nodes : min(col0 + COLS - 1, ncol - 1) / a.n_rep + 1;
    if (makes) {
      const int r0 = (nodes0 - pt) * TREE_KEYS, rows = min((t1 - pt) * TREE_KEYS, a.nodes) - r0;
      const NodeRows<KT, NT> x(a, g, r0, rows);
      nsx_lds_barrier();
      tree_turns<NT>(freq, a.amp, P, sdep, na, nb, turn);
      nsx_lds_barrier();
      x.each(r0, rows, turn, [&](int row, int d, float k0, float k1, float v0, float v1) {
        uint8_t* to = &lds[NODES_AT + row * NROW];
        store_row<KT>(to, to + NBYTES, 0, d, k0, k1, v0, v1);
        if (cb == 0) store_row<KT>(a.wk, a.wv, (int64_t)g * a.max_nodes + r0 + row, d, k0, k1, v0, v1);
      });
    } else {
      nsx_lds_barrier();
      tree_turns<NT>(freq, a.amp, P, sdep, na, nb, turn);
      nsx_lds_barrier();
    }
  }
  bool spread = false;
  auto leave = [&](const v4u (&tm)[QT]) {
#pragma unroll
    for (int k = 0; k < QT; ++k) *(v4u*)&lds[(k * COLS + qc) * QROW + (4 * qj + qg) * 16] = tm[k];
  };
  if (qc < COLS) {
    if constexpr (ROPE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (a.bq) qx[e] += bx[e], qy[e] += by[e];
        const float2 w = turn[qnode * HALF + R::dim(0, qg, e)];
        const float ps = qy[e] * w.y;
        qx[e] = fmaf(qx[e], w.x, qj ? ps : -ps);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) qx[e] *= a.scale2;
    v4u tm[QT];
    if constexpr (Q::SCALED) {
      float most = 0.f, x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(qx[e]));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor(most, o, 64));  // (a column's eight threads)
      const int up = query_shift(most);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = ldexpf(qx[e], up);
      if (t % 8 == 0) sunit[qc] = ldexpf(1.f, -up);
      Q::split(x, tm);
      float lost = query_lost(x, tm);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) lost += __shfl_xor(lost, o, 64);
      spread = query_spread(lost, up);
    } else {
      Q::split(qx, tm);
    }
    leave(tm);
  }
  if constexpr (Q::SCALED) {
    const int any = __any(spread);
    if (lane == 0) sspread[wave] = any;
  }
  nsx_lds_barrier();
  bool exact = false;  // the queries are in LDS as fp32 values, four in place of each term
  if constexpr (Q::SCALED) {
    int some = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) some |= sspread[w];
    exact = __builtin_amdgcn_readfirstlane(some) != 0;
    if (exact) {
      if (qc < COLS) {
        v4u x[QT];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = __builtin_bit_cast(uint32_t, qx[e]);
        leave(x);
        if (t % 8 == 0) sunit[qc] = 1.f;
      }
      nsx_lds_barrier();
    }
  }
  const int q0 = i16 * QROW + kq * 16;
  auto query = [&](int k, int ct, int j) { return *(const v4u*)&lds[q0 + (k * COLS + 16 * ct) * QROW + 64 * j]; };
  // a column's node: what it sees of the nodes, its first visible row of the cache
  auto node_of = [&](int ct) { return min(col0 + 16 * ct + i16, ncol - 1) / a.n_rep; };
  float unit[NC];
  if constexpr (Q::SCALED) {
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) unit[ct] = sunit[16 * ct + i16];
  }
  int deepest = 0;  // the last of the columns' first rows
  if (a.window > 0) {
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) deepest = max(deepest, P + sdep[node_of(ct)] + 1 - a.window);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) deepest = max(deepest, __shfl_xor(deepest, o, 64));
    deepest = __builtin_amdgcn_readfirstlane(deepest);
  }

  float m[NC], l[NC];
  v4f acc[NC][4];
  float* sp = (float*)&lds[QBYTES + wave * PBYTES];  // the second way's weights, [key][column]
  auto start = [&] {
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) {
      m[ct] = ATTN_LOWEST;
      l[ct] = 0.f;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) acc[ct][dt] = v4f{0.f, 0.f, 0.f, 0.f};
    }
  };
  // scores in powers of two -> weights; what a column does not see has none
  auto weights = [&](int tile, v4f (&s)[NC][2]) {
    if constexpr (Q::SCALED) {
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int n = 0; n < 2; ++n) s[ct][n] *= unit[ct];
    }
    const bool own = tile >= pt;
    const int r0 = own ? (tile - pt) * TREE_KEYS : lo + tile * TREE_KEYS;
    if (own) {
#pragma unroll
      for (int ct = 0; ct < NC; ++ct) {
        const uint64_t vis = svis[node_of(ct)];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint32_t bits = (uint32_t)(vis >> (r0 + 16 * n + 4 * kq));
#pragma unroll
          for (int r = 0; r < 4; ++r) s[ct][n][r] = bits & (1u << r) ? s[ct][n][r] : -INFINITY;
        }
      }
    } else if (r0 + TREE_KEYS > P || r0 < deepest) {
#pragma unroll
      for (int ct = 0; ct < NC; ++ct) {
        const int from = a.window > 0 ? P + sdep[node_of(ct)] + 1 - a.window : 0;
        const int lo_k = from - r0 - 4 * kq, hi_k = P - r0 - 4 * kq;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int k = 16 * (e >> 2) + (e & 3);
          s[ct][e >> 2][e & 3] = k >= lo_k && k < hi_k ? s[ct][e >> 2][e & 3] : -INFINITY;
        }
      }
    }
    float mx[NC];
    bool move = false;
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) {
      mx[ct] = fmaxf(s[ct][0][0], s[ct][0][1]);
#pragma unroll
      for (int e = 2; e < 8; ++e) mx[ct] = fmaxf(mx[ct], s[ct][e >> 2][e & 3]);
      move = move || mx[ct] > m[ct] + 8.f;
    }
    if (__any(move)) {
#pragma unroll
      for (int ct = 0; ct < NC; ++ct) {
        float mn = fmaxf(mx[ct], __shfl_xor(mx[ct], 16, 64));
        mn = fmaxf(m[ct], fmaxf(mn, __shfl_xor(mn, 32, 64)));
        const float corr = __builtin_amdgcn_exp2f(m[ct] - mn);  // (first tile: of nothing)
        m[ct] = mn;
        l[ct] *= corr;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) acc[ct][dt] *= corr;
      }
    }
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = __builtin_amdgcn_exp2f(s[ct][e >> 2][e & 3] - m[ct]);
        s[ct][e >> 2][e & 3] = w;
        l[ct] += w;  // this lane group's keys; the groups are added at the end
      }
    }
  };

  // scores of the keys in kr by fp32 products
  auto scores32 = [&](v4f (&s)[NC][2]) {
#pragma unroll
    for (int ct = 0; ct < NC; ++ct)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        v4u qt[QT];
#pragma unroll
        for (int k = 0; k < QT; ++k) qt[k] = query(k, ct, j);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float q = Q::term(qt[QT - 1], e);
#pragma unroll
          for (int k = QT - 2; k >= 0; --k) q += Q::term(qt[k], e);
          if (exact) q = __builtin_bit_cast(float, (uint32_t)qt[e >> 2][e & 3]);
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
            s[ct][kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(R::k(kr[kt][j], e), q, s[ct][kt], 0, 0, 0);
        }
      }
  };
  // a tile whose rows are in kr and vr, the next one's loads on their way as soon as they are free
  auto take = [&](int tile, auto next_k, auto next_v) {
    v4f s[NC][2] = {};
    if (Q::SCALED && exact) {
      scores32(s);
      next_k();
    } else {
      v4u kt_[2][2][KTN];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int j = 0; j < 2; ++j) key_terms<KT>(kr[kt][j], kt_[kt][j]);
      next_k();
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) {
          v4u q[QT];
#pragma unroll
          for (int k = 0; k < QT; ++k) q[k] = query(k, ct, j);
#pragma unroll
          for (int o = QT - 1; o >= 0; --o)  // (the small products first)
#pragma unroll
            for (int k = 0; k <= o; ++k)
              if (o - k < KTN) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
                  s[ct][kt] = Q::dot(kt_[kt][j][o - k], q[k], s[ct][kt]);
              }
        }
    }
    weights(tile, s);
    v4u pw[NC][PT];
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s[ct][e >> 2][e & 3];
      split8(x, pw[ct]);
    }
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      v4u vt[VT];
      value_terms<KT>(vr, dt, vt);
      if (dt == 3) next_v();
#pragma unroll
      for (int o = PT - 1; o >= 0; --o)
#pragma unroll
        for (int k = 0; k <= o; ++k)
          if (o - k < VT) {
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) acc[ct][dt] = dot_bf16(vt[o - k], pw[ct][k], acc[ct][dt]);
          }
    }
  };

  start();
  int tile = first;
  for (; tile < end; tile += NW) {
    const int next = min(tile + NW, last);
    take(tile, [&] { load_k(next); }, [&] { load_v(next); });
  }
  if constexpr (ROPE) {
#pragma unroll 1
    for (; tile < t1; tile += NW) {
      node_k(tile);
      node_v(tile);
      take(tile, [] {}, [] {});
    }
  }
  bool ok = true;
#pragma unroll
  for (int ct = 0; ct < NC; ++ct)
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) ok = ok && finite(acc[ct][dt][r]);
  if (!__all(ok)) {
    start();
#pragma unroll 1
    for (int tile = first; tile < t1; tile += NW) {
      const bool in_lds = ROPE && tile >= pt;
      if (in_lds) node_k(tile);
      else load_k(tile);
      v4f s[NC][2] = {};
      scores32(s);
      weights(tile, s);
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int e = 0; e < 8; ++e) sp[(16 * (e >> 2) + 4 * kq + (e & 3)) * COLS + 16 * ct + i16] = s[ct][e >> 2][e & 3];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const auto r = rsrc(in_lds ? t0 - 1 : tile, true);
#pragma unroll 1
      for (int k = 0; k < TREE_KEYS; ++k) {
        typename R::V4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = in_lds ? R::v4(node_row(tile, k, true), 4 * kq + u) : R::v4(r, k, 4 * kq + u);
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) {
          const float w = sp[k * COLS + 16 * ct + i16];
          if (w != 0.f) {
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
              for (int u = 0; u < 4; ++u) acc[ct][dt][u] = fmaf(w, R::v(v[u], dt), acc[ct][dt][u]);
          }
        }
      }
    }
  }

  nsx_lds_barrier();  // (the sums take the query terms' place)
  float(*sacc)[COLS][OROW] = (float(*)[COLS][OROW])lds;
#pragma unroll
  for (int ct = 0; ct < NC; ++ct) {
    l[ct] += __shfl_xor(l[ct], 16, 64);
    l[ct] += __shfl_xor(l[ct], 32, 64);
    if (kq == 0) {
      sm[wave][16 * ct + i16] = m[ct];
      sl[wave][16 * ct + i16] = l[ct];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *(v4f*)&sacc[wave][16 * ct + i16][16 * kq + 4 * r] = v4f{acc[ct][0][r], acc[ct][1][r], acc[ct][2][r], acc[ct][3][r]};
  }
  nsx_lds_barrier();
  const bool whole = a.nsplit == 1;
  for (int i = t; i < min(COLS, ncol - col0) * ATTN_D; i += NT) {
    const int cc = i / ATTN_D, d = i % ATTN_D, col = col0 + cc;
    const int h = g * a.n_rep + col % a.n_rep;
    const int64_t row = (int64_t)(col / a.n_rep) * a.n_head + h;
    const float sink = whole && a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
    float M = sink;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w][cc]);
    float Z = whole && a.sinks ? __builtin_amdgcn_exp2f(sink - M) : 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {  // (a wave without a tile has weight 0)
      const float e = __builtin_amdgcn_exp2f(sm[w][cc] - M);
      Z = fmaf(e, sl[w][cc], Z);
      v = fmaf(e, sacc[w][cc][d], v);
    }
    if (whole) {
      a.out[row * ATTN_D + d] = v / Z;
    } else {
      a.part[(row * a.nsplit + c) * ATTN_D + d] = v;
      if (d == 0) {
        float* ml = a.part + ((int64_t)a.nodes * a.n_head * ATTN_D + row * 2) * a.nsplit + 2 * c;
        ml[0] = M;
        ml[1] = Z;
      }
    }
  }
}

// The same attention for many columns: a workgroup of 8 waves takes 128 columns and a split of the keys. Four waves (32
// columns each) make a group, the two groups share the split's tiles of KEYS keys, and a tile's rows become terms once
// for the group: each wave loads a part of them, splits it and leaves it in LDS as the operands that every wave of the
// group then reads.
//
// A tile takes two phases: products (the scores of tile i, the values of tile i - 1) and the rest (the weights of
// tile i, the terms of keys i + 1 and values i). Waves w and w + 4 share a SIMD, and their groups are one phase apart, kept
// so by the barrier between phases: the matrix cores have one group's products while the VALU has the other's weights.
//
// Bound by the phases' shared issue: 64 nodes over 65536 bf16 keys (64 / 8 heads, three products a term pair: 206 GFLOP of
// bf16) 184 us back to back, 1120 TFLOP/s, what a large library product reaches here (1108; a call at a time under a profiler
// took 206 to 250); 64 nodes over 6000 fp32 keys (six products)
// 48 us, 16 over 16384 38; 64 over 32000 fp16 keys (two of the scores, five of the values) 116. Of an iteration's 5450 cycles over fp32 rows the products take
// 1870 and the rest 2530, the VALU issuing an instruction in 8 beside the other group's products. Both groups in one phase
// 188 for an earlier 160, no offset between them 184; scheduler groups, one barrier a tile, 32 x 32 products, two workgroups of
// four waves: all within 5 % or slower.
//
// ROPE as above, the table where the first tiles come afterwards; a split with nodes' rows writes them beside the cache
// and loads them back as it does the cache's.
template <typename KT, bool ROPE>
__global__ __launch_bounds__(512, 2) void tree_wide_kernel(TreeArgs a) {
  using R = Rows<KT>;
  using Q = Meets<KT>;
  constexpr int KTN = R::NT, VT = R::VT, QT = Q::QT, PT = 3, NC = 2, CW = 4, NG = 2, COLS = 16 * NC * CW;
  constexpr int TPP = KTN == 1 ? 2 : 1, KEYS = 32 * TPP;  // 16-bit rows: two tiles a phase, as their phases are short
  constexpr int KF = TPP * 4 * KTN, VF = TPP * 4 * VT;    // operands (64 lanes x 16 bytes) of a tile's keys and values
  constexpr int GROUP = (KF + VF) * 1024, OROW = ATTN_D + 4;
  constexpr int PBYTES = 32 * 16 * NC * 4;  // a wave's weights of 32 keys (the second way)
  constexpr int LDS = std::max(std::max(NG * GROUP, 8 * PBYTES), CW * 16 * NC * OROW * 4);
  __shared__ __align__(16) uint8_t lds[LDS];
  __shared__ float sm[CW][16 * NC], sl[CW][16 * NC];
  __shared__ uint64_t svis[64];
  __shared__ int sdep[64];
  const int t = threadIdx.x, lane = t & 63, i16 = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int group = wave / CW, cw = wave % CW;  // waves w and w + 4 lie on one SIMD
  const int g = blockIdx.x % a.n_kv, cb = blockIdx.x / a.n_kv, c = blockIdx.y;
  // what does not wait for the position: the wave's parents, a thread's frequency, its queries
  constexpr int HALF = ATTN_D / 2;
  const int heads = ROPE ? a.n_head + 2 * a.n_kv : a.n_head;  // rows of a node in q
  const int ncol = a.nodes * a.n_rep, col0 = cb * COLS + 16 * NC * cw;
  const int up = wave == 0 ? tree_parent(a.parents, a.nodes, lane) : -1;
  const float freq = ROPE ? a.inv_freq[t % HALF] : 0.f;
  float qx[NC][2][8], qb[NC][2][8];
#pragma unroll
  for (int ct = 0; ct < NC; ++ct) {
    const int col = min(col0 + 16 * ct + i16, ncol - 1), h = g * a.n_rep + col % a.n_rep;
    const float* qp = a.q + ((int64_t)(col / a.n_rep) * heads + h) * ATTN_D;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const v4f x0 = *(const v4f*)(qp + R::dim(j, kq, 0)), x1 = *(const v4f*)(qp + R::dim(j, kq, 4));
#pragma unroll
      for (int e = 0; e < 8; ++e) qx[ct][j][e] = e < 4 ? x0[e & 3] : x1[e & 3];
    }
    if (ROPE && a.bq) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) qb[ct][j][e] = a.bq[h * ATTN_D + R::dim(j, kq, e)];
    }
  }
  const int P = *a.pos;
  if (P < 0 || P > a.ctx_max) return;
  const Tiles tl(a, P, KEYS, 1);
  const int lo = tl.lo, pt = tl.cache, t0 = c * tl.per, t1 = min(tl.all, t0 + tl.per);
  if (t0 >= t1) return;
  const int phases = (t1 - t0 + 1) / 2;               // tiles of the first group, the most
  const int mine = (t1 - t0 + 1 - group) / 2;  // of this one: t0 + group, + 2, ..

  uint8_t* kl = lds + group * GROUP;
  uint8_t* vl = kl + KF * 1024;
  // where tile i of the group lies; rows past the last, and tiles past the group's, read as zero
  struct Source {
    int64_t at;  // bytes from the start of the rows
    uint32_t bytes;
    bool own;
  };
  auto source = [&](int i) {
    const int tile = t0 + group + 2 * i;
    const bool own = tile >= pt;
    const int r0 = own ? (tile - pt) * KEYS : lo + tile * KEYS, rows = min((own ? a.nodes : P) - r0, KEYS);
    const int64_t head = (int64_t)g * (own ? a.max_nodes : a.ctx_max);
    return i < mine ? Source{(head + r0) * R::BYTES, (uint32_t)(rows * R::BYTES), own} : Source{0, 0, false};
  };
  auto rsrc = [&](const Source& x, bool values) {
    return nsx_rsrc((const char*)(x.own ? (values ? a.dv : a.dk) : (values ? a.vc : a.kc)) + x.at, x.bytes);
  };
  // This wave's part of a tile: items cw, cw + CW, .. of 4 a subtile. Of the keys an item is 16 rows x 32 dimensions; of the
  // values 16 rows x 32 dimensions too, a lane holding rows 4 kq .. + 3 of dimensions 2 i16, 2 i16 + 1.
  constexpr int ITEMS = TPP * 4 / CW;
  using V2 = std::conditional_t<std::is_same_v<KT, float>, v2u, uint32_t>;
  typename R::K8 kr[ITEMS];
  V2 vr[ITEMS][4];
  auto load_k = [&](const Source& x) {
    const auto r = rsrc(x, false);
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int n = cw + CW * it;  // [subtile][kt][j]
      kr[it] = R::k8(r, 16 * (n >> 1) + i16, n & 1, kq);
    }
  };
  auto load_v = [&](const Source& x) {
    const auto r = rsrc(x, true);
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int n = cw + CW * it;  // [subtile][kt][half of the dimensions]
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int o = (16 * (n >> 1) + 4 * kq + k) * R::BYTES + (n & 1) * (R::BYTES / 2) + i16 * (R::BYTES / 32);
        if constexpr (std::is_same_v<KT, float>) vr[it][k] = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(r, o, 0, 0));
        else vr[it][k] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, o, 0, 0);
      }
    }
  };
  auto store_k = [&] {
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      v4u x[KTN];
      key_terms<KT>(kr[it], x);
#pragma unroll
      for (int k = 0; k < KTN; ++k) *(v4u*)(kl + ((cw + CW * it) * KTN + k) * 1024 + lane * 16) = x[k];
    }
  };
  auto store_v = [&] {  // operand [subtile][half][dimension's parity]: the kt'th 8 bytes of a lane
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int n = cw + CW * it, sub = n >> 2, kt = (n >> 1) & 1, half = n & 1;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        v2u x[VT];
        if constexpr (VT == 1) {
          const uint32_t sel = b ? 0x07060302u : 0x05040100u;
          x[0] = v2u{__builtin_amdgcn_perm(vr[it][1], vr[it][0], sel), __builtin_amdgcn_perm(vr[it][3], vr[it][2], sel)};
        } else {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            float f[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              if constexpr (std::is_same_v<KT, float>) f[q] = __builtin_bit_cast(float, (uint32_t)vr[it][2 * p + q][b]);
              else f[q] = nsx_h2f(b ? vr[it][2 * p + q] >> 16 : vr[it][2 * p + q] & 0xffffu);
            }
#pragma unroll
            for (int k = 0; k < VT; ++k) {
              x[k][p] = top2(f[0], f[1]);
              if (k + 1 < VT) f[0] = below(f[0]), f[1] = below(f[1]);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < VT; ++k)
          *(v2u*)(vl + (((sub * 2 + half) * 2 + b) * VT + k) * 1024 + lane * 16 + kt * 8) = x[k];
      }
    }
  };
  // ROPE: a split with nodes' rows makes them first
  const bool makes = ROPE && t1 > pt;
  Source src = source(0);
  if (!makes || !src.own) {
    load_k(src);
    load_v(src);
  }
  if (wave == 0) {
    uint64_t line = tree_lineage(up, lane);
    const int dep = __popcll(line) - 1;
    if (a.window > 0 && a.window < a.nodes) {  // ancestors out of the window
      for (int j = 0; j < a.nodes; ++j)
        if (dep - __shfl(dep, j, 64) >= a.window) line &= ~(1ull << j);
    }
    svis[lane] = line;
    sdep[lane] = dep;
  }
  static_assert(!ROPE || NSX_TREE_MAX_NODES * HALF * (int)sizeof(float2) <= LDS);
  float2* turn = (float2*)lds;  // amplitude times (cosine, sine); the first tiles come over it, a barrier later
  if constexpr (ROPE) {
    const int na = makes ? 0 : cb * COLS / a.n_rep, nb = makes ? a.nodes : min(cb * COLS + COLS - 1, ncol - 1) / a.n_rep + 1;
    if (makes) {
      const int r0 = (max(t0, pt) - pt) * KEYS, rows = min((t1 - pt) * KEYS, a.nodes) - r0;
      const NodeRows<KT, 512> x(a, g, r0, rows);
      nsx_lds_barrier();
      tree_turns<512>(freq, a.amp, P, sdep, na, nb, turn);
      nsx_lds_barrier();
      x.each(r0, rows, turn, [&](int row, int d, float k0, float k1, float v0, float v1) {
        store_row<KT>(a.wk, a.wv, (int64_t)g * a.max_nodes + r0 + row, d, k0, k1, v0, v1);  // (every block the same)
      });
      __syncthreads();  // this workgroup's stores, ahead of its loads
      if (src.own) {
        load_k(src);
        load_v(src);
      }
    } else {
      nsx_lds_barrier();
      tree_turns<512>(freq, a.amp, P, sdep, na, nb, turn);
      nsx_lds_barrier();
    }
  }
  v4u q[NC][2][QT];
  float unit[NC];  // scaled queries: what a column's scores are in units of
  bool exact = false;  // q holds the queries as fp32 values, four in place of each term
#pragma unroll
  for (int ct = 0; ct < NC; ++ct) {
    if constexpr (ROPE) {
      const int node = min(col0 + 16 * ct + i16, ncol - 1) / a.n_rep;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (a.bq) qx[ct][0][e] += qb[ct][0][e], qx[ct][1][e] += qb[ct][1][e];
        const float2 w = turn[node * HALF + R::dim(0, kq, e)];
        const float x0 = qx[ct][0][e], x1 = qx[ct][1][e];
        qx[ct][0][e] = fmaf(x0, w.x, -(x1 * w.y)), qx[ct][1][e] = fmaf(x1, w.x, x0 * w.y);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) qx[ct][j][e] *= a.scale2;
    if constexpr (Q::SCALED) {
      float most = 0.f, lost = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(qx[ct][j][e]));
      most = fmaxf(most, __shfl_xor(most, 16, 64));
      const int up = query_shift(fmaxf(most, __shfl_xor(most, 32, 64)));
      unit[ct] = ldexpf(1.f, -up);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = ldexpf(qx[ct][j][e], up);
        Q::split(x, q[ct][j]);
        lost += query_lost(x, q[ct][j]);
      }
      lost += __shfl_xor(lost, 16, 64);
      lost += __shfl_xor(lost, 32, 64);
      exact = exact || query_spread(lost, up);
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) Q::split(qx[ct][j], q[ct][j]);
    }
  }
  if constexpr (Q::SCALED) {
    exact = __any(exact);
    if (exact) {
#pragma unroll
      for (int ct = 0; ct < NC; ++ct) {
        unit[ct] = 1.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) q[ct][j][e >> 2][e & 3] = __builtin_bit_cast(uint32_t, qx[ct][j][e]);
      }
    }
  }
  nsx_lds_barrier();
  uint64_t vis[NC];
  int from[NC], deepest = 0;  // the columns' first visible cache rows, and the last of them
#pragma unroll
  for (int ct = 0; ct < NC; ++ct) {
    const int node = min(col0 + 16 * ct + i16, ncol - 1) / a.n_rep;
    vis[ct] = svis[node];
    from[ct] = a.window > 0 ? P + sdep[node] + 1 - a.window : 0;
    deepest = max(deepest, from[ct]);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) deepest = max(deepest, __shfl_xor(deepest, o, 64));
  deepest = __builtin_amdgcn_readfirstlane(deepest);

  float m[NC], l[NC];
  v4f acc[NC][4];  // [dimension's half, parity]
  v4f s[NC][2 * TPP];
  v4u pw[NC][TPP][PT];
  auto start = [&] {
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) {
      m[ct] = ATTN_LOWEST;
      l[ct] = 0.f;
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[ct][f] = v4f{0.f, 0.f, 0.f, 0.f};
    }
  };
  // scores in powers of two -> weights, 16 keys each of N; r0: the first key's row (own: of the nodes)
  auto weights = [&](auto& x, auto n_tag, bool own, int r0) {
    constexpr int N = decltype(n_tag)::value;
    if constexpr (Q::SCALED) {
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int n = 0; n < N; ++n) x[ct][n] *= unit[ct];
    }
    if (own) {
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const uint32_t bits = (uint32_t)(vis[ct] >> (r0 + 16 * n + 4 * kq));
#pragma unroll
          for (int r = 0; r < 4; ++r) x[ct][n][r] = bits & (1u << r) ? x[ct][n][r] : -INFINITY;
        }
    } else if (r0 + 16 * N > P || r0 < deepest) {
#pragma unroll
      for (int ct = 0; ct < NC; ++ct) {
        const int lo_k = from[ct] - r0 - 4 * kq, hi_k = P - r0 - 4 * kq;
#pragma unroll
        for (int e = 0; e < 4 * N; ++e) {
          const int k = 16 * (e >> 2) + (e & 3);
          x[ct][e >> 2][e & 3] = k >= lo_k && k < hi_k ? x[ct][e >> 2][e & 3] : -INFINITY;
        }
      }
    }
    float mx[NC];
    bool move = false;
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) {
      mx[ct] = fmaxf(x[ct][0][0], x[ct][0][1]);
#pragma unroll
      for (int e = 2; e < 4 * N; ++e) mx[ct] = fmaxf(mx[ct], x[ct][e >> 2][e & 3]);
      move = move || mx[ct] > m[ct] + 8.f;
    }
    if (__any(move)) {
#pragma unroll
      for (int ct = 0; ct < NC; ++ct) {
        float mn = fmaxf(mx[ct], __shfl_xor(mx[ct], 16, 64));
        mn = fmaxf(m[ct], fmaxf(mn, __shfl_xor(mn, 32, 64)));
        const float corr = __builtin_amdgcn_exp2f(m[ct] - mn);  // (first tile: of nothing)
        m[ct] = mn;
        l[ct] *= corr;
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[ct][f] *= corr;
      }
    }
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) {
#pragma unroll
      for (int e = 0; e < 4 * N; ++e) {
        const float w = __builtin_amdgcn_exp2f(x[ct][e >> 2][e & 3] - m[ct]);
        x[ct][e >> 2][e & 3] = w;
        l[ct] += w;  // this lane group's keys; the groups are added at the end
      }
    }
  };
  // query e of 8, for fp32 products
  auto query32 = [&](int ct, int j, int e) {
    float x = Q::term(q[ct][j][QT - 1], e);
#pragma unroll
    for (int k = QT - 2; k >= 0; --k) x += Q::term(q[ct][j][k], e);
    return exact ? __builtin_bit_cast(float, (uint32_t)q[ct][j][e >> 2][e & 3]) : x;
  };
  auto phase = [] {
    __builtin_amdgcn_sched_barrier(0);
    nsx_lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };

  // The products of a tile step by step, an operand set each: the values of tile i - 1 (the first time: zeros under no
  // weights), then the keys of tile i (the last time: what is there, unused). A step's operands are read AHEAD steps early.
  constexpr int STEPS = 8 * TPP, VSTEPS = 4 * TPP, AHEAD = VT == 1 ? 4 : 1, MOST = VT > KTN ? VT : KTN;
  auto products = [&] {
    v4u x[AHEAD + 1][MOST];
    auto read = [&](int n) {
      const uint8_t* at = n < VSTEPS ? vl + n * VT * 1024 : kl + (n - VSTEPS) * KTN * 1024;
#pragma unroll
      for (int k = 0; k < (n < VSTEPS ? VT : KTN); ++k) x[n % (AHEAD + 1)][k] = *(const v4u*)(at + k * 1024 + lane * 16);
    };
#pragma unroll
    for (int ct = 0; ct < NC; ++ct)
#pragma unroll
      for (int n = 0; n < 2 * TPP; ++n) s[ct][n] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) read(n);
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
      if (n + AHEAD < STEPS) read(n + AHEAD);
      const v4u(&y)[MOST] = x[n % (AHEAD + 1)];
      if (n < VSTEPS) {
#pragma unroll
        for (int o = PT - 1; o >= 0; --o)  // (the small products first)
#pragma unroll
          for (int k = 0; k <= o; ++k)
            if (o - k < VT) {
#pragma unroll
              for (int ct = 0; ct < NC; ++ct) acc[ct][n % 4] = dot_bf16(y[o - k], pw[ct][n / 4][k], acc[ct][n % 4]);
            }
      } else {
        const int kn = n - VSTEPS;
#pragma unroll
        for (int o = QT - 1; o >= 0; --o)
#pragma unroll
          for (int k = 0; k <= o; ++k)
            if (o - k < KTN) {
#pragma unroll
              for (int ct = 0; ct < NC; ++ct) s[ct][kn / 2] = Q::dot(y[o - k], q[ct][kn % 2][k], s[ct][kn / 2]);
            }
      }
    }
    // the order above, kept by the scheduler: LDS reads (0x100) ahead of the products (0x8); of the first and second kind
    constexpr int VPRODUCTS = NC * (VT == 3 ? 6 : VT == 2 ? 5 : 3), KPRODUCTS = NC * (KTN == 3 ? 6 : QT);
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * VT, 0);
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
      if (n + AHEAD < VSTEPS) __builtin_amdgcn_sched_group_barrier(0x100, VT, 0);
      else if (n + AHEAD < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, KTN, 0);
      if (n < VSTEPS) __builtin_amdgcn_sched_group_barrier(0x8, VPRODUCTS, 0);
      else __builtin_amdgcn_sched_group_barrier(0x8, KPRODUCTS, 0);
    }
  };

  // the scores of the tile in LDS by fp32 products, in place of those above
  auto scores32 = [&] {
    if constexpr (Q::SCALED) {
#pragma unroll
      for (int n = 0; n < 4 * TPP; ++n) {
        const auto x = __builtin_bit_cast(typename R::K8, *(const v4u*)(kl + n * 1024 + lane * 16));
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) {
          if (n % 2 == 0) s[ct][n / 2] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 8; ++e)
            s[ct][n / 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(R::k(x, e), query32(ct, n % 2, e), s[ct][n / 2], 0, 0, 0);
        }
      }
    }
  };

  start();
#pragma unroll
  for (int ct = 0; ct < NC; ++ct)
#pragma unroll
    for (int u = 0; u < TPP; ++u) {
#pragma unroll
      for (int k = 0; k < PT; ++k) pw[ct][u][k] = v4u{0, 0, 0, 0};
    }
#pragma unroll
  for (int n = 0; n < VF / CW; ++n) *(v4u*)(vl + (cw + CW * n) * 1024 + lane * 16) = v4u{0, 0, 0, 0};
  store_k();
  src = source(1);  // the tile whose keys are in registers and whose values are next
  load_k(src);
  if (group) phase();
  phase();
#pragma unroll 1
  for (int i = 0; i <= phases; ++i) {
    if (i <= mine) {
      __builtin_amdgcn_s_setprio(1);
      products();
      __builtin_amdgcn_s_setprio(0);
      if (Q::SCALED && exact) scores32();
    }
    phase();
    if (i < mine) {
      const int tile = t0 + group + 2 * i;
      const bool own = tile >= pt;
      store_v();
      store_k();
      load_v(src);
      src = source(i + 2);
      load_k(src);
      weights(s, std::integral_constant<int, 2 * TPP>{}, own, own ? (tile - pt) * KEYS : lo + tile * KEYS);
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int u = 0; u < TPP; ++u) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = s[ct][2 * u + (e >> 2)][e & 3];
          split8(x, pw[ct][u]);
        }
    }
    phase();
  }
  if (!group) phase();

  bool ok = true;
#pragma unroll
  for (int ct = 0; ct < NC; ++ct)
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r) ok = ok && finite(acc[ct][f][r]);
  if (!__all(ok)) {  // the second way, by this wave alone
    float* sp = (float*)&lds[wave * PBYTES];
    start();
#pragma unroll 1
    for (int i = 0; i < mine * TPP; ++i) {
      const int tile = t0 + group + 2 * (i / TPP);
      const bool own = tile >= pt;
      const Source tile_at = source(i / TPP);
      const auto rk = rsrc(tile_at, false), rv = rsrc(tile_at, true);
      const int sub = 32 * (i % TPP), r0 = (own ? (tile - pt) * KEYS : lo + tile * KEYS) + sub;
      v4f x[NC][2] = {};
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const auto kk = R::k8(rk, sub + 16 * kt + i16, j, kq);
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int ct = 0; ct < NC; ++ct)
              x[ct][kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(R::k(kk, e), query32(ct, j, e), x[ct][kt], 0, 0, 0);
        }
      weights(x, std::integral_constant<int, 2>{}, own, r0);
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int e = 0; e < 8; ++e) sp[(16 * (e >> 2) + 4 * kq + (e & 3)) * (16 * NC) + 16 * ct + i16] = x[ct][e >> 2][e & 3];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
      for (int k = 0; k < 32; ++k) {
        typename R::V4 v[2][2];  // dimensions 32 h + 8 kq ..
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int u = 0; u < 2; ++u) v[h][u] = R::v4(rv, sub + k, 8 * h + 2 * kq + u);
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) {
          const float w = sp[k * (16 * NC) + 16 * ct + i16];
          if (w != 0.f) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int d = 0; d < 8; ++d)
                acc[ct][2 * h + (d & 1)][d >> 1] = fmaf(w, R::v(v[h][d >> 2], d & 3), acc[ct][2 * h + (d & 1)][d >> 1]);
          }
        }
      }
    }
  }

  // the second group's sums join the first's
#pragma unroll
  for (int ct = 0; ct < NC; ++ct) {
    l[ct] += __shfl_xor(l[ct], 16, 64);
    l[ct] += __shfl_xor(l[ct], 32, 64);
  }
  float(*so)[16 * NC][OROW] = (float(*)[16 * NC][OROW])lds;
  nsx_lds_barrier();
  if (group) {
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) {
      if (kq == 0) sm[cw][16 * ct + i16] = m[ct], sl[cw][16 * ct + i16] = l[ct];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          *(v4f*)&so[cw][16 * ct + i16][32 * h + 8 * kq + 4 * u] =
              v4f{acc[ct][2 * h][2 * u], acc[ct][2 * h + 1][2 * u], acc[ct][2 * h][2 * u + 1], acc[ct][2 * h + 1][2 * u + 1]};
    }
  }
  nsx_lds_barrier();
  if (group) return;
  const bool whole = a.nsplit == 1;
#pragma unroll
  for (int ct = 0; ct < NC; ++ct) {
    const int cc = 16 * ct + i16, col = col0 + cc;
    if (col >= ncol) continue;
    const int h = g * a.n_rep + col % a.n_rep;
    const int64_t row = (int64_t)(col / a.n_rep) * a.n_head + h;
    const float sink = whole && a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
    const float M = fmaxf(sink, fmaxf(m[ct], sm[cw][cc]));
    const float e0 = __builtin_amdgcn_exp2f(m[ct] - M), e1 = __builtin_amdgcn_exp2f(sm[cw][cc] - M);  // (no tile: 0)
    const float Z = (whole && a.sinks ? __builtin_amdgcn_exp2f(sink - M) : 0.f) + fmaf(e0, l[ct], e1 * sl[cw][cc]);
    float* to = whole ? a.out + row * ATTN_D : a.part + (row * a.nsplit + c) * ATTN_D;
    const float div = whole ? Z : 1.f;
#pragma unroll
    for (int d = 0; d < 16; d += 4) {
      const int at = 32 * (d >> 3) + 8 * kq + (d & 7);
      const v4f x = *(const v4f*)&so[cw][cc][at];
      v4f v;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int dd = d + k;
        v[k] = fmaf(e1, x[k], e0 * acc[ct][2 * (dd >> 3) + (dd & 1)][(dd & 7) >> 1]) / div;
      }
      *(v4f*)(to + at) = v;
    }
    if (!whole && kq == 0) {
      float* ml = a.part + ((int64_t)a.nodes * a.n_head * ATTN_D + row * 2) * a.nsplit + 2 * c;
      ml[0] = M;
      ml[1] = Z;
    }
  }
}

// WPR waves per (node, query head): merge the live splits with the sink. Every wave forms all the splits' weights (lane =
// split); then 16 lanes take a split's 64 values, so a wave adds four splits a load, WPR waves 4 WPR, and the lanes' and
// waves' sums meet. Bound by its two rounds of loads and the launch: 4.7 us for 1024 rows of 32 splits (one wave each), 4.9
// for 448 rows of 64 (four).
template <int WPR>
__global__ __launch_bounds__(256) void tree_combine_kernel(TreeArgs a) {
  constexpr int LPS = TREE_MAX_SPLIT / 64;  // splits per lane
  __shared__ float ws[4][TREE_MAX_SPLIT];
  __shared__ v4f red[4][16];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, part = wave % WPR, i16 = lane & 15, kq = lane >> 4;
  const int64_t rows = (int64_t)a.nodes * a.n_head, row = min((int64_t)blockIdx.x * (4 / WPR) + wave / WPR, rows - 1);
  const int P = *a.pos;
  if (P < 0 || P > a.ctx_max) return;
  const Tiles tl(a, P, a.keys, a.round);
  const int nc = (tl.all + tl.per - 1) / tl.per;  // 1 <= nc <= nsplit
  const float* ml = a.part + (rows * ATTN_D + row * 2) * a.nsplit;
  const float sink = a.sinks ? a.sinks[row % a.n_head] * LOG2E : -INFINITY;
  float mv[LPS], lv[LPS], M = sink;
#pragma unroll
  for (int i = 0; i < LPS; ++i) {
    const int s = min(lane + 64 * i, nc - 1);
    mv[i] = ml[2 * s];
    lv[i] = ml[2 * s + 1];
    M = fmaxf(M, mv[i]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  float z = 0.f;
#pragma unroll
  for (int i = 0; i < LPS; ++i) {
    const float e = lane + 64 * i < nc ? __builtin_amdgcn_exp2f(mv[i] - M) : 0.f;
    ws[wave][lane + 64 * i] = e;  // (splits past the last: weight 0)
    z = fmaf(e, lv[i], z);
  }
  const float Z = nsx_wave_sum(z) + (a.sinks ? __builtin_amdgcn_exp2f(sink - M) : 0.f);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own weights
  const float* pv = a.part + row * a.nsplit * ATTN_D + 4 * i16;
  v4f v = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = 4 * part + kq; c0 < nc; c0 += 16 * WPR) {
    v4f x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = *(const v4f*)(pv + (int64_t)min(c0 + 4 * WPR * u, nc - 1) * ATTN_D);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = c0 + 4 * WPR * u;
      const float e = s < nc ? ws[wave][s] : 0.f;
#pragma unroll
      for (int d = 0; d < 4; ++d) v[d] = fmaf(e, x[u][d], v[d]);
    }
  }
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    v[d] += __shfl_xor(v[d], 16, 64);
    v[d] += __shfl_xor(v[d], 32, 64);
  }
  if constexpr (WPR > 1) {
    if (kq == 0) red[wave][i16] = v;
    __syncthreads();
    v = (red[0][i16] + red[1][i16]) + (red[2][i16] + red[3][i16]);
  }
  if (part == 0 && kq == 0) *(v4f*)(a.out + row * ATTN_D + 4 * i16) = v / Z;
}

// Accepted nodes' rows into the caches: path[j] to row pos + j for j < count, then pos moves on. A thread takes one
// 16-byte piece of a key row and the same of the value row, over (layer and kv head, j, piece). Every workgroup reads pos
// and counts itself out; the last one moves it and leaves the counter at zero for the next call. (Nothing else passes
// between workgroups, so no fence: what the last one knows is that all others have pos.) Latency, two rounds of loads: 3.8
// us for 6 rows of 36 layers.
__global__ __launch_bounds__(256) void tree_commit_kernel(char* __restrict__ kc, char* __restrict__ vc,
                                                          const char* __restrict__ dk, const char* __restrict__ dv,
                                                          int row_bytes, int heads, int nodes, int max_nodes,
                                                          const int32_t* __restrict__ path,
                                                          const int32_t* __restrict__ count, int32_t* pos,
                                                          int64_t ctx_max, uint32_t* out) {
  const int pieces = row_bytes / 16;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(i % pieces), j = (int)(i / pieces % nodes);
  const int64_t h = i / pieces / nodes;
  const int src = path[j], p = *pos, n = max(0, min(*count, nodes));
  if (h < heads && j < n && p >= 0 && (int64_t)p + j < ctx_max && src >= 0 && src < max_nodes) {
    const int64_t from = (h * max_nodes + src) * row_bytes + 16 * c, to = (h * ctx_max + p + j) * row_bytes + 16 * c;
    const v4u k = *(const v4u*)(dk + from), v = *(const v4u*)(dv + from);
    *(v4u*)(kc + to) = k;
    *(v4u*)(vc + to) = v;
  }
  __syncthreads();  // every wave of the workgroup has pos
  if (threadIdx.x == 0 && atomicAdd(out, 1u) == gridDim.x - 1) {
    *out = 0;
    if (p >= 0 && p <= ctx_max) *pos = (int32_t)min((int64_t)p + n, ctx_max);
  }
}

// ---------------------------------------------------------------------------

enum { TREE_16, TREE_32, TREE_WIDE };  // kernel by the columns of its workgroups: 16, 32, 128

// Which kernel a call runs, and its grid.
struct TreePlan {
  int kind, ncb, nsplit, keys, round;
  bool alone;  // 16 columns, all keys: eight waves
};

// `work` counts pieces of 32 keys x 16 columns. Below 12288, twelve for each SIMD of the chip, the kernel of 16 columns has
// the most workgroups and the shortest way through one (us for 16 / 32 / 128 columns at 64 / 8 heads, fp32, 4000 keys:
// 16 nodes 22.9 / 23.7 / 26.3, 32 nodes 30.1 / 27.6 / 31.0; bf16 17.6 / 20.2 / 24.6 and 21.7 / 21.2 / 27.5). Past it, more
// than 64 columns go to the wide kernel once its sharing of terms outweighs its longer way, the sooner the more terms an
// element has: three from 32768 pieces on (fp32, 64 nodes, 4000 keys 52.3 / 41.3 / 42.6, 8000 keys 86.4 / 64.8 / 60.0), two from
// 49152 (fp16 values; 64 nodes, 8000 keys 54.8 / 44.9 / 43.5; 16 nodes, 32000 keys 54.7 / 44.5 / 41.8, 16000 keys 33.3 / 28.6 /
// 29.1), one from 98304 (bf16, 64 nodes, 16000 keys 95.0 / 59.8 / 60.6, 32000 keys 177 / 104 / 101, 8000 keys 52.7 / 36.8 /
// 42.5).
//
// The columns themselves do not enter below that: with 16 or fewer the kernel of 16 stays ahead past 12288 pieces too (8
// columns over 32000 rows: by 7 % over fp32, 16 over 16-bit rows), which takes 8 kv heads and 49152 rows to reach. And the
// choice goes by the capacity, so that a captured call serves every position: a cache a tenth full costs up to half as much
// again (us full / a tenth full of the capacity's choice, from projections: one node, 13107 rows, fp32 18.0 / 19.6, bf16 13.3 /
// 14.4; 16 nodes, 1638 rows 17.2 / 23.2 and 13.8 / 16.7; 64 nodes, 600 rows 22.0 / 26.8 and 12.4 / 20.4, 6000 rows 49.3 / 49.2 and
// 33.4 / 38.0).
//
// Few tiles are one workgroup's, of eight waves, rather than splits with a merge behind them: with up to 96 KB of keys, where
// the merge costs as much as the longer way, and some more where the grid is large (us alone / split: one node of 64 / 8
// heads, bf16, 17 tiles 9.1 / 10.0, 33 tiles 11.2 / 10.0; fp32, 11 tiles 10.6 / 10.9, 17 tiles 12.9 / 10.8; 40 nodes, fp32, 15
// tiles 13.0 / 20.7, 21 tiles 15.5 / 18.2). Four waves do for four tiles (one node, 3 tiles, fp32 8.2, with eight 8.8).
TreePlan tree_plan(int n_kv, int n_rep, int nodes, int64_t ctx_max, int window, int kv_dtype) {
  const int64_t cols = (int64_t)nodes * n_rep, rows = window > 0 ? std::min<int64_t>(ctx_max, window) : ctx_max;
  const int64_t work = n_kv * nsx_cdiv(cols, 16) * nsx_cdiv(rows, 32);
  const int terms = kv_dtype == NSX_DT_F32 ? 3 : kv_dtype == NSX_DT_F16 ? 2 : 1;  // of a value
  TreePlan p;
  p.kind = work < 12288 ? TREE_16 : cols > 64 && work * terms >= 98304 ? TREE_WIDE : TREE_32;
  const bool wide = p.kind == TREE_WIDE;
  p.keys = wide && terms < 3 ? 2 * TREE_KEYS : TREE_KEYS;
  p.round = wide ? 1 : TREE_NW;
  p.ncb = (int)nsx_cdiv(cols, p.kind == TREE_16 ? 16 : p.kind == TREE_32 ? 32 : 128);
  const int64_t tiles = nsx_cdiv(rows, p.keys) + nsx_cdiv(nodes, p.keys);
  const int64_t step = wide ? 2 : TREE_NW;  // tiles that a workgroup takes at a time
  // workgroups that the chip holds at once: two of four waves a CU, or one of eight
  const int64_t fill = wide ? TREE_GRID / 2 : TREE_GRID;
  p.alone = p.kind == TREE_16 && tiles > TREE_NW && tiles <= (terms == 3 ? 12 : 24) + (n_kv * p.ncb >= 64 ? 8 : 0);
  p.nsplit = tiles <= 2 * step || p.alone ? 1
      : (int)std::min<int64_t>({nsx_cdiv(tiles, step), nsx_cdiv(fill, n_kv * (int64_t)p.ncb), TREE_MAX_SPLIT});
  return p;
}

int64_t tree_bytes(int n_head, int n_kv, int nodes, int64_t ctx_max, int window, int kv_dtype) {
  // a split's values and (maximum, sum) per row
  return (int64_t)nodes * n_head * tree_plan(n_kv, n_head / n_kv, nodes, ctx_max, window, kv_dtype).nsplit * (ATTN_D + 2) * 4;
}

int tree_shapes(int n_head, int n_kv, int head_dim, int nodes, int max_nodes, int64_t ctx_max, int window) {
  NSX_REQUIRE(head_dim == ATTN_D, NSX_ENOTIMPL, "head_dim %d (the kernels are written for 64)", head_dim);
  NSX_REQUIRE(n_head > 0 && n_kv > 0 && n_head % n_kv == 0 && n_head / n_kv <= ATTN_MAX_REP, NSX_EINVAL,
              "n_head=%d, n_kv=%d: n_head must be a multiple of n_kv, at most %d per kv head", n_head, n_kv,
              ATTN_MAX_REP);
  NSX_REQUIRE(n_kv <= 65536, NSX_EINVAL, "n_kv=%d", n_kv);
  NSX_REQUIRE(nodes > 0 && nodes <= max_nodes && max_nodes <= NSX_TREE_MAX_NODES, NSX_EINVAL,
              "%d nodes of at most %d (limit %d)", nodes, max_nodes, NSX_TREE_MAX_NODES);
  NSX_REQUIRE(ctx_max > 0 && ctx_max < (1ll << 31) - 64 && window >= 0, NSX_EINVAL, "ctx_max=%lld window=%d",
              (long long)ctx_max, window);
  return NSX_OK;
}

template <typename KT, bool ROPE>
int tree_attn_typed(TreeArgs& a, const TreePlan& p, hipStream_t st) {
  a.nsplit = p.nsplit;
  a.ncb = p.ncb;
  a.keys = p.keys;
  a.round = p.round;
  const dim3 grid(a.n_kv * a.ncb, a.nsplit);
  if (p.alone) {
    hipLaunchKernelGGL((tree_attn_kernel<KT, 1, 2 * TREE_NW, ROPE>), grid, dim3(128 * TREE_NW), 0, st, a);
  } else if (p.kind == TREE_16) {
    hipLaunchKernelGGL((tree_attn_kernel<KT, 1, TREE_NW, ROPE>), grid, dim3(64 * TREE_NW), 0, st, a);
  } else if (p.kind == TREE_32) {
    hipLaunchKernelGGL((tree_attn_kernel<KT, 2, TREE_NW, ROPE>), grid, dim3(64 * TREE_NW), 0, st, a);
  } else {
    hipLaunchKernelGGL((tree_wide_kernel<KT, ROPE>), grid, dim3(512), 0, st, a);
  }
  NSX_LAUNCHED();
  if (a.nsplit > 1) {
    // a wave per row, or four where the rows are few and their splits many
    const int rows = a.nodes * a.n_head;
    if (a.nsplit > 32) hipLaunchKernelGGL(tree_combine_kernel<4>, dim3(rows), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(tree_combine_kernel<1>, dim3((rows + 3) / 4), dim3(256), 0, st, a);
    NSX_LAUNCHED();
  }
  return NSX_OK;
}

template <bool ROPE>
int tree_attn_launch(TreeArgs& a, int kv_dtype, hipStream_t st) {
  const TreePlan p = tree_plan(a.n_kv, a.n_rep, a.nodes, a.ctx_max, a.window, kv_dtype);
  if (kv_dtype == NSX_DT_F32) return tree_attn_typed<float, ROPE>(a, p, st);
  if (kv_dtype == NSX_DT_F16) return tree_attn_typed<_Float16, ROPE>(a, p, st);
  return tree_attn_typed<Bf16, ROPE>(a, p, st);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int64_t kv_elem(int dt) { return dt == NSX_DT_F32 ? 4 : 2; }

}  // namespace

extern "C" int64_t nsx_tree_workspace_bytes(int n_head, int n_kv, int head_dim, int max_nodes, int64_t ctx_max) {
  if (tree_shapes(n_head, n_kv, head_dim, max_nodes, max_nodes, ctx_max, 0) != NSX_OK) return -1;
  int64_t most = 0;  // fewer nodes or a window may take more splits, never more than the cache's rows do
  for (int n = 1; n <= max_nodes; ++n)
    for (const int dt : {NSX_DT_F32, NSX_DT_F16, NSX_DT_BF16})
      most = std::max(most, tree_bytes(n_head, n_kv, n, ctx_max, 0, dt));
  return most;
}

static int tree_checks(const void* kc, const void* vc, int kv_dtype, const void* dk, const void* dv, const int32_t* pos,
                       const void* workspace, int64_t workspace_bytes, const float* out, int n_head, int n_kv,
                       int nodes, int64_t ctx_max, int window) {
  NSX_REQUIRE(kv_dtype == NSX_DT_F32 || kv_dtype == NSX_DT_F16 || kv_dtype == NSX_DT_BF16, NSX_ETYPE,
              "cache element type %d", kv_dtype);
  NSX_REQUIRE(kc && vc && dk && dv && pos && workspace && out, NSX_EINVAL, "null buffer");
  NSX_REQUIRE(aligned16(kc) && aligned16(vc) && aligned16(dk) && aligned16(dv) && aligned16(workspace) && aligned16(out),
              NSX_EINVAL, "the caches, the nodes' rows, the workspace and out must be 16-byte aligned");
  const int64_t need = tree_bytes(n_head, n_kv, nodes, ctx_max, window, kv_dtype);
  NSX_REQUIRE(workspace_bytes >= need, NSX_EINVAL, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
              (long long)need);
  return NSX_OK;
}

extern "C" int nsx_tree_attn(const float* q, const void* k_cache, const void* v_cache, int kv_dtype,
                             const void* node_k, const void* node_v, const int32_t* parents, int n_nodes,
                             int max_nodes, const float* sinks, int n_head, int n_kv, int head_dim,
                             const int32_t* pos, int64_t ctx_max, int window, float scale, void* workspace,
                             int64_t workspace_bytes, float* out, void* stream) {
  if (const int rc = tree_shapes(n_head, n_kv, head_dim, n_nodes, max_nodes, ctx_max, window)) return rc;
  NSX_REQUIRE(q && aligned16(q), NSX_EINVAL, "q must be a 16-byte aligned buffer");
  if (const int rc = tree_checks(k_cache, v_cache, kv_dtype, node_k, node_v, pos, workspace, workspace_bytes, out,
                                 n_head, n_kv, n_nodes, ctx_max, window))
    return rc;
  TreeArgs a{q, k_cache, v_cache, node_k, node_v, parents, pos, ctx_max, window, n_head / n_kv, n_kv, n_head, n_nodes,
             max_nodes, 0, 0, 0, 0, scale * LOG2E, (float*)workspace, sinks, out, nullptr,
             nullptr, nullptr, nullptr, 0.f, nullptr, nullptr};
  return tree_attn_launch<false>(a, kv_dtype, (hipStream_t)stream);
}

extern "C" int nsx_tree_attn_qkv(const float* qkv, const float* q_bias, const float* k_bias, const float* v_bias,
                                 const float* inv_freq, float amplitude, const void* k_cache, const void* v_cache,
                                 int kv_dtype, void* node_k, void* node_v, const int32_t* parents, int n_nodes,
                                 int max_nodes, const float* sinks, int n_head, int n_kv, int head_dim,
                                 const int32_t* pos, int64_t ctx_max, int window, float scale, void* workspace,
                                 int64_t workspace_bytes, float* out, void* stream) {
  if (const int rc = tree_shapes(n_head, n_kv, head_dim, n_nodes, max_nodes, ctx_max, window)) return rc;
  NSX_REQUIRE(qkv && aligned16(qkv) && inv_freq, NSX_EINVAL, "qkv must be a 16-byte aligned buffer, inv_freq not null");
  if (const int rc = tree_checks(k_cache, v_cache, kv_dtype, node_k, node_v, pos, workspace, workspace_bytes, out,
                                 n_head, n_kv, n_nodes, ctx_max, window))
    return rc;
  TreeArgs a{qkv, k_cache, v_cache, node_k, node_v, parents, pos, ctx_max, window, n_head / n_kv, n_kv, n_head, n_nodes,
             max_nodes, 0, 0, 0, 0, scale * LOG2E, (float*)workspace, sinks, out, q_bias,
             k_bias, v_bias, inv_freq, amplitude, node_k, node_v};
  return tree_attn_launch<true>(a, kv_dtype, (hipStream_t)stream);
}

extern "C" int nsx_tree_commit(void* k_caches, void* v_caches, const void* node_k, const void* node_v, int kv_dtype,
                               int n_layer, int n_kv, int head_dim, int n_nodes, int max_nodes, const int32_t* path,
                               const int32_t* count, int32_t* pos, int64_t ctx_max, uint32_t* counter,
                               void* stream) {
  if (const int rc = tree_shapes(n_kv, n_kv, head_dim, n_nodes, max_nodes, ctx_max, 0)) return rc;
  NSX_REQUIRE(n_layer > 0 && (int64_t)n_layer * n_kv < (1 << 24), NSX_EINVAL, "n_layer=%d", n_layer);
  NSX_REQUIRE(kv_dtype == NSX_DT_F32 || kv_dtype == NSX_DT_F16 || kv_dtype == NSX_DT_BF16, NSX_ETYPE,
              "cache element type %d", kv_dtype);
  NSX_REQUIRE(k_caches && v_caches && node_k && node_v && path && count && pos && counter, NSX_EINVAL, "null buffer");
  NSX_REQUIRE(aligned16(k_caches) && aligned16(v_caches) && aligned16(node_k) && aligned16(node_v), NSX_EINVAL,
              "the caches and the nodes' rows must be 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  const int row = (int)(ATTN_D * kv_elem(kv_dtype)), heads = n_layer * n_kv;
  const int64_t work = (int64_t)heads * n_nodes * (row / 16);
  hipLaunchKernelGGL(tree_commit_kernel, dim3((unsigned)nsx_cdiv(work, 256)), dim3(256), 0, st, (char*)k_caches,
                     (char*)v_caches, (const char*)node_k, (const char*)node_v, row, heads, n_nodes, max_nodes, path,
                     count, pos, ctx_max, counter);
  NSX_LAUNCHED();
  return NSX_OK;
}
