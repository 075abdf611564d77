// Dense softmax attention over packed short sequences (walks of a few nodes), forward and backward.
//
// A matrix tile of 32 rows by 32 keys holds six walks of five nodes: a sixth of its products count, and float32's are
// slow besides. Here a row of one head is a group of LPR lanes with 16 bytes of the row each, which walks the few keys
// that the row sees: dot products by shuffles within the group, the softmax's maximum and sum running in registers.
// Neighbouring groups are a token's heads, so q, out and every k and v row are read in whole cache lines, and rows of
// one sequence find its keys in the caches: what is left is one read and one write of each tensor.
//
// The backward in float32 does rows (dQ) and keys (dK, dV) of one range in one launch, so that the second finds in the
// caches what the first read; Delta of a row is formed again from out for each of its keys instead of making a round trip
// through memory. In 16-bit types out is rounded, and Delta, the second part of a difference, would carry that rounding (dQ
// of bfloat16 walks of 5 was off by up to 27 times what its own rounding allows). There the rows' launch forms it from
// the scores, and the keys' launch reads it: fewer rows are read for each pair of row and key, four tensors are read
// twice. One launch : two in us, forward and backward: 338,686 walks of 5, 8 heads of 16, bfloat16 1447 : 1400; 140,000
// rows in sequences of 2 to 5, 8 of 64, float16 404 : 422; 100,000 rows of 5, float16, 32 of 16 over 8 378 : 339.
// 338,686 walks of 5, 8 heads of 16, float32: forward 0.65 ms for 3.5 GB (5.4 TB/s), backward 1.65 ms for 6.9 GB (4.2
// TB/s); in tiles both took 8.1 ms together.
#include "packed_short.h"

#include "packed_tile.h"

namespace bf {
namespace {

struct ShortArgs {
  const void *q, *k, *v, *out, *dout;
  void *o, *dq, *dk, *dv;
  float *lse, *delta;
  const int2 *row_span, *key_span;
  int64_t qs_t, qs_h, ks_t, ks_h, vs_t, vs_h;
  int32_t n_rows, n_keys;          // (token, head) pairs of the queries, of the keys
  int32_t n_q, n_k, hq, hk, group, dim;
  Div by_hq, by_hk, by_group;
  float scale, c;
};

template <typename T> struct Chunk {               // a lane's 16 bytes of a row
  static constexpr int kN = 16 / int(sizeof(T));
  float x[kN];
  static __device__ __forceinline__ uint4 raw(const T* p) { return *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void set(const uint4& r) {
    typedef T V __attribute__((ext_vector_type(kN)));
    const V v = __builtin_bit_cast(V, r);
#pragma unroll
    for (int j = 0; j < kN; ++j) x[j] = float(v[j]);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < kN; ++j) x[j] = 0.f;
  }
  __device__ __forceinline__ float dot(const Chunk& o) const {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kN; ++j) s = fmaf(x[j], o.x[j], s);
    return s;
  }
  __device__ __forceinline__ void add(float w, const Chunk& o) {
#pragma unroll
    for (int j = 0; j < kN; ++j) x[j] = fmaf(w, o.x[j], x[j]);
  }
  __device__ __forceinline__ void store(T* p, float by) const {
    typedef T V __attribute__((ext_vector_type(kN)));
    V v;
#pragma unroll
    for (int j = 0; j < kN; ++j) v[j] = T(x[j] * by);
    *reinterpret_cast<V*>(p) = v;
  }
};

template <int LPR> __device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}

constexpr int kShortThreads = 256;
constexpr int kAhead = 4;          // keys whose loads are on their way together

template <typename T, int LPR>
__global__ __launch_bounds__(kShortThreads) void short_fwd(const ShortArgs a) {
  using Ch = Chunk<T>;
  const int part = threadIdx.x % LPR, at = part * Ch::kN;
  const int64_t item = int64_t(blockIdx.x) * (kShortThreads / LPR) + threadIdx.x / LPR;
  if (item >= a.n_rows) return;                      // whole groups: shuffles stay within them
  const bool mine = at < a.dim;
  const int d = mine ? at : 0;                       // lanes behind the row read its first values and add zeros
  const int token = int(a.by_hq(uint32_t(item))), head = int(item) - token * a.hq, h = int(a.by_group(uint32_t(head)));
  const int2 span = a.row_span[token];
  const int lo = max(span.x, 0), hi = min(span.y, a.n_k);
  Ch q, acc;
  q.set(Ch::raw(static_cast<const T*>(a.q) + token * a.qs_t + head * a.qs_h + d));
  if (!mine) q.zero();
  acc.zero();
  const T* kp = static_cast<const T*>(a.k) + h * a.ks_h + d;
  const T* vp = static_cast<const T*>(a.v) + h * a.vs_h + d;
  float mc = -INFINITY, l = 0.f;
  for (int j = lo; j < hi; j += kAhead) {
    uint4 kr[kAhead], vr[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t key = min(j + u, hi - 1);
      kr[u] = Ch::raw(kp + key * a.ks_t);
      vr[u] = Ch::raw(vp + key * a.vs_t);
    }
    float s[kAhead], top = mc;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      Ch k;
      k.set(kr[u]);
      if (!mine) k.zero();
      s[u] = row_sum<LPR>(q.dot(k)) * a.c;
      if (j + u >= hi) s[u] = -INFINITY;
      top = fmaxf(top, s[u]);
    }
    const float base = top == -INFINITY ? 0.f : top, alpha = exp2_fast(mc - base);
    mc = top;
    l *= alpha;
#pragma unroll
    for (int k = 0; k < Ch::kN; ++k) acc.x[k] *= alpha;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float p = exp2_fast(s[u] - base);
      l += p;
      Ch v;
      v.set(vr[u]);
      if (j + u < hi) acc.add(p, v);
    }
  }
  if (mine) acc.store(static_cast<T*>(a.o) + item * a.dim + at, l == 0.f ? 0.f : 1.f / l);
  if (part == 0) a.lse[item] = l == 0.f ? -INFINITY : mc + __log2f(l);
}

// float32: dQ of rows, and dK and dV of keys, of one range.
template <typename T, int LPR>
__global__ __launch_bounds__(kShortThreads) void short_bwd(const ShortArgs a) {
  using Ch = Chunk<T>;
  const int part = threadIdx.x % LPR, at = part * Ch::kN;
  const int64_t item = int64_t(blockIdx.x) * (kShortThreads / LPR) + threadIdx.x / LPR;
  const bool mine = at < a.dim;
  const int d = mine ? at : 0;
  const T* qp = static_cast<const T*>(a.q) + d;
  const T* gp = static_cast<const T*>(a.dout) + d;
  const T* op = static_cast<const T*>(a.out) + d;
  if (item < a.n_rows) {                             // dQ of a row
    const int token = int(a.by_hq(uint32_t(item))), head = int(item) - token * a.hq, h = int(a.by_group(uint32_t(head)));
    const int2 span = a.row_span[token];
    const int lo = max(span.x, 0), hi = min(span.y, a.n_k);
    Ch q, g, o, acc;
    q.set(Ch::raw(qp + token * a.qs_t + head * a.qs_h));
    g.set(Ch::raw(gp + item * a.dim));
    o.set(Ch::raw(op + item * a.dim));
    if (!mine) q.zero(), g.zero(), o.zero();
    acc.zero();
    const float delta = row_sum<LPR>(g.dot(o)), stat = a.lse[item], lse = stat == -INFINITY ? INFINITY : stat;
    const T* kp = static_cast<const T*>(a.k) + h * a.ks_h + d;
    const T* vp = static_cast<const T*>(a.v) + h * a.vs_h + d;
    for (int j = lo; j < hi; j += kAhead) {
      uint4 kr[kAhead], vr[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t key = min(j + u, hi - 1);
        kr[u] = Ch::raw(kp + key * a.ks_t);
        vr[u] = Ch::raw(vp + key * a.vs_t);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        Ch k, v;
        k.set(kr[u]);
        v.set(vr[u]);
        if (!mine) k.zero(), v.zero();
        const float s = row_sum<LPR>(q.dot(k)), dp = row_sum<LPR>(g.dot(v));
        const float ds = exp2_fast(fmaf(s, a.c, -lse)) * (dp - delta);
        if (j + u < hi) acc.add(ds, k);
      }
    }
    if (mine) acc.store(static_cast<T*>(a.dq) + item * a.dim + at, a.scale);
  }
  if (item < a.n_keys) {                             // dK and dV of a key, over its rows and their heads of the group
    const int key = int(a.by_hk(uint32_t(item))), h = int(item) - key * a.hk;
    const int2 span = a.key_span[key];
    const int lo = max(span.x, 0), hi = min(span.y, a.n_q);
    Ch k, v, dk, dv;
    k.set(Ch::raw(static_cast<const T*>(a.k) + key * a.ks_t + h * a.ks_h + d));
    v.set(Ch::raw(static_cast<const T*>(a.v) + key * a.vs_t + h * a.vs_h + d));
    if (!mine) k.zero(), v.zero();
    dk.zero(), dv.zero();
    constexpr int U = 2;
    for (int head = h * a.group; head < (h + 1) * a.group; ++head) {
      for (int i = lo; i < hi; i += U) {
        uint4 qr[U], gr[U], orr[U];
        float stat[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int row = min(i + u, hi - 1);
          const int64_t r = int64_t(row) * a.hq + head;
          qr[u] = Ch::raw(qp + row * a.qs_t + head * a.qs_h);
          gr[u] = Ch::raw(gp + r * a.dim);
          orr[u] = Ch::raw(op + r * a.dim);
          stat[u] = a.lse[r];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          Ch q, g, o;
          q.set(qr[u]), g.set(gr[u]), o.set(orr[u]);
          if (!mine) q.zero(), g.zero(), o.zero();
          const float s = row_sum<LPR>(q.dot(k)), dp = row_sum<LPR>(g.dot(v)), delta = row_sum<LPR>(g.dot(o));
          const float p = exp2_fast(fmaf(s, a.c, stat[u] == -INFINITY ? -INFINITY : -stat[u]));
          if (i + u < hi) {
            dv.add(p, g);
            dk.add(p * (dp - delta), q);
          }
        }
      }
    }
    if (mine) {
      dk.store(static_cast<T*>(a.dk) + item * a.dim + at, a.scale);
      dv.store(static_cast<T*>(a.dv) + item * a.dim + at, 1.f);
    }
  }
}

// 16-bit types: dQ and Delta of a row in one walk of its keys, without the rounded out. With Delta = sum P dP,
// sum P (dP - Delta) k is sum P dP' k - (sum P dP') (sum P k); dP' is relative to the first key's dP, so that nothing
// large cancels where the values have a part in common (and a row of one key has dQ = 0).
template <typename T, int LPR>
__global__ __launch_bounds__(kShortThreads) void short_bwd_rows(const ShortArgs a) {
  using Ch = Chunk<T>;
  const int part = threadIdx.x % LPR, at = part * Ch::kN;
  const int64_t item = int64_t(blockIdx.x) * (kShortThreads / LPR) + threadIdx.x / LPR;
  if (item >= a.n_rows) return;
  const bool mine = at < a.dim;
  const int d = mine ? at : 0;
  const int token = int(a.by_hq(uint32_t(item))), head = int(item) - token * a.hq, h = int(a.by_group(uint32_t(head)));
  const int2 span = a.row_span[token];
  const int lo = max(span.x, 0), hi = min(span.y, a.n_k);
  Ch q, g, pdk, pk;
  q.set(Ch::raw(static_cast<const T*>(a.q) + token * a.qs_t + head * a.qs_h + d));
  g.set(Ch::raw(static_cast<const T*>(a.dout) + item * a.dim + d));
  if (!mine) q.zero(), g.zero();
  pdk.zero(), pk.zero();
  const float stat = a.lse[item], lse = stat == -INFINITY ? INFINITY : stat;
  const T* kp = static_cast<const T*>(a.k) + h * a.ks_h + d;
  const T* vp = static_cast<const T*>(a.v) + h * a.vs_h + d;
  float first = 0.f, mean = 0.f;
  for (int j = lo; j < hi; j += kAhead) {
    uint4 kr[kAhead], vr[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t key = min(j + u, hi - 1);
      kr[u] = Ch::raw(kp + key * a.ks_t);
      vr[u] = Ch::raw(vp + key * a.vs_t);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      Ch k, v;
      k.set(kr[u]);
      v.set(vr[u]);
      if (!mine) k.zero(), v.zero();
      const float s = row_sum<LPR>(q.dot(k)), dp = row_sum<LPR>(g.dot(v));
      if (u == 0 && j == lo) first = dp;
      const float p = exp2_fast(fmaf(s, a.c, -lse)), pd = p * (dp - first);
      if (j + u < hi) {
        mean += pd;
        pdk.add(pd, k);
        pk.add(p, k);
      }
    }
  }
  pdk.add(-mean, pk);
  if (mine) pdk.store(static_cast<T*>(a.dq) + item * a.dim + at, a.scale);
  if (part == 0) a.delta[item] = first + mean;
}

// dK and dV of a key, over its rows and their heads of the group, with the rows' Delta from memory.
template <typename T, int LPR>
__global__ __launch_bounds__(kShortThreads) void short_bwd_keys(const ShortArgs a) {
  using Ch = Chunk<T>;
  const int part = threadIdx.x % LPR, at = part * Ch::kN;
  const int64_t item = int64_t(blockIdx.x) * (kShortThreads / LPR) + threadIdx.x / LPR;
  if (item >= a.n_keys) return;
  const bool mine = at < a.dim;
  const int d = mine ? at : 0;
  const T* qp = static_cast<const T*>(a.q) + d;
  const T* gp = static_cast<const T*>(a.dout) + d;
  const int key = int(a.by_hk(uint32_t(item))), h = int(item) - key * a.hk;
  const int2 span = a.key_span[key];
  const int lo = max(span.x, 0), hi = min(span.y, a.n_q);
  Ch k, v, dk, dv;
  k.set(Ch::raw(static_cast<const T*>(a.k) + key * a.ks_t + h * a.ks_h + d));
  v.set(Ch::raw(static_cast<const T*>(a.v) + key * a.vs_t + h * a.vs_h + d));
  if (!mine) k.zero(), v.zero();
  dk.zero(), dv.zero();
  constexpr int U = 4;
  for (int head = h * a.group; head < (h + 1) * a.group; ++head) {
    for (int i = lo; i < hi; i += U) {
      uint4 qr[U], gr[U];
      float stat[U], delta[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = min(i + u, hi - 1);
        const int64_t r = int64_t(row) * a.hq + head;
        qr[u] = Ch::raw(qp + row * a.qs_t + head * a.qs_h);
        gr[u] = Ch::raw(gp + r * a.dim);
        stat[u] = a.lse[r], delta[u] = a.delta[r];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        Ch q, g;
        q.set(qr[u]), g.set(gr[u]);
        if (!mine) q.zero(), g.zero();
        const float s = row_sum<LPR>(q.dot(k)), dp = row_sum<LPR>(g.dot(v));
        const float p = exp2_fast(fmaf(s, a.c, stat[u] == -INFINITY ? -INFINITY : -stat[u]));
        if (i + u < hi) {
          dv.add(p, g);
          dk.add(p * (dp - delta[u]), q);
        }
      }
    }
  }
  if (mine) {
    dk.store(static_cast<T*>(a.dk) + item * a.dim + at, a.scale);
    dv.store(static_cast<T*>(a.dv) + item * a.dim + at, 1.f);
  }
}

ShortArgs make_args(const bf_packed_attn* p, const void* q, const void* k, const void* v) {
  ShortArgs a{};
  a.q = q, a.k = k, a.v = v;
  a.row_span = reinterpret_cast<const int2*>(p->row_span);
  a.key_span = reinterpret_cast<const int2*>(p->key_span);
  a.qs_t = p->q_stride[0], a.qs_h = p->q_stride[1];
  a.ks_t = p->k_stride[0], a.ks_h = p->k_stride[1];
  a.vs_t = p->v_stride[0], a.vs_h = p->v_stride[1];
  a.hq = p->heads_q, a.hk = p->heads_k, a.group = p->heads_q / p->heads_k, a.dim = p->head_dim;
  a.n_rows = int32_t(p->n_q * a.hq);
  a.n_keys = int32_t(p->n_k * a.hk);
  a.n_q = int32_t(p->n_q), a.n_k = int32_t(p->n_k);
  a.by_hq = make_div(uint32_t(a.hq)), a.by_hk = make_div(uint32_t(a.hk)), a.by_group = make_div(uint32_t(a.group));
  a.scale = p->scale, a.c = p->scale * kLog2e;
  return a;
}

// f(T(), lanes of a row) for a call.
template <typename F> int with_lanes(const bf_packed_attn* p, F&& f) {
  return with_type(p->dtype, [&](auto t) -> int {
    using T = decltype(t);
    const int lanes = p->head_dim * int(sizeof(T)) / 16;
    if (lanes <= 1) return f(t, std::integral_constant<int, 1>());
    if (lanes <= 2) return f(t, std::integral_constant<int, 2>());
    if (lanes <= 4) return f(t, std::integral_constant<int, 4>());
    if (lanes <= 8) return f(t, std::integral_constant<int, 8>());
    if (lanes <= 16) return f(t, std::integral_constant<int, 16>());
    return f(t, std::integral_constant<int, 32>());
  });
}

}  // namespace

// A row costs a key's lanes for every key it sees here, and its share of whole tiles otherwise. Forward and backward of
// 25,000 to 1.6 million rows took, as lanes : tiles in us, causal and not,
//   float32, heads of 16:  8 keys 299..345 : 743, 16 keys 426..544 : 745, 24 keys 499..727 : 949..1036, 32 keys 692..906 : 698..744
//   bfloat16, heads of 16: 8 keys 170..188 : 488, 16 keys 220..276 : 491, 24 keys 281..372 : 492, 32 keys 359..512 : 465
//   bfloat16, heads of 64: 4 keys 141..144 : 268, 8 keys 194..209 : 270, 16 keys 270..367 : 233
//   bfloat16, heads of 128: 4 keys 203..249 : 308, 8 keys 318..473 : 253
//   float32, heads of 64:  4 keys 285..329 : 665, 8 keys 403..509 : 669, 16 keys 663..916 : 668
// Heads that share keys fill a tile with fewer tokens, which masks less of it (100,000 rows, 5, 12 and 24 tokens):
//   float16, 32 heads of 16 over 8: 343, 524, 880 : 461, 441, 447; bfloat16, 32 of 32 over 4: 642, 906, 1562 : 559, 560, 573
//   float32, 16 heads of 16 over 1: 271, 365, 601 : 399, 413, 462; 16 of 64 over 2: 1123, 1657, 2899 : 1284, 1296, 1359
// A call of few rows leaves most of the chip idle either way and is as long as its longest chain, for lanes the rows of a
// key's group (2000 rows, 12 and 24 tokens; float16, 8 heads of 128 over 4: 39, 60 : 78, 80; bfloat16, 16 of 64 over 8: 38, 56 : 36, 37):
//   bfloat16, 8 of 64: 27, 41 : 44, 46; float32, 8 of 128: 87, 103 : 123, 123
bool packed_is_short(const bf_packed_attn* p) {
  const bool wide = p->dtype == BF_DTYPE_F32;
  const int64_t row = int64_t(p->head_dim) * (wide ? 4 : 2), group = p->heads_q / p->heads_k;
  if (p->longest <= 0 || p->longest > 24 || p->n_k >= kMaxRows / p->heads_k) return false;
  const int64_t most = group > 2 ? (wide ? 1280 : 256) : (wide ? 2048 : 1024);
  const bool few = p->longest * group <= 40 && p->n_q * p->heads_q * row <= (int64_t(wide ? 8 : 4) << 20);
  return few || p->longest * row <= most;
}

int packed_short_fwd(const bf_packed_attn* p, const void* q, const void* k, const void* v, void* out, float* lse,
                     hipStream_t st) {
  ShortArgs a = make_args(p, q, k, v);
  a.o = out, a.lse = lse;
  return with_lanes(p, [&](auto t, auto lanes) -> int {
    using T = decltype(t);
    constexpr int LPR = decltype(lanes)::value;
    auto kern = short_fwd<T, LPR>;
    BF_LAUNCH("packed_attn_fwd_short", kern, dim3(unsigned(ceil_div(a.n_rows, kShortThreads / LPR))), dim3(kShortThreads), 0, st,
              a);
    BF_CHECK_LAUNCH();
    return BF_OK;
  });
}

int packed_short_bwd(const bf_packed_attn* p, const void* q, const void* k, const void* v, const void* out, const float* lse,
                     const void* dout, void* dq, void* dk, void* dv, float* delta, hipStream_t st) {
  ShortArgs a = make_args(p, q, k, v);
  a.out = out, a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv;
  a.lse = const_cast<float*>(lse), a.delta = delta;
  return with_lanes(p, [&](auto t, auto lanes) -> int {
    using T = decltype(t);
    constexpr int LPR = decltype(lanes)::value;
    const dim3 block(kShortThreads);
    if constexpr (sizeof(T) == 2) {
      if (a.n_rows > 0) {
        auto rows = short_bwd_rows<T, LPR>;
        BF_LAUNCH("packed_attn_bwd_short_rows", rows, dim3(unsigned(ceil_div(a.n_rows, kShortThreads / LPR))), block, 0, st, a);
        BF_CHECK_LAUNCH();
      }
      if (a.n_keys > 0) {
        auto keys = short_bwd_keys<T, LPR>;
        BF_LAUNCH("packed_attn_bwd_short_keys", keys, dim3(unsigned(ceil_div(a.n_keys, kShortThreads / LPR))), block, 0, st, a);
        BF_CHECK_LAUNCH();
      }
    } else {
      const int64_t most = a.n_rows > a.n_keys ? a.n_rows : a.n_keys;
      if (most == 0) return BF_OK;
      auto kern = short_bwd<T, LPR>;
      BF_LAUNCH("packed_attn_bwd_short", kern, dim3(unsigned(ceil_div(most, kShortThreads / LPR))), block, 0, st, a);
      BF_CHECK_LAUNCH();
    }
    return BF_OK;
  });
}

}  // namespace bf
