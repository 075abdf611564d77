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

constexpr int kFar = 24;                        // short sequences' distances: -kFar .. kFar

struct ShortBias {
  const float* table;                           // [hq, buckets]
  const int32_t *map, *positions;
  float* part;
  int32_t buckets, reach;
};

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
  ShortBias bias;
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

// With a bias (BIAS) a workgroup takes several ranges of rows (or keys), so that what it keeps in LDS is formed once: the heads' values
// by distance in log2 units, and for the table's gradient a column of sums for each of its keys, by head of the group and bucket. The next
// range's keys are of the same heads (the workgroups are a multiple of them), and nobody else adds to a column.
constexpr int kShortGroups = 2048;
constexpr int kByDistance = 2 * kFar + 1;

__device__ __forceinline__ int short_bucket(const ShortBias& b, int x) {       // of distance x - kFar
  const int at = min(max(x - kFar, -b.reach), b.reach) + b.reach;
  return min(max(b.map[at], 0), b.buckets - 1);
}
__device__ __forceinline__ void stage_short(const ShortArgs& a, float* values, int* buckets) {
  for (int x = threadIdx.x; x < kByDistance; x += kShortThreads) {
    const int b = short_bucket(a.bias, x);
    if (buckets) buckets[x] = b;
    for (int h = 0; h < a.hq; ++h) values[h * kByDistance + x] = a.bias.table[int64_t(h) * a.bias.buckets + b] * kLog2e;
  }
}
__device__ __forceinline__ int short_at(int distance) { return min(max(distance, -kFar), kFar) + kFar; }

// f(item) for the workgroup's items; without a bias one each.
template <bool BIAS, int PER, typename F> __device__ __forceinline__ void each_item(int64_t n, F&& f) {
  int64_t block = blockIdx.x;
  f(block * PER + threadIdx.x / (kShortThreads / PER));
  if constexpr (BIAS)
    for (block += gridDim.x; block * PER < n; block += gridDim.x) f(block * PER + threadIdx.x / (kShortThreads / PER));
}
constexpr int kAhead = 4;          // keys whose loads are on their way together

template <typename T, int LPR, bool BIAS>
__global__ __launch_bounds__(kShortThreads) void short_fwd(const ShortArgs a) {
  using Ch = Chunk<T>;
  extern __shared__ float short_lds[];
  const int part = threadIdx.x % LPR, at = part * Ch::kN;
  if constexpr (BIAS) {
    stage_short(a, short_lds, nullptr);
    __syncthreads();
  }
  each_item<BIAS, kShortThreads / LPR>(a.n_rows, [&](int64_t item) {
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
    int place = 0;
    if constexpr (BIAS) place = span.x + a.bias.positions[token];
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
        if constexpr (BIAS) s[u] += short_lds[head * kByDistance + short_at(j + u - place)];
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
  });
}

// The columns of the table's gradient: by head of the group and bucket, a key's beside its neighbours'.
template <int PER> __device__ __forceinline__ float* short_cols(const ShortArgs& a, float* lds) {
  float* cols = lds + a.hq * kByDistance + kByDistance;
  for (int i = threadIdx.x; i < a.group * a.bias.buckets * PER; i += kShortThreads) cols[i] = 0.f;
  return cols;
}
template <int PER> __device__ __forceinline__ void store_cols(const ShortArgs& a, const float* cols) {
  __syncthreads();
  const int nb = a.bias.buckets, base = int(int64_t(blockIdx.x) * PER % a.hk);
  float* part = a.bias.part + int64_t(blockIdx.x) * a.hq * nb;
  for (int o = threadIdx.x; o < a.hq * nb; o += kShortThreads) {
    const int head = o / nb, h = head / a.group, g = head - h * a.group;
    const float* c = cols + (g * nb + (o - head * nb)) * PER;
    float sum = 0.f;
    for (int i = h >= base ? h - base : h - base + a.hk; i < PER; i += a.hk) sum += c[i];
    part[o] = sum;
  }
}

// float32: dQ of rows, and dK and dV of keys, of one range.
template <typename T, int LPR, bool BIAS>
__global__ __launch_bounds__(kShortThreads) void short_bwd(const ShortArgs a) {
  using Ch = Chunk<T>;
  extern __shared__ float short_lds[];
  constexpr int PER = kShortThreads / LPR;
  const int part = threadIdx.x % LPR, at = part * Ch::kN;
  int* buckets = nullptr;
  float* cols = nullptr;
  if constexpr (BIAS) {
    buckets = reinterpret_cast<int*>(short_lds + a.hq * kByDistance);
    stage_short(a, short_lds, buckets);
    cols = short_cols<PER>(a, short_lds) + threadIdx.x / LPR;
    __syncthreads();
  }
  each_item<BIAS, PER>(max(a.n_rows, a.n_keys), [&](int64_t item) {
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
      int place = 0;
      if constexpr (BIAS) place = span.x + a.bias.positions[token];
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
          const float less = BIAS ? lse - short_lds[head * kByDistance + short_at(j + u - place)] : lse;
          const float ds = exp2_fast(fmaf(s, a.c, -less)) * (dp - delta);
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
      int first = 0;                                   // the place that stands at the first row; the others follow
      if constexpr (BIAS) first = lo < hi ? a.row_span[lo].x + a.bias.positions[lo] : 0;
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
            const int x = BIAS ? short_at(key - first - (i + u - lo)) : 0;
            const float more = BIAS ? short_lds[head * kByDistance + x] : 0.f;
            const float p = exp2_fast(fmaf(s, a.c, stat[u] == -INFINITY ? -INFINITY : BIAS ? more - stat[u] : -stat[u]));
            if (i + u < hi) {
              const float ds = p * (dp - delta);
              dv.add(p, g);
              dk.add(ds, q);
              if (BIAS && part == 0) cols[((head - h * a.group) * a.bias.buckets + buckets[x]) * PER] += ds;
            }
          }
        }
      }
      if (mine) {
        dk.store(static_cast<T*>(a.dk) + item * a.dim + at, a.scale);
        dv.store(static_cast<T*>(a.dv) + item * a.dim + at, 1.f);
      }
    }
  });
  if constexpr (BIAS) store_cols<PER>(a, cols - threadIdx.x / LPR);
}

// 16-bit types: dQ and Delta of a row in one walk of its keys, without the rounded out. With Delta = sum P dP,
// sum P (dP - Delta) k is sum P dP' k - (sum P dP') (sum P k); dP' is relative to the first key's dP, so that nothing
// large cancels where the values have a part in common (and a row of one key has dQ = 0).
template <typename T, int LPR, bool BIAS>
__global__ __launch_bounds__(kShortThreads) void short_bwd_rows(const ShortArgs a) {
  using Ch = Chunk<T>;
  extern __shared__ float short_lds[];
  const int part = threadIdx.x % LPR, at = part * Ch::kN;
  if constexpr (BIAS) {
    stage_short(a, short_lds, nullptr);
    __syncthreads();
  }
  each_item<BIAS, kShortThreads / LPR>(a.n_rows, [&](int64_t item) {
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
    int place = 0;
    if constexpr (BIAS) place = span.x + a.bias.positions[token];
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
        const float less = BIAS ? lse - short_lds[head * kByDistance + short_at(j + u - place)] : lse;
        const float p = exp2_fast(fmaf(s, a.c, -less)), pd = p * (dp - first);
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
  });
}

// dK and dV of a key, over its rows and their heads of the group, with the rows' Delta from memory.
template <typename T, int LPR, bool BIAS>
__global__ __launch_bounds__(kShortThreads) void short_bwd_keys(const ShortArgs a) {
  using Ch = Chunk<T>;
  extern __shared__ float short_lds[];
  constexpr int PER = kShortThreads / LPR;
  const int part = threadIdx.x % LPR, at = part * Ch::kN;
  int* buckets = nullptr;
  float* cols = nullptr;
  if constexpr (BIAS) {
    buckets = reinterpret_cast<int*>(short_lds + a.hq * kByDistance);
    stage_short(a, short_lds, buckets);
    cols = short_cols<PER>(a, short_lds) + threadIdx.x / LPR;
    __syncthreads();
  }
  each_item<BIAS, PER>(a.n_keys, [&](int64_t item) {
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
    int first = 0;                                     // as in short_bwd
    if constexpr (BIAS) first = lo < hi ? a.row_span[lo].x + a.bias.positions[lo] : 0;
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
          const int x = BIAS ? short_at(key - first - (i + u - lo)) : 0;
          const float more = BIAS ? short_lds[head * kByDistance + x] : 0.f;
          const float p = exp2_fast(fmaf(s, a.c, stat[u] == -INFINITY ? -INFINITY : BIAS ? more - stat[u] : -stat[u]));
          if (i + u < hi) {
            const float ds = p * (dp - delta[u]);
            dv.add(p, g);
            dk.add(ds, q);
            if (BIAS && part == 0) cols[((head - h * a.group) * a.bias.buckets + buckets[x]) * PER] += ds;
          }
        }
      }
    }
    if (mine) {
      dk.store(static_cast<T*>(a.dk) + item * a.dim + at, a.scale);
      dv.store(static_cast<T*>(a.dv) + item * a.dim + at, 1.f);
    }
  });
  if constexpr (BIAS) store_cols<PER>(a, cols - threadIdx.x / LPR);
}

ShortArgs make_args(const bf_packed_attn* p, const bf_packed_bias* bias, const void* q, const void* k, const void* v) {
  ShortArgs a{};
  if (bias) a.bias = ShortBias{bias->table, bias->map, bias->positions, nullptr, bias->buckets, bias->reach};
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

int lanes_of(const bf_packed_attn* p) {
  const int lanes = p->head_dim * (p->dtype == BF_DTYPE_F32 ? 4 : 2) / 16;
  return lanes <= 1 ? 1 : lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32;
}

// f(T(), lanes of a row, whether with a bias) for a call.
template <typename F> int with_lanes(const bf_packed_attn* p, const bf_packed_bias* bias, F&& f) {
  return with_type(p->dtype, [&](auto t) -> int {
    auto both = [&](auto lanes) -> int { return bias ? f(t, lanes, std::true_type()) : f(t, lanes, std::false_type()); };
    switch (lanes_of(p)) {
      case 1: return both(std::integral_constant<int, 1>());
      case 2: return both(std::integral_constant<int, 2>());
      case 4: return both(std::integral_constant<int, 4>());
      case 8: return both(std::integral_constant<int, 8>());
      case 16: return both(std::integral_constant<int, 16>());
      default: return both(std::integral_constant<int, 32>());
    }
  });
}

// Workgroups over n items: one range each, or with a bias at most some kShortGroups, a multiple of the key heads.
int64_t groups_of(const bf_packed_attn* p, int64_t n, bool bias) {
  const int64_t blocks = ceil_div(n, kShortThreads / lanes_of(p)), most = ceil_div(kShortGroups, p->heads_k) * p->heads_k;
  return bias && blocks > most ? most : blocks;
}

// Floats of LDS: the heads' values by distance, the buckets, and in the keys' pass the columns.
int64_t short_floats(const bf_packed_attn* p, const bf_packed_bias* bias, bool columns) {
  if (!bias) return 0;
  const int64_t cols = int64_t(p->heads_q / p->heads_k) * bias->buckets * (kShortThreads / lanes_of(p));
  return (p->heads_q + 1) * int64_t(kByDistance) + (columns ? cols : 0);
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
// With a bias what a workgroup keeps in LDS has to leave room for a second one.
bool packed_is_short(const bf_packed_attn* p, const bf_packed_bias* bias) {
  if (short_floats(p, bias, true) > 16384) return false;
  const bool wide = p->dtype == BF_DTYPE_F32;
  const int64_t row = int64_t(p->head_dim) * (wide ? 4 : 2), group = p->heads_q / p->heads_k;
  if (p->longest <= 0 || p->longest > 24 || p->n_k >= kMaxRows / p->heads_k) return false;
  const int64_t most = group > 2 ? (wide ? 1280 : 256) : (wide ? 2048 : 1024);
  const bool few = p->longest * group <= 40 && p->n_q * p->heads_q * row <= (int64_t(wide ? 8 : 4) << 20);
  return few || p->longest * row <= most;
}

int64_t packed_short_parts(const bf_packed_attn* p) {
  const int64_t rows = p->n_q * p->heads_q, keys = p->n_k * p->heads_k;
  return groups_of(p, p->dtype == BF_DTYPE_F32 && rows > keys ? rows : keys, true);
}

int packed_short_fwd(const bf_packed_attn* p, const bf_packed_bias* bias, const void* q, const void* k, const void* v, void* out,
                     float* lse, hipStream_t st) {
  ShortArgs a = make_args(p, bias, q, k, v);
  a.o = out, a.lse = lse;
  const unsigned lds = 4u * unsigned(short_floats(p, bias, false));
  return with_lanes(p, bias, [&](auto t, auto lanes, auto biased) -> int {
    using T = decltype(t);
    constexpr int LPR = decltype(lanes)::value;
    auto kern = short_fwd<T, LPR, decltype(biased)::value>;
    BF_LAUNCH("packed_attn_fwd_short", kern, dim3(unsigned(groups_of(p, a.n_rows, bias))), dim3(kShortThreads), lds, st, a);
    BF_CHECK_LAUNCH();
    return BF_OK;
  });
}

int packed_short_bwd(const bf_packed_attn* p, const bf_packed_bias* bias, const void* q, const void* k, const void* v, const void* out,
                     const float* lse, const void* dout, void* dq, void* dk, void* dv, float* delta, float* bias_part, hipStream_t st) {
  ShortArgs a = make_args(p, bias, q, k, v);
  a.out = out, a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv;
  a.lse = const_cast<float*>(lse), a.delta = delta, a.bias.part = bias_part;
  const unsigned lds = 4u * unsigned(short_floats(p, bias, false)), more = 4u * unsigned(short_floats(p, bias, true));
  return with_lanes(p, bias, [&](auto t, auto lanes, auto biased) -> int {
    using T = decltype(t);
    constexpr int LPR = decltype(lanes)::value;
    constexpr bool BIAS = decltype(biased)::value;
    const dim3 block(kShortThreads);
    if constexpr (sizeof(T) == 2) {
      if (a.n_rows > 0) {
        auto rows = short_bwd_rows<T, LPR, BIAS>;
        BF_LAUNCH("packed_attn_bwd_short_rows", rows, dim3(unsigned(groups_of(p, a.n_rows, bias))), block, lds, st, a);
        BF_CHECK_LAUNCH();
      }
      if (a.n_keys > 0) {
        auto keys = short_bwd_keys<T, LPR, BIAS>;
        BF_LAUNCH("packed_attn_bwd_short_keys", keys, dim3(unsigned(groups_of(p, a.n_keys, bias))), block, more, st, a);
        BF_CHECK_LAUNCH();
      }
    } else {
      const int64_t most = a.n_rows > a.n_keys ? a.n_rows : a.n_keys;
      if (most == 0) return BF_OK;
      auto kern = short_bwd<T, LPR, BIAS>;
      BF_LAUNCH("packed_attn_bwd_short", kern, dim3(unsigned(groups_of(p, most, bias))), block, more, st, a);
      BF_CHECK_LAUNCH();
    }
    return BF_OK;
  });
}

}  // namespace bf
