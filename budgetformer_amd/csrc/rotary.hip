// Rotary positions of one or two tensors of heads (q and k), and their gradient (the same turn backwards).
//
// A pair (a, b) of a head's values becomes (a cos t - b sin t, a sin t + b cos t), t = 2 pi pos * turns[pair]. A
// token's angles serve all its heads: a workgroup forms those of its tokens once, in LDS, and its lanes then stream
// the heads. Angles are formed in 64 bits and reduced to one turn there (at position 10^6 a float32 angle is off
// by 0.06), sin and cos of the rest in 32. What bounds it is one read and one write of the tensors:
// 16,411 tokens, 32 heads of 64 (half turned) in float32, 269 MB in 57 us (4.7 TB/s); 32,768 tokens, 40 heads of 128 in
// bfloat16, 671 MB in 125 us (5.4 TB/s); 64 tokens of those 7 us, a launch's latency.
#include <type_traits>

#include "bf_common.h"

namespace bf {
namespace {

struct RotaryArgs {
  const void *x, *y;
  void *ox, *oy;
  int64_t xs_t, xs_h, ys_t, ys_h;
  int64_t n;
  int32_t hx, hy, dim, rot;
  const void* positions;
  const double* turns;
  float amplitude;
  int32_t wide, inverse;
  int32_t tokens, heads;          // of a workgroup
};

constexpr int kRotaryThreads = 256;
constexpr int kAhead = 4;
constexpr int kRotaryAngles = 512;     // angles of a workgroup at most (4 KB of LDS)

// V: values a lane moves at a time (16 bytes, or 1 where the sizes or addresses do not allow that).
template <typename T, int V, bool PAIRS>
__global__ __launch_bounds__(kRotaryThreads) void rotary(const RotaryArgs a) {
  typedef T Vec __attribute__((ext_vector_type(V)));
  __shared__ float2 turn[kRotaryAngles];
  const int half = a.rot >> 1;
  const int64_t t0 = int64_t(blockIdx.x) * a.tokens;
  const int nt = int(min(int64_t(a.tokens), a.n - t0));
  for (int i = threadIdx.x; i < nt * half; i += kRotaryThreads) {
    const int t = i / half;
    const int64_t pos = a.wide ? static_cast<const int64_t*>(a.positions)[t0 + t]
                               : int64_t(static_cast<const int32_t*>(a.positions)[t0 + t]);
    const double u = double(pos) * a.turns[i - t * half];
    float s, c;
    sincospif(2.f * float(u - rint(u)), &s, &c);
    turn[i] = make_float2(c * a.amplitude, (a.inverse ? -s : s) * a.amplitude);
  }
  __syncthreads();

  // a head's work: its turned pairs V values at a time, then the values that are copied
  const int turned = (PAIRS ? a.rot : half) / V, rest = (a.dim - a.rot) / V, per = turned + rest;
  const int h0 = blockIdx.y * a.heads, nh = min(a.heads, a.hx + a.hy - h0);
  // kAhead pieces of work a lane at a time, their loads on their way together
  const int all = nt * nh * per;
  for (int i0 = threadIdx.x; i0 < all; i0 += kRotaryThreads * kAhead) {
    const T* src[kAhead];
    T* dst[kAhead];
    const float2* tn[kAhead];
    int at[kAhead];
    Vec x[kAhead], y[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = min(i0 + k * kRotaryThreads, all - 1), u = i % per, th = i / per, t = th / nh;
      int h = h0 + th - t * nh;
      if (h < a.hx) {
        src[k] = static_cast<const T*>(a.x) + (t0 + t) * a.xs_t + h * a.xs_h;
        dst[k] = static_cast<T*>(a.ox) + ((t0 + t) * a.hx + h) * a.dim;
      } else {
        h -= a.hx;
        src[k] = static_cast<const T*>(a.y) + (t0 + t) * a.ys_t + h * a.ys_h;
        dst[k] = static_cast<T*>(a.oy) + ((t0 + t) * a.hy + h) * a.dim;
      }
      const bool turns = u < turned;
      at[k] = turns ? u * V : a.rot + (u - turned) * V;
      tn[k] = turns ? turn + t * half : nullptr;
      x[k] = *reinterpret_cast<const Vec*>(src[k] + at[k]);
      // the other value of each pair: elsewhere in the head, or (single values of neighbouring pairs) next to it
      if constexpr (!PAIRS)
        y[k] = *reinterpret_cast<const Vec*>(src[k] + at[k] + (turns ? half : 0));
      else if constexpr (V == 1)
        y[k] = *reinterpret_cast<const Vec*>(src[k] + (turns ? at[k] ^ 1 : at[k]));
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 + k * kRotaryThreads >= all) break;
      Vec o = x[k];
      if (tn[k]) {
        if constexpr (!PAIRS) {
          Vec r;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float2 w = tn[k][at[k] + j];
            const float p = float(x[k][j]), q = float(y[k][j]);
            o[j] = T(fmaf(p, w.x, -q * w.y));
            r[j] = T(fmaf(p, w.y, q * w.x));
          }
          *reinterpret_cast<Vec*>(dst[k] + half + at[k]) = r;
        } else if constexpr (V == 1) {
          const float2 w = tn[k][at[k] >> 1];
          const float p = float(x[k][0]), q = float(y[k][0]);
          o[0] = T(at[k] & 1 ? fmaf(q, w.y, p * w.x) : fmaf(p, w.x, -q * w.y));
        } else {
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            const float2 w = tn[k][(at[k] + j) >> 1];
            const float p = float(x[k][j]), q = float(x[k][j + 1]);
            o[j] = T(fmaf(p, w.x, -q * w.y));
            o[j + 1] = T(fmaf(p, w.y, q * w.x));
          }
        }
      }
      *reinterpret_cast<Vec*>(dst[k] + at[k]) = o;
    }
  }
}

bool rotary_vectors(const RotaryArgs& a, int per, int elem, bool pairs) {
  if (a.dim % per || (pairs ? a.rot : a.rot / 2) % per || a.rot % per) return false;
  for (int64_t s : {a.xs_t, a.xs_h, a.hy ? a.ys_t : 0, a.hy ? a.ys_h : 0})
    if (s % per) return false;
  for (const void* p : {a.x, static_cast<const void*>(a.ox), a.hy ? a.y : nullptr, a.hy ? static_cast<const void*>(a.oy) : nullptr})
    if (reinterpret_cast<uintptr_t>(p) % (per * elem)) return false;
  return true;
}

template <typename T> int launch_rotary(RotaryArgs a, bool pairs, hipStream_t st) {
  constexpr int V = 16 / int(sizeof(T));
  const bool vec = rotary_vectors(a, V, sizeof(T), pairs);
  const int half = a.rot / 2, all = a.hx + a.hy;
  // tokens: about a workgroup's lanes' worth of angles; heads: all of a token's, except that calls of few tokens spread
  // them over the chip
  a.tokens = kRotaryThreads / half > 0 ? kRotaryThreads / half : 1;
  if (a.tokens > 16) a.tokens = 16;
  a.heads = all;
  while (a.tokens > 1 && ceil_div(a.n, a.tokens) < 1024) a.tokens >>= 1;
  while (a.heads > 1 && ceil_div(a.n, a.tokens) * ceil_div(all, a.heads) < 512) a.heads = (a.heads + 1) / 2;
  const dim3 grid(unsigned(ceil_div(a.n, a.tokens)), unsigned(ceil_div(all, a.heads)));
  const dim3 block(kRotaryThreads);
#define BF_ROTARY(VV, PP)                                                     \
  do {                                                                        \
    auto kern = rotary<T, VV, PP>;                                            \
    BF_LAUNCH("rotary", kern, grid, block, 0, st, a);                         \
  } while (0)
  if (vec && pairs) BF_ROTARY(V, true);
  else if (vec) BF_ROTARY(V, false);
  else if (pairs) BF_ROTARY(1, true);
  else BF_ROTARY(1, false);
#undef BF_ROTARY
  BF_CHECK_LAUNCH();
  return BF_OK;
}

}  // namespace
}  // namespace bf

using namespace bf;

extern "C" int bf_rotary(const void* x, const void* y, int64_t n, int32_t heads_x, int32_t heads_y, int32_t dim, int32_t rot,
                         int32_t dtype, const int64_t x_stride[2], const int64_t y_stride[2], const void* positions,
                         int32_t wide, const double* turns, float amplitude, int32_t interleaved, int32_t inverse, void* out_x,
                         void* out_y, void* stream) {
  BF_CHECK_ARG(n >= 0 && n < (int64_t(1) << 31) && heads_x >= 1 && heads_y >= 0 && heads_x <= (1 << 20) && heads_y <= (1 << 20) &&
                   dim >= 1 && dim <= (1 << 20),
               "rotary: bad sizes (%lld rows of %d and %d heads of %d)", (long long)n, heads_x, heads_y, dim);
  BF_CHECK_ARG(rot >= 2 && rot % 2 == 0 && rot <= dim && rot <= 2 * kRotaryAngles,
               "rotary: %d of %d values (an even number up to the head and %d expected)", rot, dim, 2 * kRotaryAngles);
  BF_CHECK_ARG(dtype == BF_DTYPE_F32 || dtype == BF_DTYPE_BF16 || dtype == BF_DTYPE_F16, "rotary: dtype %d", dtype);
  if (n == 0) return BF_OK;
  BF_CHECK_ARG(x && out_x && x_stride && (heads_y == 0 || (y && out_y && y_stride)) && positions && turns,
               "rotary: bad arguments");
  // one workgroup's items are counted in 32 bits
  BF_CHECK_ARG(int64_t(16) * (int64_t(heads_x) + heads_y) * dim <= (int64_t(1) << 30), "rotary: a token of %d heads of %d",
               heads_x + heads_y, dim);
  RotaryArgs a{};
  a.x = x, a.y = y, a.ox = out_x, a.oy = out_y;
  a.xs_t = x_stride[0], a.xs_h = x_stride[1];
  if (heads_y) a.ys_t = y_stride[0], a.ys_h = y_stride[1];
  a.n = n, a.hx = heads_x, a.hy = heads_y, a.dim = dim, a.rot = rot;
  a.positions = positions, a.turns = turns, a.amplitude = amplitude, a.wide = wide, a.inverse = inverse;
  const hipStream_t st = as_stream(stream);
  const bool pairs = interleaved != 0;
  if (dtype == BF_DTYPE_F32) return launch_rotary<float>(a, pairs, st);
  if (dtype == BF_DTYPE_BF16) return launch_rotary<__bf16>(a, pairs, st);
  return launch_rotary<_Float16>(a, pairs, st);
}
