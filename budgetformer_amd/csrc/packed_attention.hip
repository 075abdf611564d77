// Dense softmax attention inside each sequence of a packed batch, forward and backward, on the matrix cores.
//
//   S = scale * q k^T over the keys a row sees, P = exp(S - m) / l, O = P V, lse = m + log l
//   Delta = sum_d dO O, dV = P^T dO, dP = dO V^T, dS = P (dP - Delta), dQ = scale dS K, dK = scale dS^T Q
//
// What a row sees is one interval of keys, [lo, hi), and both ends never fall along the packed axis: own sequence,
// causal or not, empty sequences and rows behind the last one are all the same to the kernels. Tiles are therefore
// cut from the packed axis and not from the sequences (a batch of 5-token walks fills its tiles as a long sequence
// does, and the grid is known without reading a length back): a tile walks the keys from its first row's lo to its
// last row's hi and compares indices only where a wave's rows do not all see the whole tile. The rows of one key
// head are (token, head of its group) pairs, token-major, so a group shares its K and V tiles, and dK and dV sum the
// group in registers. Nothing is added atomically: dQ has a pass of its own (rows own their sums), as dK/dV has (keys
// own theirs), so results repeat bit for bit; that costs two of seven matrix products and saves the float32
// dQ buffer with its atomics.
//
// Layout. v_mfma 32x32x16 takes 8 values a lane along the contraction (lane l: row or column l % 32, half l / 32) and
// leaves column l % 32, rows (r % 4) + 8 (r / 4) + 4 (l / 32) of the product in register r. The kernels form S^T
// (keys by rows) so that a lane owns one row: its maximum and sum are a register loop and one exchange between the
// halves. Registers 8t .. 8t+7 are then, as they stand, the second operand of the next product over 16 keys, if
// that product counts its keys as the registers do: value j of half h is key 16t + (j % 4) + 8 (j / 4) + 4 h. The
// transposed operand (V^T, K^T, Q^T, dO^T) is read from LDS in that order by the transposing LDS reads of 4 x 16
// blocks. LDS rows are padded by 32 bytes: the 4 rows of such a read, and the 8 rows of a 16-byte read, then
// fall on different banks. float32 uses the same layout with eight 32x32x2 products for one of 16.
//
// A wave that multiplies goes before one that forms exponentials (s_setprio around the products of the forward and of
// dQ): 0.34 -> 0.32 and 0.45 -> 0.42 ms on one causal sequence of 8192, 16 heads of 128 over 4; dK and dV gain nothing.
//
// What bounds it: long wide heads, the matrix cores with exponentials and LDS reads between their products (one causal
// sequence of 8192, 16 heads of 128 over 4, bfloat16: forward 0.32 ms, 860 TFLOP/s of what the mask leaves; dQ 0.42, 980;
// dK and dV 0.60, 910); few rows, the keys' bytes (64 next tokens over 0.5 to 8 thousand keys each: 5.0 TB/s); narrow heads, the
// exponentials and masks of a tile.
//
// Precision: scores, softmax statistics and all sums are float32. P and dS are rounded to the activations' type as
// operands of the second products (half a step of each term, as the inputs' own rounding); float32 rounds nothing. float16
// loses bits below 2^-14 and ends at 65504, where a long row's P and a gradient's dS need not: there both are operands in
// units of a power of 2 (kLift, kLiftBack). Delta is a difference's second part: a forward that trains keeps
// what the rounding of out left (`rest`), for it.
//
// NaN and infinities in places a row does not see: a masked P is 0, but 0 * inf is not. Where a tile is masked its
// staged operand is checked; one that holds such a value takes a path that multiplies the finite values only, and
// finds by a second product of indicators which rows do see one.
#include "packed_short.h"
#include "packed_tile.h"

namespace bf {
namespace {

// ---------------------------------------------------------------- arguments
struct Args {
  const void *q, *k, *v, *out, *dout;
  void *o, *rest, *dq, *dk, *dv;                   // rest: what the rounding of out left, or NULL
  float *lse, *delta, *part, *stat;
  const int2 *row_span, *key_span;
  int64_t qs_t, qs_h, ks_t, ks_h, vs_t, vs_h;      // strides in values
  int32_t rows, n_q, n_k, hq, hk, group, dim;      // rows: (token, head of the group) pairs of one key head
  int32_t tiles, pieces;
  const int32_t* order;                            // of the tiles, or NULL: the last one first
  float scale, c;                                  // c = scale * log2(e)
  Div by_group;
  int32_t xcd_groups;                              // of heads, dealt to the XCDs (place)
};

struct Row {
  int32_t token, head;     // of the query tensor
};

__device__ __forceinline__ Row row_of(const Args& a, int h, int rho) {
  const int32_t t = int32_t(a.by_group(uint32_t(rho)));
  return Row{t, h * a.group + (rho - t * a.group)};
}

__device__ __forceinline__ int2 span_at(const int2* s, int i) {
  const int2 x = s[i];
  return make_int2(__builtin_amdgcn_readfirstlane(x.x), __builtin_amdgcn_readfirstlane(x.y));
}

// A row's bound among the keys, and the rows of the group that a key's span names: inside the tensors whatever a span holds.
__device__ __forceinline__ int in_keys(const Args& a, int x) { return min(max(x, 0), a.n_k); }
__device__ __forceinline__ int2 group_rows(const Args& a, int2 s) {
  return make_int2(min(max(s.x, 0), a.n_q) * a.group, min(max(s.y, 0), a.n_q) * a.group);
}

// Which (tile, key head, piece) a workgroup takes; false: none. Workgroup i runs on XCD i % 8, each with an L2 of its own.
// The heads are dealt to groups of XCDs (as many groups as divide both), a group's heads follow each other, and its XCDs
// take their tiles in turn: an XCD reads few heads' keys at a time, and each gets its share of a causal mask's long and
// short tiles, the long ones (later rows) first. One contiguous run of tiles an XCD instead, which shares its keys as
// well, leaves the XCDs unevenly loaded: 0.49 instead of 0.36 ms forward on one causal sequence of 8192 (16 heads of 128).
__device__ __forceinline__ bool place(const Args& a, int& tile, int& h, int& piece) {
  const int per = a.tiles * a.pieces;
  const int x = blockIdx.x % kXcds, groups = a.xcd_groups, each = kXcds / groups, heads = a.hk / groups;
  const int64_t at = int64_t(blockIdx.x / kXcds) * each + x % each;
  if (at >= int64_t(heads) * per) return false;
  h = x / each * heads + int(at / per);
  const int t = int(at % per);
  piece = t % a.pieces;
  tile = a.order ? a.order[t / a.pieces] : a.tiles - 1 - t / a.pieces;
  return true;
}

// A row's fragments straight from memory (the operand a wave keeps in registers).
template <typename T, int DP>
__device__ __forceinline__ void load_row(Frag<T> (&f)[DP / 16], const T* p, int dim, int half) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int at = 16 * s + 8 * half;
    if (p && at < dim) {
      f[s] = *reinterpret_cast<const Frag<T>*>(p + at);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[s][j] = T(0.f);
    }
  }
}

// A product's columns (one row of the result a lane) to memory, scaled.
template <int DP, typename O>
__device__ __forceinline__ void store_cols(O* p, const F32x16 (&acc)[(DP + 31) / 32], float by, int dim, int half) {
#pragma unroll
  for (int n = 0; n < (DP + 31) / 32; ++n) store_block<O>(p, acc[n], by, n, dim, half);
}

// ---------------------------------------------------------------- forward
// A row's terms are taken relative to a maximum that is raised only when a score passes it by 2^kLazy: the sums, then
// up to 2^kLazy times larger, lose nothing in float32, and most tiles skip the rescaling of the accumulators.
constexpr float kLazy = 6.f;

// float16: terms are given times 2^9, at most 2^(9 + kLazy) then, and keep their bits down to 2^-23 of the row's maximum
// (half a step is 2^-34 below that). The factor is in the exponent (free) and in the sum, so the quotient does not see it.
template <typename T> constexpr float kLift = std::is_same<T, _Float16>::value ? 9.f : 0.f;

template <typename T, int DP, int NW, int BN, bool SPLIT>
__global__ __launch_bounds__(64 * NW, SPLIT || (sizeof(T) == 4 && DP == 128) ? 1 : 2) void packed_fwd(const Args a) {
  using TL = Tile<T, DP>;
  constexpr int NT = 64 * NW, BM = 32 * NW;
  __shared__ __attribute__((aligned(16))) char k_lds[TL::bytes(BN)];
  __shared__ __attribute__((aligned(16))) char v_lds[TL::bytes(BN)];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
  int tile, h, piece;
  if (!place(a, tile, h, piece)) return;

  const int row0 = tile * BM, last = min(row0 + BM, a.rows) - 1;
  const int2 first_span = span_at(a.row_span, a.by_group(row0)), last_span = span_at(a.row_span, a.by_group(last));
  int kbeg = in_keys(a, first_span.x), kend = in_keys(a, last_span.y);
  if constexpr (SPLIT) {
    const int width = (max(kend - kbeg, 0) + a.pieces * BN - 1) / (a.pieces * BN) * BN;
    kbeg += piece * width;
    kend = min(kend, kbeg + width);
  }
  // this wave's rows, and what they see together
  const int w_row0 = row0 + 32 * wave, w_last = min(w_row0 + 31, a.rows - 1);
  const bool w_any = w_row0 < a.rows;
  const int2 wf = span_at(a.row_span, a.by_group(min(w_row0, a.rows - 1))), wl = span_at(a.row_span, a.by_group(w_last));
  const int rho = w_row0 + col;
  const bool valid = rho < a.rows;
  const Row row = row_of(a, h, valid ? rho : a.rows - 1);
  const int2 span = a.row_span[row.token];
  const int lo = span.x, hi = valid ? span.y : span.x;

  Frag<T> qf[TL::kSteps];
  load_row<T, DP>(qf, valid ? static_cast<const T*>(a.q) + row.token * a.qs_t + row.head * a.qs_h : nullptr, a.dim, half);
  F32x16 o[TL::kBlocks];
#pragma unroll
  for (int n = 0; n < TL::kBlocks; ++n) o[n] = zero16();
  float mc = -INFINITY, l = 0.f;      // c * maximum, and this half's part of the sum

  const T* kp = static_cast<const T*>(a.k) + h * a.ks_h;
  const T* vp = static_cast<const T*>(a.v) + h * a.vs_h;
  Stage<T, DP, BN, NT> ks, vs;
  auto fetch = [&](int j0) {
    ks.load(tid, kend - j0, a.dim, [&](int r) { return kp + (j0 + r) * a.ks_t; });
    vs.load(tid, kend - j0, a.dim, [&](int r) { return vp + (j0 + r) * a.vs_t; });
  };
  if (kbeg < kend) fetch(kbeg);
  for (int j0 = kbeg; j0 < kend; j0 += BN) {
    ks.clip(tid, kend - j0, a.dim);
    vs.clip(tid, kend - j0, a.dim);
    __syncthreads();
    ks.store(tid, k_lds);
    vs.store(tid, v_lds);
    bool odd = false;
    if (j0 < last_span.x || j0 + BN > first_span.y)
      odd = __syncthreads_or(vs.tainted());
    else
      __syncthreads();
    if (j0 + BN < kend) fetch(j0 + BN);
    if (!w_any || j0 >= wl.y || j0 + BN <= wf.x) continue;

    float s[BN / 32][16];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int b = 0; b < BN / 32; ++b) {
      F32x16 acc = zero16();
#pragma unroll
      for (int st = 0; st < TL::kSteps; ++st) acc = Mat<T>::mma(TL::row_frag(k_lds, 32 * b + col, st, half), qf[st], acc);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = acc[r];
    }
    __builtin_amdgcn_s_setprio(0);
    const bool masked = j0 < wl.x || j0 + BN > wf.y || w_last < w_row0 + 31;
    if (masked) {
#pragma unroll
      for (int b = 0; b < BN / 32; ++b) {
        const uint32_t seen = seen_bits(lo - j0 - 32 * b, hi - j0 - 32 * b, half);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = where_seen(seen, r, s[b][r], -INFINITY);
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < BN / 32; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    float mc_new = fmaxf(mc, top * a.c);
    if (__any(mc_new > mc + kLazy)) {
      const float alpha = mc_new == -INFINITY ? 1.f : exp2_fast(mc - mc_new);
      l *= alpha;
#pragma unroll
      for (int n = 0; n < TL::kBlocks; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] *= alpha;
      mc = mc_new;
    }
    const float base = mc == -INFINITY ? 0.f : mc - kLift<T>;
#pragma unroll
    for (int b = 0; b < BN / 32; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[b][r] = exp2_fast(fmaf(s[b][r], a.c, -base));
        l += s[b][r];
      }
    if (masked && odd) {
#pragma unroll
      for (int n = 0; n < TL::kBlocks; ++n) {
#pragma unroll
        for (int t = 0; t < BN / 16; ++t)
          o[n] = Mat<T>::mma(finite<T>(TL::col_frag(v_lds, t, n, lane)), pack8<T>(s[t / 2], t & 1), o[n]);
        add_infinite<BN / 16>(o[n], [&](int t, F32x16 x, float sign) {
          return Mat<T>::mma(is_infinite<T>(TL::col_frag(v_lds, t, n, lane), sign), pack8<T>(s[t / 2], t & 1), x);
        });
      }
    } else {
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < BN / 16; ++t) {
        const Frag<T> p = pack8<T>(s[t / 2], t & 1);
#pragma unroll
        for (int n = 0; n < TL::kBlocks; ++n) o[n] = Mat<T>::mma(TL::col_frag(v_lds, t, n, lane), p, o[n]);
      }
      __builtin_amdgcn_s_setprio(0);
    }
  }

  l += __shfl_xor(l, 32, 64);
  mc -= kLift<T>;                      // what the sums are relative to
  if (!valid) return;
  const int64_t at = int64_t(row.token) * a.hq + row.head;
  if constexpr (SPLIT) {
    const int64_t slot = at * a.pieces + piece;
    if (half == 0) {
      a.stat[2 * slot] = mc;
      a.stat[2 * slot + 1] = l;
    }
    if (l != 0.f) store_cols<DP>(a.part + slot * a.dim, o, 1.f, a.dim, half);
  } else {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (a.rest) {
#pragma unroll
      for (int n = 0; n < TL::kBlocks; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] *= inv;
      store_cols<DP>(static_cast<T*>(a.o) + at * a.dim, o, 1.f, a.dim, half);
#pragma unroll
      for (int n = 0; n < TL::kBlocks; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] -= float(T(o[n][r]));
      store_cols<DP>(static_cast<T*>(a.rest) + at * a.dim, o, 1.f, a.dim, half);
    } else {
      store_cols<DP>(static_cast<T*>(a.o) + at * a.dim, o, inv, a.dim, half);
    }
    if (half == 0) a.lse[at] = l == 0.f ? -INFINITY : mc + __log2f(l);
  }
}

// Joins the pieces of a row: one wave a row. out = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p. A lane has a piece's
// statistics (kMaxPieces is a wave); only pieces that hold keys of the row were written and are read.
template <typename T>
__global__ __launch_bounds__(256) void packed_join(const float* part, const float* stat, int64_t n_rows, int pieces, int dim,
                                                   T* out, T* rest, float* lse) {
  const int lane = threadIdx.x & 63;
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= n_rows) return;
  const float2 st = lane < pieces ? *reinterpret_cast<const float2*>(stat + (row * pieces + lane) * 2) : make_float2(-INFINITY, 0.f);
  float top = st.x;
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float w = exp2_fast(st.x - (top == -INFINITY ? 0.f : top));
  float l = st.y == 0.f ? 0.f : w * st.y;
  for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o, 64);
  const int d = 2 * lane;
  float a0 = 0.f, a1 = 0.f;
  for (uint64_t left = __ballot(st.y != 0.f); left; left &= left - 1) {
    const int p = __ffsll((unsigned long long)left) - 1;
    const float wp = __shfl(w, p, 64);
    if (d < dim) {
      const float2 x = *reinterpret_cast<const float2*>(part + (row * pieces + p) * dim + d);
      a0 = fmaf(wp, x.x, a0);
      a1 = fmaf(wp, x.y, a1);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (d < dim) {
    typedef T V2 __attribute__((ext_vector_type(2)));
    const V2 v = {T(a0 * inv), T(a1 * inv)};
    *reinterpret_cast<V2*>(out + row * dim + d) = v;
    if (rest) {
      const V2 w = {T(a0 * inv - float(v[0])), T(a1 * inv - float(v[1]))};
      *reinterpret_cast<V2*>(rest + row * dim + d) = w;
    }
  }
  if (lane == 0) lse[row] = l == 0.f ? -INFINITY : top + __log2f(l);
}

// ---------------------------------------------------------------- float16's units of the backward
// P and dS are operands times 2^12, by their exponent: P fits and keeps its bits down to 2^-26, dS down to 2^-26 of a
// gradient of ordinary size (half a step is 2^-37, where a result's own is 2^-25). A dS that would pass 2^15 shrinks the
// factor of its lane's row (or key), and what is summed so far, to bring it to 2^13. Training without : with it in us: one causal
// sequence of 8192, 16 heads of 128 over 4: 1380 : 1416; 256 graphs of 9 to 250 nodes, 8 heads of 32: 146 : 150; eight causal
// sequences of 400 to 2000, 16 heads of 64: 313 : 319.
template <typename T> constexpr bool kUnits = std::is_same<T, _Float16>::value;
template <typename T> constexpr int kLiftBack = kUnits<T> ? 12 : 0;
constexpr float kMost = 32768.f;

// Whether some lane's dS pass kMost; they then are brought to 2^13, by 2^`by` (0 for the other lanes).
__device__ __forceinline__ bool shrink(float (&ds)[16], int& by) {
  float big = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) big = fmaxf(big, fabsf(ds[r]));
  if (!__any(big > kMost)) return false;
  big = fmaxf(big, __shfl_xor(big, 32, 64));           // the row's (or key's) other half
  by = big > kMost && big < INFINITY ? 13 - __builtin_amdgcn_frexp_expf(big) : 0;
#pragma unroll
  for (int r = 0; r < 16; ++r) ds[r] = ldexpf(ds[r], by);
  return true;
}

// ---------------------------------------------------------------- backward: dQ (and Delta)
template <typename T, int DP, int NW, int BN>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 4 && DP == 128 ? 1 : 2) void packed_bwd_q(const Args a) {
  using TL = Tile<T, DP>;
  constexpr int NT = 64 * NW, BM = 32 * NW;
  __shared__ __attribute__((aligned(16))) char k_lds[TL::bytes(BN)];
  __shared__ __attribute__((aligned(16))) char v_lds[TL::bytes(BN)];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
  int tile, h, piece;
  if (!place(a, tile, h, piece)) return;

  const int row0 = tile * BM, last = min(row0 + BM, a.rows) - 1;
  const int2 first_span = span_at(a.row_span, a.by_group(row0)), last_span = span_at(a.row_span, a.by_group(last));
  const int kbeg = in_keys(a, first_span.x), kend = in_keys(a, last_span.y);
  const int w_row0 = row0 + 32 * wave, w_last = min(w_row0 + 31, a.rows - 1);
  const bool w_any = w_row0 < a.rows;
  const int2 wf = span_at(a.row_span, a.by_group(min(w_row0, a.rows - 1))), wl = span_at(a.row_span, a.by_group(w_last));
  const int rho = w_row0 + col;
  const bool valid = rho < a.rows;
  const Row row = row_of(a, h, valid ? rho : a.rows - 1);
  const int2 span = a.row_span[row.token];
  const int lo = span.x, hi = valid ? span.y : span.x;
  const int64_t at = int64_t(row.token) * a.hq + row.head;

  Frag<T> qf[TL::kSteps], gf[TL::kSteps];
  load_row<T, DP>(qf, valid ? static_cast<const T*>(a.q) + row.token * a.qs_t + row.head * a.qs_h : nullptr, a.dim, half);
  load_row<T, DP>(gf, valid ? static_cast<const T*>(a.dout) + at * a.dim : nullptr, a.dim, half);
  float delta = 0.f;
  {
    Frag<T> of[TL::kSteps];
    load_row<T, DP>(of, valid ? static_cast<const T*>(a.out) + at * a.dim : nullptr, a.dim, half);
#pragma unroll
    for (int s = 0; s < TL::kSteps; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf(float(gf[s][j]), float(of[s][j]), delta);
    if (a.rest) {
      load_row<T, DP>(of, valid ? static_cast<const T*>(a.rest) + at * a.dim : nullptr, a.dim, half);
#pragma unroll
      for (int s = 0; s < TL::kSteps; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) delta = fmaf(float(gf[s][j]), float(of[s][j]), delta);
    }
    delta += __shfl_xor(delta, 32, 64);
    if (valid && half == 0) a.delta[at] = delta;
  }
  // a row without a finite score has lse = -inf and P = 0: +inf in the exponent's place gives that
  float lse = a.lse[at];
  if (lse == -INFINITY) lse = INFINITY;
  int lift = kLiftBack<T>;             // P, dS and the sums are times 2^lift
  lse -= float(lift);

  F32x16 dq[TL::kBlocks];
#pragma unroll
  for (int n = 0; n < TL::kBlocks; ++n) dq[n] = zero16();
  const T* kp = static_cast<const T*>(a.k) + h * a.ks_h;
  const T* vp = static_cast<const T*>(a.v) + h * a.vs_h;
  Stage<T, DP, BN, NT> ks, vs;
  auto fetch = [&](int j0) {
    ks.load(tid, kend - j0, a.dim, [&](int r) { return kp + (j0 + r) * a.ks_t; });
    vs.load(tid, kend - j0, a.dim, [&](int r) { return vp + (j0 + r) * a.vs_t; });
  };
  if (kbeg < kend) fetch(kbeg);
  for (int j0 = kbeg; j0 < kend; j0 += BN) {
    ks.clip(tid, kend - j0, a.dim);
    vs.clip(tid, kend - j0, a.dim);
    __syncthreads();
    ks.store(tid, k_lds);
    vs.store(tid, v_lds);
    bool odd = false;
    if (j0 < last_span.x || j0 + BN > first_span.y)
      odd = __syncthreads_or(ks.tainted());
    else
      __syncthreads();
    if (j0 + BN < kend) fetch(j0 + BN);
    if (!w_any || j0 >= wl.y || j0 + BN <= wf.x) continue;
    const bool masked = j0 < wl.x || j0 + BN > wf.y || w_last < w_row0 + 31;
#pragma unroll
    for (int b = 0; b < BN / 32; ++b) {
      F32x16 sa = zero16(), pa = zero16();
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int st = 0; st < TL::kSteps; ++st) {
        sa = Mat<T>::mma(TL::row_frag(k_lds, 32 * b + col, st, half), qf[st], sa);
        pa = Mat<T>::mma(TL::row_frag(v_lds, 32 * b + col, st, half), gf[st], pa);
      }
      __builtin_amdgcn_s_setprio(0);
      float ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = exp2_fast(fmaf(sa[r], a.c, -lse)) * (pa[r] - delta);
      if (masked) {
        const uint32_t seen = seen_bits(lo - j0 - 32 * b, hi - j0 - 32 * b, half);
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] = where_seen(seen, r, ds[r], 0.f);
      }
      if constexpr (kUnits<T>) {
        int by;
        if (shrink(ds, by)) {
#pragma unroll
          for (int n = 0; n < TL::kBlocks; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) dq[n][r] = ldexpf(dq[n][r], by);
          lse -= float(by);                        // for the tiles that follow
          lift += by;
        }
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Frag<T> f = pack8<T>(ds, t);
#pragma unroll
        for (int n = 0; n < TL::kBlocks; ++n) {
          Frag<T> kt = TL::col_frag(k_lds, 2 * b + t, n, lane);
          if (masked && odd) kt = finite<T>(kt);      // a key with such a value has no finite score: the rows that see it get theirs by dS
          dq[n] = Mat<T>::mma(kt, f, dq[n]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
  }
  if (valid) store_cols<DP>(static_cast<T*>(a.dq) + at * a.dim, dq, kUnits<T> ? ldexpf(a.scale, -lift) : a.scale, a.dim, half);
}

// ---------------------------------------------------------------- backward: dK and dV
// A wave owns 32 keys (a lane one of them); Q and dO tiles of BR rows pass through LDS with their rows' lse and Delta.
template <typename T, int DP, int NW, int BR>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 4 && DP >= 64 ? 1 : 2) void packed_bwd_kv(const Args a) {
  using TL = Tile<T, DP>;
  constexpr int NT = 64 * NW, BK = 32 * NW;
  __shared__ __attribute__((aligned(16))) char q_lds[TL::bytes(BR)];
  __shared__ __attribute__((aligned(16))) char g_lds[TL::bytes(BR)];
  __shared__ __attribute__((aligned(16))) float lse_lds[BR], delta_lds[BR];
  constexpr bool kVLds = sizeof(T) == 2 && DP == 128;
  __shared__ __attribute__((aligned(16))) char v_lds[kVLds ? TL::bytes(BK) : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
  int tile, h, piece;
  if (!place(a, tile, h, piece)) return;
  if (!a.order) tile = a.tiles - 1 - tile;         // with a causal mask the first keys are seen by the most rows

  const int key0 = tile * BK, last = min(key0 + BK, a.n_k) - 1;
  // rows of the group: token * group + head
  const int2 first_span = group_rows(a, span_at(a.key_span, key0)), last_span = group_rows(a, span_at(a.key_span, last));
  int rbeg = first_span.x, rend = last_span.y;
  if (a.pieces > 1) {                             // equal parts of the tile's own rows
    const int width = int(ceil_div(max(rend - rbeg, 0), a.pieces * BR)) * BR;
    rbeg = min(rbeg + piece * width, rend);
    rend = min(rend, rbeg + width);
  }
  const int w_key0 = key0 + 32 * wave, w_last = min(w_key0 + 31, a.n_k - 1);
  const bool w_any = w_key0 < a.n_k;
  const int2 wf = group_rows(a, span_at(a.key_span, min(w_key0, a.n_k - 1))), wl = group_rows(a, span_at(a.key_span, w_last));
  const int w_beg = wf.x, w_end = wl.y, w_full_beg = wl.x, w_full_end = wf.y;
  const int key = w_key0 + col;
  const bool valid = key < a.n_k;
  const int2 span = group_rows(a, a.key_span[valid ? key : a.n_k - 1]);
  const int lo = span.x, hi = valid ? span.y : lo;

  Frag<T> kf[TL::kSteps], vf[TL::kSteps];
  load_row<T, DP>(kf, valid ? static_cast<const T*>(a.k) + key * a.ks_t + h * a.ks_h : nullptr, a.dim, half);
  load_row<T, DP>(vf, valid ? static_cast<const T*>(a.v) + key * a.vs_t + h * a.vs_h : nullptr, a.dim, half);
  if constexpr (kVLds) {       // the wave's own rows of the tile: nobody else reads them
#pragma unroll
    for (int st = 0; st < TL::kSteps; ++st)
      *reinterpret_cast<Frag<T>*>(v_lds + (32 * wave + col) * TL::kPitch + (16 * st + 8 * half) * int(sizeof(T))) = vf[st];
  }
  F32x16 dk[TL::kBlocks], dv[TL::kBlocks];
#pragma unroll
  for (int n = 0; n < TL::kBlocks; ++n) dk[n] = zero16(), dv[n] = zero16();
  int less = 0;                        // float16: dS, and dK's sums, are times 2^less besides
  bool shrunk = false;                 // whether some lane's are

  const T* qp = static_cast<const T*>(a.q);
  const T* gp = static_cast<const T*>(a.dout);
  Stage<T, DP, BR, NT> qs, gs;
  float stat = 0.f;
  auto fetch = [&](int i0) {
    qs.load(tid, rend - i0, a.dim, [&](int r) {
      const Row w = row_of(a, h, i0 + r);
      return qp + w.token * a.qs_t + w.head * a.qs_h;
    });
    gs.load(tid, rend - i0, a.dim, [&](int r) {
      const Row w = row_of(a, h, i0 + r);
      return gp + (int64_t(w.token) * a.hq + w.head) * a.dim;
    });
    if (tid < 2 * BR) {          // rows behind rend read the last one's: their P and dS are masked
      const Row w = row_of(a, h, min(i0 + (tid & (BR - 1)), rend - 1));
      stat = (tid < BR ? a.lse : a.delta)[int64_t(w.token) * a.hq + w.head];
    }
  };
  static_assert(2 * BR <= NT, "one statistic a lane");
  if (rbeg < rend) fetch(rbeg);
  for (int i0 = rbeg; i0 < rend; i0 += BR) {
    qs.clip(tid, rend - i0, a.dim);
    gs.clip(tid, rend - i0, a.dim);
    __syncthreads();
    qs.store(tid, q_lds);
    gs.store(tid, g_lds);
    if (tid < BR)
      lse_lds[tid] = stat == -INFINITY ? INFINITY : stat - float(kLiftBack<T>);       // as in the dQ pass; not looked at before: nothing waits in fetch
    else if (tid < 2 * BR)
      delta_lds[tid - BR] = stat;
    bool odd = false;
    if (i0 < last_span.x || i0 + BR > first_span.y) {
      const bool mine = qs.tainted() || gs.tainted();
      odd = __syncthreads_or(mine);
    } else {
      __syncthreads();
    }
    if (i0 + BR < rend) fetch(i0 + BR);
    if (!w_any || i0 >= w_end || i0 + BR <= w_beg) continue;
    const bool masked = i0 < w_full_beg || i0 + BR > w_full_end || w_last < w_key0 + 31;
#pragma unroll
    for (int b = 0; b < BR / 32; ++b) {
      F32x16 sa = zero16(), pa = zero16();
#pragma unroll
      for (int st = 0; st < TL::kSteps; ++st) {
        sa = Mat<T>::mma(TL::row_frag(q_lds, 32 * b + col, st, half), kf[st], sa);
        pa = Mat<T>::mma(TL::row_frag(g_lds, 32 * b + col, st, half),
                         kVLds ? TL::row_frag(v_lds, 32 * wave + col, st, half) : vf[st], pa);
      }
      float p[16], ds[16];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 ls = *reinterpret_cast<const float4*>(&lse_lds[32 * b + 8 * g + 4 * half]);
        const float4 de = *reinterpret_cast<const float4*>(&delta_lds[32 * b + 8 * g + 4 * half]);
        const float lv[4] = {ls.x, ls.y, ls.z, ls.w}, dl[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[4 * g + j] = exp2_fast(fmaf(sa[4 * g + j], a.c, -lv[j]));
          ds[4 * g + j] = p[4 * g + j] * (pa[4 * g + j] - dl[j]);
        }
      }
      if (masked) {
        const uint32_t seen = seen_bits(lo - i0 - 32 * b, hi - i0 - 32 * b, half);
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = where_seen(seen, r, p[r], 0.f), ds[r] = where_seen(seen, r, ds[r], 0.f);
      }
      if constexpr (kUnits<T>) {
        if (shrunk) {
#pragma unroll
          for (int r = 0; r < 16; ++r) ds[r] = ldexpf(ds[r], less);
        }
        int by;
        if (shrink(ds, by)) {
#pragma unroll
          for (int n = 0; n < TL::kBlocks; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) dk[n][r] = ldexpf(dk[n][r], by);
          less += by;
          shrunk = true;
        }
      }
      if (masked && odd) {
#pragma unroll
        for (int n = 0; n < TL::kBlocks; ++n) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            dv[n] = Mat<T>::mma(finite<T>(TL::col_frag(g_lds, 2 * b + t, n, lane)), pack8<T>(p, t), dv[n]);
            dk[n] = Mat<T>::mma(finite<T>(TL::col_frag(q_lds, 2 * b + t, n, lane)), pack8<T>(ds, t), dk[n]);
          }
          add_infinite<2>(dv[n], [&](int t, F32x16 x, float sign) {
            return Mat<T>::mma(is_infinite<T>(TL::col_frag(g_lds, 2 * b + t, n, lane), sign), pack8<T>(p, t), x);
          });
        }
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const Frag<T> pf = pack8<T>(p, t), df = pack8<T>(ds, t);
#pragma unroll
          for (int n = 0; n < TL::kBlocks; ++n) {
            dv[n] = Mat<T>::mma(TL::col_frag(g_lds, 2 * b + t, n, lane), pf, dv[n]);
            dk[n] = Mat<T>::mma(TL::col_frag(q_lds, 2 * b + t, n, lane), df, dk[n]);
          }
        }
      }
    }
  }
  if (!valid) return;
  const float dv_by = kUnits<T> ? ldexpf(1.f, -kLiftBack<T>) : 1.f;
  const float dk_by = kUnits<T> ? ldexpf(a.scale, -kLiftBack<T> - less) : a.scale;
  const int64_t at = (int64_t(key) * a.hk + h) * a.dim;
  if (a.pieces > 1) {
    const int64_t all = int64_t(a.n_k) * a.hk * a.dim;
    store_cols<DP>(a.part + 2 * piece * all + at, dk, dk_by, a.dim, half);
    store_cols<DP>(a.part + (2 * piece + 1) * all + at, dv, dv_by, a.dim, half);
    return;
  }
  store_cols<DP>(static_cast<T*>(a.dk) + at, dk, dk_by, a.dim, half);
  store_cols<DP>(static_cast<T*>(a.dv) + at, dv, dv_by, a.dim, half);
}

// Sums the pieces of dK and dV, in their order: 4 values a lane.
template <typename T>
__global__ __launch_bounds__(256) void packed_join_kv(const float* part, int64_t all, int pieces, T* dk, T* dv) {
  const int64_t i = 4 * (int64_t(blockIdx.x) * 256 + threadIdx.x);
  if (i >= 2 * all) return;
  float4 s = *reinterpret_cast<const float4*>(part + i);          // dK's and dV's values lie behind each other, as a piece's do
  for (int p = 1; p < pieces; ++p) {
    const float4 x = *reinterpret_cast<const float4*>(part + 2 * p * all + i);
    s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
  }
  store4<T>(i < all ? dk + i : dv + (i - all), s.x, s.y, s.z, s.w);
}

// ---------------------------------------------------------------- spans
// The keys each query row sees, and the query rows that see each key, from the sequences' offsets (one thread a row:
// a binary search for its sequence). Rows behind the last sequence see nothing. Offsets are taken as they are and
// every span is clamped to the tensors, so bad ones give wrong results and no access outside.
__global__ __launch_bounds__(256) void packed_spans(const int32_t* q_off, const int32_t* k_off, int32_t n_seq, int32_t n_q,
                                                    int32_t n_k, int causal, int2* row_span, int2* key_span, int32_t* positions) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const bool is_q = i < n_q;
  if (i >= int64_t(n_q) + n_k) return;
  const int32_t x = int32_t(is_q ? i : i - n_q);
  const int32_t* off = is_q ? q_off : k_off;
  int lo = 0, hi = n_seq;                       // the last s with off[s] <= x
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);      // their sum may pass 32 bits
    if (off[mid + 1] <= x)
      lo = mid + 1;
    else
      hi = mid;
  }
  const int32_t lim = is_q ? n_k : n_q;
  int2 s;
  if (lo == n_seq || x < off[0]) {
    const int32_t end = lo == n_seq ? (is_q ? k_off : q_off)[n_seq] : 0;
    s = make_int2(end, end);
    if (is_q && positions) positions[x] = 0;
  } else {
    const int32_t q0 = q_off[lo], q1 = q_off[lo + 1], k0 = k_off[lo], k1 = k_off[lo + 1];
    const int32_t past = (k1 - k0) - (q1 - q0);
    if (is_q && positions) positions[x] = x - q0 + past;
    if (is_q)
      s = make_int2(k0, causal ? max(k0, min(k1, k0 + (x - q0) + past + 1)) : k1);
    else
      s = make_int2(causal ? max(q0, min(q1, q0 + (x - k0) - past)) : q0, q1);
  }
  s.x = min(max(s.x, 0), lim);
  s.y = min(max(s.y, s.x), lim);
  (is_q ? row_span : key_span)[x] = s;
}

// ---------------------------------------------------------------- launches
// Waves of a workgroup, of 32 rows (or keys) each. Two walk fewer keys that only a neighbour's rows see and start sooner;
// more share a tile's loads, which pays where the products of wide 16-bit heads leave time for little else. Forward, dQ,
// dK and dV with four : two waves, 32,768 rows, 8 heads, not causal, in us: float32 heads of 16, length 50: 60, 80, 103 : 45,
// 61, 75, length 500: 193, 252, 352 : 180, 238, 311; bfloat16 heads of 64, length 500: 123, 127, 165 : 104, 114, 144, length
// 2000: 233, 250, 350 : 239, 265, 373; bfloat16 heads of 128 (over 2), length 500: 156, 202, 318 : 198, 198, 318; float16
// heads of 32, length 130: 47, 59, 57 : 50, 56, 56; float32 heads of 128 (over 2), length 500: 828, 1164, 2039 : 767, 1071, 2704.
constexpr int fwd_waves(int elem, int dp) { return elem == 2 && (dp == 128 || dp == 32) ? 4 : 2; }
constexpr int dq_waves(int elem, int dp) { return elem == 2 && dp == 128 ? 4 : 2; }
// Keys of a tile of the dQ pass: more where their products are short (32 : 64 keys in us; 8 heads of 16, bfloat16, 256
// graphs of 9 to 250 nodes 55 : 49, two causal sequences of 8000 181 : 159; heads of 32, float16: 63 : 61, 192 : 188; heads of 64:
// 72 : 75, 264 : 260).
constexpr int dq_keys(int elem, int dp) { return elem == 2 && dp <= 32 ? 64 : 32; }
// dK and dV of 32 keys of 128 16-bit values fill a wave's registers: eight waves a workgroup stage little enough each that
// two of them fit a SIMD (with four, some of it leaves the registers, or one wave a SIMD runs: 0.75 and 0.87 instead
// of 0.61 ms on one causal sequence of 8192, 16 heads over 4).
constexpr int kv_waves(int elem, int dp) { return dp == 128 ? (elem == 2 ? 8 : 4) : 2; }
constexpr int kMaxPieces = 64;    // a wave joins them

template <typename T> constexpr int tile_rows() { return sizeof(T) == 2 ? 64 : 32; }
template <typename T> constexpr int tile_keys() { return sizeof(T) == 2 ? 64 : 32; }

template <typename F> int with_dim(int dim, F&& f) {
  if (dim <= 16) return f(std::integral_constant<int, 16>());
  if (dim <= 32) return f(std::integral_constant<int, 32>());
  if (dim <= 64) return f(std::integral_constant<int, 64>());
  return f(std::integral_constant<int, 128>());
}

int check(const bf_packed_attn* p, const char* fn, bool backward) {
  BF_CHECK_ARG(p != nullptr, "%s: no arguments", fn);
  BF_CHECK_ARG(p->dtype == BF_DTYPE_F32 || p->dtype == BF_DTYPE_BF16 || p->dtype == BF_DTYPE_F16, "%s: dtype %d", fn,
               p->dtype);
  BF_CHECK_ARG(p->heads_q >= 1 && p->heads_k >= 1 && p->heads_q % p->heads_k == 0,
               "%s: %d query heads over %d key heads (a multiple expected)", fn, p->heads_q, p->heads_k);
  if (p->head_dim < 8 || p->head_dim > 128 || p->head_dim % 8) {
    set_error("%s: head_dim %d (a multiple of 8 up to 128 is supported)", fn, p->head_dim);
    return BF_ERR_UNSUPPORTED;
  }
  BF_CHECK_ARG(p->n_q >= 0 && p->n_k >= 0 && p->n_k < kMaxRows && p->n_q < kMaxRows / p->heads_q,
               "%s: %lld rows of %d heads, %lld keys (below 2^31 - 2^17 each)", fn, (long long)p->n_q, p->heads_q, (long long)p->n_k);
  BF_CHECK_ARG(p->longest >= 0, "%s: longest sequence %d", fn, p->longest);
  // its product with log2 e has to be finite too
  BF_CHECK_ARG(p->scale > 0.f && p->scale <= 2e38f, "%s: scale %g (positive, up to 2e38 expected)", fn, double(p->scale));
  const int64_t per16 = p->dtype == BF_DTYPE_F32 ? 4 : 8;
  for (const int64_t* s : {p->q_stride, p->k_stride, p->v_stride})
    BF_CHECK_ARG(s[0] >= 0 && s[1] >= 0 && s[0] % per16 == 0 && s[1] % per16 == 0,
                 "%s: strides (%lld, %lld) are not whole 16-byte steps", fn, (long long)s[0], (long long)s[1]);
  BF_CHECK_ARG(p->n_q == 0 || p->row_span, "%s: no row spans", fn);
  BF_CHECK_ARG(!backward || p->n_k == 0 || p->key_span, "%s: no key spans", fn);
  return BF_OK;
}

Args make_args(const bf_packed_attn* p, const void* q, const void* k, const void* v) {
  Args a{};
  a.q = q, a.k = k, a.v = v;
  a.row_span = reinterpret_cast<const int2*>(p->row_span);
  a.key_span = reinterpret_cast<const int2*>(p->key_span);
  a.qs_t = p->q_stride[0], a.qs_h = p->q_stride[1];
  a.ks_t = p->k_stride[0], a.ks_h = p->k_stride[1];
  a.vs_t = p->v_stride[0], a.vs_h = p->v_stride[1];
  a.hq = p->heads_q, a.hk = p->heads_k, a.group = p->heads_q / p->heads_k, a.dim = p->head_dim;
  a.rows = int32_t(p->n_q * a.group);
  a.n_q = int32_t(p->n_q), a.n_k = int32_t(p->n_k);
  a.scale = p->scale;
  a.c = p->scale * kLog2e;
  a.by_group = make_div(uint32_t(a.group));
  a.pieces = 1;
  a.xcd_groups = 1;
  while (a.xcd_groups < kXcds && a.hk % (2 * a.xcd_groups) == 0) a.xcd_groups *= 2;
  return a;
}

// Workgroups that cover every (tile, key head, piece).
dim3 grid_of(const Args& a) {
  const int64_t per = int64_t(a.tiles) * a.pieces;
  const int64_t each = kXcds / a.xcd_groups;
  return dim3(unsigned(ceil_div(a.hk / a.xcd_groups * per, each) * kXcds));
}

// Pieces a tile's keys are cut into. From some number of rows on, workgroups over whole rows fill the chip (256 CUs); below
// that, one-wave workgroups over pieces of the keys do. Whole : pieces in us, one causal sequence of keys with the last
// (workgroups of 128 rows) of them as rows:
//   16 bits, heads of 128 (16 over 4): 2000 keys (64) 58 : 49, (96) 57 : 67, (136) 60 : 82; 8192 keys (72) 204 : 167, (96) 203 :
//     211, (136) 208 : 298, (248) 209 : 383
//   16 bits, heads of 64: 2000 keys (136) 42 : 38, (248) 43 : 43, (264) 43 : 52; 8192 keys (136) 158 : 141, (264) 160 : 177;
//     heads of 32: 2000 keys (136) 34 : 31, (264) 35 : 42; 8192 keys (136) 125 : 83, (264) 127 : 125, (504) 129 : 136
//   float32, heads of 16: 2000 keys (264) 81 : 67, (504) 82 : 72; 8192 keys (264) 427 : 311; heads of 128 (16 over 2): 2000
//     keys (264) 307 : 194, (504) 309 : 201; 8192 keys (264) 1902 : 1666, (504) 1898 : 2049
int pieces_of(const bf_packed_attn* p) {
  const int64_t rows = p->n_q * (p->heads_q / p->heads_k);
  const int64_t enough = p->dtype == BF_DTYPE_F32 ? 512 : p->head_dim > 64 ? 96 : 256;
  if (ceil_div(rows, 128) * p->heads_k >= enough) return 1;
  const int64_t tiles = ceil_div(rows, 32) * p->heads_k;
  const int64_t want = ceil_div(2048, tiles);
  const int64_t most = ceil_div(p->n_k, 64);
  int64_t n = want < most ? want : most;
  if (n > kMaxPieces) n = kMaxPieces;
  return n < 1 ? 1 : int(n);
}

// Pieces a key tile's rows are cut into (float32 partial sums, joined in order), where the key tiles are too few to fill
// the chip and to even out what a causal mask gives them. Equal parts of each tile's own rows, the longest tiles first:
// parts of one width for all, in either order, read less of the rows together and took 0.71 to 1.0 instead of 0.61 ms on
// one causal sequence of 8192 (16 heads of 128 over 4). Whole : pieces in us, forward and backward: 500 rows in sequences
// of 5, 32 heads of 128 over 2, bfloat16 289 : 72; in sequences of 100, 16 heads of 64 over 2, float32 319 : 123. Tiles that fill
// the chip once gain by pieces only what a long mask leaves uneven: 20,000 rows in sequences of 500, 8 heads of 128 over 4,
// float16 456 : 520. Short walks of narrow 16-bit heads do not earn the second launch: 640 rows of one causal sequence, 8 heads
// of 64, float16, dK and dV 24 : 25, 900 rows 33 : 29 (float32 heads of 16: 43 : 32, 60 : 36).
int kv_pieces_of(const bf_packed_attn* p) {
  const int elem = p->dtype == BF_DTYPE_F32 ? 4 : 2;
  const int64_t keys = 32 * kv_waves(elem, p->head_dim > 64 ? 128 : 64), groups = ceil_div(p->n_k, keys) * p->heads_k;
  if (groups >= 512 || groups == 0) return 1;
  if (groups >= 256 && p->longest > 0 && p->longest < p->n_q / 4) return 1;
  // what a tile of several sequences walks: its keys' sequences
  const int64_t walks = p->longest > 0 && p->longest + keys < p->n_q ? p->longest + keys : p->n_q;
  const int64_t rows = walks * (p->heads_q / p->heads_k);
  if (elem == 2 && p->head_dim <= 64 && rows < 768) return 1;
  int64_t n = ceil_div(512, groups);
  if (n > rows / 256) n = rows / 256;
  if (n > kMaxPieces) n = kMaxPieces;
  return n < 1 ? 1 : int(n);
}

// Order of the tiles of rows (or keys) by the keys (rows) that they walk, most first, in 256 classes: one workgroup.
__global__ __launch_bounds__(1024) void packed_order(const int2* span, int tiles, int per_tile, Div by_group, int last_row,
                                                     int32_t* order) {
  __shared__ int count[256], top;
  const int tid = threadIdx.x;
  if (tid < 256) count[tid] = 0;
  if (tid == 0) top = 1;
  __syncthreads();
  constexpr int kEach = 8;
  int cost[kEach];
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int t = tid + 1024 * u;
    cost[u] = 0;
    if (t < tiles) {
      const int first = t * per_tile, last = min(first + per_tile - 1, last_row);
      cost[u] = max(span[by_group(last)].y - span[by_group(first)].x, 0);
      atomicMax(&top, cost[u]);
    }
  }
  __syncthreads();
  const float by = 255.f / float(top);
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    cost[u] = 255 - int(float(cost[u]) * by);
    if (tid + 1024 * u < tiles) atomicAdd(&count[cost[u]], 1);
  }
  __syncthreads();
  if (tid < 64) {                      // where each class begins: a wave's scan over 4 classes a lane
    int c[4], sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = count[4 * tid + k], sum += c[k];
    int before = sum;
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(before, o, 64);
      if (tid >= o) before += x;
    }
    before -= sum;
#pragma unroll
    for (int k = 0; k < 4; ++k) count[4 * tid + k] = before, before += c[k];
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kEach; ++u)
    if (tid + 1024 * u < tiles) order[atomicAdd(&count[cost[u]], 1)] = tid + 1024 * u;
}

constexpr int kMaxOrder = 8192;        // tiles that a workgroup orders; beyond, the chip evens out by itself

// Whether a call's tiles are put in order: several sequences, some of them long (one sequence's are in order as they lie).
// An ordering takes some 6 us. Four causal sequences of 4096, 8 heads of 128, with and without it: forward 180 and 216 us,
// dQ 237 and 288, dK and dV 314 and 460; eight of 2048, 16 heads over 4: 186 and 207, 255 and 263, 339 and 534.
bool orders_tiles(const bf_packed_attn* p) {
  return p->longest != p->n_q && (p->longest == 0 || p->longest >= 512) && p->n_q >= 2048;
}

int64_t order_ints(const bf_packed_attn* p) { return orders_tiles(p) ? kMaxOrder : 0; }

// Sets a.order: the order of the call's tiles, in the head of its scratch, or NULL.
int order_tiles(Args& a, const bf_packed_attn* p, const int2* span, int group, int per_tile, int n, float* scratch,
                hipStream_t st) {
  a.order = nullptr;
  if (!orders_tiles(p) || a.tiles > kMaxOrder) return BF_OK;
  BF_CHECK_ARG(scratch != nullptr, "packed_attn: no scratch (bf_packed_attn_fwd_floats, bf_packed_attn_bwd_floats)");
  int32_t* order = reinterpret_cast<int32_t*>(scratch);
  BF_LAUNCH("packed_attn_order", packed_order, dim3(1), dim3(1024), 0, st, span, a.tiles, per_tile, make_div(uint32_t(group)),
            n - 1, order);
  BF_CHECK_LAUNCH();
  a.order = order;
  return BF_OK;
}

}  // namespace
}  // namespace bf

using namespace bf;

extern "C" int bf_packed_spans(const int32_t* q_offsets, const int32_t* k_offsets, int64_t n_seq, int64_t n_q, int64_t n_k,
                               int32_t causal, int32_t* row_span, int32_t* key_span, int32_t* positions,
                               void* stream) {
  BF_CHECK_ARG(n_seq >= 0 && n_q >= 0 && n_k >= 0 && n_seq < (int64_t(1) << 31) - 1 && n_q < (int64_t(1) << 31) - 1 &&
                   n_k < (int64_t(1) << 31) - 1,
               "packed_spans: sizes must fit 32 bits");
  if (n_q + n_k == 0) return BF_OK;
  BF_CHECK_ARG(q_offsets && k_offsets && (n_q == 0 || row_span) && (n_k == 0 || key_span), "packed_spans: bad arguments");
  BF_LAUNCH("packed_spans", packed_spans, dim3(unsigned(ceil_div(n_q + n_k, 256))), dim3(256), 0, as_stream(stream),
            q_offsets, k_offsets, int32_t(n_seq), int32_t(n_q), int32_t(n_k), int(causal != 0),
            reinterpret_cast<int2*>(row_span), reinterpret_cast<int2*>(key_span), positions);
  BF_CHECK_LAUNCH();
  return BF_OK;
}

extern "C" int64_t bf_packed_attn_fwd_floats(const bf_packed_attn* p) {
  if (check(p, "packed_attn_fwd_floats", false) != BF_OK) return -1;
  if (p->n_q == 0 || packed_is_short(p)) return 0;
  const int n = pieces_of(p);
  return n == 1 ? order_ints(p) : p->n_q * p->heads_q * n * (int64_t(p->head_dim) + 2);
}

extern "C" int bf_packed_attn_rest(const bf_packed_attn* p) {
  return check(p, "packed_attn_rest", false) == BF_OK && p->dtype != BF_DTYPE_F32 && !packed_is_short(p);
}

extern "C" int bf_packed_attn_fwd(const bf_packed_attn* p, const void* q, const void* k, const void* v, void* out, void* rest,
                                  float* lse, float* scratch, void* stream) {
  BF_CHECK_OK(check(p, "packed_attn_fwd", false));
  if (p->n_q == 0) return BF_OK;
  BF_CHECK_ARG(q && out && lse && (p->n_k == 0 || (k && v)), "packed_attn_fwd: bad arguments");
  BF_CHECK_ARG(aligned16({q, k, v, out}), "packed_attn_fwd: q, k, v and out must be 16-byte aligned");
  BF_CHECK_ARG(aligned16({rest, scratch}), "packed_attn_fwd: rest and scratch must be 16-byte aligned");
  if (packed_is_short(p)) return packed_short_fwd(p, q, k, v, out, lse, as_stream(stream));
  Args a = make_args(p, q, k, v);
  a.o = out, a.rest = rest, a.lse = lse;
  a.pieces = pieces_of(p);
  const hipStream_t st = as_stream(stream);
  if (a.pieces == 1) {
    return with_type(p->dtype, [&](auto t) -> int {
      using T = decltype(t);
      return with_dim(a.dim, [&](auto dp) -> int {
        constexpr int DP = decltype(dp)::value, BN = tile_keys<T>(), NW = fwd_waves(sizeof(T), DP);
        a.tiles = int(ceil_div(a.rows, 32 * NW));
        BF_CHECK_OK(order_tiles(a, p, a.row_span, a.group, 32 * NW, a.rows, scratch, st));
        auto kern = packed_fwd<T, DP, NW, BN, false>;
        BF_LAUNCH("packed_attn_fwd", kern, grid_of(a), dim3(64 * NW), 0, st, a);
        BF_CHECK_LAUNCH();
        return BF_OK;
      });
    });
  }
  BF_CHECK_ARG(scratch != nullptr, "packed_attn_fwd: no scratch (bf_packed_attn_fwd_floats)");
  const int64_t n_rows = p->n_q * p->heads_q;
  a.part = scratch;
  a.stat = scratch + n_rows * a.pieces * a.dim;
  a.tiles = int(ceil_div(a.rows, 32));
  return with_type(p->dtype, [&](auto t) -> int {
    using T = decltype(t);
    return with_dim(a.dim, [&](auto dp) -> int {
      constexpr int DP = decltype(dp)::value;
      auto kern = packed_fwd<T, DP, 1, 32, true>;
      BF_LAUNCH("packed_attn_fwd_pieces", kern, grid_of(a), dim3(64), 0, st, a);
      BF_CHECK_LAUNCH();
      BF_LAUNCH("packed_attn_join", (packed_join<T>), dim3(unsigned(ceil_div(n_rows, 4))), dim3(256), 0, st, a.part, a.stat,
                n_rows, a.pieces, a.dim, static_cast<T*>(out), static_cast<T*>(rest), lse);
      BF_CHECK_LAUNCH();
      return BF_OK;
    });
  });
}

extern "C" int64_t bf_packed_attn_bwd_floats(const bf_packed_attn* p) {
  if (check(p, "packed_attn_bwd_floats", true) != BF_OK) return -1;
  if (packed_is_short(p)) return 0;
  const int n = kv_pieces_of(p);
  return order_ints(p) + (n == 1 ? 0 : 2 * p->n_k * p->heads_k * p->head_dim * n);
}

extern "C" int bf_packed_attn_bwd(const bf_packed_attn* p, const void* q, const void* k, const void* v, const void* out,
                                  const void* rest, const float* lse, const void* dout, void* dq, void* dk, void* dv, float* delta,
                                  float* scratch, void* stream) {
  BF_CHECK_OK(check(p, "packed_attn_bwd", true));
  BF_CHECK_ARG((p->n_q == 0 || (q && out && lse && dout && dq && delta)) && (p->n_k == 0 || (k && v && dk && dv)),
               "packed_attn_bwd: bad arguments");
  BF_CHECK_ARG(aligned16({q, k, v, out, dout, dq, dk, dv}), "packed_attn_bwd: tensors must be 16-byte aligned");
  BF_CHECK_ARG(aligned16({rest, scratch}), "packed_attn_bwd: rest and scratch must be 16-byte aligned");
  if (packed_is_short(p)) return packed_short_bwd(p, q, k, v, out, lse, dout, dq, dk, dv, delta, as_stream(stream));
  Args a = make_args(p, q, k, v);
  a.out = out, a.rest = const_cast<void*>(rest), a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv, a.delta = delta;
  a.lse = const_cast<float*>(lse);
  const hipStream_t st = as_stream(stream);
  return with_type(p->dtype, [&](auto t) -> int {
    using T = decltype(t);
    return with_dim(a.dim, [&](auto dp) -> int {
      constexpr int DP = decltype(dp)::value;
      if (a.rows > 0) {
        constexpr int NW = dq_waves(sizeof(T), DP);
        a.tiles = int(ceil_div(a.rows, 32 * NW));
        BF_CHECK_OK(order_tiles(a, p, a.row_span, a.group, 32 * NW, a.rows, scratch, st));
        auto kern = packed_bwd_q<T, DP, NW, dq_keys(sizeof(T), DP)>;
        BF_LAUNCH("packed_attn_bwd_q", kern, grid_of(a), dim3(64 * NW), 0, st, a);
        BF_CHECK_LAUNCH();
      }
      if (a.n_k > 0) {
        constexpr int NWK = kv_waves(sizeof(T), DP);
        a.tiles = int(ceil_div(a.n_k, 32 * NWK));
        a.pieces = kv_pieces_of(p);
        BF_CHECK_OK(order_tiles(a, p, a.key_span, 1, 32 * NWK, a.n_k, scratch, st));
        BF_CHECK_ARG(a.pieces == 1 || scratch, "packed_attn_bwd: no scratch (bf_packed_attn_bwd_floats)");
        a.part = scratch + order_ints(p);
        auto kern = packed_bwd_kv<T, DP, NWK, DP == 128 ? 32 : tile_rows<T>()>;
        BF_LAUNCH("packed_attn_bwd_kv", kern, grid_of(a), dim3(64 * NWK), 0, st, a);
        BF_CHECK_LAUNCH();
        if (a.pieces > 1) {
          const int64_t all = p->n_k * p->heads_k * p->head_dim;
          BF_LAUNCH("packed_attn_join_kv", (packed_join_kv<T>), dim3(unsigned(ceil_div(2 * all, 1024))), dim3(256), 0, st,
                    a.part, all, a.pieces, static_cast<T*>(dk), static_cast<T*>(dv));
          BF_CHECK_LAUNCH();
        }
      }
      return BF_OK;
    });
  });
}
