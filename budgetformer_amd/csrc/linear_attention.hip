// Linear attention with a decay for each head over packed sequences, on the matrix cores.
//
//   out_i = scale sum_{j <= i, same sequence} g^(i - j) (x_i . y_j) z_j
//
// One pass in three uses: the forward is (x, y, z) = (q, k, v); the gradients are (dout, v, k) for dq and, with the
// packed axis read backwards, (v, dout, q) for dk and (k, q, dout) for dv.
//
// Chunked form. A workgroup walks a segment of the packed axis in tiles of 32 tokens, the state M = sum g^(t - j) y_j z_j^T
// in the accumulators of its waves (wave w owns the columns 32w .. 32w+31 of z, so a column of M is a lane's, its rows
// are registers). Per tile [t0, t1):
//   W_ij = scale (x_i . y_j) g^(i - j) for j <= i of the same sequence
//   out_i = sum_j W_ij z_j + scale g^(i - t0 + 1) x_i M                   the second only if the sequence began before t0
//   M = g^(t1 - t0) M + sum_j g^(t1 - 1 - j) y_j z_j^T                    only the last row's sequence
// The registers of W and of M are, packed, operands of the next product as they stand (packed_tile.h): every wave forms
// W for itself, and the state never moves. (Tiles of 64 tokens share W's four blocks through LDS; their loads on the way
// leave fewer waves and two barriers more: 90 instead of 57 us for the pass over 8192 tokens, 16 heads of 128, and 110
// instead of 64 us over 40,000, 8 heads of 16.) Tiles are cut from the packed axis, not from the sequences: a boundary is
// a comparison of indices, and short sequences fill tiles. Where states come in or go out (init, final) tiles end at the
// sequences' ends instead.
//
// Calls of few heads cut the axis into segments: one launch forms each segment's own contribution to the state, one
// carries it from segment to segment, and the pass starts from there. States are float32 throughout; as operands of x M
// and W z, M and W are rounded to the activations' type (half a step, as the inputs' own rounding; in float32 not at all);
// the decayed z that enters the state is given in parts that keep its float32 value. float16 ends at 65504 and loses bits
// below 2^-14, where a score or a state need not: there both are operands in units of a power of 2 (kScoreUnit, kStateUnit).
//
// What bounds it is the wait for a tile's loads with two waves a SIMD: 8192 tokens, 16 heads of 128, bfloat16 with a final
// state take 29 (segments) + 12 (carry) + 52 us (pass), where the tensors' bytes are 26 us of a copy.
#include "packed_tile.h"

namespace bf {
namespace {

struct LinArgs {
  const void *x, *y, *z;
  void* out;
  int64_t xs_t, xs_h, ys_t, ys_h, zs_t, zs_h;
  const int2 *row_span, *key_span;
  const int32_t* offsets;
  const float *log_decay, *init;
  float *final_state, *carry;
  int64_t init_sx, init_sz;
  int32_t n, n_seq, heads, dx, dz;
  int32_t seg_len, n_seg;
  float scale;
  bool reverse, states;
  bool warm;                       // segments begin with the sequence that their first token is in: nothing is carried
};

template <typename T> __device__ __forceinline__ Frag<T> pack8_by(const F32x16& x, int t, float by) {
  Frag<T> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = T(x[8 * t + j] * by);
  return f;
}

struct LinRoles {
  LinArgs role[3];
};

constexpr int kTile = 32;        // tokens of a tile

// float16's units of scores and of states as operands: what is 64 times (512 times) a score or state of ordinary size still
// fits, and the gradients' small ones keep their bits (a state's rounding is then 2^-31 at most, a score's 2^-34, where the
// result's own is 2^-25). Larger ones take a unit of their own, that brings the largest to 2^15.
constexpr float kScoreUnit = 1.f / 512.f, kStateUnit = 1.f / 64.f, kUnitMost = 32768.f;

// The unit, a power of 2, in which `big` is at most 2^15.
__device__ __forceinline__ float unit_of(float big) { return ldexpf(1.f, __builtin_amdgcn_frexp_expf(big) - 15); }

// A head's log decay; one of 0 (log -inf) stays finite, so that its power 0 is 1; a NaN stays one
__device__ __forceinline__ float finite_decay(float x) { return x < -1e4f ? -1e4f : x; }
__device__ __forceinline__ float decay_log2(const LinArgs& a, int h) { return finite_decay(a.log_decay[h]) * kLog2e; }

// the token at a place of the axis as the pass reads it, its span, and where its sequence starts on that axis
__device__ __forceinline__ int token_at(const LinArgs& a, int p) { return a.reverse ? a.n - 1 - p : p; }
__device__ __forceinline__ int2 span_at(const LinArgs& a, int p) { return (a.reverse ? a.key_span : a.row_span)[token_at(a, p)]; }
__device__ __forceinline__ int start_of(const LinArgs& a, int2 s) {
  if (a.reverse) return a.n - s.y;                     // behind the last sequence: after its own place
  return s.y > s.x ? s.x : a.n;                        // a row behind the last sequence sees nothing
}

// Last s with offsets[s] <= p; n_seq behind the last sequence, -1 before the first.
__device__ __forceinline__ int sequence_of(const LinArgs& a, int p) {
  int lo = -1, hi = a.n_seq;
  while (lo < hi) {
    const int mid = hi - ((hi - lo) >> 1);      // their sum may pass 32 bits; lo + 1 at least
    if (a.offsets[mid] <= p)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// The same value, unknown to the compiler: the addresses of a state's 64 values a lane are then formed where a sequence
// begins or ends, and not kept in registers through the loop.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The final state of sequences without tokens is their initial one: each workgroup its share of the sequences.
template <int NT> __device__ __forceinline__ void empty_states(const LinArgs& a, int tid) {
  const int64_t per = int64_t(a.heads) * a.dx * a.dz;
  for (int64_t s0 = int64_t(blockIdx.x) * 64; s0 < a.n_seq; s0 += int64_t(gridDim.x) * 64) {
    const int64_t mine = s0 + (tid & 63);
    const bool empty = mine < a.n_seq && a.offsets[mine + 1] <= a.offsets[mine];
    for (uint64_t left = __ballot(empty); left; left &= left - 1) {
      const int64_t s = s0 + __ffsll((unsigned long long)left) - 1;
      for (int64_t i = tid; i < per; i += NT) {
        const int64_t h = i / (a.dx * a.dz), x = i / a.dz % a.dx, z = i % a.dz;
        a.final_state[s * per + i] = a.init ? a.init[(s * a.heads + h) * a.dx * a.dz + x * a.init_sx + z * a.init_sz] : 0.f;
      }
    }
  }
}

template <typename T, int DX, int DZ, bool OUT, bool STATES>
__global__ __launch_bounds__(2 * DZ, 2) void linear_pass(const LinRoles all) {
  const LinArgs a = all.role[blockIdx.y];
  constexpr int C = kTile, NW = DZ / 32, NT = 64 * NW, XB = DX / 32;
  // parts of the decayed z (see below): the third only for a state that goes out
  const bool third = STATES && a.final_state != nullptr;
  constexpr bool kUnits = std::is_same<T, _Float16>::value;
  constexpr int kParts = sizeof(T) == 4 ? 1 : std::is_same<T, __bf16>::value ? 3 : 2;
  using TX = Tile<T, DX>;
  using TZ = Tile<T, DZ>;
  __shared__ __attribute__((aligned(16))) char x_lds[OUT ? TX::bytes(C) : 16];
  __shared__ __attribute__((aligned(16))) char y_lds[TX::bytes(C)];
  __shared__ __attribute__((aligned(16))) char z_lds[TZ::bytes(C)];
  __shared__ int start_lds[C];
  __shared__ __attribute__((aligned(16))) float power[C];       // g^0 .. g^(C - 1), last first: a tile's weights towards its end
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
  const int64_t slot = xcd_slot(blockIdx.x, gridDim.x);
  const int h = int(slot % a.heads), seg = int(slot / a.heads);     // the heads of a token share its cache lines
  const int own = seg * a.seg_len, end = min(own + a.seg_len, a.n);
  const int begin = a.warm && seg > 0 ? max(min(own, start_of(a, span_at(a, own))), 0) : own;      // rows before `own` are another's
  const float ld = decay_log2(a, h);
  // the axis as the pass reads it: from the last token with steps back, or from the first
  const int64_t back = a.reverse ? a.n - 1 : 0;
  const T* xp = static_cast<const T*>(a.x) + h * a.xs_h + back * a.xs_t;
  const T* yp = static_cast<const T*>(a.y) + h * a.ys_h + back * a.ys_t;
  const T* zp = static_cast<const T*>(a.z) + h * a.zs_h + back * a.zs_t;
  const int64_t xs_t = a.reverse ? -a.xs_t : a.xs_t, ys_t = a.reverse ? -a.ys_t : a.ys_t, zs_t = a.reverse ? -a.zs_t : a.zs_t;
  const int2* spans = a.reverse ? a.key_span : a.row_span;

  F32x16 m[XB];
#pragma unroll
  for (int b = 0; b < XB; ++b) m[b] = zero16();
  float* carry = a.carry + ((int64_t(seg) * a.heads + h) * XB * NW + wave) * 1024 + lane;       // register r of block b: + (b * NW * 16 + r) * 64
  if (OUT && seg > 0 && !a.warm) {
#pragma unroll
    for (int b = 0; b < XB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) m[b][r] = carry[(int64_t(b) * NW * 16 + r) * 64];
  }
  // with states: the sequence of the next tile and its bounds (read again only where one ends)
  int seq = STATES ? sequence_of(a, begin) : -1, seq_begin = -1, seq_end = a.n;
  auto bounds = [&]() {
    const bool in = seq >= 0 && seq < a.n_seq;
    seq_begin = in ? a.offsets[seq] : -1;
    seq_end = seq < a.n_seq ? a.offsets[seq + 1] : a.n;
  };
  if (STATES) bounds();
  // at least one token on, whatever the offsets hold
  auto tile_end = [&](int t0) { return max(min(min(t0 + C, end), seq_end), t0 + 1); };

  Stage<T, DX, C, NT> xs, ys;
  Stage<T, DZ, C, NT> zs;
  int2 span = make_int2(0, 0);
  auto fetch = [&](int t0, int t1) {
    if constexpr (OUT) xs.load(tid, t1 - t0, a.dx, [&](int r) { return xp + (t0 + r) * xs_t; });
    ys.load(tid, t1 - t0, a.dx, [&](int r) { return yp + (t0 + r) * ys_t; });
    zs.load(tid, t1 - t0, a.dz, [&](int r) { return zp + (t0 + r) * zs_t; });
    if (tid < C) span = spans[token_at(a, min(t0 + tid, t1 - 1))];      // not looked at before the tile is stored: nothing waits here
  };

  if (tid < C) power[tid] = exp2_fast(ld * float(C - 1 - tid));
  int t1 = begin < end ? tile_end(begin) : begin;
  if (begin < end) fetch(begin, t1);
  for (int t0 = begin; t0 < end;) {
    const int len = t1 - t0;
    if constexpr (OUT) xs.clip(tid, len, a.dx);
    ys.clip(tid, len, a.dx);
    zs.clip(tid, len, a.dz);
    __syncthreads();
    if constexpr (OUT) xs.store(tid, x_lds);
    ys.store(tid, y_lds);
    zs.store(tid, z_lds);
    if (tid < C) start_lds[tid] = start_of(a, span);
    bool odd = false;
    if constexpr (OUT)
      odd = __syncthreads_or(zs.tainted());
    else
      __syncthreads();
    if (STATES && t0 == seq_begin) {                                  // with states: a sequence begins with its tile
      const int z = fresh(32 * wave + col), x0 = fresh(4 * half);
      const float* s0 = a.init ? a.init + (int64_t(seq) * a.heads + h) * a.dx * a.dz : nullptr;
#pragma unroll
      for (int b = 0; b < XB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int x = x0 + 32 * b + acc_row(r, 0);
          const float v = s0 ? s0[min(x, a.dx - 1) * a.init_sx + min(z, a.dz - 1) * a.init_sz] : 0.f;
          m[b][r] = x < a.dx && z < a.dz ? v : 0.f;
        }
    }
    const bool ends = STATES && seq_begin >= 0 && t1 == seq_end;
    const int this_seq = seq;
    if (STATES && t1 == seq_end && t1 < end) {
      while (seq < a.n_seq && a.offsets[seq + 1] <= t1) ++seq;
      bounds();
    }
    const int next = t1 < end ? tile_end(t1) : t1;
    if (t1 < end) fetch(t1, next);

    const int first_start = start_lds[0], last_start = start_lds[len - 1];
    // z towards the wave's columns, for out and for the state
    Frag<T> zf[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) zf[t] = TZ::template col_frag<true>(z_lds, t, wave, lane);
    if constexpr (OUT) {
      const int i = col, from = start_lds[i] - t0;
      F32x16 acc = zero16(), o = zero16();
#pragma unroll
      for (int s = 0; s < TX::kSteps; ++s)
        acc = Mat<T>::mma(TX::row_frag(y_lds, col, s, half), TX::row_frag(x_lds, col, s, half), acc);
      // with states the tile is one sequence's, whose state came in or was begun above
      if (STATES || first_start < t0) {
        float unit = 1.f;
        if constexpr (kUnits) {                // one for the wave: the state's rows are other lanes' contractions
          unit = kStateUnit;
          float big = 0.f;
#pragma unroll
          for (int b = 0; b < XB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) big = fmaxf(big, fabsf(m[b][r]));
          if (__any(big > kUnitMost * kStateUnit)) {
            if (!(big < INFINITY)) {           // a column that is not finite is no reason for the others to overflow
              big = 0.f;
#pragma unroll
              for (int b = 0; b < XB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) big = fmaxf(big, fabsf(m[b][r]) < INFINITY ? fabsf(m[b][r]) : 0.f);
            }
            for (int n = 32; n; n >>= 1) big = fmaxf(big, __shfl_xor(big, n, 64));
            if (big > kUnitMost * kStateUnit) unit = unit_of(big);
          }
        }
        const float per_unit = 1.f / unit;
#pragma unroll
        for (int b = 0; b < XB; ++b)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            Frag<T> mf;
            if constexpr (kUnits)
              mf = pack8_by<T>(m[b], t, per_unit);
            else
              mf = pack8<T>(m[b], t);
            o = Mat<T>::mma(mf, TX::row_frag_regs(x_lds, i, 2 * b + t, half), o);
          }
        const bool mine = from < int(STATES);
        const float f = a.scale * exp2_fast(ld * float(i + 1)) * unit;
#pragma unroll
        for (int r = 0; r < 16; ++r) o[r] = mine ? o[r] * f : 0.f;
      }
      float w[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = acc_row(r, half);
        w[r] = j <= i && j >= from ? acc[r] * (a.scale * exp2_fast(ld * float(i - j))) : 0.f;
      }
      float unit = 1.f;
      if constexpr (kUnits) {                  // a row's own: it is the lane's (and its other half's)
        unit = kScoreUnit;
        float big = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) big = fmaxf(big, fabsf(w[r]));
        if (__any(big > kUnitMost * kScoreUnit)) {
          big = fmaxf(big, __shfl_xor(big, 32, 64));
          if (big > kUnitMost * kScoreUnit && big < INFINITY) unit = unit_of(big);
        }
        const float per_unit = 1.f / unit;
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] *= per_unit, o[r] *= per_unit;
      }
      if (!odd) {
#pragma unroll
        for (int t = 0; t < 2; ++t) o = Mat<T>::mma(zf[t], pack8<T>(w, t), o);
      } else {                            // some z is not finite: NaN for the rows that see it, nothing for the others
        F32x16 bad = zero16();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          o = Mat<T>::mma(finite<T>(zf[t]), pack8<T>(w, t), o);
          Frag<T> sees;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int j = 16 * t + acc_row(k, half);
            sees[k] = T(j <= i && j >= from ? 1.f : 0.f);
          }
          bad = Mat<T>::mma(is_infinite<T>(zf[t], 1.f), sees, bad);
          bad = Mat<T>::mma(is_infinite<T>(zf[t], -1.f), sees, bad);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (bad[r] > 0.f) o[r] = NAN;
      }
      if (i < len && t0 + i >= own)
        store_block<T>(static_cast<T*>(a.out) + (int64_t(token_at(a, t0 + i)) * a.heads + h) * a.dz, o, unit, wave, a.dz, half);
    }

    if (!OUT || t1 < end || ends) {
      const bool keep = STATES || last_start < t0;
      const float f = exp2_fast(ld * float(len));
#pragma unroll
      for (int b = 0; b < XB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) m[b][r] = keep ? m[b][r] * f : 0.f;
      const int from = STATES ? 0 : last_start - t0;
      const bool cut = from > 0;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        // the decayed z in two or three parts of the activations' type, which add up to (nearly) its float32 value
        Frag<T> part[3];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int j = 16 * t + acc_row(k, half);
          float x = j >= from && j < len ? float(zf[t][k]) * power[min(j + C - len, C - 1)] : 0.f;
#pragma unroll
          for (int n = 0; n < kParts; ++n) {
            part[n][k] = T(x);
            x -= float(part[n][k]);
          }
        }
#pragma unroll
        for (int b = 0; b < XB; ++b) {
          Frag<T> yf = TX::template col_frag<true>(y_lds, t, b, lane);
          if (cut) {                      // what another sequence holds there may not be finite
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (16 * t + acc_row(k, half) < from) yf[k] = T(0.f);
          }
#pragma unroll
          for (int n = 0; n < kParts; ++n)
            if (n < 2 || third) m[b] = Mat<T>::mma(yf, part[n], m[b]);
        }
      }
      if (OUT && ends && a.final_state) {
        const int z = fresh(32 * wave + col), x0 = fresh(4 * half);
        float* fs = a.final_state + (int64_t(this_seq) * a.heads + h) * a.dx * a.dz;
#pragma unroll
        for (int b = 0; b < XB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int x = x0 + 32 * b + acc_row(r, 0);
            if (x < a.dx && z < a.dz) fs[x * a.dz + z] = m[b][r];
          }
      }
    }
    t0 = t1;
    t1 = next;
  }
  if constexpr (OUT && STATES) {
    if (a.final_state) empty_states<NT>(a, tid);
  }
  if constexpr (!OUT) {
#pragma unroll
    for (int b = 0; b < XB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) carry[(int64_t(b) * NW * 16 + r) * 64] = m[b][r];
  }
}

// Segments' own contributions -> the state each segment starts from, in place: a workgroup 256 values of a head's state, a
// wave kCarry segments of them, held in registers. What a wave's segments make of the state before them goes to the
// others through LDS (times a factor, or dropped where a sequence began, plus a sum), so one trip to memory serves up to 256
// segments. (A lane that walks all segments of a value instead, 16 at a time: 27 instead of 13.5 us for 250 segments of 8 heads
// of 32, 20 instead of 16 for 126 of 8 of 64, 26 instead of 25 for 32 of 16 of 128.)
constexpr int kCarry = 16, kCarryWaves = 16;

__global__ __launch_bounds__(64 * kCarryWaves) void linear_carry(const LinRoles all, int64_t values) {
  typedef float V4 __attribute__((ext_vector_type(4)));
  __shared__ V4 sum_lds[kCarryWaves][64];
  __shared__ float by_lds[kCarryWaves];
  constexpr float kDropped = -1.f;
  const LinArgs a = all.role[blockIdx.y];
  const int lane = threadIdx.x, wave = threadIdx.y, waves = blockDim.y;
  const int64_t i = int64_t(blockIdx.x) * 256 + 4 * lane, step = values * a.heads;      // values is a multiple of 256
  const float f = exp2_fast(decay_log2(a, int(i / values)) * float(a.seg_len));
  float* c = a.carry + i;
  V4 into = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.n_seg; s0 += kCarry * waves) {
    const int first = s0 + wave * kCarry;
    V4 mine[kCarry];
#pragma unroll
    for (int k = 0; k < kCarry; ++k)     // segments behind the last read it again
      mine[k] = *reinterpret_cast<const V4*>(c + min(first + k, a.n_seg - 1) * step);
    // bit k: segment k's last sequence began in it
    const int s = min(first + (lane & (kCarry - 1)), a.n_seg - 1);
    const uint64_t began = __ballot(start_of(a, span_at(a, min((s + 1) * a.seg_len, a.n) - 1)) >= s * a.seg_len);
    float by = 1.f;
    V4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kCarry; ++k) {
      if (first + k >= a.n_seg) continue;
      const bool b = began >> k & 1;
      by = b || by == kDropped ? kDropped : by * f;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = b ? mine[k][j] : fmaf(sum[j], f, mine[k][j]);
    }
    sum_lds[wave][lane] = sum;
    if (lane == 0) by_lds[wave] = by;
    __syncthreads();
    V4 run = into;
    for (int p = 0; p < waves; ++p) {
      const V4 x = sum_lds[p][lane];
      const float w = by_lds[p];
      if (p == wave) run = into;
#pragma unroll
      for (int j = 0; j < 4; ++j) into[j] = w == kDropped ? x[j] : fmaf(into[j], w, x[j]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kCarry; ++k) {
      if (first + k < a.n_seg) *reinterpret_cast<V4*>(c + (first + k) * step) = run;
      const bool b = began >> k & 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) run[j] = b ? mine[k][j] : fmaf(run[j], f, mine[k][j]);
    }
  }
}

// The final states of sequences without tokens where no pass runs.
__global__ __launch_bounds__(256) void linear_empty(const LinArgs a) { empty_states<256>(a, threadIdx.x); }

// One token a sequence: a workgroup a state; 256 lanes take 4 columns of 1024 / dz rows at a time. Bound by the states'
// bytes: 64 sequences, 16 heads of 128 x 128, 135 MB in 21 us (part of it out of the last-level cache).
template <typename T>
__global__ __launch_bounds__(256) void linear_step(const T* q, const T* k, const T* v, const float* log_decay, const float* state,
                                                   int heads, int dk, int dv, float scale, T* out, float* new_state) {
  __shared__ float part[256 * 4];
  const int64_t nh = blockIdx.x;
  const int h = int(nh % heads), cols = dv / 4, rows = 256 / cols, tid = threadIdx.x;
  const int c = tid % cols, r0 = tid / cols;
  const float g = __expf(finite_decay(log_decay[h]));
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  if (r0 < rows) {
    float vv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) vv[j] = float(v[nh * dv + 4 * c + j]);
    const float* s = state + nh * dk * dv + 4 * c;
    float* n = new_state + nh * dk * dv + 4 * c;
    for (int r = r0; r < dk; r += rows) {
      const float kr = float(k[nh * dk + r]), qr = float(q[nh * dk + r]);
      float4 x = *reinterpret_cast<const float4*>(s + int64_t(r) * dv);
      x.x = fmaf(x.x, g, kr * vv[0]);
      x.y = fmaf(x.y, g, kr * vv[1]);
      x.z = fmaf(x.z, g, kr * vv[2]);
      x.w = fmaf(x.w, g, kr * vv[3]);
      *reinterpret_cast<float4*>(n + int64_t(r) * dv) = x;
      o[0] = fmaf(qr, x.x, o[0]);
      o[1] = fmaf(qr, x.y, o[1]);
      o[2] = fmaf(qr, x.z, o[2]);
      o[3] = fmaf(qr, x.w, o[3]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) part[r0 * dv + 4 * c + j] = o[j];
  }
  __syncthreads();
  for (int d = tid; d < dv; d += 256) {
    float sum = 0.f;
    for (int r = 0; r < rows; ++r) sum += part[r * dv + d];
    out[nh * dv + d] = T(sum * scale);
  }
}

// ---------------------------------------------------------------- launches
int pad32(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

template <typename F> int with_pad(int d, F&& f) {
  if (d <= 32) return f(std::integral_constant<int, 32>());
  if (d <= 64) return f(std::integral_constant<int, 64>());
  return f(std::integral_constant<int, 128>());
}

int check(const bf_linear_attn* p, const char* fn) {
  BF_CHECK_ARG(p != nullptr, "%s: no arguments", fn);
  BF_CHECK_ARG(p->dtype == BF_DTYPE_F32 || p->dtype == BF_DTYPE_BF16 || p->dtype == BF_DTYPE_F16, "%s: dtype %d", fn,
               p->dtype);
  for (int d : {p->dim_k, p->dim_v})
    if (d < 8 || d > 128 || d % 8) {
      set_error("%s: head dims (%d, %d) (multiples of 8 up to 128 are supported)", fn, p->dim_k, p->dim_v);
      return BF_ERR_UNSUPPORTED;
    }
  BF_CHECK_ARG(p->n >= 0 && p->n < kMaxRows && p->n_seq >= 0 && p->n_seq < (int64_t(1) << 31) - 1 &&
                   p->heads >= 1 && p->heads <= (1 << 20),
               "%s: bad sizes (%lld rows, %lld sequences, %d heads)", fn, (long long)p->n, (long long)p->n_seq, p->heads);
  const int64_t per16 = p->dtype == BF_DTYPE_F32 ? 4 : 8;
  for (const int64_t* s : {p->q_stride, p->k_stride, p->v_stride})
    BF_CHECK_ARG(s[0] >= 0 && s[1] >= 0 && s[0] % per16 == 0 && s[1] % per16 == 0,
                 "%s: strides (%lld, %lld) are not whole 16-byte steps", fn, (long long)s[0], (long long)s[1]);
  BF_CHECK_ARG(p->scale == p->scale && p->scale <= 3e38f && p->scale >= -3e38f, "%s: scale %g", fn, double(p->scale));
  BF_CHECK_ARG(p->longest >= 0, "%s: longest sequence %d", fn, p->longest);
  BF_CHECK_ARG(p->log_decay && (p->n == 0 || (p->row_span && p->key_span)), "%s: no decays or no spans", fn);
  BF_CHECK_ARG(!(p->init || p->final_state) || p->offsets, "%s: states need the offsets", fn);
  return BF_OK;
}

// Tokens of a segment: whole tiles, so many that some 2048 waves share the axis, but at least twice as many as a state
// has columns (a segment's own contribution and its carry are a state each, written and read, against its tokens' rows).
int64_t segment_of(const bf_linear_attn* p) {
  const int64_t columns = pad32(p->dim_k > p->dim_v ? p->dim_k : p->dim_v);
  const int64_t want = ceil_div(int64_t(2048), p->heads * (columns / 32));
  const int64_t len = ceil_div(ceil_div(p->n, want), kTile) * kTile;
  return len < 2 * columns ? 2 * columns : len;
}

// Whether a segment begins with the whole sequence that its first token is in, instead of being handed that one's state:
// where no sequence is longer than half a segment (it then walks a quarter more tokens on average, and less when they
// are shorter; the two launches for the states go).
bool warms(const bf_linear_attn* p) { return p->longest > 0 && 2 * int64_t(p->longest) <= segment_of(p); }

// Floats that one pass's segments carry.
int64_t carry_floats(const bf_linear_attn* p) {
  const int64_t segs = ceil_div(p->n, segment_of(p));
  return segs <= 1 || warms(p) ? 0 : segs * p->heads * pad32(p->dim_k) * pad32(p->dim_v);
}

LinArgs make_args(const bf_linear_attn* p) {
  LinArgs a{};
  a.row_span = reinterpret_cast<const int2*>(p->row_span);
  a.key_span = reinterpret_cast<const int2*>(p->key_span);
  a.offsets = p->offsets, a.log_decay = p->log_decay;
  a.n = int32_t(p->n), a.n_seq = int32_t(p->n_seq), a.heads = p->heads;
  a.scale = p->scale;
  a.seg_len = int32_t(segment_of(p));
  a.n_seg = int32_t(ceil_div(p->n, a.seg_len));
  a.warm = warms(p);
  return a;
}

// One launch (three with segments) for passes of the same head sizes.
int launch(const LinRoles& roles, int n_roles, int32_t dtype, hipStream_t st) {
  const LinArgs& a = roles.role[0];
  const int64_t groups = int64_t(a.n_seg) * a.heads;
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return with_pad(a.dx, [&](auto px) -> int {
      return with_pad(a.dz, [&](auto pz) -> int {
        constexpr int DX = decltype(px)::value, DZ = decltype(pz)::value;
        const dim3 grid = dim3(unsigned(groups), unsigned(n_roles));
        if (a.n_seg > 1 && !a.warm) {
          auto own = a.states ? linear_pass<T, DX, DZ, false, true> : linear_pass<T, DX, DZ, false, false>;
          BF_LAUNCH("linear_attn_segments", own, grid, dim3(2 * DZ), 0, st, roles);
          BF_CHECK_LAUNCH();
          const int64_t values = DX * DZ;
          const int64_t waves = ceil_div(a.n_seg, kCarry) < kCarryWaves ? ceil_div(a.n_seg, kCarry) : kCarryWaves;
          BF_LAUNCH("linear_attn_carry", linear_carry, dim3(unsigned(values * a.heads / 256), unsigned(n_roles)),
                    dim3(64, unsigned(waves)), 0, st, roles, values);
          BF_CHECK_LAUNCH();
        }
        auto pass = a.states ? linear_pass<T, DX, DZ, true, true> : linear_pass<T, DX, DZ, true, false>;
        BF_LAUNCH("linear_attn_pass", pass, grid, dim3(2 * DZ), 0, st, roles);
        BF_CHECK_LAUNCH();
        return BF_OK;
      });
    });
  });
}

// The passes of a call: those of the same padded head sizes together.
int run(LinArgs (&pass)[3], int n, int32_t dtype, hipStream_t st) {
  bool done[3] = {false, false, false};
  for (int i = 0; i < n; ++i) {
    if (done[i]) continue;
    LinRoles r{};
    int m = 0;
    for (int j = i; j < n; ++j)
      if (!done[j] && pad32(pass[j].dx) == pad32(pass[i].dx) && pad32(pass[j].dz) == pad32(pass[i].dz) &&
          pass[j].states == pass[i].states) {
        r.role[m++] = pass[j];
        done[j] = true;
      }
    BF_CHECK_OK(launch(r, m, dtype, st));
  }
  return BF_OK;
}

void set_x(LinArgs& a, const void* x, const int64_t (&s)[2], int d) { a.x = x, a.xs_t = s[0], a.xs_h = s[1], a.dx = d; }
void set_y(LinArgs& a, const void* y, const int64_t (&s)[2]) { a.y = y, a.ys_t = s[0], a.ys_h = s[1]; }
void set_z(LinArgs& a, const void* z, const int64_t (&s)[2], int d) { a.z = z, a.zs_t = s[0], a.zs_h = s[1], a.dz = d; }

}  // namespace
}  // namespace bf

using namespace bf;

extern "C" int64_t bf_linear_attn_fwd_floats(const bf_linear_attn* p) {
  if (check(p, "linear_attn_fwd_floats") != BF_OK) return -1;
  return carry_floats(p);
}

extern "C" int bf_linear_attn_fwd(const bf_linear_attn* p, const void* q, const void* k, const void* v, void* out,
                                  float* scratch, void* stream) {
  BF_CHECK_OK(check(p, "linear_attn_fwd"));
  BF_CHECK_ARG(p->n == 0 || (q && k && v && out), "linear_attn_fwd: bad arguments");
  BF_CHECK_ARG(aligned16({q, k, v, out, scratch}), "linear_attn_fwd: q, k, v, out and scratch must be 16-byte aligned");
  LinArgs pass[3] = {make_args(p)};
  LinArgs& a = pass[0];
  set_x(a, q, p->q_stride, p->dim_k);
  set_y(a, k, p->k_stride);
  set_z(a, v, p->v_stride, p->dim_v);
  a.out = out, a.carry = scratch;
  a.init = p->init, a.final_state = p->final_state, a.states = (p->init || p->final_state) && p->n_seq > 0;
  a.init_sx = p->dim_v, a.init_sz = 1;
  const hipStream_t st = as_stream(stream);
  if (a.n == 0) {
    if (!a.states || !a.final_state) return BF_OK;
    BF_LAUNCH("linear_attn_empty", linear_empty, dim3(unsigned(ceil_div(a.n_seq, 64))), dim3(256), 0, st, a);
    BF_CHECK_LAUNCH();
    return BF_OK;
  }
  BF_CHECK_ARG(a.n_seg == 1 || a.warm || scratch, "linear_attn_fwd: no scratch (bf_linear_attn_fwd_floats)");
  return run(pass, 1, p->dtype, st);
}

extern "C" int64_t bf_linear_attn_bwd_floats(const bf_linear_attn* p) {
  if (check(p, "linear_attn_bwd_floats") != BF_OK) return -1;
  return 3 * carry_floats(p);
}

extern "C" int bf_linear_attn_bwd(const bf_linear_attn* p, const void* q, const void* k, const void* v, const void* dout,
                                  void* dq, void* dk, void* dv, float* scratch, void* stream) {
  BF_CHECK_OK(check(p, "linear_attn_bwd"));
  if (p->n == 0) return BF_OK;
  BF_CHECK_ARG(q && k && v && dout && dq && dk && dv, "linear_attn_bwd: bad arguments");
  BF_CHECK_ARG(aligned16({q, k, v, dout, dq, dk, dv, scratch}), "linear_attn_bwd: tensors must be 16-byte aligned");
  const int64_t ds[2] = {int64_t(p->heads) * p->dim_v, p->dim_v};
  LinArgs pass[3] = {make_args(p), make_args(p), make_args(p)};
  const int64_t carry = carry_floats(p);
  BF_CHECK_ARG(carry == 0 || scratch, "linear_attn_bwd: no scratch (bf_linear_attn_bwd_floats)");
  for (int i = 0; i < 3; ++i) pass[i].carry = scratch + i * carry, pass[i].reverse = i > 0;
  set_x(pass[0], dout, ds, p->dim_v);                 // dq = (dout, v, k), from the initial state's transpose
  set_y(pass[0], v, p->v_stride);
  set_z(pass[0], k, p->k_stride, p->dim_k);
  pass[0].out = dq;
  pass[0].init = p->init, pass[0].states = p->init && p->n_seq > 0;
  pass[0].init_sx = 1, pass[0].init_sz = p->dim_v;
  set_x(pass[1], v, p->v_stride, p->dim_v);           // dk = reverse (v, dout, q)
  set_y(pass[1], dout, ds);
  set_z(pass[1], q, p->q_stride, p->dim_k);
  pass[1].out = dk;
  set_x(pass[2], k, p->k_stride, p->dim_k);           // dv = reverse (k, q, dout)
  set_y(pass[2], q, p->q_stride);
  set_z(pass[2], dout, ds, p->dim_v);
  pass[2].out = dv;
  return run(pass, 3, p->dtype, as_stream(stream));
}

extern "C" int bf_linear_attn_step(const void* q, const void* k, const void* v, const float* log_decay, const float* state,
                                   int64_t n, int32_t heads, int32_t dim_k, int32_t dim_v, int32_t dtype, float scale, void* out,
                                   float* new_state, void* stream) {
  BF_CHECK_ARG(dtype == BF_DTYPE_F32 || dtype == BF_DTYPE_BF16 || dtype == BF_DTYPE_F16, "linear_attn_step: dtype %d", dtype);
  for (int d : {dim_k, dim_v})
    if (d < 8 || d > 128 || d % 8) {
      set_error("linear_attn_step: head dims (%d, %d) (multiples of 8 up to 128 are supported)", dim_k, dim_v);
      return BF_ERR_UNSUPPORTED;
    }
  BF_CHECK_ARG(n >= 0 && heads >= 1 && n < (int64_t(1) << 24) / heads, "linear_attn_step: %lld sequences of %d heads",
               (long long)n, heads);
  if (n == 0) return BF_OK;
  BF_CHECK_ARG(q && k && v && log_decay && state && out && new_state, "linear_attn_step: bad arguments");
  BF_CHECK_ARG(aligned16({state, new_state}), "linear_attn_step: states must be 16-byte aligned");
  const hipStream_t st = as_stream(stream);
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    BF_LAUNCH("linear_attn_step", (linear_step<T>), dim3(unsigned(n * heads)), dim3(256), 0, st, static_cast<const T*>(q),
              static_cast<const T*>(k), static_cast<const T*>(v), log_decay, state, heads, dim_k, dim_v, scale,
              static_cast<T*>(out), new_state);
    BF_CHECK_LAUNCH();
    return BF_OK;
  });
}
