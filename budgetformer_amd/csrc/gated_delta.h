// The gated delta rule over packed sequences: kernels and launches of one activation type (gated_delta_*.hip hold one each).
//
//   S'_t = a_t S_{t-1},  e_t = v_t - S'_t^T k_t,  S_t = S'_t + b_t k_t e_t^T,  out_t = scale S_t^T q_t,   a = exp(log_gate), b = beta
//
// Chunks of C = 32 tokens of one sequence. With G_i the sum of log_gate over the chunk up to token i, D_ij = exp(G_i - G_j)
// and S the state before the chunk, the unknown e of a chunk solve a triangular system:
//   (1 + L) e = v - exp(G) (K S),   L_ij = D_ij (k_i . k_j) b_j  for j < i
//   out_i = scale exp(G_i) S^T q_i + sum_{j <= i} P_ij b_j e_j,   P_ij = scale D_ij (q_i . k_j)
//   S <- exp(G_C) S + sum_j exp(G_C - G_j) k_j (b_j e_j)^T
// Backwards, with dS the gradient of the state behind the chunk:
//   du = P^T dout + exp(G_C - G) (K dS),  z = (1 + L')^-T du,  L'_ij = b_i D_ij (k_i . k_j),  dv = b z,  db = e . z
//   dS <- exp(G_C) dS + sum_i scale exp(G_i) q_i dout_i^T - b_i exp(G_i) k_i z_i^T
// With e and z known, the gradients of q and k are passes of linear attention over b e and b z, and the gate's is
//   dlog_gate_t = <S, dS> behind the segment + sum over its tokens i >= t of (q_i . dq_i + k_i . dk_i' - k_i . dk_i"),
// dk' the part of dk that k_i gets as the reader of a state (in e_i), dk" that as its writer.
//
// The inverses are formed by substitution in float32, a lane a column (delta_prep): backward stable, where the product
// (1 - L)(1 + L^2)(1 + L^4).. of a nilpotent L cancels sums of 3e8 for keys that repeat. They and P are kept for the passes, as operands.
//
// Sequences of more than a segment (seg_chunks chunks) are walked by segments at once: delta_pass<kMaps> forms what a
// segment makes of a state, S -> M S + B (M's columns are as many more state columns that begin as the identity),
// delta_carry hands the states from segment to segment, delta_pass walks the segments from there. Chunk x of the call's
// chunks (segment alike) is found without a table: sequence s has the places offsets[s] / 32 + s and on, which never meet the
// next one's; a wave searches 64 sequences at a time. Chunks do not hold two sequences: what is not finite stays in its own.
//
// Arithmetic. Every product is of bfloat16 matrix instructions over operands in parts: a float32 value is the sum of two bfloat16
// ones to 2^-17, of three to 2^-25, and a product of operands in parts adds the products of parts that matter. bfloat16
// activations are one part, float16's two, float32's three (six instructions; float32's own matrix instructions take
// sixteen times as long each). States, e, z, the inverses and P are operands in two parts (float32: three): nothing but the results is
// rounded to the activations' type, and the range is float32's whatever the type.
#pragma once

#include "packed_tile.h"

namespace bf {

constexpr int kDeltaChunk = 32;

struct DeltaArgs {
  const void *q, *k, *v, *dout;
  int64_t qs_t, qs_h, ks_t, ks_h, vs_t, vs_h;
  const float *log_gate, *beta;                // [n, heads]
  const int32_t* offsets;
  float *g2, *gin, *gout;                      // [n, heads]: log2 of the gates up to the token in its chunk; exp(G), exp(G_C - G)
  uint4 *inv, *score, *inv_t, *score_t;        // operands of each (chunk, head); the transposed ones for the backward, or NULL
  uint4 *map_f, *map_b;                        // M and M^T of each (segment, head), operands (the latter for the backward, or NULL)
  float *state, *dstate;                       // [segments, heads, dk, dv]: before each segment; the gradient behind it
  const float* init;
  float* final_state;
  float *e, *z;                                // [n, heads, dv]
  void *out, *dq, *dk, *dv;
  float *dq32, *dk32;                          // [n, heads, dk]: a value head's gradients of q (or NULL) and of k
  float *dgate, *dbeta;
  int64_t n_chunk, n_seg;                      // places
  int32_t n, n_seq, heads, heads_k, group, dim_k, dim_v, seg_chunks;
  float scale;
  bool carried;                                // states are handed from segment to segment
};

enum DeltaPass { kMaps, kForward, kTrain };
enum DeltaBack { kBackMaps, kBack };

template <typename T> struct DeltaLaunch {
  static int prep(const DeltaArgs& a, hipStream_t st);
  static int forward(const DeltaArgs& a, hipStream_t st);
  static int backward(const DeltaArgs& a, hipStream_t st);
  static int step(const DeltaArgs& a, int64_t n, hipStream_t st);
};

inline int delta_pad(int dk, int dv) { return dk > 64 || dv > 64 ? 128 : dk > 32 || dv > 32 ? 64 : 32; }

// Parts of an operand: of the activations, of anything else.
template <typename T> struct DeltaParts;
template <> struct DeltaParts<__bf16> { static constexpr int kIn = 1, kMid = 2; };
template <> struct DeltaParts<_Float16> { static constexpr int kIn = 2, kMid = 2; };
template <> struct DeltaParts<float> { static constexpr int kIn = 3, kMid = 3; };

inline int delta_mid_parts(int32_t dtype) { return dtype == BF_DTYPE_F32 ? 3 : 2; }

}  // namespace bf

#ifdef BF_DELTA_KERNELS
namespace bf {
namespace {

constexpr int C = kDeltaChunk;
using BFrag = Frag<__bf16>;

template <int N> struct Split { BFrag p[N]; };

// Two values' parts, a word each (one conversion instruction for both).
template <int N> __device__ __forceinline__ void split_two(float a, float b, uint32_t (&w)[N]) {
  typedef float F2 __attribute__((ext_vector_type(2)));
  typedef __bf16 B2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const F2 f = {a, b};
    w[n] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, B2));
    a -= __uint_as_float(w[n] << 16);
    b -= __uint_as_float(w[n] & 0xffff0000u);
  }
}

template <int N> __device__ __forceinline__ Split<N> split(const float (&x)[8]) {
  uint32_t w[4][N];
#pragma unroll
  for (int j = 0; j < 4; ++j) split_two<N>(x[2 * j], x[2 * j + 1], w[j]);
  Split<N> s;
#pragma unroll
  for (int n = 0; n < N; ++n) s.p[n] = __builtin_bit_cast(BFrag, make_uint4(w[0][n], w[1][n], w[2][n], w[3][n]));
  return s;
}

// Registers 8t .. 8t+7.
template <int N, typename X> __device__ __forceinline__ Split<N> split_regs(const X& x, int t) {
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = x[8 * t + j];
  return split<N>(y);
}

// acc += a b over operands in parts, without the products that are below both operands' last part.
template <int NA, int NB> __device__ __forceinline__ F32x16 mul(const Split<NA>& a, const Split<NB>& b, F32x16 acc) {
  constexpr int kMost = NA > NB ? NA : NB;
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < kMost) acc = Mat<__bf16>::mma(a.p[i], b.p[j], acc);
  return acc;
}

// A tile of C rows in N parts, a bfloat16 tile each. (Of 32 values in parts with half the padding: a CU then holds four of float32's
// gradient passes instead of three.)
template <int N, int D> struct PartTile {
  using TL = Tile<__bf16, D, (D == 32 && N > 1 ? 16 : 32)>;
  static constexpr int kPart = (TL::bytes(C) + 15) / 16 * 16, kBytes = N * kPart;
  static __device__ __forceinline__ Split<N> rows(const char* lds, int row, int s, int half) {
    Split<N> f;
#pragma unroll
    for (int n = 0; n < N; ++n) f.p[n] = TL::row_frag(lds + n * kPart, row, s, half);
    return f;
  }
  static __device__ __forceinline__ Split<N> rows_regs(const char* lds, int row, int s, int half) {
    Split<N> f;
#pragma unroll
    for (int n = 0; n < N; ++n) f.p[n] = TL::row_frag_regs(lds + n * kPart, row, s, half);
    return f;
  }
  static __device__ __forceinline__ Split<N> cols(const char* lds, int t, int block, int lane) {
    Split<N> f;
#pragma unroll
    for (int n = 0; n < N; ++n) f.p[n] = TL::template col_frag<true>(lds + n * kPart, t, block, lane);
    return f;
  }
  // values 4 i .. 4 i + 3 of a row
  static __device__ __forceinline__ void four(const char* lds, int row, int i, float (&x)[4]) {
    typedef __bf16 V4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = 0.f;
#pragma unroll
    for (int n = N - 1; n >= 0; --n) {
      const V4 v = *reinterpret_cast<const V4*>(lds + n * kPart + row * TL::kPitch + i * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] += float(v[j]);
    }
  }
};

template <int N> __device__ __forceinline__ void values(const Split<N>& s, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = float(s.p[N - 1][j]);
#pragma unroll
    for (int n = N - 2; n >= 0; --n) x[j] += float(s.p[n][j]);
  }
}

// A staged tile to LDS in parts, its rows times by(row).
template <int N, typename T, int D, int NT, typename F>
__device__ __forceinline__ void store_parts(const Stage<T, D, C, NT>& st, int tid, char* lds, F&& by) {
  using S = Stage<T, D, C, NT>;
  using PT = PartTile<N, D>;
  typedef __bf16 Out __attribute__((ext_vector_type(S::kPer)));
  typedef T In __attribute__((ext_vector_type(S::kPer)));
#pragma unroll
  for (int i = 0; i < S::kN; ++i) {
    const int c = i * NT + tid, row = c / S::kChunks;
    if (C * S::kChunks % NT && row >= C) continue;
    char* p = lds + row * PT::TL::kPitch + (c % S::kChunks) * int(sizeof(Out));
    const In v = __builtin_bit_cast(In, st.r[i]);
    const float w = by(row);
    uint32_t o[S::kPer / 2][N];
#pragma unroll
    for (int j = 0; j < S::kPer / 2; ++j) split_two<N>(float(v[2 * j]) * w, float(v[2 * j + 1]) * w, o[j]);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      typedef uint32_t Words __attribute__((ext_vector_type(S::kPer / 2)));
      Words q;
#pragma unroll
      for (int j = 0; j < S::kPer / 2; ++j) q[j] = o[j][n];
      *reinterpret_cast<Words*>(p + n * PT::kPart) = q;
    }
  }
}

template <int N, typename T, int D, int NT>
__device__ __forceinline__ void store_parts(const Stage<T, D, C, NT>& st, int tid, char* lds) {
  if constexpr (std::is_same<T, __bf16>::value && N == 1)
    st.store(tid, lds);
  else
    store_parts<N>(st, tid, lds, [](int) { return 1.f; });
}

// ---------------------------------------------------------------- places
struct Place {
  int seq, idx;            // n_seq: the rows behind the last sequence
  int begin, end;          // its rows
  int seq_end;
  bool none;               // no rows, and not an empty sequence's only place
};

// The unit (chunk or segment) of `per` tokens at place x. Offsets are taken as they are, clamped to the tensors.
__device__ __forceinline__ int clamped(const DeltaArgs& a, int64_t s) { return min(max(a.offsets[s], 0), a.n); }

__device__ __forceinline__ Place find(const DeltaArgs& a, int64_t x, int per) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, hi = int64_t(a.n_seq) + 1;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 63) / 64, s = lo + lane * step;
    const bool ok = s < hi && clamped(a, s) / per + s <= x;
    const int n = max(__popcll(__ballot(ok)), 1);
    lo += (n - 1) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  Place p;
  lo = __builtin_amdgcn_readfirstlane(int(lo));
  const int from = __builtin_amdgcn_readfirstlane(clamped(a, lo));
  p.seq = int(lo);
  p.seq_end = __builtin_amdgcn_readfirstlane(lo < a.n_seq ? max(clamped(a, lo + 1), from) : a.n);
  const int64_t idx = x - (from / per + lo), at = from + idx * per;
  p.none = idx < 0 || (idx > 0 && at >= p.seq_end);
  p.idx = int(idx);
  p.begin = int(at < p.seq_end ? at : p.seq_end);
  p.end = int(at + per < p.seq_end ? at + per : p.seq_end);
  return p;
}

__device__ __forceinline__ int64_t chunk_place(const DeltaArgs& a, const Place& p, int row) {      // of the sequence's chunk at `row`
  const int from = clamped(a, p.seq);
  return int64_t(from / C) + p.seq + (row - from) / C;
}

// Places that lie behind the last sequence: their share of a result's rows is 0.
template <typename O> __device__ __forceinline__ void clear_rows(O* p, const Place& at, int64_t row, int64_t head, int dim, int tid, int nt) {
  if (p == nullptr) return;
  for (int r = at.begin; r < at.end; ++r)
    for (int d = tid; d < dim; d += nt) p[r * row + head + d] = O(0.f);
}

// A chunk's rows of a result, as a buffer: stores need no branch, since what lies behind the last row, or at kNowhere, is dropped.
struct Rows {
  __amdgpu_buffer_rsrc_t r;
  int stride;                  // of a row, in values
};
constexpr int kNowhere = 0x7ffe0000;          // also with a state's bytes added
template <typename O> __device__ __forceinline__ Rows rows_at(O* p, int len, int stride, int dim) {
  return Rows{__builtin_amdgcn_make_buffer_rsrc(p, 0, len > 0 ? ((len - 1) * stride + dim) * int(sizeof(O)) : 0, 0x20000), stride};
}
template <typename O> __device__ __forceinline__ void put(const Rows& w, int row, int at, bool in, float x) {
  const int off = in ? (row * w.stride + at) * int(sizeof(O)) : kNowhere;
  if constexpr (sizeof(O) == 2)
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, O(x)), w.r, off, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), w.r, off, 0, 0);
}
template <typename O> __device__ __forceinline__ void put4(const Rows& w, int row, int at, bool in, float a, float b, float c, float d) {
  typedef O V4 __attribute__((ext_vector_type(4)));
  typedef uint32_t U2 __attribute__((ext_vector_type(2)));
  typedef uint32_t U4 __attribute__((ext_vector_type(4)));
  const int off = in ? (row * w.stride + at) * int(sizeof(O)) : kNowhere;
  const V4 v = {O(a), O(b), O(c), O(d)};
  if constexpr (sizeof(O) == 2)
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(U2, v), w.r, off, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(U4, v), w.r, off, 0, 0);
}

// Stores that are dropped, as many as follow a loop's loads each time round: the first wait for loads then counts what the others do.
template <int N> __device__ __forceinline__ void no_stores(void* p) {
  const Rows none = rows_at(static_cast<float*>(p), 0, 0, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) put<float>(none, 0, 0, false, 0.f);
}

// ---------------------------------------------------------------- inverses and scores of the chunks
__device__ __forceinline__ float finite_gate2(float g) { return (g < -150.f ? -150.f : g) * kLog2e; }      // -inf too; NaN stays

// Eight values of a row as an operand; `in`: else zeros.
template <typename T> __device__ __forceinline__ Split<DeltaParts<T>::kIn> row_parts(Frag<T> f, bool in) {
  if constexpr (sizeof(T) == 2) {
    uint4 w = __builtin_bit_cast(uint4, f);
    f = __builtin_bit_cast(Frag<T>, in ? w : make_uint4(0, 0, 0, 0));
  }
  if constexpr (std::is_same<T, __bf16>::value) {
    Split<1> s;
    s.p[0] = f;
    return s;
  }
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = sizeof(T) == 2 || in ? float(f[j]) : 0.f;
  return split<DeltaParts<T>::kIn>(x);
}

// A wave a (chunk, head). Lanes 0 .. 31 solve for the columns of (1 + L)^-1, the others for those of (1 + L')^-1.
template <typename T, int D>
__global__ __launch_bounds__(64, 4) void delta_prep(const DeltaArgs a) {
  constexpr int kMid = DeltaParts<T>::kMid, kPitch = C + 4;
  __shared__ __attribute__((aligned(16))) float l_lds[2][C][kPitch];       // L and L' by columns, then the inverses by rows
  __shared__ __attribute__((aligned(16))) double g_lds[C];
  __shared__ float beta_lds[C];
  const int lane = threadIdx.x, half = lane >> 5, col = lane & 31;
  const int64_t x = blockIdx.x / a.heads;
  const int h = int(blockIdx.x % a.heads);
  const Place at = find(a, x, C);
  if (at.none || at.seq >= a.n_seq || at.begin >= at.end) return;
  const int len = at.end - at.begin;
  const bool row_in = col < len;
  const int64_t row = at.begin + min(col, len - 1);
  // all loads at once, and without branches, which would wait for each by itself
  const T* kp = static_cast<const T*>(a.k) + row * a.ks_t + (h / a.group) * a.ks_h;
  const T* qp = static_cast<const T*>(a.q) + row * a.qs_t + (h / a.group) * a.qs_h;
  constexpr int kMost = std::is_same<T, __bf16>::value ? 8 : sizeof(T) == 2 ? 4 : 2, kAhead = D / 16 < kMost ? D / 16 : kMost;
  Frag<T> ks[kAhead], qs[kAhead];
  auto fetch = [&](int s) {
    const int from = min(16 * s + 8 * half, a.dim_k - 8);
    ks[s % kAhead] = *reinterpret_cast<const Frag<T>*>(kp + from);
    qs[s % kAhead] = *reinterpret_cast<const Frag<T>*>(qp + from);
  };
#pragma unroll
  for (int s = 0; s < kAhead; ++s) fetch(s);

  const float gate = a.log_gate[row * a.heads + h], strength = a.beta[row * a.heads + h];

  double g = row_in ? double(finite_gate2(gate)) : 0.0;
  for (int o = 1; o < C; o <<= 1) {
    const double up = __shfl_up(g, o, 32);
    if (col >= o) g += up;
  }
  const double all = __shfl(g, C - 1, 32);
  const float beta = row_in ? strength : 0.f;
  if (half == 0) {
    g_lds[col] = g;
    beta_lds[col] = beta;
    if (row_in) {
      a.g2[row * a.heads + h] = float(g);
      a.gin[row * a.heads + h] = exp2_fast(float(g));
      a.gout[row * a.heads + h] = exp2_fast(float(all - g));
    }
  }
  F32x16 kk = zero16(), kq = zero16(), qk = zero16();
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const bool in = row_in && 16 * s + 8 * half < a.dim_k;
    const auto k = row_parts<T>(ks[s % kAhead], in), q = row_parts<T>(qs[s % kAhead], in);
    if (s + kAhead < D / 16) fetch(s + kAhead);
    kk = mul(k, k, kk);
    kq = mul(k, q, kq);                          // lane: the row i, registers: the columns j
    if (a.score_t) qk = mul(q, k, qk);
  }
  __syncthreads();
  float p[16], pt[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int i = acc_row(r, half), j = col;     // of kk and qk: registers i, lane j; of kq the other way round
    const double gi = g_lds[i];
    const float ahead = exp2_fast(float(i >= j ? gi - g : g - gi));
    const float l = i > j ? kk[r] * ahead : 0.f;
    l_lds[0][j][i] = l * beta;
    l_lds[1][j][i] = l * beta_lds[i];
    p[r] = i <= j ? kq[r] * (a.scale * ahead) : 0.f;
    pt[r] = i >= j ? qk[r] * (a.scale * ahead) : 0.f;
  }
  __syncthreads();
  float t[C];
#pragma unroll
  for (int i = 0; i < C; ++i) t[i] = i == col ? 1.f : 0.f;
#pragma unroll
  for (int j = 0; j < C - 1; ++j) {
#pragma unroll
    for (int i0 = (j + 1) / 4 * 4; i0 < C; i0 += 4) {
      const float4 l = *reinterpret_cast<const float4*>(&l_lds[half][j][i0]);
      const float lv[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (i0 + n > j) t[i0 + n] = fmaf(-lv[n], t[j], t[i0 + n]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < C; ++i) l_lds[half][i][col] = t[i];
  __syncthreads();
  const int64_t slot = (x * a.heads + h) * (2 * kMid * 64) + lane;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = l_lds[0][col][16 * u + acc_row(j, half)];
    const Split<kMid> inv = split<kMid>(y), sc = split_regs<kMid>(p, u);
#pragma unroll
    for (int n = 0; n < kMid; ++n) {
      a.inv[slot + (u * kMid + n) * 64] = __builtin_bit_cast(uint4, inv.p[n]);
      a.score[slot + (u * kMid + n) * 64] = __builtin_bit_cast(uint4, sc.p[n]);
    }
    if (a.score_t) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = l_lds[1][16 * u + acc_row(j, half)][col];
      const Split<kMid> ti = split<kMid>(y), ts = split_regs<kMid>(pt, u);
#pragma unroll
      for (int n = 0; n < kMid; ++n) {
        a.inv_t[slot + (u * kMid + n) * 64] = __builtin_bit_cast(uint4, ti.p[n]);
        a.score_t[slot + (u * kMid + n) * 64] = __builtin_bit_cast(uint4, ts.p[n]);
      }
    }
  }
}

// A chunk's operand of two steps on its way from memory to LDS; all waves read it there. (A workgroup of one wave has it in its
// registers as it stands.)
template <int N, int NT> struct ChunkFrag {
  static constexpr int kAll = 2 * N * 64, kN = (kAll + NT - 1) / NT;
  uint4 r[kN];
  __device__ __forceinline__ void load(const uint4* p, int tid) {
#pragma unroll
    for (int i = 0; i < kN; ++i) r[i] = p[min(i * NT + tid, kAll - 1)];
  }
  __device__ __forceinline__ void store(uint4* lds, int tid) const {
    if constexpr (NT == 64) return;
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (kAll % NT == 0 || i * NT + tid < kAll) lds[i * NT + tid] = r[i];
  }
  __device__ __forceinline__ Split<N> get(const uint4* lds, int u, int lane) const {
    Split<N> s;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if constexpr (NT == 64)
        s.p[n] = __builtin_bit_cast(BFrag, r[u * N + n]);
      else
        s.p[n] = __builtin_bit_cast(BFrag, lds[(u * N + n) * 64 + lane]);
    }
    return s;
  }
};

// Four tokens' scalars, of registers 4g .. 4g + 3.
__device__ __forceinline__ void four_of(const float* lds, int g, int half, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(lds + 8 * g + 4 * half);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}

// x[r] *= lds[token of register r]
__device__ __forceinline__ void by_token(float (&x)[16], const float* lds, int half) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float w[4];
    four_of(lds, g, half, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[4 * g + j] *= w[j];
  }
}

// A state's block of 32 rows, row-major [dk, dv] float32 in memory: register r row 32 b + acc_row(r, half), lane the column.
// (A state has at most 2^14 values. `fresh`: the addresses are formed where they are used, and not kept through a loop.)
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
// Rows 32 b .. 32 b + 31 of a state, a lane column z: as a buffer without branches, since what lies outside of it (of NULL all) reads 0 and
// is not written. The state's address is one for the workgroup.
__device__ __forceinline__ void load_state(F32x16& m, const float* s, int b, int z, int half, int dk, int dv) {
  const auto from = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(s), 0, s ? dk * dv * 4 : 0, 0x20000);
  const int at = fresh(z < dv ? ((32 * b + 4 * half) * dv + z) * 4 : kNowhere);
#pragma unroll
  for (int r = 0; r < 16; ++r) m[r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(from, at + acc_row(r, 0) * dv * 4, 0, 0));
}
__device__ __forceinline__ void store_state(const F32x16& m, float* s, int b, int z, int half, int dk, int dv) {
  const auto to = __builtin_amdgcn_make_buffer_rsrc(s, 0, dk * dv * 4, 0x20000);
  const int at = fresh(z < dv ? ((32 * b + 4 * half) * dv + z) * 4 : kNowhere);
#pragma unroll
  for (int r = 0; r < 16; ++r) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(m[r]), to, at + acc_row(r, 0) * dv * 4, 0, 0);
}

// An infinity or NaN among a wave's values by token is the tokens' from its own on, not the ones before, which a product with the
// inverse's (or P's) zeros would make NaN as well: there the finite values are multiplied, and a product of marks tells the
// tokens that follow.
__device__ __forceinline__ bool odd_values(const float (&x)[16]) {
  float odd = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) odd = fmaf(x[r], 0.f, odd);
  return __any(odd != odd);
}
template <int N> struct Marked {
  Split<N> finite;
  BFrag odd, up;           // 1 where a value is not finite; 1 for the tokens up to the lane's
};
template <int N> __device__ __forceinline__ Marked<N> marked(const float (&x)[16], int t, int half, int col) {
  Marked<N> m;
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool fin = fabsf(x[8 * t + j]) < INFINITY;
    y[j] = fin ? x[8 * t + j] : 0.f;
    m.odd[j] = __bf16(fin ? 0.f : 1.f);
    m.up[j] = __bf16(16 * t + acc_row(j, half) <= col ? 1.f : 0.f);
  }
  m.finite = split<N>(y);
  return m;
}

// ---------------------------------------------------------------- the forward pass over a segment
// A wave owns 32 columns of the state (a lane one, its rows in registers). kMaps: the waves behind those of the values' columns
// own M's.
template <typename T, int D, int MODE>
__global__ __launch_bounds__((MODE == kMaps ? 4 : 2) * D, sizeof(T) == 2 || (MODE == kMaps && D == 128) ? 2 : 1) void delta_pass(const DeltaArgs a) {
  constexpr int NW = D / 32 * (MODE == kMaps ? 2 : 1), NT = 64 * NW, XB = D / 32;
  constexpr int kIn = DeltaParts<T>::kIn, kMid = DeltaParts<T>::kMid;
  constexpr bool OUT = MODE != kMaps;
  using PX = PartTile<kIn, D>;
  using TZ = Tile<T, D>;
  __shared__ __attribute__((aligned(16))) char k_lds[PX::kBytes];
  __shared__ __attribute__((aligned(16))) char q_lds[OUT ? PX::kBytes : 16];
  __shared__ __attribute__((aligned(16))) char v_lds[TZ::bytes(C)];
  __shared__ uint4 inv_lds[NT > 64 ? 2 * kMid * 64 : 1], sc_lds[OUT && NT > 64 ? 2 * kMid * 64 : 1];
  __shared__ __attribute__((aligned(16))) float gin_lds[C], gout_lds[C], beta_lds[C];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
  const int64_t slot = blockIdx.x, x = slot / a.heads;
  const int h = int(slot % a.heads);
  const Place at = find(a, x, C * a.seg_chunks);
  if (at.none) return;
  if (at.seq >= a.n_seq) {
    if (OUT) clear_rows(static_cast<T*>(a.out), at, int64_t(a.heads) * a.dim_v, int64_t(h) * a.dim_v, a.dim_v, tid, NT);
    return;
  }
  const bool last = at.end == at.seq_end;
  if (MODE == kMaps && last) return;             // nothing follows
  const bool own = MODE != kMaps || wave < XB;   // columns of the values, not of M
  const int z = 32 * (wave % XB) + col;
  const int64_t per = int64_t(a.dim_k) * a.dim_v, sx = x * a.heads + h;

  F32x16 m[XB];
  if constexpr (MODE == kMaps) {
#pragma unroll
    for (int b = 0; b < XB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) m[b][r] = !own && 32 * b + acc_row(r, half) == z ? 1.f : 0.f;
  } else {
    const float* s0 = a.carried ? a.state + sx * per : a.init ? a.init + (int64_t(at.seq) * a.heads + h) * per : nullptr;
#pragma unroll
    for (int b = 0; b < XB; ++b) load_state(m[b], s0, b, z, half, a.dim_k, a.dim_v);
  }

  const T* kp = static_cast<const T*>(a.k) + (h / a.group) * a.ks_h;
  const T* qp = static_cast<const T*>(a.q) + (h / a.group) * a.qs_h;
  const T* vp = static_cast<const T*>(a.v) + h * a.vs_h;
  const int64_t c0 = chunk_place(a, at, at.begin);
  Stage<T, D, C, NT> ks, qs, vs;
  ChunkFrag<kMid, NT> inv, sc;
  float gi = 0.f, go = 0.f, be = 0.f;
  auto fetch = [&](int t0) {
    const int n = min(C, at.end - t0);
    ks.load(tid, n, a.dim_k, [&](int r) { return kp + int64_t(t0 + r) * a.ks_t; });
    if constexpr (OUT) qs.load(tid, n, a.dim_k, [&](int r) { return qp + int64_t(t0 + r) * a.qs_t; });
    vs.load(tid, n, a.dim_v, [&](int r) { return vp + int64_t(t0 + r) * a.vs_t; });
    const int64_t i = int64_t(t0 + min(tid & (C - 1), n - 1)) * a.heads + h;      // all waves: no branch between loads
    gi = a.gin[i], go = a.gout[i], be = a.beta[i];
    const int64_t c = ((c0 + (t0 - at.begin) / C) * a.heads + h) * (2 * kMid * 64);
    inv.load(a.inv + c, tid);
    if constexpr (OUT) sc.load(a.score + c, tid);
  };
  if (at.begin < at.end) fetch(at.begin);
  if constexpr (OUT) no_stores<MODE == kTrain ? 20 : 4>(a.out);
  for (int t0 = at.begin; t0 < at.end; t0 += C) {
    const int len = min(C, at.end - t0);
    ks.clip(tid, len, a.dim_k);
    if constexpr (OUT) qs.clip(tid, len, a.dim_k);
    vs.clip(tid, len, a.dim_v);
    __syncthreads();
    store_parts<kIn>(ks, tid, k_lds);
    if constexpr (OUT) store_parts<kIn>(qs, tid, q_lds);
    vs.store(tid, v_lds);
    inv.store(inv_lds, tid);
    if constexpr (OUT) sc.store(sc_lds, tid);
    const ChunkFrag<kMid, NT> now = inv, scn = sc;
    if (tid < C) gin_lds[tid] = gi, gout_lds[tid] = go, beta_lds[tid] = tid < len ? be : 0.f;
    __syncthreads();
    if (t0 + C < at.end) fetch(t0 + C);

    const float whole = gin_lds[C - 1];          // the last token's, where there are fewer
    F32x16 ksum = zero16(), o = zero16();
#pragma unroll
    for (int b = 0; b < XB; ++b)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Split<kMid> s = split_regs<kMid>(m[b], t);
        ksum = mul(PX::rows_regs(k_lds, col, 2 * b + t, half), s, ksum);
        if constexpr (OUT) o = mul(s, PX::rows_regs(q_lds, col, 2 * b + t, half), o);
      }
    float w[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = ksum[r];
    by_token(w, gin_lds, half);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Frag<T> f = TZ::template col_frag<true>(v_lds, t, wave % XB, lane);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[8 * t + j] = (own ? float(f[j]) : 0.f) - w[8 * t + j];
    }
    F32x16 e = zero16();
    if (!odd_values(w)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) e = mul(now.get(inv_lds, t, lane), split_regs<kMid>(w, t), e);
    } else {
      F32x16 seen = zero16();
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Marked<kMid> y = marked<kMid>(w, t, half, col);
        e = mul(now.get(inv_lds, t, lane), y.finite, e);
        seen = Mat<__bf16>::mma(y.up, y.odd, seen);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (seen[r] > 0.f) e[r] = NAN;
    }
    float u[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) u[r] = e[r];
    if constexpr (MODE == kTrain) {
      const Rows to = rows_at(a.e + (int64_t(t0) * a.heads + h) * a.dim_v, len, a.heads * a.dim_v, a.dim_v);
#pragma unroll
      for (int r = 0; r < 16; ++r) put<float>(to, acc_row(r, half), z, z < a.dim_v, e[r]);
    }
    by_token(u, beta_lds, half);
    if constexpr (OUT) {
      const float f = a.scale * gin_lds[col];
#pragma unroll
      for (int r = 0; r < 16; ++r) o[r] *= f;
      if (!odd_values(u)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) o = mul(split_regs<kMid>(u, t), scn.get(sc_lds, t, lane), o);
      } else {
        F32x16 seen = zero16();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const Marked<kMid> y = marked<kMid>(u, t, half, col);
          o = mul(y.finite, scn.get(sc_lds, t, lane), o);
          seen = Mat<__bf16>::mma(y.odd, y.up, seen);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (seen[r] > 0.f) o[r] = NAN;
      }
      const Rows to = rows_at(static_cast<T*>(a.out) + (int64_t(t0) * a.heads + h) * a.dim_v, len, a.heads * a.dim_v, a.dim_v);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * wave + 8 * g + 4 * half;
        put4<T>(to, col, d, d < a.dim_v, o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
      }
    }
    by_token(u, gout_lds, half);
#pragma unroll
    for (int b = 0; b < XB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) m[b][r] *= whole;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Split<kMid> s = split_regs<kMid>(u, t);
#pragma unroll
      for (int b = 0; b < XB; ++b) m[b] = mul(PX::cols(k_lds, t, b, lane), s, m[b]);
    }
  }
  if constexpr (MODE == kMaps) {
    if (own) {
#pragma unroll
      for (int b = 0; b < XB; ++b) store_state(m[b], a.state + sx * per, b, z, half, a.dim_k, a.dim_v);
    }
    __syncthreads();                             // the tile of keys is no longer read
    if (!own) {                                  // M as the carries' operands, by blocks of its rows and steps over its columns
      const int w = wave % XB;
      uint4* mf = a.map_f + sx * (kMid * D * D / 8) + lane;
      uint4* mb = a.map_b ? a.map_b + sx * (kMid * D * D / 8) + lane : nullptr;
      __bf16* mine = reinterpret_cast<__bf16*>(k_lds) + w * 1024;          // a 32 x 32 block, the wave's own
#pragma unroll
      for (int b = 0; b < XB; ++b) {
        Split<kMid> s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          s[t] = split_regs<kMid>(m[b], t);
          if (mb) {                              // M^T's rows are the lanes' columns: as the registers stand
#pragma unroll
            for (int n = 0; n < kMid; ++n) mb[((w * 2 * XB + 2 * b + t) * kMid + n) * 64] = __builtin_bit_cast(uint4, s[t].p[n]);
          }
        }
#pragma unroll
        for (int n = 0; n < kMid; ++n) {
#pragma unroll
          for (int r = 0; r < 16; ++r) mine[acc_row(r, half) * 32 + col] = s[r / 8].p[n][r % 8];
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const uint2 lo = *reinterpret_cast<const uint2*>(mine + col * 32 + 16 * t + 4 * half);
            const uint2 hi = *reinterpret_cast<const uint2*>(mine + col * 32 + 16 * t + 8 + 4 * half);
            mf[((b * 2 * XB + 2 * w + t) * kMid + n) * 64] = make_uint4(lo.x, lo.y, hi.x, hi.y);
          }
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
  } else if (last && a.final_state) {
    float* fs = a.final_state + (int64_t(at.seq) * a.heads + h) * per;
#pragma unroll
    for (int b = 0; b < XB; ++b) store_state(m[b], fs, b, z, half, a.dim_k, a.dim_v);
  }
}

// Sequences that the carry takes at once: of some thousand workgroups at most, which take several each.
__host__ __device__ inline int carry_seqs(const DeltaArgs& a) {
  const int seqs = 1 + 2048 / a.heads;
  return seqs < a.n_seq ? seqs : a.n_seq;
}

// ---------------------------------------------------------------- states from segment to segment
// A workgroup 32 columns of a (sequence, head)'s state: wave b forms rows 32 b of M S + B. Its rows of M and of B are on their way
// two segments ahead; the blocks of S pass through LDS as operands. BACK: from the last segment, with M^T. The workgroups of one
// state are 8 apart: on one XCD, whose L2 then holds M for all of them.
template <typename T, int D, bool BACK>
__global__ __launch_bounds__(2 * D) void delta_carry(const DeltaArgs a) {
  constexpr int XB = D / 32, kMid = DeltaParts<T>::kMid, kSteps = 2 * XB;
  __shared__ uint4 s_lds[2][kSteps][kMid][64];
  const int tid = threadIdx.x, lane = tid & 63, b = tid >> 6, half = lane >> 5, col = lane & 31;
  const int z = 32 * int(blockIdx.x / 8 % XB) + col;
  const int64_t unit = int64_t(blockIdx.x / (8 * XB)) * 8 + blockIdx.x % 8;
  const int step_seqs = carry_seqs(a), h = int(unit % a.heads);
  if (unit >= int64_t(step_seqs) * a.heads) return;
  const int64_t per = int64_t(a.dim_k) * a.dim_v;
  const int seg = C * a.seg_chunks;
  for (int64_t seq = unit / a.heads; seq < a.n_seq; seq += step_seqs) {
    const int from = clamped(a, seq), to = max(clamped(a, seq + 1), from);
    const int64_t x0 = from / seg + seq;
    const int n = max((to - from + seg - 1) / seg, 1);
    auto place_of = [&](int k) { return (x0 + (BACK ? n - 1 - k : k)) * a.heads + h; };
    float* states = BACK ? a.dstate : a.state;
    const uint4* maps = (BACK ? a.map_b : a.map_f) + b * kSteps * kMid * 64 + lane;
    // The last segment visited hands nothing on. What is on its way is counted by the waits only without branches around loads and stores,
    // so those behind the last segment read it again.
    struct Ahead {
      uint4 map[kSteps][kMid];
      F32x16 part;
    } ahead[2];
    auto fetch = [&](int k, Ahead& to) {
      const int64_t sx = place_of(k < n ? k : n - 1);
      load_state(to.part, states + sx * per, b, z, half, a.dim_k, a.dim_v);
      const uint4* p = maps + sx * (kMid * D * D / 8);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int x = 0; x < kMid; ++x) to.map[s][x] = p[(s * kMid + x) * 64];
    };
    F32x16 m;
    load_state(m, !BACK && a.init ? a.init + (seq * a.heads + h) * per : nullptr, b, z, half, a.dim_k, a.dim_v);
    auto step = [&](int k, Ahead& mine) {
      store_state(m, states + place_of(k) * per, b, z, half, a.dim_k, a.dim_v);
      F32x16 sum = zero16();
      uint4(*lds)[kMid][64] = s_lds[k & 1];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Split<kMid> s = split_regs<kMid>(m, t);
#pragma unroll
        for (int p = 0; p < kMid; ++p) lds[2 * b + t][p][lane] = __builtin_bit_cast(uint4, s.p[p]);
      }
      __syncthreads();                           // one a segment: the other half of s_lds is written next
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        Split<kMid> f, g;
#pragma unroll
        for (int p = 0; p < kMid; ++p) f.p[p] = __builtin_bit_cast(BFrag, mine.map[s][p]), g.p[p] = __builtin_bit_cast(BFrag, lds[s][p][lane]);
        sum = mul(f, g, sum);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) m[r] = sum[r] + mine.part[r];       // not as what is added to: the registers would change their roles
      fetch(k + 2, mine);
      __builtin_amdgcn_sched_barrier(0);
    };
    int k = 0;
    if (BACK && n > 1) {                         // the last segment begins from 0: no map
      F32x16 part;
      load_state(part, states + place_of(0) * per, b, z, half, a.dim_k, a.dim_v);
      store_state(m, states + place_of(0) * per, b, z, half, a.dim_k, a.dim_v);
      m = part;
      k = 1;
    }
    if (k + 1 < n) {
      fetch(k, ahead[0]);
      fetch(k + 1, ahead[1]);
      for (;;) {
        step(k, ahead[0]);
        if (++k + 1 >= n) break;
        step(k, ahead[1]);
        if (++k + 1 >= n) break;
      }
    }
    store_state(m, states + place_of(k) * per, b, z, half, a.dim_k, a.dim_v);
    __syncthreads();
  }
}

// ---------------------------------------------------------------- the backward pass over a segment: z, dv
template <typename T, int D, int MODE>
__global__ __launch_bounds__(2 * D, sizeof(T) == 2 ? 2 : 1) void delta_back(const DeltaArgs a) {
  constexpr int NW = D / 32, NT = 64 * NW, XB = D / 32;
  constexpr int kIn = DeltaParts<T>::kIn, kMid = DeltaParts<T>::kMid;
  using PX = PartTile<kIn, D>;
  using TZ = Tile<T, D>;
  __shared__ __attribute__((aligned(16))) char k_lds[PX::kBytes];
  __shared__ __attribute__((aligned(16))) char q_lds[PX::kBytes];
  __shared__ __attribute__((aligned(16))) char g_lds[TZ::bytes(C)];
  __shared__ uint4 inv_lds[NT > 64 ? 2 * kMid * 64 : 1], sc_lds[NT > 64 ? 2 * kMid * 64 : 1];
  __shared__ __attribute__((aligned(16))) float gin_lds[C], gout_lds[C], beta_lds[C];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
  const int64_t slot = blockIdx.x, x = slot / a.heads;
  const int h = int(slot % a.heads);
  const Place at = find(a, x, C * a.seg_chunks);
  if (at.none) return;
  if (at.seq >= a.n_seq) {
    if (MODE == kBack) clear_rows(static_cast<T*>(a.dv), at, int64_t(a.heads) * a.dim_v, int64_t(h) * a.dim_v, a.dim_v, tid, NT);
    return;
  }
  if (MODE == kBackMaps && at.idx == 0) return;       // nothing goes before
  const int z = 32 * wave + col;
  const int64_t per = int64_t(a.dim_k) * a.dim_v, sx = x * a.heads + h;
  F32x16 m[XB];
#pragma unroll
  for (int b = 0; b < XB; ++b)
    load_state(m[b], MODE == kBack && a.carried ? a.dstate + sx * per : nullptr, b, z, half, a.dim_k, a.dim_v);

  const T* kp = static_cast<const T*>(a.k) + (h / a.group) * a.ks_h;
  const T* qp = static_cast<const T*>(a.q) + (h / a.group) * a.qs_h;
  const T* gp = static_cast<const T*>(a.dout) + int64_t(h) * a.dim_v;
  const int64_t c0 = chunk_place(a, at, at.begin), gs_t = int64_t(a.heads) * a.dim_v;
  Stage<T, D, C, NT> ks, qs, gs;
  ChunkFrag<kMid, NT> inv, sc;
  float gi = 0.f, go = 0.f, be = 0.f;
  auto fetch = [&](int t0) {
    const int n = min(C, at.end - t0);
    ks.load(tid, n, a.dim_k, [&](int r) { return kp + int64_t(t0 + r) * a.ks_t; });
    qs.load(tid, n, a.dim_k, [&](int r) { return qp + int64_t(t0 + r) * a.qs_t; });
    gs.load(tid, n, a.dim_v, [&](int r) { return gp + int64_t(t0 + r) * gs_t; });
    const int64_t i = int64_t(t0 + min(tid & (C - 1), n - 1)) * a.heads + h;      // all waves: no branch between loads
    gi = a.gin[i], go = a.gout[i], be = a.beta[i];
    const int64_t c = ((c0 + (t0 - at.begin) / C) * a.heads + h) * (2 * kMid * 64);
    inv.load(a.inv_t + c, tid);
    sc.load(a.score_t + c, tid);
  };
  const int chunks = (at.end - at.begin + C - 1) / C;
  if (chunks > 0) fetch(at.begin + (chunks - 1) * C);
  if constexpr (MODE == kBack) no_stores<32>(a.dv);
  for (int c = chunks - 1; c >= 0; --c) {
    const int t0 = at.begin + c * C, len = min(C, at.end - t0);
    ks.clip(tid, len, a.dim_k);
    qs.clip(tid, len, a.dim_k);
    gs.clip(tid, len, a.dim_v);
    __syncthreads();
    store_parts<kIn>(ks, tid, k_lds);
    store_parts<kIn>(qs, tid, q_lds);
    gs.store(tid, g_lds);
    inv.store(inv_lds, tid);
    sc.store(sc_lds, tid);
    const ChunkFrag<kMid, NT> now = inv, scn = sc;
    if (tid < C) gin_lds[tid] = gi, gout_lds[tid] = go, beta_lds[tid] = tid < len ? be : 0.f;
    __syncthreads();
    if (c > 0) fetch(t0 - C);

    const float whole = gin_lds[C - 1];
    F32x16 ksum = zero16();
#pragma unroll
    for (int b = 0; b < XB; ++b)
#pragma unroll
      for (int t = 0; t < 2; ++t) ksum = mul(PX::rows_regs(k_lds, col, 2 * b + t, half), split_regs<kMid>(m[b], t), ksum);
    float w[16], g[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = ksum[r];
    by_token(w, gout_lds, half);
    F32x16 du;
#pragma unroll
    for (int r = 0; r < 16; ++r) du[r] = w[r];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Frag<T> f = TZ::template col_frag<true>(g_lds, t, wave, lane);
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) g[8 * t + j] = y[j] = float(f[j]);
      du = mul(scn.get(sc_lds, t, lane), split<kIn>(y), du);
    }
    F32x16 zz = zero16();
#pragma unroll
    for (int t = 0; t < 2; ++t) zz = mul(now.get(inv_lds, t, lane), split_regs<kMid>(du, t), zz);
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = zz[r];
    by_token(w, beta_lds, half);
    if constexpr (MODE == kBack) {
      const int64_t o = (int64_t(t0) * a.heads + h) * a.dim_v;
      const Rows to_z = rows_at(a.z + o, len, a.heads * a.dim_v, a.dim_v);
      const Rows to_v = rows_at(static_cast<T*>(a.dv) + o, len, a.heads * a.dim_v, a.dim_v);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        put<float>(to_z, acc_row(r, half), z, z < a.dim_v, zz[r]);
        put<T>(to_v, acc_row(r, half), z, z < a.dim_v, w[r]);
      }
    }
    if (MODE == kBack && c == 0) break;            // nobody reads the state's gradient before the segment
    by_token(w, gin_lds, half);
    by_token(g, gin_lds, half);
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = -w[r], g[r] *= a.scale;
#pragma unroll
    for (int b = 0; b < XB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) m[b][r] *= whole;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Split<kMid> ws = split_regs<kMid>(w, t), ys = split_regs<kMid>(g, t);
#pragma unroll
      for (int b = 0; b < XB; ++b) {
        m[b] = mul(PX::cols(k_lds, t, b, lane), ws, m[b]);
        m[b] = mul(PX::cols(q_lds, t, b, lane), ys, m[b]);
      }
    }
  }
  if (MODE == kBackMaps) {
#pragma unroll
    for (int b = 0; b < XB; ++b) store_state(m[b], a.dstate + sx * per, b, z, half, a.dim_k, a.dim_v);
  }
}

template <int CTRL> __device__ __forceinline__ float add_lane(float x) {
  return x + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
// The sum of N lanes beside each other (8, 16 or 32), in all of them: by rows of 16 without LDS.
template <int N> __device__ __forceinline__ float add_neighbours(float x) {
  static_assert(N == 8 || N == 16 || N == 32, "lanes");
  x = add_lane<0xb1>(x);                         // the other of a pair
  x = add_lane<0x4e>(x);                         // the other pair of four
  x = add_lane<0x141>(x);                        // the other four of eight, mirrored
  if constexpr (N > 8) x = add_lane<0x140>(x);   // the other eight of a row
  if constexpr (N > 16) x += __shfl_xor(x, 16, 64);
  return x;
}

// ---------------------------------------------------------------- gradients of q and k, of gates and strengths
// Passes of linear attention over a segment, with the state transposed: a wave owns 32 of the keys' values (a lane one), the rows of
// its columns are the values' values. BACK false: dq, dk' and db from the state before the segment on; true: dk", and from all of
// them the gates', from the gradient behind the segment back.
template <typename T, int D, bool BACK>
__global__ __launch_bounds__(2 * D, sizeof(T) == 2 && (DeltaParts<T>::kIn == 1 || D < 128) ? 2 : 1) void delta_grad(const DeltaArgs a) {
  constexpr int NW = D / 32, NT = 64 * NW, XB = D / 32;
  constexpr int kIn = DeltaParts<T>::kIn, kMid = DeltaParts<T>::kMid;
  // The gates' gradient is a sum of differences that nearly cancel, of what follows from these operands, so they keep a part more than
  // elsewhere; they are registers only. 17.5K tokens, 8 heads of 64, float16, in segments of 6: dlog_gate 6e-6 off instead of 3e-5, both
  // passes 162 us instead of 147 (5.9K tokens, 16 heads of 128, bfloat16, segments of 8: 260 instead of 226). With u and z in three parts
  // too: 5e-6, and 212 (371), by their LDS.
  constexpr int kFine = 3;
  using PX = PartTile<kIn, D>;
  using PM = PartTile<kMid, D>;
  __shared__ __attribute__((aligned(16))) char k_lds[PX::kBytes];
  __shared__ __attribute__((aligned(16))) char q_lds[PX::kBytes];
  __shared__ __attribute__((aligned(16))) char g_lds[PX::kBytes];
  __shared__ __attribute__((aligned(16))) char u_lds[PM::kBytes];       // b e
  __shared__ __attribute__((aligned(16))) char z_lds[PM::kBytes];
  __shared__ __attribute__((aligned(16))) float gin_lds[C], gout_lds[C], beta_lds[C], g2_lds[C];
  __shared__ float sum_lds[NW][C];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
  const int64_t slot = blockIdx.x, x = slot / a.heads;
  const int h = int(slot % a.heads);
  const Place at = find(a, x, C * a.seg_chunks);
  if (at.none) return;
  const int64_t row_v = int64_t(a.heads) * a.dim_v, row_k = int64_t(a.heads) * a.dim_k;
  T* dq_out = a.dq32 ? nullptr : static_cast<T*>(a.dq);
  T* dk_out = a.dq32 ? nullptr : static_cast<T*>(a.dk);
  if (at.seq >= a.n_seq) {
    if (!BACK) {
      clear_rows(dq_out, at, row_k, int64_t(h) * a.dim_k, a.dim_k, tid, NT);
      clear_rows(a.dq32, at, row_k, int64_t(h) * a.dim_k, a.dim_k, tid, NT);
      clear_rows(a.dbeta, at, a.heads, h, 1, tid, NT);
    } else {
      clear_rows(dk_out, at, row_k, int64_t(h) * a.dim_k, a.dim_k, tid, NT);
      if (a.dq32) clear_rows(a.dk32, at, row_k, int64_t(h) * a.dim_k, a.dim_k, tid, NT);
      clear_rows(a.dgate, at, a.heads, h, 1, tid, NT);
    }
    return;
  }
  const int64_t per = int64_t(a.dim_k) * a.dim_v, sx = x * a.heads + h;
  const int kd = 32 * wave + col;                // the lane's value of a key
  const bool last = at.end == at.seq_end;
  // the transposed state: rows dv, four in a row of memory
  const float* s0 = BACK ? (a.carried && !last ? a.dstate + sx * per : nullptr)
                         : a.carried ? a.state + sx * per : a.init ? a.init + (int64_t(at.seq) * a.heads + h) * per : nullptr;
  const float* s1 = BACK && s0 ? a.state + (sx + a.heads) * per : nullptr;      // the state behind the segment
  F32x16 m[XB];
  float running = 0.f;
#pragma unroll
  for (int b = 0; b < XB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * b + 8 * g + 4 * half;
      const bool in = s0 && kd < a.dim_k && d < a.dim_v;
      const float4 v = in ? *reinterpret_cast<const float4*>(s0 + int64_t(kd) * a.dim_v + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      m[b][4 * g] = v.x, m[b][4 * g + 1] = v.y, m[b][4 * g + 2] = v.z, m[b][4 * g + 3] = v.w;
      if (BACK && in) {
        const float4 y = *reinterpret_cast<const float4*>(s1 + int64_t(kd) * a.dim_v + d);
        running += v.x * y.x + v.y * y.y + v.z * y.z + v.w * y.w;
      }
    }
  if constexpr (BACK) {
    for (int o = 32; o; o >>= 1) running += __shfl_xor(running, o, 64);
    if (lane == 0) sum_lds[wave][0] = running;
    __syncthreads();
    running = 0.f;
    for (int w = 0; w < NW; ++w) running += sum_lds[w][0];
  }

  const T* kp = static_cast<const T*>(a.k) + (h / a.group) * a.ks_h;
  const T* qp = static_cast<const T*>(a.q) + (h / a.group) * a.qs_h;
  const T* gp = static_cast<const T*>(a.dout) + int64_t(h) * a.dim_v;
  const float* ep = a.e + int64_t(h) * a.dim_v;
  const float* zp = a.z + int64_t(h) * a.dim_v;
  Stage<T, D, C, NT> ks, qs, gs;
  Stage<float, D, C, NT> es, zs;
  float gi = 0.f, go = 0.f, be = 0.f, g2 = 0.f;
  auto fetch = [&](int t0) {
    const int n = min(C, at.end - t0), tid = D > 32 ? fresh(threadIdx.x) : threadIdx.x;
    ks.load(tid, n, a.dim_k, [&](int r) { return kp + int64_t(t0 + r) * a.ks_t; });
    qs.load(tid, n, a.dim_k, [&](int r) { return qp + int64_t(t0 + r) * a.qs_t; });
    gs.load(tid, n, a.dim_v, [&](int r) { return gp + int64_t(t0 + r) * row_v; });
    es.load(tid, n, a.dim_v, [&](int r) { return ep + int64_t(t0 + r) * row_v; });
    zs.load(tid, n, a.dim_v, [&](int r) { return zp + int64_t(t0 + r) * row_v; });
    const int64_t i = int64_t(t0 + min(tid & (C - 1), n - 1)) * a.heads + h;
    gi = a.gin[i], go = a.gout[i], be = a.beta[i], g2 = a.g2[i];
  };
  const int chunks = (at.end - at.begin + C - 1) / C;
  auto begin_of = [&](int c) { return at.begin + (BACK ? chunks - 1 - c : c) * C; };
  if (chunks > 0) fetch(begin_of(0));
  for (int c = 0; c < chunks; ++c) {
    const int t0 = begin_of(c), len = min(C, at.end - t0);
    // formed anew each time round for wide heads: the addresses of all tiles, kept through the loop, do not fit the registers
    const int tid = D > 32 ? fresh(threadIdx.x) : threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
    ks.clip(tid, len, a.dim_k);
    qs.clip(tid, len, a.dim_k);
    gs.clip(tid, len, a.dim_v);
    es.clip(tid, len, a.dim_v);
    zs.clip(tid, len, a.dim_v);
    __syncthreads();
    if (tid < C) gin_lds[tid] = gi, gout_lds[tid] = go, beta_lds[tid] = tid < len ? be : 0.f, g2_lds[tid] = g2;
    store_parts<kIn>(ks, tid, k_lds);
    store_parts<kIn>(qs, tid, q_lds);
    store_parts<kIn>(gs, tid, g_lds);
    store_parts<kMid>(zs, tid, z_lds);
    if constexpr (!BACK) {                       // db: a row's chunks are neighbouring lanes
      using S = Stage<float, D, C, NT>;
      const Rows to = rows_at(a.dbeta + int64_t(t0) * a.heads + h, len, a.heads, 1);
#pragma unroll
      for (int i = 0; i < S::kN; ++i) {
        const float4 y = __builtin_bit_cast(float4, es.r[i]), w = __builtin_bit_cast(float4, zs.r[i]);
        float s = y.x * w.x + y.y * w.y + y.z * w.z + y.w * w.w;
        s = add_neighbours<S::kChunks>(s);
        const int n = i * NT + tid;
        put<float>(to, n / S::kChunks, 0, n % S::kChunks == 0, s);
      }
    }
    __syncthreads();
    store_parts<kMid>(es, tid, u_lds, [&](int r) { return beta_lds[r]; });
    __syncthreads();

    const float whole = gin_lds[C - 1];
    // products of the chunk's rows with each other: the lane's token against the registers'
    F32x16 fa = zero16(), ea = zero16();
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const Split<kMid> us = PM::rows(u_lds, col, s, half), zr = PM::rows(z_lds, col, s, half);
      const Split<kIn> gr = PX::rows(g_lds, col, s, half);
      if constexpr (BACK) {
        fa = mul(gr, us, fa);
        ea = mul(zr, us, ea);
      } else {
        fa = mul(us, gr, fa);
        ea = mul(us, zr, ea);
      }
    }
    float f[16], ee[16];
    const float mine = g2_lds[col], beta = beta_lds[col];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float other[4], bo[4];
      four_of(g2_lds, g, half, other);
      four_of(beta_lds, g, half, bo);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * g + j, i = acc_row(r, half);                // BACK: the reader i in the registers, the writer in the lane
        const bool sees = BACK ? i >= col : i <= col;
        const float d = exp2_fast(BACK ? other[j] - mine : mine - other[j]);
        f[r] = sees ? fa[r] * (a.scale * d) : 0.f;
        ee[r] = sees && i != col ? -ea[r] * d * (BACK ? bo[j] : beta) : 0.f;
      }
    }
    F32x16 o1 = zero16(), o2 = zero16();
#pragma unroll
    for (int b = 0; b < XB; ++b)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Split<kFine> s = split_regs<kFine>(m[b], t);
        if constexpr (BACK) {
          o1 = mul(s, PM::rows_regs(u_lds, col, 2 * b + t, half), o1);
        } else {
          o1 = mul(s, PX::rows_regs(g_lds, col, 2 * b + t, half), o1);
          o2 = mul(s, PM::rows_regs(z_lds, col, 2 * b + t, half), o2);
        }
      }
    // what the other pass found, on its way while the products are formed
    float before = 0.f;
    float4 other_k[4];
    if constexpr (BACK) {
      const int64_t row = t0 + min(col, len - 1);
      before = a.dgate[row * a.heads + h];
      const float* from = a.dk32 + (row * a.heads + h) * a.dim_k;
#pragma unroll
      for (int g = 0; g < 4; ++g) other_k[g] = *reinterpret_cast<const float4*>(from + min(32 * wave + 8 * g + 4 * half, a.dim_k - 4));
    }
    const float by1 = BACK ? gout_lds[col] : a.scale * gin_lds[col], by2 = -beta * gin_lds[col];
#pragma unroll
    for (int r = 0; r < 16; ++r) o1[r] *= by1, o2[r] *= by2;
    Split<kIn> kc[2], qc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      kc[t] = PX::cols(k_lds, t, wave, lane);
      if constexpr (BACK) {
        qc[t] = PX::cols(q_lds, t, wave, lane);
        o1 = mul(qc[t], split_regs<kFine>(f, t), o1);
        o1 = mul(kc[t], split_regs<kFine>(ee, t), o1);
      } else {
        o1 = mul(kc[t], split_regs<kFine>(f, t), o1);
        o2 = mul(kc[t], split_regs<kFine>(ee, t), o2);
      }
    }
    // results: a lane has a token's values 32 wave + 8 g + 4 half + (0 .. 3)
    const int64_t at0 = int64_t(t0) * row_k + int64_t(h) * a.dim_k;
    // with value heads that share a key head the sums over them follow
    const Rows wide = rows_at((BACK || !a.dq32 ? a.dk32 : a.dq32) + at0, a.dq32 ? len : 0, int(row_k), a.dq32 ? a.dim_k : 0);
    const Rows narrow = rows_at((BACK ? static_cast<T*>(a.dk) : static_cast<T*>(a.dq)) + (a.dq32 ? 0 : at0), a.dq32 ? 0 : len, int(row_k),
                                a.dq32 ? 0 : a.dim_k);
    const Rows reader = rows_at(a.dk32 + at0, len, int(row_k), a.dim_k);
    float dot = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * wave + 8 * g + 4 * half;
      float kv[4], qv[4];
      PX::four(k_lds, col, d / 4, kv);
      if constexpr (!BACK) PX::four(q_lds, col, d / 4, qv);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        dot += BACK ? -kv[j] * o1[4 * g + j] : qv[j] * o1[4 * g + j] + kv[j] * o2[4 * g + j];
      const bool in = d < a.dim_k;
      float x[4] = {o1[4 * g], o1[4 * g + 1], o1[4 * g + 2], o1[4 * g + 3]};
      if constexpr (!BACK) {
        put4<float>(reader, col, d, in, o2[4 * g], o2[4 * g + 1], o2[4 * g + 2], o2[4 * g + 3]);
      } else {
        x[0] += other_k[g].x, x[1] += other_k[g].y, x[2] += other_k[g].z, x[3] += other_k[g].w;
      }
      put4<float>(wide, col, d, in, x[0], x[1], x[2], x[3]);
      put4<T>(narrow, col, d, in, x[0], x[1], x[2], x[3]);
    }
    dot += __shfl_xor(dot, 32, 64);
    if (half == 0) sum_lds[wave][col] = dot;
    if (c + 1 < chunks) fetch(begin_of(c + 1));      // not before: the registers were the chunk's products'
    // the state
#pragma unroll
    for (int b = 0; b < XB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) m[b][r] *= whole;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float kx[8], qx[8];
      values(kc[t], kx);
      if constexpr (BACK) values(qc[t], qx);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float gv[4], bo[4];
        four_of(BACK ? gin_lds : gout_lds, 2 * t + g, half, gv);
        four_of(beta_lds, 2 * t + g, half, bo);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (BACK) {
            qx[4 * g + j] *= a.scale * gv[j];
            kx[4 * g + j] *= -bo[j] * gv[j];
          } else {
            kx[4 * g + j] *= gv[j];
          }
        }
      }
      const Split<kFine> ksp = split<kFine>(kx);
      Split<kFine> qsp;
      if constexpr (BACK) qsp = split<kFine>(qx);
#pragma unroll
      for (int b = 0; b < XB; ++b) {
        if constexpr (BACK) {
          m[b] = mul(PX::cols(g_lds, t, b, lane), qsp, m[b]);
          m[b] = mul(PM::cols(z_lds, t, b, lane), ksp, m[b]);
        } else {
          m[b] = mul(PM::cols(u_lds, t, b, lane), ksp, m[b]);
        }
      }
    }
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) s += sum_lds[w][col];
    if constexpr (BACK) {                        // the sum from the token to the chunk's end, and behind it
      s = col < len ? s + before : 0.f;
#pragma unroll
      for (int n = 1; n < C; n <<= 1) {
        const float y = __shfl_down(s, n, 32);
        if (col + n < C) s += y;
      }
      s += running;
      running = __shfl(s, 0, 64);
    }
    put<float>(rows_at(a.dgate + int64_t(t0) * a.heads + h, len, a.heads, 1), col, 0, tid < C, s);
  }
}

// A key head's gradients: the sums over its value heads. Four values a lane.
template <typename T>
__global__ __launch_bounds__(256) void delta_sum_heads(const float* dq32, const float* dk32, int64_t values, int group, int dim, T* dq, T* dk) {
  const int64_t i = 4 * (int64_t(blockIdx.x) * 256 + threadIdx.x);
  if (i >= 2 * values) return;
  const bool is_k = i >= values;
  const int64_t at = is_k ? i - values : i, head = at / dim, d = at % dim;
  const float* p = (is_k ? dk32 : dq32) + head * group * dim + d;
  float4 s = *reinterpret_cast<const float4*>(p);
  for (int g = 1; g < group; ++g) {
    const float4 y = *reinterpret_cast<const float4*>(p + int64_t(g) * dim);
    s.x += y.x, s.y += y.y, s.z += y.z, s.w += y.w;
  }
  store4<T>((is_k ? dk : dq) + at, s.x, s.y, s.z, s.w);
}

// ---------------------------------------------------------------- one token a sequence
// A workgroup a state: lane group c has four columns, each thread up to 16 rows of them in registers; two sums over the
// rows (S'^T k, S^T q) go through LDS.
template <typename T, int D>
__global__ __launch_bounds__(256) void delta_step(const DeltaArgs a) {
  constexpr int kCols = D / 4, kRows = 256 / kCols, kEach = D / kRows;
  __shared__ __attribute__((aligned(16))) float part[kRows][D + 4];
  __shared__ float k_lds[D], q_lds[D];
  const int tid = threadIdx.x, c = tid % kCols, r0 = tid / kCols;
  const int64_t nh = blockIdx.x, token = nh / a.heads;
  const int h = int(nh % a.heads);
  const float* s = a.init + nh * a.dim_k * a.dim_v + 4 * c;
  const bool in = 4 * c < a.dim_v;
  const float gate = a.log_gate[nh], f = exp2_fast(finite_gate2(gate)), beta = a.beta[nh];
  float4 x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int r = r0 + i * kRows;
    x[i] = in && r < a.dim_k ? *reinterpret_cast<const float4*>(s + int64_t(r) * a.dim_v) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (tid < D) {
    const int64_t kh = h / a.group;
    k_lds[tid] = tid < a.dim_k ? float(static_cast<const T*>(a.k)[token * a.ks_t + kh * a.ks_h + tid]) : 0.f;
    q_lds[tid] = tid < a.dim_k ? float(static_cast<const T*>(a.q)[token * a.qs_t + kh * a.qs_h + tid]) : 0.f;
  }
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const float k = k_lds[r0 + i * kRows];
    x[i].x *= f, x[i].y *= f, x[i].z *= f, x[i].w *= f;
    o.x = fmaf(k, x[i].x, o.x), o.y = fmaf(k, x[i].y, o.y), o.z = fmaf(k, x[i].z, o.z), o.w = fmaf(k, x[i].w, o.w);
  }
  auto sum_rows = [&]() {
    *reinterpret_cast<float4*>(&part[r0][4 * c]) = o;
    __syncthreads();
    float4 t = *reinterpret_cast<const float4*>(&part[0][4 * c]);
#pragma unroll
    for (int r = 1; r < kRows; ++r) {
      const float4 y = *reinterpret_cast<const float4*>(&part[r][4 * c]);
      t.x += y.x, t.y += y.y, t.z += y.z, t.w += y.w;
    }
    return t;
  };
  const float4 got = sum_rows();
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (in) {
    const T* vp = static_cast<const T*>(a.v) + token * a.vs_t + h * a.vs_h + 4 * c;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = float(vp[j]);
  }
  const float u[4] = {beta * (v[0] - got.x), beta * (v[1] - got.y), beta * (v[2] - got.z), beta * (v[3] - got.w)};
  float* fs = a.final_state + nh * a.dim_k * a.dim_v + 4 * c;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int r = r0 + i * kRows;
    const float k = k_lds[r], q = q_lds[r];
    x[i].x = fmaf(k, u[0], x[i].x), x[i].y = fmaf(k, u[1], x[i].y), x[i].z = fmaf(k, u[2], x[i].z), x[i].w = fmaf(k, u[3], x[i].w);
    o.x = fmaf(q, x[i].x, o.x), o.y = fmaf(q, x[i].y, o.y), o.z = fmaf(q, x[i].z, o.z), o.w = fmaf(q, x[i].w, o.w);
    if (in && r < a.dim_k) *reinterpret_cast<float4*>(fs + int64_t(r) * a.dim_v) = x[i];
  }
  __syncthreads();
  const float4 y = sum_rows();
  if (in && r0 == 0) store4<T>(static_cast<T*>(a.out) + nh * a.dim_v + 4 * c, y.x * a.scale, y.y * a.scale, y.z * a.scale, y.w * a.scale);
}

template <typename F> int with_delta_pad(const DeltaArgs& a, F&& f) {
  switch (delta_pad(a.dim_k, a.dim_v)) {
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    default: return f(std::integral_constant<int, 128>());
  }
}

dim3 carry_grid(const DeltaArgs& a) {
  const int64_t units = int64_t(carry_seqs(a)) * a.heads;
  return dim3(unsigned(ceil_div(units, int64_t(8)) * 8 * (delta_pad(a.dim_k, a.dim_v) / 32)));
}

}  // namespace

template <typename T> int DeltaLaunch<T>::prep(const DeltaArgs& a, hipStream_t st) {
  return with_delta_pad(a, [&](auto d) -> int {
    constexpr int D = decltype(d)::value;
    BF_LAUNCH("delta_prep", (delta_prep<T, D>), dim3(unsigned(a.n_chunk * a.heads)), dim3(64), 0, st, a);
    BF_CHECK_LAUNCH();
    return BF_OK;
  });
}

template <typename T> int DeltaLaunch<T>::forward(const DeltaArgs& a, hipStream_t st) {
  return with_delta_pad(a, [&](auto d) -> int {
    constexpr int D = decltype(d)::value;
    const dim3 grid = dim3(unsigned(a.n_seg * a.heads));
    if (a.carried) {
      BF_LAUNCH("delta_maps", (delta_pass<T, D, kMaps>), grid, dim3(4 * D), 0, st, a);
      BF_CHECK_LAUNCH();
      BF_LAUNCH("delta_carry", (delta_carry<T, D, false>), carry_grid(a), dim3(2 * D), 0, st, a);
      BF_CHECK_LAUNCH();
    }
    auto pass = a.e ? delta_pass<T, D, kTrain> : delta_pass<T, D, kForward>;
    BF_LAUNCH("delta_pass", pass, grid, dim3(2 * D), 0, st, a);
    BF_CHECK_LAUNCH();
    return BF_OK;
  });
}

template <typename T> int DeltaLaunch<T>::backward(const DeltaArgs& a, hipStream_t st) {
  return with_delta_pad(a, [&](auto d) -> int {
    constexpr int D = decltype(d)::value;
    const dim3 grid = dim3(unsigned(a.n_seg * a.heads));
    if (a.carried) {
      BF_LAUNCH("delta_back_maps", (delta_back<T, D, kBackMaps>), grid, dim3(2 * D), 0, st, a);
      BF_CHECK_LAUNCH();
      BF_LAUNCH("delta_back_carry", (delta_carry<T, D, true>), carry_grid(a), dim3(2 * D), 0, st, a);
      BF_CHECK_LAUNCH();
    }
    BF_LAUNCH("delta_back", (delta_back<T, D, kBack>), grid, dim3(2 * D), 0, st, a);
    BF_CHECK_LAUNCH();
    BF_LAUNCH("delta_grad_q", (delta_grad<T, D, false>), grid, dim3(2 * D), 0, st, a);
    BF_CHECK_LAUNCH();
    BF_LAUNCH("delta_grad_k", (delta_grad<T, D, true>), grid, dim3(2 * D), 0, st, a);
    BF_CHECK_LAUNCH();
    if (a.dq32) {
      const int64_t values = int64_t(a.n) * a.heads_k * a.dim_k;
      BF_LAUNCH("delta_sum_heads", (delta_sum_heads<T>), dim3(unsigned(ceil_div(2 * values, 1024))), dim3(256), 0, st, a.dq32,
                a.dk32, values, a.group, a.dim_k, static_cast<T*>(a.dq), static_cast<T*>(a.dk));
      BF_CHECK_LAUNCH();
    }
    return BF_OK;
  });
}

template <typename T> int DeltaLaunch<T>::step(const DeltaArgs& a, int64_t n, hipStream_t st) {
  return with_delta_pad(a, [&](auto d) -> int {
    constexpr int D = decltype(d)::value;
    BF_LAUNCH("delta_step", (delta_step<T, D>), dim3(unsigned(n * a.heads)), dim3(256), 0, st, a);
    BF_CHECK_LAUNCH();
    return BF_OK;
  });
}

}  // namespace bf
#endif  // BF_DELTA_KERNELS
