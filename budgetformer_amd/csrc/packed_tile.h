// Matrix-core operands and LDS tiles shared by the operators over packed sequences.
//
// v_mfma 32x32x16 takes 8 values a lane along the contraction (lane l: row or column l % 32, half l / 32) and leaves
// column l % 32, rows (r % 4) + 8 (r / 4) + 4 (l / 32) of the product in register r. Registers 8t .. 8t+7 are then, as
// they stand, an operand of another product over the 16 rows 16t .. 16t+15, if that product counts its contraction as
// the registers do: value j of half h is row 16t + (j % 4) + 8 (j / 4) + 4 h ("register order"). float32 uses the same
// layout with eight 32x32x2 products for one of 16.
#pragma once

#include <type_traits>

#include "bf_common.h"

namespace bf {

typedef float F32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;

// Rows of an axis at most: the end of a tile, of a piece of one or of a segment may lie behind the last row, in 32 bits.
constexpr int64_t kMaxRows = (int64_t(1) << 31) - (1 << 17);

template <typename T> struct Mat;

template <> struct Mat<__bf16> {
  typedef __bf16 Frag __attribute__((ext_vector_type(8)));
  typedef __bf16 Frag4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ F32x16 mma(const Frag& a, const Frag& b, const F32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // acc, or a NaN if the 16 bytes hold an infinity or a NaN (0 * x is then a NaN)
  static __device__ __forceinline__ float taint(const uint4& v, float acc) {
    typedef __bf16 P2 __attribute__((ext_vector_type(2)));
    const P2 z = {__bf16(0.f), __bf16(0.f)};
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(P2, v.x), z, acc, false);
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(P2, v.y), z, acc, false);
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(P2, v.z), z, acc, false);
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(P2, v.w), z, acc, false);
  }
};

template <> struct Mat<_Float16> {
  typedef _Float16 Frag __attribute__((ext_vector_type(8)));
  typedef _Float16 Frag4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ F32x16 mma(const Frag& a, const Frag& b, const F32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float taint(const uint4& v, float acc) {
    typedef _Float16 P2 __attribute__((ext_vector_type(2)));
    const P2 z = {_Float16(0.f), _Float16(0.f)};
    acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(P2, v.x), z, acc, false);
    acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(P2, v.y), z, acc, false);
    acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(P2, v.z), z, acc, false);
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(P2, v.w), z, acc, false);
  }
};

template <> struct Mat<float> {
  typedef float Frag __attribute__((ext_vector_type(8)));
  typedef float Frag4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ F32x16 mma(const Frag& a, const Frag& b, F32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ float taint(const uint4& v, float acc) {
    acc = fmaf(__uint_as_float(v.x), 0.f, acc);
    acc = fmaf(__uint_as_float(v.y), 0.f, acc);
    acc = fmaf(__uint_as_float(v.z), 0.f, acc);
    return fmaf(__uint_as_float(v.w), 0.f, acc);
  }
};

template <typename T> using Frag = typename Mat<T>::Frag;

__device__ __forceinline__ F32x16 zero16() {
  F32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

template <typename T> __device__ __forceinline__ Frag<T> zero_frag() {
  Frag<T> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = T(0.f);
  return f;
}

// Row (of 32) that register r of a product holds, for the lane's half; also value r's row in register order.
__device__ __forceinline__ int acc_row(int r, int half) { return (r & 3) + 8 * (r >> 2) + 4 * half; }

// The places of a 32 block that lie in [lo, hi), a bit each, as the lane's half sees them: register r's place is bit
// acc_row(r, 0).
__device__ __forceinline__ uint32_t seen_bits(int lo, int hi, int half) {
  const uint32_t below_hi = hi >= 32 ? ~0u : hi <= 0 ? 0u : (1u << hi) - 1u;
  const uint32_t below_lo = lo >= 32 ? ~0u : lo <= 0 ? 0u : (1u << lo) - 1u;
  return (below_hi & ~below_lo) >> (4 * half);
}

// x where register r's bit is set, else `other` (two instructions: the bit spread over a word, and a bitwise choice).
__device__ __forceinline__ float where_seen(uint32_t bits, int r, float x, float other) {
  const uint32_t all = uint32_t(__builtin_amdgcn_sbfe(int(bits), uint32_t(acc_row(r, 0)), 1u));
  return __uint_as_float((__float_as_uint(x) & all) | (__float_as_uint(other) & ~all));
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Registers 8t .. 8t+7 as an operand of the next product.
template <typename T, typename X> __device__ __forceinline__ Frag<T> pack8(const X& x, int t) {
  Frag<T> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = T(x[8 * t + j]);
  return f;
}

// A fragment's finite values, the others as 0.
template <typename T> __device__ __forceinline__ Frag<T> finite(const Frag<T>& f) {
  Frag<T> o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = fabsf(float(f[j])) < INFINITY ? f[j] : T(0.f);
  return o;
}

// 1 where a fragment holds an infinity of this sign or a NaN, else 0.
template <typename T> __device__ __forceinline__ Frag<T> is_infinite(const Frag<T>& f, float sign) {
  Frag<T> o;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = float(f[j]) * sign;
    o[j] = T(x < INFINITY ? 0.f : 1.f);
  }
  return o;
}

// What infinite values add to a product of weights that are not negative: mma(t, x, sign) multiplies the indicators of
// that sign in step t; where their sum is positive an infinity of that sign is added (of both: a NaN).
template <int STEPS, typename F> __device__ __forceinline__ void add_infinite(F32x16& acc, F&& mma) {
#pragma unroll
  for (int way = 0; way < 2; ++way) {
    const float sign = way ? -1.f : 1.f;
    F32x16 x = zero16();
#pragma unroll
    for (int t = 0; t < STEPS; ++t) x = mma(t, x, sign);
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] += x[r] > 0.f ? sign * INFINITY : 0.f;
  }
}

// A tile of rows of DP values in LDS. Rows are padded by 32 bytes: the 4 rows of a transposing read, and the 8 rows that
// a cycle of 16-byte reads touches, then fall on different banks.
template <typename T, int DP> struct Tile {
  static constexpr int kPitch = DP * int(sizeof(T)) + 32;       // bytes of a row
  static constexpr int kSteps = DP / 16;                        // contractions of 16 over the row
  static constexpr int kBlocks = (DP + 31) / 32;                // blocks of 32 values of the row
  // DP 16 reads columns 16 .. 31 too (values that only reach product rows nobody stores): in bounds up to this slack
  static constexpr int bytes(int rows) { return rows * kPitch + (DP < 32 ? 64 : 0); }

  // values [16 s + 8 half, + 8) of a row: the operand whose rows are the tile's rows
  static __device__ __forceinline__ Frag<T> row_frag(const char* lds, int row, int s, int half) {
    return *reinterpret_cast<const Frag<T>*>(lds + row * kPitch + (16 * s + 8 * half) * int(sizeof(T)));
  }
  // the same 16 values in register order
  static __device__ __forceinline__ Frag<T> row_frag_regs(const char* lds, int row, int s, int half) {
    typedef typename Mat<T>::Frag4 F4;
    const char* p = lds + row * kPitch + (16 * s + 4 * half) * int(sizeof(T));
    const F4 a = *reinterpret_cast<const F4*>(p), b = *reinterpret_cast<const F4*>(p + 8 * sizeof(T));
    const Frag<T> f = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return f;
  }
  // the operand whose rows are the values 32 n + lane % 32 of the tile's rows, over the tile's rows 16 t .. 16 t + 15: in
  // register order, or (REGS false) in their own. Two transposing reads of 4 x 16 blocks in 16-bit types.
  template <bool REGS = true>
  static __device__ __forceinline__ Frag<T> col_frag(const char* lds, int t, int n, int lane) {
    constexpr int kHalf = REGS ? 4 : 8, kSecond = REGS ? 8 : 4;
    if constexpr (sizeof(T) == 2) {
      typedef short S4 __attribute__((ext_vector_type(4)));
      typedef short S8 __attribute__((ext_vector_type(8)));
      typedef __attribute__((address_space(3))) S4 LdsS4;
      const int i = lane & 15, row = 16 * t + kHalf * (lane >> 5) + (i >> 2);
      const char* p = lds + row * kPitch + (32 * n + (lane & 16) + 4 * (i & 3)) * 2;
      const S4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4*)p);
      const S4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4*)(p + kSecond * kPitch));
      const S8 ab = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      return __builtin_bit_cast(Frag<T>, ab);
    } else {
      Frag<T> f;
      const char* p = lds + (16 * t + kHalf * (lane >> 5)) * kPitch + (32 * n + (lane & 31)) * 4;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = *reinterpret_cast<const T*>(p + ((j & 3) + kSecond * (j >> 2)) * kPitch);
      return f;
    }
  }
};

// A tile on its way from memory to LDS, in registers: 16 bytes a lane and step, a row's chunks side by side. Nothing in
// load depends on a value it reads and nothing branches, so that all of a tile's loads are on their way at once.
template <typename T, int DP, int ROWS, int NT> struct Stage {
  static constexpr int kChunks = DP * int(sizeof(T)) / 16, kPer = 16 / int(sizeof(T));
  static constexpr int kN = (ROWS * kChunks + NT - 1) / NT;
  uint4 r[kN];
  // rows 0 .. n - 1 of the tile (1 <= n) are at row_at(row); the others read row n - 1 again
  template <typename F> __device__ __forceinline__ void load(int tid, int n, int dim, F&& row_at) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = i * NT + tid, row = c / kChunks, at = (c % kChunks) * kPer;
      r[i] = *reinterpret_cast<const uint4*>(row_at(min(row, n - 1)) + (at < dim ? at : 0));
    }
  }
  // zeros in the place of rows n and on and of values dim and on
  __device__ __forceinline__ void clip(int tid, int n, int dim) {
    if (n >= ROWS && dim == DP) return;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = i * NT + tid, row = c / kChunks, at = (c % kChunks) * kPer;
      if (row >= n || at >= dim) r[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  __device__ __forceinline__ void store(int tid, char* lds) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = i * NT + tid, row = c / kChunks;
      if (ROWS * kChunks % NT == 0 || row < ROWS) *reinterpret_cast<uint4*>(lds + row * Tile<T, DP>::kPitch + (c % kChunks) * 16) = r[i];
    }
  }
  // whether the lane's part holds an infinity or a NaN
  __device__ __forceinline__ bool tainted() const {
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < kN; ++i) acc = Mat<T>::taint(r[i], acc);
    return acc != acc;
  }
};

// Four values of a row, rounded to its type.
template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  typedef T V4 __attribute__((ext_vector_type(4)));
  const V4 v = {T(a), T(b), T(c), T(d)};
  *reinterpret_cast<V4*>(p) = v;
}

// A product's columns (a lane has one row of the result) to memory, scaled: values 32 n + 8 g + 4 half + (0 .. 3).
template <typename T> __device__ __forceinline__ void store_block(T* p, const F32x16& acc, float by, int n, int dim, int half) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int at = 32 * n + 8 * g + 4 * half;
    if (at < dim) store4<T>(p + at, acc[4 * g] * by, acc[4 * g + 1] * by, acc[4 * g + 2] * by, acc[4 * g + 3] * by);
  }
}

struct Div {           // n / d for n < 2^31 by a multiplication
  uint32_t magic, shift;
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(n, magic) + n) >> shift; }
};

inline Div make_div(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  return Div{uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << s) - d)) / d + 1), s};
}

// f(T()) for a dtype code.
template <typename F> int with_type(int32_t dtype, F&& f) {
  switch (dtype) {
    case BF_DTYPE_F32: return f(float());
    case BF_DTYPE_BF16: return f(__bf16());
    default: return f(_Float16());
  }
}

inline bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}

}  // namespace bf
