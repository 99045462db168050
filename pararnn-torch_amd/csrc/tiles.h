// Matrix tiles in registers and LDS for kernels on gfx950's matrix instructions, in bf16 or fp32.
//
// A wave's tile has NC rows and columns (32 or 16).  A product leaves lane l with column l % NC and,
// with G = 64 / NC groups of lanes, g = l / NC, in register 4 q + r of the tile row 4 G q + 4 g + r.
// An operand gives lane l row (or column) l % NC and 8 places of a contraction of 8 G.  The order of
// a contraction is free, so these places are the rows that the lane holds of a product,
// {4 g + r, 4 G + 4 g + r}: what one product leaves in registers is the next one's operand, its
// registers 8 f .. 8 f + 7 the operand of step f.
#pragma once

#include "prnn_common.h"

namespace prnn {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

template <int NC>
struct Shape;
template <>
struct Shape<32> {
  using Acc = f16v;
};
template <>
struct Shape<16> {
  using Acc = f4;
};
template <int NC>
using Acc = typename Shape<NC>::Acc;

struct InBf16 {
  using E = uint16_t;
};
struct InF32 {
  using E = float;
};

// Operands: of P parts that add up to the value (fp32: one, whatever P).
template <class M, int P>
struct Op;
template <int P>
struct Op<InBf16, P> {
  b8 p[P];
};
template <int P>
struct Op<InF32, P> {
  float x[8];
};

template <int NC>
__device__ __forceinline__ Acc<NC> mfma_bf16(b8 a, b8 b, Acc<NC> c) {
  if constexpr (NC == 32)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <int NC>
__device__ __forceinline__ Acc<NC> mfma_f32(float a, float b, Acc<NC> c) {
  if constexpr (NC == 32)
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// c += a b; of several parts on both sides the products that count (the first with all of the
// other's, the second with the first).
template <int NC, int P, int R>
__device__ __forceinline__ void mul(Acc<NC>& c, const Op<InBf16, P>& a, const Op<InBf16, R>& b) {
#pragma unroll
  for (int i = 0; i < P; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (i + j < (P > R ? P : R)) c = mfma_bf16<NC>(a.p[i], b.p[j], c);
}
template <int NC, int P, int R>
__device__ __forceinline__ void mul(Acc<NC>& c, const Op<InF32, P>& a, const Op<InF32, R>& b) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = mfma_f32<NC>(a.x[i], b.x[i], c);
}

// The same product by product, so that several sums can take turns (a matrix instruction waits for the
// last one of its own sum): products kPairs<P, R> of operands of P and R parts, number k of them.
template <int P, int R>
constexpr int kPairs = P == 1 || R == 1 ? P * R : P == 3 ? 6 : 3;  // (of two or three parts each the largest)
template <int NC, int P, int R>
__device__ __forceinline__ void mul_one(Acc<NC>& c, const Op<InBf16, P>& a, const Op<InBf16, R>& b, int k) {
  static_assert(P == 1 || R == 1 || (P == R && P < 4), "products are listed for these");
  const int i = P == 1 ? 0 : R == 1 ? k : k == 5 ? 2 : k == 2 || k == 4;
  const int j = P == 1 ? k : R == 1 ? 0 : k == 3 ? 2 : k == 1 || k == 4;
  c = mfma_bf16<NC>(a.p[i], b.p[j], c);
}
template <int NC, int P, int R>
__device__ __forceinline__ void mul_one(Acc<NC>& c, const Op<InF32, P>& a, const Op<InF32, R>& b, int k) {
  if (k == 0) mul<NC>(c, a, b);
}

__device__ __forceinline__ b8 pack8(const float* x) {
  union {
    uint32_t w[4];
    b8 v;
  } r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  return r.v;
}
// x as bf16, and what that leaves of it in x.
__device__ __forceinline__ b8 split8(float* x) {
  union {
    uint32_t w[4];
    b8 v;
  } r;
  r.v = pack8(x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] -= lo_bf16(r.w[i]);
    x[2 * i + 1] -= hi_bf16(r.w[i]);
  }
  return r.v;
}

// Eight floats as an operand of P parts (x is used up).
template <class M, int P>
__device__ __forceinline__ Op<M, P> parts_of(float* x) {
  Op<M, P> r;
  if constexpr (sizeof(typename M::E) == 2) {
#pragma unroll
    for (int i = 0; i + 1 < P; ++i) r.p[i] = split8(x);
    r.p[P - 1] = pack8(x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.x[i] = x[i];
  }
  return r;
}

// The eight values of an exact operand.
__device__ __forceinline__ void values(const Op<InBf16, 1>& o, float* x) {
  union {
    b8 v;
    uint32_t w[4];
  } u;
  u.v = o.p[0];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = lo_bf16(u.w[i]);
    x[2 * i + 1] = hi_bf16(u.w[i]);
  }
}
__device__ __forceinline__ void values(const Op<InF32, 1>& o, float* x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = o.x[i];
}

// Step f of a contraction along a row in memory, `g` the lane's group.
template <class M, int G>
__device__ __forceinline__ Op<M, 1> row_op(const char* row, int f, int g) {
  using E = typename M::E;
  const char* at = row + (8 * G * f + 4 * g) * static_cast<int>(sizeof(E));
  Op<M, 1> r;
  if constexpr (sizeof(E) == 2) {
    union {
      u2 h[2];
      b8 v;
    } x;
    x.h[0] = *reinterpret_cast<const u2*>(at);
    x.h[1] = *reinterpret_cast<const u2*>(at + 4 * G * 2);
    r.p[0] = x.v;
  } else {
    const f4 a = *reinterpret_cast<const f4*>(at), b = *reinterpret_cast<const f4*>(at + 4 * G * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.x[i] = a[i];
      r.x[4 + i] = b[i];
    }
  }
  return r;
}

// A contraction down the rows of an LDS tile of RB bytes a row: the 8 G rows from t0, this lane's
// column c0 + l % NC.  `at`: the tile with the lane's share of the address, col_share.
template <class M, int G, int RB>
__device__ __forceinline__ int col_share(int lane) {
  if constexpr (sizeof(typename M::E) == 2) {
    const int i = lane & 15, gg = lane >> 4;
    if constexpr (G == 2)
      return (4 * (gg >> 1) + (i >> 2)) * RB + (16 * (gg & 1) + 4 * (i & 3)) * 2;
    else
      return (4 * gg + (i >> 2)) * RB + 4 * (i & 3) * 2;
  } else {
    constexpr int NC = 64 / G;
    return 4 * (lane / NC) * RB + (lane % NC) * 4;
  }
}
template <class M, int G, int RB>
__device__ __forceinline__ Op<M, 1> col_op(const char* at, int t0, int c0) {
  Op<M, 1> r;
  if constexpr (sizeof(typename M::E) == 2) {
    union {
      s4 h[2];
      b8 v;
    } x;
    x.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + t0 * RB + c0 * 2));
    x.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + (t0 + 4 * G) * RB + c0 * 2));
    r.p[0] = x.v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      r.x[i] = *reinterpret_cast<const float*>(at + (t0 + (i >> 2) * 4 * G + (i & 3)) * RB + c0 * 4);
  }
  return r;
}

}  // namespace prnn
