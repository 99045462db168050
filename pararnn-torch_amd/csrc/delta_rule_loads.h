// Gated delta rule: rows of tokens from memory, to LDS or as operands.
#pragma once

#include <type_traits>
#include <utility>

#include "delta_rule.h"
#include "tiles.h"

namespace prnn {

constexpr int dr_row_k(bool narrow, int cols) {
  return narrow ? (cols >= 128 ? cols * 2 + 48 : cols * 2 + 16) : (cols + 4) * 4;
}
constexpr int dr_row_z(bool narrow, int cols) {
  return narrow ? (cols == 32 ? 64 : cols == 64 ? 144 : cols * 2 + 48) : (cols + 4) * 4;
}

// Rows of 64 tokens of a head on their way from memory to LDS: 16-byte units in bf16, single
// elements of any storage type to floats.
template <class M, int COLS, int NT>
struct Staged {
  static constexpr bool kNarrow = sizeof(typename M::E) == 2;
  static constexpr int U = kNarrow ? COLS / 8 : COLS;  // units of a row
  static constexpr int N = kDrC * U / NT;
  static_assert(kDrC * U % NT == 0, "whole units");
  std::conditional_t<kNarrow, u4, uint32_t> r[N];

  // `width` columns from c0; tokens [0, n) from `p` are there: the others lie behind the buffer's end (a
  // row is at most a stride wide, or they are told by a comparison).
  __device__ __forceinline__ void fetch(const char* p, long long st, int n, int c0, int width, int dtype,
                                        int tid = threadIdx.x) {
    if constexpr (kNarrow) {
      constexpr int D = NT / U;  // rows between a thread's loads
      static_assert(NT % U == 0, "whole rows");
      const int step = static_cast<int>(st) * 2, c = c0 + tid % U * 8;
      const rsrc_t b = make_rsrc(p, n > 0 ? (n - 1) * step + width * 2 : 0);
      const uint32_t at = la_in(c < width, tid / U * step + c * 2);
#pragma unroll
      for (int k = 0; k < N; ++k) r[k] = __builtin_amdgcn_raw_buffer_load_b128(b, at + k * D * step, 0, 0);
    } else {
      const rsrc_t b = make_rsrc(p, 0x7fffffffu);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int e = tid + k * NT, row = e / U, c = e % U;
        if (dtype == PRNN_F32)
          r[k] = __builtin_amdgcn_raw_buffer_load_b32(
              b, la_in((row < n) & (c0 + c < width), (row * static_cast<int>(st) + c0 + c) * 4), 0, 0);
        else
          r[k] = __builtin_amdgcn_raw_buffer_load_b16(
              b, la_in((row < n) & (c0 + c < width), (row * static_cast<int>(st) + c0 + c) * 2), 0, 0);
      }
    }
  }
  template <int RB>
  __device__ __forceinline__ void put(char* tile, int dtype, int tid = threadIdx.x) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int e = tid + k * NT, row = e / U, c = e % U;
      if constexpr (kNarrow) {
        *reinterpret_cast<u4*>(tile + row * RB + c * 16) = r[k];
      } else {
        const float v = dtype == PRNN_F32   ? __uint_as_float(r[k])
                        : dtype == PRNN_F16 ? Narrow<f16>::val(r[k])
                                            : Narrow<bf16>::val(r[k]);
        *reinterpret_cast<float*>(tile + row * RB + c * 4) = v;
      }
    }
  }
};

// Operand `which` of an array of them (dr_operand_at), its parts `part` bytes apart.
template <class M>
__device__ __forceinline__ Op<M, M::kParts> global_op(rsrc_t r, bool in, int which, int part) {
  constexpr int ES = static_cast<int>(sizeof(typename M::E));
  const int lane = threadIdx.x & 63;
  Op<M, M::kParts> o;
  if constexpr (ES == 2) {
#pragma unroll
    for (int k = 0; k < M::kParts; ++k)
      o.p[k] = __builtin_bit_cast(
          b8, __builtin_amdgcn_raw_buffer_load_b128(r, la_in(in, (which * 64 + lane) * 16 + k * part), 0, 0));
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const u4 w = __builtin_amdgcn_raw_buffer_load_b128(r, la_in(in, (which * 64 + lane) * 32 + 16 * k), 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) o.x[4 * k + i] = __uint_as_float(w[i]);
    }
  }
  return o;
}

}  // namespace prnn
