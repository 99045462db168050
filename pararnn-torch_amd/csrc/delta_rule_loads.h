// Gated delta rule: rows of tokens from memory, to LDS or as operands.
#pragma once

#include <type_traits>
#include <utility>

#include "delta_rule.h"
#include "tiles.h"

namespace prnn {

// Bytes of a row in LDS.  (Keys of 128 and values of 64 leave no room for more: two chunks of them fill it.)
constexpr int dr_row_k(bool narrow, int cols) {
  return narrow ? (cols > 128 ? cols * 2 + 48 : cols * 2 + 16) : (cols + 4) * 4;
}
constexpr int dr_row_z(bool narrow, int cols, int keys) {
  return !narrow ? (cols + 4) * 4 : cols == 32 || (cols == 64 && keys == 128) ? cols * 2 : cols == 64 ? 144 : cols * 2 + 48;
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

// Dense rows of floats, widths in fours, on their way from memory to LDS rows of RB bytes.
template <int COLS, int NT>
struct StagedFloats {
  static constexpr int U = COLS / 4, N = kDrC * U / NT;
  static_assert(NT % U == 0 && kDrC * U % NT == 0, "whole rows and units");
  u4 r[N];
  __device__ __forceinline__ void fetch(const float* p, int st, int n, int c0, int width) {
    const int c = c0 + threadIdx.x % U * 4;
    const rsrc_t b = make_rsrc(p, n > 0 ? ((n - 1) * st + width) * 4 : 0);
    const uint32_t at = la_in(c < width, (threadIdx.x / U * st + c) * 4);
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] = __builtin_amdgcn_raw_buffer_load_b128(b, at + k * (NT / U) * st * 4, 0, 0);
  }
  template <int RB>
  __device__ __forceinline__ void put(char* tile) const {
#pragma unroll
    for (int k = 0; k < N; ++k)
      *reinterpret_cast<u4*>(tile + (threadIdx.x / U + k * (NT / U)) * RB + threadIdx.x % U * 16) = r[k];
  }
  // The rows to memory, rounded to bf16.
  __device__ __forceinline__ void as_bf16(uint16_t* p, int st, int n, int c0, int width) const {
    const int c = c0 + threadIdx.x % U * 4;
    const rsrc_t b = make_rsrc(p, n > 0 ? ((n - 1) * st + width) * 2 : 0);
    const uint32_t at = la_in(c < width, (threadIdx.x / U * st + c) * 2);
#pragma unroll
    for (int k = 0; k < N; ++k)
      __builtin_amdgcn_raw_buffer_store_b64(u2{pack_bf16x2(__uint_as_float(r[k][0]), __uint_as_float(r[k][1])),
                                               pack_bf16x2(__uint_as_float(r[k][2]), __uint_as_float(r[k][3]))},
                                            b, at + k * (NT / U) * st * 2, 0, 0);
  }
};

// The eight floats that a lane has of operand `which` of an array of them (dr_operand_at).
struct Eight {
  float x[8];
};
__device__ __forceinline__ Eight global_op(rsrc_t r, bool in, int which) {
  Eight o;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const u4 w = __builtin_amdgcn_raw_buffer_load_b128(r, la_in(in, (which * 64 + (threadIdx.x & 63)) * 32 + 16 * k), 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) o.x[4 * k + i] = __uint_as_float(w[i]);
  }
  return o;
}
// As an operand of 24 bits.
template <class M>
__device__ __forceinline__ Op<M, 3> whole(Eight o) {
  return parts_of<M, 3>(o.x);
}

}  // namespace prnn
