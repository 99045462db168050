// Residual norm: the norms behind and before a block with its gate and residual scale.
//
//   f = norm(y) p  or  y        a = act(gate)  or  1        h = x + s a f
//   z = norm(h) w + b           norm(t) = (t - mean) rstd, or without the mean (rms)
//
// backwards, with n2 = norm(h), n1 = norm(y), r their rstd, m(.) the mean over a row:
//
//   dn2 = gz w,   dh = gh + r2 (dn2 - [m(dn2)] - n2 m(dn2 n2)),   dx = dh,   df = dh s a,
//   dy = r1 (df p - [m(df p)] - n1 m(df p n1))  or  df,   dgate = dh s f act'(gate),
//   and sums over rows: dw = gz n2, db = gz, dp = df n1, ds = dh a f.
//
// A row lies in the registers of NT threads, E elements each: every array is read once and written
// once, the statistics are two-pass and the backward pass forms them again from x, y and the gate.
// Bound by memory where rows are many: 16384 rows of 1024 in bf16 with gate and both norms take 41 us
// forwards (168 MB, 4.1 TB/s) and 61 backwards (268 MB, 4.4 TB/s); a launch's latency where they are few
// (32 rows 6.4 us).
#pragma once

#include <algorithm>

#include "prnn_host.h"

namespace prnn {

constexpr int kRnMax = 16384;  // channels: 1024 threads of 16

struct RnArgs {
  const void *x, *y, *w, *b, *pw, *gate, *scale;  // scale NULL: `number`
  void *h, *z;
  const void *gh, *gz;
  void *dx, *dy, *dgate;
  float* parts;   // (workgroup, 4, C): sums of dw, db, dp, ds over its rows
  int N, C;
  int layer, post, act, w_dtype;
  int want;       // which of the sums (bits 0 .. 3)
  float number, eps;
};

int rn_forward(const RnArgs& a, int dtype, bool vec, hipStream_t stream);
int rn_backward(const RnArgs& a, int dtype, bool vec, int groups, hipStream_t stream);

// Threads of a row: 8 elements each, of rows over 8192 16.
inline int rn_threads(int C) {
  int nt = 64;
  while (nt < 1024 && nt * 8 < C) nt *= 2;
  return nt;
}
// The backward pass holds more of a row, and 1024 threads have 128 registers each: rows of 4097 .. 8192
// elements of 16 bits take 512 threads of 16 (4096 x 8192 with all options: 232 us, 309 with 1024 of 8;
// fp32 564 and 418).  Over 8192 registers spill (1 TB/s of such rows).
inline int rn_back_threads(int C, bool narrow) { return narrow && C > 4096 && C <= 8192 ? 512 : rn_threads(C); }
// Workgroups of the backward pass: as many as run at a time, 12 waves a CU of 16-byte accesses, 8 of
// single elements (16384 x 1024 in bf16: 61 us, with 8 waves 69; a workgroup's sums over its rows are
// written and read once more).
inline int rn_groups(int N, int C, bool vec, bool narrow) {
  const int nt = rn_back_threads(C, narrow), rows = nt >= 256 ? 1 : 256 / nt;
  const long long groups = (static_cast<long long>(N) + rows - 1) / rows;
  const int most = (vec ? 768 : 512) * 256 / std::max(256, nt);
  return static_cast<int>(std::min<long long>(groups, most));
}

template <typename T, int V, int E, int NT>
struct RnRow {
  static constexpr int K = E / V;
  int C, lane;
  __device__ __forceinline__ int col(int i) const { return ((i / V) * NT + lane) * V + i % V; }
  // A row on its way: 16-byte units, or elements one by one.  Zeros behind the width and where there is
  // no array.
  static constexpr int U = V == 1 ? E : E * static_cast<int>(sizeof(T)) / 4;
  struct Raw {
    uint32_t w[U];
  };
  __device__ __forceinline__ Raw fetch(const void* p, long long row) const {
    Raw r;
    const rsrc_t b = make_rsrc(p ? static_cast<const T*>(p) + row * C : nullptr, p ? C * static_cast<uint32_t>(sizeof(T)) : 0u);
    if constexpr (V == 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) r.w[k] = ldb_bits(static_cast<T*>(nullptr), b, (k * NT + lane) * sizeof(T), 0);
    } else {
      typedef uint32_t u4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const u4 w = __builtin_amdgcn_raw_buffer_load_b128(b, (k * NT + lane) * 16, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[4 * k + i] = w[i];
      }
    }
    return r;
  }
  __device__ __forceinline__ void values(const Raw& r, float* v) const {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if constexpr (V == 1)
        v[i] = bits_to_f32(static_cast<T*>(nullptr), r.w[i]);
      else if constexpr (sizeof(T) == 4)
        v[i] = __uint_as_float(r.w[i]);
      else
        v[i] = i & 1 ? Narrow<T>::hi(r.w[i / 2]) : Narrow<T>::lo(r.w[i / 2]);
    }
  }
  __device__ __forceinline__ void store(void* p, long long row, const float* v) const {
    if (p == nullptr) return;
    T* at = static_cast<T*>(p) + row * C;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * NT + lane) * V;
      if constexpr (V == 1) {
        if (c < C) at[c] = from_f32<T>(v[k]);
      } else {
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (sizeof(T) == 4)
            w[i] = __float_as_uint(v[k * V + i]);
          else
            w[i] = Narrow<T>::pack(v[k * V + 2 * i], v[k * V + 2 * i + 1]);
        }
        if (c < C) *reinterpret_cast<u4*>(at + c) = w;
      }
    }
  }
  // a parameter per channel, `none` where there is none
  __device__ __forceinline__ void param(float* v, const void* p, int dtype, float none) const {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = col(i);
      v[i] = none;
      if (p != nullptr && c < C)
        v[i] = dtype == PRNN_F32 ? static_cast<const float*>(p)[c] : to_f32(static_cast<const T*>(p)[c]);
    }
  }
};

// Sum over the wave, in all lanes: rows of 16 by shifts, the rows' last lanes handed on.
template <int CTRL, int ROWS>
__device__ __forceinline__ float rn_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float rn_wave_sum(float v) {
  v = rn_add<0x111, 0xf>(v);
  v = rn_add<0x112, 0xf>(v);
  v = rn_add<0x114, 0xf>(v);
  v = rn_add<0x118, 0xf>(v);
  v = rn_add<0x142, 0xa>(v);
  v = rn_add<0x143, 0xc>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Sums of two values over the NT threads of a row, in all of them; `turn` alternates the LDS places,
// so one barrier a sum is enough.
template <int NT>
__device__ __forceinline__ void rn_sum(float& a, float& b, float* lds, int& turn) {
  a = rn_wave_sum(a);
  b = rn_wave_sum(b);
  if constexpr (NT > 64) {
    constexpr int W = NT / 64;
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    float* at = lds + turn * 32;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
      at[wave * 2] = a;
      at[wave * 2 + 1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      a += at[(first + w) * 2];
      b += at[(first + w) * 2 + 1];
    }
  }
}

// t -> (t - mean) rstd in place; returns rstd.
template <typename R, int E, int NT>
__device__ __forceinline__ float rn_norm(const R& row, float* t, int layer, float eps, float* lds, int& turn) {
  const float inv = 1.0f / static_cast<float>(row.C);
  if (layer) {
    float s = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += t[i];  // zeros behind the width
    rn_sum<NT>(s, none, lds, turn);
    s *= inv;
#pragma unroll
    for (int i = 0; i < E; ++i) t[i] = row.col(i) < row.C ? t[i] - s : 0.0f;
  }
  float q = 0.0f, none = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) q = fmaf(t[i], t[i], q);
  rn_sum<NT>(q, none, lds, turn);
  // not v_rsq_f32: the statistics keep all bits
  const float r = 1.0f / sqrtf(fmaf(q, inv, eps));
#pragma unroll
  for (int i = 0; i < E; ++i) t[i] *= r;
  return r;
}

// act(g) in a, its derivative in d.
__device__ __forceinline__ void rn_act(float g, int act, float& a, float& d) {
  if (act == 0) {
    a = g;
    d = 1.0f;
    return;
  }
  const float e = fexp(-fabsf(g)), s = 1.0f / (1.0f + e);  // of |g|: e is at most 1
  const float sig = g >= 0.0f ? s : e * s, com = g >= 0.0f ? e * s : s;
  a = act == 1 ? g * sig : sig;
  d = act == 1 ? sig * fmaf(g, com, 1.0f) : sig * com;
}

}  // namespace prnn
