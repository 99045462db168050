// Residual norm (residual_norm.h), the backward pass.
//
// A workgroup takes rows in strides of the grid and keeps the parameters' gradients of its columns in
// registers over them; rows side by side in a workgroup are added through LDS, the workgroups' sums
// by a second launch, both in a fixed order.
#include "residual_norm.h"

namespace prnn {
namespace {

template <typename T, int V, int E, int NT>
__global__ __launch_bounds__(NT < 256 ? 256 : NT, E == 8 && V > 1 && NT <= 256 ? 3 : 1) void rn_backward_kernel(RnArgs A) {
  constexpr int R = NT < 256 ? 256 / NT : 1, block = NT < 256 ? 256 : NT;
  __shared__ float lds[64];
  __shared__ float s_sum[R > 1 ? E * block : 1];
  using Row = RnRow<T, V, E, NT>;
  const Row row{A.C, static_cast<int>(threadIdx.x) % NT};
  int turn = 0;
  const float inv = 1.0f / static_cast<float>(A.C);
  float w[E], p[E], s[E], sums[4][E];
  row.param(w, A.w, A.w_dtype, 1.0f);
  row.param(p, A.pw, A.w_dtype, 1.0f);
  row.param(s, A.scale, A.w_dtype, A.number);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < E; ++i) sums[k][i] = 0.0f;
  const int step = static_cast<int>(gridDim.x) * R;
  constexpr bool kAhead = E == 8 && NT < 1024;  // registers for the row behind this one
  auto place = [&](long long base) { return min(base + static_cast<int>(threadIdx.x) / NT, A.N - 1ll); };
  typename Row::Raw rx, ry, rg, rz, rh;  // the next row's are under way
  auto fetch = [&](long long base) {
    const long long at = place(base);
    rx = row.fetch(A.x, at);
    rz = row.fetch(A.gz, at);
    rh = row.fetch(A.gh, at);
    ry = row.fetch(A.y, at);
    rg = row.fetch(A.gate, at);
  };
  if (kAhead) fetch(blockIdx.x * R);
  for (long long base = blockIdx.x * R; base < A.N; base += step) {
    if (!kAhead) fetch(base);
    const long long at = place(base);
    const bool there = base + static_cast<int>(threadIdx.x) / NT < A.N;
    float h[E], n1[E], a[E], d[E], gz[E], dh[E];
    row.values(rx, h);
    row.values(rz, gz);
    row.values(rh, dh);
    row.values(ry, n1);
    row.values(rg, d);
    if (kAhead) fetch(base + step);
    if (!there) {  // another one's row: nothing to the sums
#pragma unroll
      for (int i = 0; i < E; ++i) gz[i] = dh[i] = 0.0f;
    }
    float r1 = 1.0f;
    if (A.y) {
      if (A.gate) {
#pragma unroll
        for (int i = 0; i < E; ++i) rn_act(d[i], A.act, a[i], d[i]);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) a[i] = 1.0f;
      }
      if (A.post) r1 = rn_norm<Row, E, NT>(row, n1, A.layer, A.eps, lds, turn);
#pragma unroll
      for (int i = 0; i < E; ++i)
        h[i] = row.col(i) < A.C ? fmaf(s[i] * a[i], n1[i] * p[i], h[i]) : 0.0f;
    }
    if (A.gz) {
      const float r2 = rn_norm<Row, E, NT>(row, h, A.layer, A.eps, lds, turn);  // h: n2 from here
      float m = 0.0f, shift = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        sums[0][i] = fmaf(gz[i], h[i], sums[0][i]);
        sums[1][i] += gz[i];
        gz[i] *= w[i];
        m = fmaf(gz[i], h[i], m);
        shift += gz[i];
      }
      rn_sum<NT>(m, shift, lds, turn);
      m *= inv;
      shift = A.layer ? shift * inv : 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) dh[i] = fmaf(r2, fmaf(-h[i], m, gz[i] - shift), dh[i]);
    }
    if (there) row.store(A.dx, at, dh);
    if (A.y) {
      float m = 0.0f, shift = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (row.col(i) >= A.C) dh[i] = 0.0f;
        const float f = n1[i] * p[i], da = dh[i] * s[i];
        sums[3][i] = fmaf(dh[i] * a[i], f, sums[3][i]);
        if (A.gate) d[i] *= da * f;
        const float df = da * a[i];
        sums[2][i] = fmaf(df, n1[i], sums[2][i]);
        dh[i] = df * p[i];
        m = fmaf(dh[i], n1[i], m);
        shift += dh[i];
      }
      if (A.gate && there) row.store(A.dgate, at, d);
      if (A.post) {
        rn_sum<NT>(m, shift, lds, turn);
        m *= inv;
        shift = A.layer ? shift * inv : 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) dh[i] = r1 * fmaf(-n1[i], m, dh[i] - shift);
      }
      if (there) row.store(A.dy, at, dh);
    }
  }
  if (A.parts == nullptr) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (!(A.want >> k & 1)) continue;
    if constexpr (R > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < E; ++i) s_sum[i * block + threadIdx.x] = sums[k][i];
      __syncthreads();
      if (threadIdx.x < NT) {
#pragma unroll
        for (int i = 0; i < E; ++i)
#pragma unroll
          for (int r = 1; r < R; ++r) sums[k][i] += s_sum[i * block + r * NT + threadIdx.x];
      }
    }
    if (threadIdx.x < NT) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = row.col(i);
        if (c < A.C) A.parts[(static_cast<size_t>(blockIdx.x) * 4 + k) * A.C + c] = sums[k][i];
      }
    }
  }
}

template <typename T, int V, int E, int NT>
int launch(const RnArgs& a, int groups, hipStream_t stream) {
  rn_backward_kernel<T, V, E, NT><<<groups, NT < 256 ? 256 : NT, 0, stream>>>(a);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}
template <typename T, int V>
int launch_row(const RnArgs& a, int groups, hipStream_t stream) {
  switch (rn_back_threads(a.C, sizeof(T) == 2)) {
    case 64: return launch<T, V, 8, 64>(a, groups, stream);
    case 128: return launch<T, V, 8, 128>(a, groups, stream);
    case 256: return launch<T, V, 8, 256>(a, groups, stream);
    case 512:
      if constexpr (sizeof(T) == 2)
        if (a.C > 4096) return launch<T, V, 16, 512>(a, groups, stream);
      return launch<T, V, 8, 512>(a, groups, stream);
  }
  if constexpr (sizeof(T) == 4)
    if (a.C <= 8192) return launch<T, V, 8, 1024>(a, groups, stream);
  return launch<T, V, 16, 1024>(a, groups, stream);
}

}  // namespace

int rn_backward(const RnArgs& a, int dtype, bool vec, int groups, hipStream_t stream) {
  return with_storage(dtype, [&](auto z) {
    using T = decltype(z);
    return vec ? launch_row<T, 16 / sizeof(T)>(a, groups, stream) : launch_row<T, 1>(a, groups, stream);
  });
}

}  // namespace prnn
