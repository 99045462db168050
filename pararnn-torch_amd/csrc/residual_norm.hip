// Residual norm (residual_norm.h): the forward pass, the sums over rows and the C entry points.
#include "residual_norm.h"

#include <algorithm>

namespace prnn {
namespace {

template <typename T, int V, int E, int NT>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void rn_forward_kernel(RnArgs A) {
  constexpr int R = NT < 256 ? 256 / NT : 1;  // rows of a workgroup
  __shared__ float lds[64];
  using Row = RnRow<T, V, E, NT>;
  const Row row{A.C, static_cast<int>(threadIdx.x) % NT};
  int turn = 0;
  float w[E], b[E], p[E], s[E];
  row.param(w, A.w, A.w_dtype, 1.0f);
  row.param(b, A.b, A.w_dtype, 0.0f);
  row.param(p, A.pw, A.w_dtype, 1.0f);
  row.param(s, A.scale, A.w_dtype, A.number);
  const int step = static_cast<int>(gridDim.x) * R;
  constexpr bool kAhead = E == 8;  // registers for the row behind this one
  auto place = [&](long long base) { return min(base + static_cast<int>(threadIdx.x) / NT, A.N - 1ll); };
  typename Row::Raw rx, ry, rg;  // the next row's are under way
  auto fetch = [&](long long base) {
    const long long at = place(base);  // behind the last row that one again: the sums meet in barriers
    rx = row.fetch(A.x, at);
    ry = row.fetch(A.y, at);
    rg = row.fetch(A.gate, at);
  };
  if (kAhead) fetch(blockIdx.x * R);
  for (long long base = blockIdx.x * R; base < A.N; base += step) {
    if (!kAhead) fetch(base);
    const long long at = place(base);
    const bool there = base + static_cast<int>(threadIdx.x) / NT < A.N;
    float h[E], f[E], g[E];
    row.values(rx, h);
    row.values(ry, f);
    row.values(rg, g);
    if (kAhead) fetch(base + step);
    if (A.y) {
      if (A.post) {
        rn_norm<Row, E, NT>(row, f, A.layer, A.eps, lds, turn);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] *= p[i];
      }
      if (A.gate) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          float a, d;
          rn_act(g[i], A.act, a, d);
          f[i] *= a;
        }
      }
#pragma unroll
      for (int i = 0; i < E; ++i) h[i] = row.col(i) < A.C ? fmaf(s[i], f[i], h[i]) : 0.0f;
      if (there) row.store(A.h, at, h);
    }
    rn_norm<Row, E, NT>(row, h, A.layer, A.eps, lds, turn);
#pragma unroll
    for (int i = 0; i < E; ++i) h[i] = fmaf(h[i], w[i], b[i]);
    if (there) row.store(A.z, at, h);
  }
}

// dst[c] = the workgroups' sums in their order: 64 columns a workgroup, its 16 waves a sixteenth of the
// parts each.
struct RnSums {
  const float* parts;
  void* dst[4];
  int groups, C, w_dtype;
};
template <typename T>
__global__ __launch_bounds__(1024) void rn_sum_kernel(RnSums A) {
  __shared__ float lds[16][64];
  const int k = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (A.dst[k] == nullptr) return;
  const int c = blockIdx.x * 64 + lane;
  float v = 0.0f;
  if (c < A.C) {
    const int each = (A.groups + 15) / 16, end = min(A.groups, (wave + 1) * each);
#pragma unroll 8
    for (int g = wave * each; g < end; ++g) v += A.parts[(static_cast<size_t>(g) * 4 + k) * A.C + c];
  }
  lds[wave][lane] = v;
  __syncthreads();
  if (wave || c >= A.C) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) v += lds[w][lane];
  if (A.w_dtype == PRNN_F32)
    static_cast<float*>(A.dst[k])[c] = v;
  else
    static_cast<T*>(A.dst[k])[c] = from_f32<T>(v);
}

template <typename T, int V, int E, int NT>
int launch(const RnArgs& a, hipStream_t stream) {
  constexpr int R = NT < 256 ? 256 / NT : 1, block = NT < 256 ? 256 : NT;
  const int groups = static_cast<int>(std::min((a.N + R - 1ll) / R, 256ll * (2048 / block)));
  rn_forward_kernel<T, V, E, NT><<<groups, block, 0, stream>>>(a);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}
template <typename T, int V>
int launch_row(const RnArgs& a, hipStream_t stream) {
  switch (rn_threads(a.C)) {
    case 64: return launch<T, V, 8, 64>(a, stream);
    case 128: return launch<T, V, 8, 128>(a, stream);
    case 256: return launch<T, V, 8, 256>(a, stream);
    case 512: return launch<T, V, 8, 512>(a, stream);
  }
  return a.C <= 8192 ? launch<T, V, 8, 1024>(a, stream) : launch<T, V, 16, 1024>(a, stream);
}

// (for any type: 16 bits and whole units have the most workgroups)
size_t parts_bytes(int N, int C) { return sizeof(float) * 4 * static_cast<size_t>(rn_groups(N, C, true, true)) * C; }

int check(int N, int C, float eps, int act, int w_dtype, int dtype) {
  if (int rc = check_dtype(dtype)) return rc;
  if (w_dtype != PRNN_F32 && w_dtype != dtype)
    return fail(PRNN_ERR_TYPE, "parameters must be float32 or of the storage type");
  if (N < 0 || C < 1 || C > kRnMax)
    return fail(PRNN_ERR_VALUE, "N=%d rows of C=%d channels: C must be in 1 .. %d", N, C, kRnMax);
  if (act < 0 || act > 2) return fail(PRNN_ERR_VALUE, "act=%d is none of 0, 1, 2", act);
  if (!(eps >= 0.0f)) return fail(PRNN_ERR_VALUE, "eps must be >= 0");
  return PRNN_OK;
}

// Rows that admit 16-byte accesses.
bool vectors(int C, int dtype, std::initializer_list<const void*> arrays) {
  uintptr_t all = static_cast<uintptr_t>(C) * (dtype == PRNN_F32 ? 4 : 2);
  for (const void* p : arrays) all |= reinterpret_cast<uintptr_t>(p);
  return (all & 15) == 0;
}

}  // namespace

int rn_forward(const RnArgs& a, int dtype, bool vec, hipStream_t stream) {
  return with_storage(dtype, [&](auto z) {
    using T = decltype(z);
    return vec ? launch_row<T, 16 / sizeof(T)>(a, stream) : launch_row<T, 1>(a, stream);
  });
}

}  // namespace prnn

using namespace prnn;

extern "C" PRNN_API int prnn_residual_norm(const void* x, const void* y, const void* w, const void* b,
                                           const void* pw, const void* gate, const void* scale,
                                           float scale_number, void* h, void* z, int N, int C, float eps,
                                           int layer, int post, int act, int w_dtype, int dtype,
                                           void* stream) {
  if (int rc = check(N, C, eps, act, w_dtype, dtype)) return rc;
  if (N == 0) return PRNN_OK;
  if (!x || !z || (y && !h)) return fail(PRNN_ERR_VALUE, "x, z and, with y, h must be non-null");
  RnArgs a{};
  a.x = x;
  a.y = y;
  a.w = w;
  a.b = b;
  a.pw = pw;
  a.gate = gate;
  a.scale = scale;
  a.h = h;
  a.z = z;
  a.N = N;
  a.C = C;
  a.layer = layer;
  a.post = post;
  a.act = act;
  a.w_dtype = w_dtype;
  a.number = scale_number;
  a.eps = eps;
  return rn_forward(a, dtype, vectors(C, dtype, {x, y, gate, h, z}), static_cast<hipStream_t>(stream));
}

extern "C" PRNN_API size_t prnn_residual_norm_backward_workspace_size(int N, int C) {
  return N < 1 || C < 1 || C > kRnMax ? 0 : parts_bytes(N, C);
}

extern "C" PRNN_API int prnn_residual_norm_backward(
    const void* gh, const void* gz, const void* x, const void* y, const void* w, const void* pw,
    const void* gate, const void* scale, float scale_number, void* dx, void* dy, void* dw, void* db,
    void* dpw, void* dgate, void* dscale, int N, int C, float eps, int layer, int post, int act,
    int w_dtype, int dtype, void* workspace, size_t bytes, void* stream) {
  if (int rc = check(N, C, eps, act, w_dtype, dtype)) return rc;
  if (N == 0) return PRNN_OK;
  if (!x || (!gh && !gz)) return fail(PRNN_ERR_VALUE, "x and one of gh and gz must be non-null");
  const size_t need = parts_bytes(N, C);
  const bool sums = dw || db || dpw || dscale;
  if (sums && (workspace == nullptr || bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(PRNN_ERR_VALUE, "the workspace must hold %zu bytes, 16-byte aligned (got %zu)", need, bytes);
  RnArgs a{};
  a.x = x;
  a.y = y;
  a.w = w;
  a.pw = pw;
  a.gate = gate;
  a.scale = scale;
  a.gh = gh;
  a.gz = gz;
  a.dx = dx;
  a.dy = dy;
  a.dgate = dgate;
  a.parts = sums ? static_cast<float*>(workspace) : nullptr;
  a.N = N;
  a.C = C;
  a.layer = layer;
  a.post = post;
  a.act = act;
  a.w_dtype = w_dtype;
  a.number = scale_number;
  a.eps = eps;
  a.want = (dw ? 1 : 0) | (db ? 2 : 0) | (dpw ? 4 : 0) | (dscale ? 8 : 0);
  const bool vec = vectors(C, dtype, {gh, gz, x, y, gate, dx, dy, dgate});
  const int groups = rn_groups(N, C, vec, dtype != PRNN_F32);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (int rc = rn_backward(a, dtype, vec, groups, st)) return rc;
  if (!sums) return PRNN_OK;
  return with_storage(dtype, [&](auto t) {
    const RnSums s{a.parts, {dw, db, dpw, dscale}, groups, C, w_dtype};
    rn_sum_kernel<decltype(t)><<<dim3((C + 63) / 64, 4), 1024, 0, st>>>(s);
    PRNN_HIP(hipGetLastError());
    return static_cast<int>(PRNN_OK);
  });
}
