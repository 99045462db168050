// Gated delta rule, one token, in place:
//   u = b (v - a S^T k),   S <- a S + k u^T,   o = scale S^T q = scale (a S^T q + (k . q) u),  a = exp(g).
//
// Bound by the state's traffic (read once, written once).  A workgroup takes 4 L columns of a head's
// state and keeps them: L lanes of four columns side by side, the rows spread over 256 / L groups of
// lanes, U rows a thread in registers.  One pass forms S^T k and S^T q; their sums over the groups
// give u and o, then the rows go back.  256 sessions of 16 heads, D = 128: 537 MB in 87 us on a pool that
// the last call has touched (half of it is still in the last-level cache), 117 otherwise (4.6 TB/s); one
// session of 8 heads 4.8 us, a launch's own time.
#include "linear_attention.h"

namespace prnn {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct StepArgs {
  LaView q, k, v;
  LaDecay g, b;
  void* out;
  float* state;
  const int* table;
  int rows;
  int H, Dk, Dv;
  float scale;
};

template <typename T, int L, int U, bool VEC>
__global__ __launch_bounds__(256) void dr_step_kernel(StepArgs A) {
  constexpr int G = 256 / L;
  __shared__ float sq[kLaMaxDim], sk[kLaMaxDim];
  __shared__ __align__(16) float s_k[4][4 * L], s_q[4][4 * L], s_kq[4];
  const int tid = threadIdx.x, lane = tid % L, grp = tid / L, wave = tid >> 6;
  const int h = blockIdx.y, b = blockIdx.z;
  const int c0 = (blockIdx.x * L + lane) * 4;
  const int r = A.table ? A.table[b] : b;
  const bool kept = r >= 0 && r < A.rows;
  const rsrc_t S = make_rsrc(A.state + (static_cast<size_t>(kept ? r : 0) * A.H + h) * A.Dk * A.Dv,
                             kept ? static_cast<uint32_t>(A.Dk * A.Dv) * 4 : 0u);
  auto offset = [&](int i, int c) {
    return i < A.Dk && c0 + c < A.Dv ? static_cast<uint32_t>(i * A.Dv + c0 + c) * 4 : kOOB;
  };
  f4 s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = grp + u * G;
    if (VEC) {
      s[u] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(S, offset(i, 0), 0, 0));
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) s[u][c] = ldb<float>(S, offset(i, c), 0);
    }
  }
  const T* q = static_cast<const T*>(A.q.p) + b * A.q.sb + (h / A.q.rep) * A.q.sh;
  const T* k = static_cast<const T*>(A.k.p) + b * A.k.sb + (h / A.k.rep) * A.k.sh;
  const T* v = static_cast<const T*>(A.v.p) + b * A.v.sb + (h / A.v.rep) * A.v.sh;
  float kq = 0.0f;
  {
    const bool in = tid < A.Dk;
    const float qi = in ? to_f32(q[tid]) : 0.0f, ki = in ? to_f32(k[tid]) : 0.0f;
    sq[tid] = qi;
    sk[tid] = ki;
    kq = qi * ki;
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) kq += __shfl_xor(kq, m);
  if ((tid & 63) == 0) s_kq[wave] = kq;
  const float a = fexp(la_decay(A.g, b, 0, h));
  const uint32_t rate_bits = la_decay_bits(A.b, b, 0, h);
  const float rate = A.b.dtype == PRNN_F32   ? __uint_as_float(rate_bits)
                     : A.b.dtype == PRNN_F16 ? Narrow<f16>::val(rate_bits)
                                             : Narrow<bf16>::val(rate_bits);
  f4 vv = {0, 0, 0, 0};
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c0 + c < A.Dv) vv[c] = to_f32(v[c0 + c]);
  __syncthreads();
  f4 xk = {0, 0, 0, 0}, xq = {0, 0, 0, 0};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = grp + u * G;
    if (i < A.Dk) {
      const float ki = sk[i], qi = sq[i];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        xk[c] = fmaf(ki, s[u][c], xk[c]);
        xq[c] = fmaf(qi, s[u][c], xq[c]);
      }
    }
  }
  // over the wave's groups, then over the waves, in a fixed order
#pragma unroll
  for (int m = L; m < 64; m <<= 1)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      xk[c] += __shfl_xor(xk[c], m);
      xq[c] += __shfl_xor(xq[c], m);
    }
  if ((tid & 63) < L) {
    *reinterpret_cast<f4*>(&s_k[wave][4 * lane]) = xk;
    *reinterpret_cast<f4*>(&s_q[wave][4 * lane]) = xq;
  }
  __syncthreads();
  kq = (s_kq[0] + s_kq[1]) + (s_kq[2] + s_kq[3]);
  f4 w;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int j = 4 * lane + c;
    const float sk4 = (s_k[0][j] + s_k[1][j]) + (s_k[2][j] + s_k[3][j]);
    const float sq4 = (s_q[0][j] + s_q[1][j]) + (s_q[2][j] + s_q[3][j]);
    w[c] = rate * fmaf(-a, sk4, vv[c]);
    xq[c] = A.scale * fmaf(kq, w[c], a * sq4);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = grp + u * G;
    const float ki = i < A.Dk ? sk[i] : 0.0f;
#pragma unroll
    for (int c = 0; c < 4; ++c) s[u][c] = fmaf(ki, w[c], a * s[u][c]);
    if (VEC) {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, s[u]), S, offset(i, 0), 0, 0);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) stb<float>(S, offset(i, c), 0, s[u][c]);
    }
  }
  if (grp == 0) {
    T* o = static_cast<T*>(A.out) + (static_cast<size_t>(b) * A.H + h) * A.Dv;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c0 + c < A.Dv) o[c0 + c] = from_f32<T>(xq[c]);
  }
}

template <typename T, int L, int U>
int launch(const StepArgs& a, int B, bool vec, hipStream_t st) {
  const dim3 grid((a.Dv + 4 * L - 1) / (4 * L), a.H, B);
  if (vec)
    dr_step_kernel<T, L, U, true><<<grid, 256, 0, st>>>(a);
  else
    dr_step_kernel<T, L, U, false><<<grid, 256, 0, st>>>(a);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

// The rows that a thread keeps, enough for all Dk.
template <typename T, int L>
int launch_rows(const StepArgs& a, int B, bool vec, hipStream_t st) {
  constexpr int G = 256 / L;
  if (a.Dk <= 2 * G) return launch<T, L, 2>(a, B, vec, st);
  if (a.Dk <= 4 * G) return launch<T, L, 4>(a, B, vec, st);
  if (L > 8 && a.Dk <= 8 * G) return launch<T, L, (L > 8 ? 8 : 4)>(a, B, vec, st);
  if (L > 16 && a.Dk <= 16 * G) return launch<T, L, (L > 16 ? 16 : 4)>(a, B, vec, st);
  return launch<T, L, kLaMaxDim / G>(a, B, vec, st);
}

}  // namespace
}  // namespace prnn

using namespace prnn;

extern "C" PRNN_API int prnn_delta_rule_step(
    const void* q, long long q_sb, long long q_sh, int q_heads, const void* k, long long k_sb,
    long long k_sh, int k_heads, const void* v, long long v_sb, long long v_sh, int v_heads,
    const void* g, long long g_sb, long long g_sh, int g_dtype, const void* beta, long long b_sb,
    long long b_sh, int b_dtype, float* state, const int* block_table, int rows, void* out, int B,
    int H, int Dk, int Dv, float scale, int dtype, void* stream) {
  if (int rc = check_dtype(dtype)) return rc;
  if (g_dtype != PRNN_F32 && g_dtype != dtype)
    return fail(PRNN_ERR_TYPE, "log_decay must be float32 or of the storage type");
  if (b_dtype != PRNN_F32 && b_dtype != dtype)
    return fail(PRNN_ERR_TYPE, "beta must be float32 or of the storage type");
  if (B < 0 || B > 65535 || H < 1 || H > 65535)
    return fail(PRNN_ERR_VALUE, "B=%d, H=%d are not in 0 .. 65535", B, H);
  if (Dk < 1 || Dk > kLaMaxDim || Dv < 1 || Dv > kLaMaxDim)
    return fail(PRNN_ERR_VALUE, "head widths (%d, %d) are not in 1 .. %d", Dk, Dv, kLaMaxDim);
  for (int heads : {q_heads, k_heads, v_heads})
    if (heads < 1 || H % heads)
      return fail(PRNN_ERR_VALUE, "%d heads do not divide H=%d", heads, H);
  if (B == 0) return PRNN_OK;
  if (!q || !k || !v || !g || !beta || !state || !out)
    return fail(PRNN_ERR_VALUE, "q, k, v, log_decay, beta, state and out must be non-null");
  StepArgs a{};
  a.q = LaView{q, q_sb, 0, q_sh, H / q_heads, 0};
  a.k = LaView{k, k_sb, 0, k_sh, H / k_heads, 0};
  a.v = LaView{v, v_sb, 0, v_sh, H / v_heads, 0};
  a.g = LaDecay{g, g_sb, 0, g_sh, g_dtype};
  a.b = LaDecay{beta, b_sb, 0, b_sh, b_dtype};
  a.out = out;
  a.state = state;
  a.table = block_table;
  a.rows = rows;
  a.H = H;
  a.Dk = Dk;
  a.Dv = Dv;
  a.scale = scale;
  const bool vec = Dv % 4 == 0 && (reinterpret_cast<uintptr_t>(state) & 15) == 0;
  return with_storage(dtype, [&](auto z) {
    using T = decltype(z);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    // narrow tiles (more workgroups) for few heads, whole rows of a head side by side for many
    const long long heads = 1ll * B * H;
    if (Dv <= 32 || heads <= 128) return launch_rows<T, 8>(a, B, vec, st);
    if (Dv <= 64 || heads < 512) return launch_rows<T, 16>(a, B, vec, st);
    return launch_rows<T, 32>(a, B, vec, st);
  });
}
