// Decayed linear attention, one token: S <- exp(g) S + k v^T in place, o = scale q^T S.
//
// Bound by the state's traffic (read once, written once: 8 bytes an element against 4 flops).
// A workgroup takes TJ columns of one head's state: L lanes of four columns side by side, the
// rows spread over 256 / L groups of lanes, so every access is 16 bytes a lane and a thread has
// U of its rows' loads in flight, and the next U's while these are worked on.
//
// 256 sessions of 16 heads of (128, 128) on a pool: 112 us, 4.8 TB/s (a large copy: 5.1); one
// session of 8 heads of (64, 64): 4.5 us on the GPU, a launch's own time.
#include "linear_attention.h"

namespace prnn {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct StepArgs {
  LaView q, k, v;
  LaDecay g;
  void* out;
  long long o_sb, o_sh;
  float* state;
  const int* table;
  int rows;
  int H, Dk, Dv;
  float scale;
};

// L lanes x 4 columns, U rows of a thread at a time.  What lies outside the head is read as zero and not written (an offset
// outside the resource).
template <typename T, int L, int U, bool VEC>
__global__ __launch_bounds__(256) void la_step_kernel(StepArgs A) {
  constexpr int G = 256 / L;  // rows at a time
  __shared__ float sq[kLaMaxDim], sk[kLaMaxDim];
  __shared__ __align__(16) float so[256 * 4];
  const int tid = threadIdx.x, lane = tid % L, grp = tid / L;
  const int h = blockIdx.y, b = blockIdx.z;
  const int c0 = (blockIdx.x * L + lane) * 4;
  const int r = A.table ? A.table[b] : b;
  const bool kept = r >= 0 && r < A.rows;
  const rsrc_t S = make_rsrc(
      A.state + (static_cast<size_t>(kept ? r : 0) * A.H + h) * A.Dk * A.Dv,
      kept ? static_cast<uint32_t>(A.Dk * A.Dv) * 4 : 0u);
  auto offset = [&](int i, int c) {
    return i < A.Dk && c0 + c < A.Dv ? static_cast<uint32_t>(i * A.Dv + c0 + c) * 4 : kOOB;
  };
  auto load = [&](f4* s, int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * G;
      if (VEC) {
        s[u] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(S, offset(i, 0), 0, 0));
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) s[u][c] = ldb<float>(S, offset(i, c), 0);
      }
    }
  };
  f4 s[U];
  load(s, grp);
  const T* q = static_cast<const T*>(A.q.p) + b * A.q.sb + (h / A.q.rep) * A.q.sh;
  const T* k = static_cast<const T*>(A.k.p) + b * A.k.sb + (h / A.k.rep) * A.k.sh;
  const T* v = static_cast<const T*>(A.v.p) + b * A.v.sb + (h / A.v.rep) * A.v.sh;
  for (int i = tid; i < A.Dk; i += 256) {
    sq[i] = to_f32(q[i]);
    sk[i] = to_f32(k[i]);
  }
  const float a = fexp(la_decay(A.g, b, 0, h));
  f4 vv = {0, 0, 0, 0};
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c0 + c < A.Dv) vv[c] = to_f32(v[c0 + c]);
  f4 o = {0, 0, 0, 0};
  __syncthreads();
  for (int i0 = grp; i0 < A.Dk; i0 += G * U) {
    f4 n[U];
    load(n, i0 + G * U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * G;
      const float ki = i < A.Dk ? sk[i] : 0.0f, qi = i < A.Dk ? sq[i] : 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[u][c] = fmaf(a, s[u][c], ki * vv[c]);
        if (i < A.Dk) o[c] = fmaf(qi, s[u][c], o[c]);
      }
      if (VEC) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, s[u]), S, offset(i, 0), 0, 0);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) stb<float>(S, offset(i, c), 0, s[u][c]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = n[u];
  }
  *reinterpret_cast<f4*>(&so[tid * 4]) = o;
  __syncthreads();
  // column j of the tile: the groups' sums in their order
  for (int j = tid; j < 4 * L; j += 256) {
    float x = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) x += so[g * 4 * L + j];
    const int col = blockIdx.x * 4 * L + j;
    if (col < A.Dv)
      static_cast<T*>(A.out)[b * A.o_sb + h * A.o_sh + col] = from_f32<T>(x * A.scale);
  }
}

template <typename T, int L, int U>
int launch(const StepArgs& a, int B, bool vec, hipStream_t st) {
  const dim3 grid((a.Dv + 4 * L - 1) / (4 * L), a.H, B);
  if (vec)
    la_step_kernel<T, L, U, true><<<grid, 256, 0, st>>>(a);
  else
    la_step_kernel<T, L, U, false><<<grid, 256, 0, st>>>(a);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

}  // namespace
}  // namespace prnn

using namespace prnn;

extern "C" PRNN_API int prnn_linear_attention_step(
    const void* q, long long q_sb, long long q_sh, int q_heads, const void* k, long long k_sb,
    long long k_sh, int k_heads, const void* v, long long v_sb, long long v_sh, int v_heads,
    const void* g, long long g_sb, long long g_sh, int g_dtype, float* state,
    const int* block_table, int rows, void* out, int B, int H, int Dk, int Dv, float scale,
    int dtype, void* stream) {
  if (int rc = check_dtype(dtype)) return rc;
  if (g_dtype != PRNN_F32 && g_dtype != dtype)
    return fail(PRNN_ERR_TYPE, "log_decay must be float32 or of the storage type");
  if (B < 0 || B > 65535 || H < 1 || H > 65535)
    return fail(PRNN_ERR_VALUE, "B=%d, H=%d are not in 0 .. 65535", B, H);
  if (Dk < 1 || Dk > kLaMaxDim || Dv < 1 || Dv > kLaMaxDim)
    return fail(PRNN_ERR_VALUE, "head widths (%d, %d) are not in 1 .. %d", Dk, Dv, kLaMaxDim);
  for (int heads : {q_heads, k_heads, v_heads})
    if (heads < 1 || H % heads)
      return fail(PRNN_ERR_VALUE, "%d heads do not divide H=%d", heads, H);
  if (B == 0) return PRNN_OK;
  if (!q || !k || !v || !g || !state || !out)
    return fail(PRNN_ERR_VALUE, "q, k, v, log_decay, state and out must be non-null");
  StepArgs a{};
  a.q = LaView{q, q_sb, 0, q_sh, H / q_heads, 0};
  a.k = LaView{k, k_sb, 0, k_sh, H / k_heads, 0};
  a.v = LaView{v, v_sb, 0, v_sh, H / v_heads, 0};
  a.g = LaDecay{g, g_sb, 0, g_sh, g_dtype};
  a.out = out;
  a.o_sb = static_cast<long long>(H) * Dv;
  a.o_sh = Dv;
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
    // Narrow tiles (more workgroups) for few heads, whole rows of a head side by side for many.
    // Of 8, 16 and 32 lanes, us: (128, 128) 64 heads 4.4, 4.9, 6.2; 128 heads 5.1, 5.6, 6.8; 256
    // heads 7.6, 7.0, 7.6; 512 heads 11.0, 9.9, 9.8; 4096 heads 93, 85, 81.  (64, 64) 8 heads 3.8,
    // 3.8, 4.8; 512 heads 5.9, 5.0, 5.8; 4096 heads 29, 25, 30.  (32, 32) 4096 heads 13, 13, 20.
    const long long heads = 1ll * B * H;
    if (Dv <= 32 || heads <= 128) return launch<T, 8, 4>(a, B, vec, st);
    if (Dv <= 64 || heads < 512) return launch<T, 16, 4>(a, B, vec, st);
    return launch<T, 32, 8>(a, B, vec, st);
  });
}
