// Gated delta rule: every chunk's triangular system and pairs, a workgroup per chunk and head.
//
// Three waves, one per tile of 32 x 32 of the lower triangle: k k^T and q k^T by rows straight from
// memory (no LDS: 16 bytes a lane are an operand), weighted by the exponentials of the decays'
// differences.  The unit triangular 1 + M is inverted in fp32: the four diagonal blocks of 16 by
// substitution, a column per lane of one wave; below them T_ij = -T_ii sum_m M_im T_mj in block
// columns, one per wave, on v_mfma_f32_16x16x4_f32 with the results as the next products' operands.
// (A product of powers (1 - M)(1 + M^2)(1 + M^4) .. has fewer steps, but the powers of keys that lie
// close together grow before they vanish.)
#include "delta_rule_loads.h"

namespace prnn {
namespace {

constexpr int kLd = 68;  // floats of a row in LDS

__device__ __forceinline__ bool not_finite(float v) {
  return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u;
}

template <class M, typename T>
__global__ __launch_bounds__(192) void dr_systems_kernel(DrSystems A) {
  using E = typename M::E;
  __shared__ __align__(16) float sM[kDrC * kLd], sT[kDrC * kLd];
  __shared__ float s_hi[kDrC], s_lo[kDrC], s_b[kDrC];
  __shared__ int s_stop;
  const int h = blockIdx.x % A.H, id = blockIdx.x / A.H;
  const DrUnit u = dr_unit(A.seqs, kDrC, id);
  if (!u.any || u.begin >= u.end) return;
  const int n = u.end - u.begin, batch = dr_batch(A.seqs, u);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
  char* sys = A.sys + (static_cast<size_t>(id) * A.H + h) * kDrSys;
  float* weights = reinterpret_cast<float*>(sys + 2 * kDrTiles);

  // ---- products: registers earlier tokens j, lanes later ones i (transposed pairs the other way)
  const int it = wave > 0, jt = wave > 1;
  auto rows = [&](const LaView& v) {
    return make_rsrc(static_cast<const T*>(v.p) + (batch * v.sb + (h / v.rep) * v.sh +
                                                   static_cast<long long>(u.begin) * v.st), 0x7fffffffu);
  };
  const rsrc_t rk = rows(A.k), rq = rows(A.q);
  const int ti = 32 * it + l32, tj = 32 * jt + l32;
  const uint32_t ki = ti * static_cast<int>(A.k.st) * sizeof(T), kj = tj * static_cast<int>(A.k.st) * sizeof(T),
                 qi = ti * static_cast<int>(A.q.st) * sizeof(T);
  if (tid == 0) s_stop = kDrC;
  f16v N, P;
#pragma unroll
  for (int r = 0; r < 16; ++r) N[r] = P[r] = 0.0f;
  bool bad = false;
  for (int c = 8 * half; c < A.Dk + 8 * half; c += 16) {
    const auto k1 = global_op<M, T>(rk, ti < n, ki, c, A.Dk), q1 = global_op<M, T>(rq, ti < n, qi, c, A.Dk);
    const auto k0 = global_op<M, T>(rk, tj < n, kj, c, A.Dk);
    mul<32>(N, k0, k1);
    if (A.transposed)
      mul<32>(P, q1, k0);
    else
      mul<32>(P, k0, q1);
    float x[8];
    values(k1, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) bad |= not_finite(x[i]);
  }
  float hi = 0.0f, lo = 0.0f, rate = 0.0f, back = 0.0f, whole = 0.0f;
  if (wave == 0) {
    const float g = lane < n ? la_decay(A.g, batch, u.begin + lane, h) : 0.0f;
    double G = g;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const double o = __shfl_up(G, k);
      if (lane >= k) G += o;
    }
    const double last = __shfl(G, 63);
    hi = static_cast<float>(G);
    lo = static_cast<float>(G - hi);
    back = static_cast<float>(last - G);
    whole = static_cast<float>(last);
    if (lane < n) rate = dr_rate(A.b, batch, u.begin + lane, h);
    s_hi[lane] = hi;
    s_lo[lane] = lo;
    s_b[lane] = rate;
    if (not_finite(g) | not_finite(rate)) atomicMin(&s_stop, lane);
  }
  __syncthreads();
  if (bad && it == jt) atomicMin(&s_stop, ti);
  if (wave == 0) {
    weights[kWg * 64 + lane] = fexp(hi);
    weights[kWr * 64 + lane] = fexp(back);
    weights[kWb * 64 + lane] = rate;
    weights[kWhi * 64 + lane] = hi;
    weights[kWlo * 64 + lane] = lo;
  }
  __syncthreads();
  const int stop = s_stop;
  if (wave == 0)
    weights[kWmeta * 64 + lane] = lane == 0 ? fexp(whole) : lane == 1 ? __int_as_float(stop) : 0.0f;

  // ---- weights; the system's matrix without what is not finite
  char* pairs = sys + kDrTiles + wave * (kDrTiles / 3 / M::kParts);
  const float Hi = s_hi[ti], Lo = s_lo[ti], Bi = s_b[ti];
  const float Hj = s_hi[tj], Lj = s_lo[tj];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int j = 32 * jt + 8 * q + 4 * half, i = 32 * it + 8 * q + 4 * half;
    f4 m, p;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float w = fexp((Hi - s_hi[j + r]) + (Lo - s_lo[j + r]));
      const float b = A.transposed ? Bi : s_b[j + r];
      m[r] = ((j + r < ti) & (ti < stop)) ? N[4 * q + r] * w * b : 0.0f;
      if (A.transposed) {  // lane: token j, registers: tokens i
        const float v = fexp((s_hi[i + r] - Hj) + (s_lo[i + r] - Lj));
        p[r] = tj <= i + r ? P[4 * q + r] * v * A.scale : 0.0f;
      } else {
        p[r] = j + r <= ti ? P[4 * q + r] * w * A.scale : 0.0f;
      }
    }
    *reinterpret_cast<f4*>(&sM[ti * kLd + j]) = m;
    const int unit = dr_unit_of<E>(l32, 2 * q + half);
    if constexpr (sizeof(E) == 2) {
      const u2 a{pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3])};
      const u2 b{pack_bf16x2(p[0] - lo_bf16(a[0]), p[1] - hi_bf16(a[0])),
                 pack_bf16x2(p[2] - lo_bf16(a[1]), p[3] - hi_bf16(a[1]))};
      *reinterpret_cast<u2*>(pairs + l32 * 64 + unit * 8) = a;
      *reinterpret_cast<u2*>(pairs + kDrTiles / 2 + l32 * 64 + unit * 8) = b;
    } else {
      *reinterpret_cast<f4*>(pairs + l32 * 128 + unit * 16) = p;
    }
  }
  __syncthreads();

  // ---- diagonal blocks
  if (wave == 0) {
    const int blk = lane >> 4, c = lane & 15;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == c ? 1.0f : 0.0f;
      const f4* row = reinterpret_cast<const f4*>(&sM[(16 * blk + i) * kLd + 16 * blk]);
#pragma unroll
      for (int j = 0; j < i; ++j) s = fmaf(-row[j >> 2][j & 3], x[j], s);
      x[i] = s;
      sT[(16 * blk + i) * kLd + 16 * blk + c] = s;
    }
  }
  __syncthreads();
  // ---- below them
  {
    const int c = lane & 15, g = lane >> 4;
    auto column = [&](auto first) {
      constexpr int J = decltype(first)::value;
      f4 X[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) X[J][r] = sT[(16 * J + 4 * g + r) * kLd + 16 * J + c];
#pragma unroll
      for (int i = J + 1; i < 4; ++i) {
        f4 sum{0, 0, 0, 0}, x{0, 0, 0, 0};
#pragma unroll
        for (int m = J; m < i; ++m) {
          const f4 a = *reinterpret_cast<const f4*>(&sM[(16 * i + c) * kLd + 16 * m + 4 * g]);
#pragma unroll
          for (int r = 0; r < 4; ++r) sum = mfma_f32<16>(a[r], X[m][r], sum);
        }
        const f4 t = *reinterpret_cast<const f4*>(&sT[(16 * i + c) * kLd + 16 * i + 4 * g]);
#pragma unroll
        for (int r = 0; r < 4; ++r) x = mfma_f32<16>(t[r], sum[r], x);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          X[i][r] = -x[r];
          sT[(16 * i + 4 * g + r) * kLd + 16 * J + c] = -x[r];
        }
      }
    };
    if (wave == 0) column(std::integral_constant<int, 0>{});
    if (wave == 1) column(std::integral_constant<int, 1>{});
    if (wave == 2) column(std::integral_constant<int, 2>{});
  }
  __syncthreads();

  // ---- the strictly triangular part of the inverse
  char* tiles = sys + wave * (kDrTiles / 3 / M::kParts);
  const int row = (A.transposed ? 32 * jt : 32 * it) + l32, col0 = A.transposed ? 32 * it : 32 * jt;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int unit = 4 * half + k, col = col0 + 4 * unit;
    f4 t;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float v = A.transposed ? sT[(col + r) * kLd + row] : sT[row * kLd + col + r];
      t[r] = (A.transposed ? col + r > row : col + r < row) ? v : 0.0f;
    }
    const int to = dr_unit_of<E>(l32, unit);
    if constexpr (sizeof(E) == 2) {
      const u2 a{pack_bf16x2(t[0], t[1]), pack_bf16x2(t[2], t[3])};
      const u2 b{pack_bf16x2(t[0] - lo_bf16(a[0]), t[1] - hi_bf16(a[0])),
                 pack_bf16x2(t[2] - lo_bf16(a[1]), t[3] - hi_bf16(a[1]))};
      *reinterpret_cast<u2*>(tiles + l32 * 64 + to * 8) = a;
      *reinterpret_cast<u2*>(tiles + kDrTiles / 2 + l32 * 64 + to * 8) = b;
    } else {
      *reinterpret_cast<f4*>(tiles + l32 * 128 + to * 16) = t;
    }
  }
}

template <class M, typename T>
int launch(const DrSystems& a, hipStream_t stream) {
  const long long groups = dr_units(a.seqs, kDrC) * a.H;
  if (int rc = check_grid("delta_rule", groups, 192)) return rc;
  dr_systems_kernel<M, T><<<static_cast<unsigned>(groups), 192, 0, stream>>>(a);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

}  // namespace

int dr_systems(const DrSystems& a, bool bf16_walk, hipStream_t stream) {
  if (bf16_walk) return launch<InBf16, bf16>(a, stream);
  return with_storage(a.dtype, [&](auto z) { return launch<InF32, decltype(z)>(a, stream); });
}

}  // namespace prnn
