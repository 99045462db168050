// Gated delta rule: every chunk's triangular system and pairs, a workgroup per chunk and head.
//
// Three waves, one per tile of 32 x 32 of the lower triangle: k k^T and q k^T, weighted by the
// exponentials of the decays' differences, which a fourth wave sums up.  Rows come through LDS: a load
// of operands straight from memory touches a line for every 32 bytes (12400 of 30000 cycles a system).
// The unit triangular 1 + M is inverted in fp32: the four diagonal blocks of 16 by substitution, a
// column per lane of one wave; below them T_ij = -T_ii sum_m M_im T_mj in block columns, one per wave,
// on v_mfma_f32_16x16x4_f32 with the results as the next products' operands.  (A product of powers
// (1 - M)(1 + M^2)(1 + M^4) .. has fewer steps, but the powers of keys that lie close together grow
// before they vanish.)
//
// Bound by what it moves and by its chain of phases, of which four workgroups a CU hide a part: 4096
// systems of bf16 keys of 64 in 54 us, 37 MB in and 104 MB out (of a workgroup's 16000 cycles 7000 are a
// wait for rows).  They are left in fp32, the walks' loading waves take them apart for bf16 products.
// Workgroups that go on to further chunks were slower: they hold the next rows in registers.
#include "delta_rule_loads.h"

namespace prnn {
namespace {

constexpr int kLd = 68;  // floats of a row in LDS

__device__ __forceinline__ bool not_finite(float v) {
  return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u;
}

constexpr int kLengths = 1024;  // that are told apart, in chunks
// Places of the pieces by their lengths, longest first, by counting.  Pieces of one length come in any
// order: it decides when they run, not what they give.
__device__ __forceinline__ void pieces_in_order(const DrSystems& A, int* count) {
  const int tid = threadIdx.x;
  auto place = [&](int i) {
    const DrUnit u = dr_unit(A.pieces, A.pieces.len, i);
    const int chunks = u.any ? (u.end - u.begin + kDrC - 1) / kDrC + 1 : 0;
    return kLengths - 1 - min(chunks, kLengths - 1);
  };
  for (int i = tid; i < kLengths; i += 256) count[i] = 0;
  __syncthreads();
  for (int i = tid; i < A.n_pieces; i += 256) atomicAdd(&count[place(i)], 1);
  __syncthreads();
  int own[kLengths / 256], sum = 0;
#pragma unroll
  for (int k = 0; k < kLengths / 256; ++k) {
    own[k] = sum;
    sum += count[tid * (kLengths / 256) + k];
  }
  // sums of the threads before: over the wave, then over the waves
  int before = sum;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(before, m);
    if ((tid & 63) >= m) before += o;
  }
  int* const waves = count + kLengths;
  if ((tid & 63) == 63) waves[tid >> 6] = before;
  __syncthreads();
  before -= sum;
  for (int w = 0; w < tid >> 6; ++w) before += waves[w];
#pragma unroll
  for (int k = 0; k < kLengths / 256; ++k) count[tid * (kLengths / 256) + k] = before + own[k];
  __syncthreads();
  for (int i = tid; i < A.n_pieces; i += 256) A.order[atomicAdd(&count[place(i)], 1)] = i;
}

template <class M>
__global__ __launch_bounds__(256) void dr_systems_kernel(DrSystems A) {
  using E = typename M::E;
  constexpr bool kNarrow = sizeof(E) == 2;
  constexpr int RB = dr_row_k(kNarrow, 64);
  __shared__ __align__(16) float lds[2 * kDrC * kLd];  // slabs of k and q, then the system and its inverse
  static_assert(2 * kDrC * RB <= static_cast<int>(sizeof(lds)), "slabs fit");
  __shared__ __align__(16) float s_hi[kDrC], s_lo[kDrC], s_b[kDrC];
  __shared__ float s_whole;
  __shared__ int s_stop;
  __shared__ bool s_bad[kDrC];
  float *const sM = lds, *const sT = lds + kDrC * kLd;
  char *const sK = reinterpret_cast<char*>(lds), *const sQ = sK + kDrC * RB;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
  const int it = wave > 0, jt = wave > 1;  // (the fourth wave's are not used)
  const int ti = 32 * it + l32, tj = 32 * jt + l32;

  static_assert((kLengths + 4) * 4 <= static_cast<int>(sizeof(lds)), "counts fit");
  if (A.order && blockIdx.x == 0) {  // a workgroup more, before the others
    pieces_in_order(A, reinterpret_cast<int*>(lds));
    return;
  }
  const int item = blockIdx.x - (A.order ? 1 : 0), h = item % A.H, id = item / A.H;
  const DrUnit u = dr_unit(A.seqs, kDrC, id);
  if (!u.any || u.begin >= u.end) return;
  const int n = u.end - u.begin, batch = dr_batch(A.seqs, u);
  auto rows = [&](const LaView& v) {
    return static_cast<const char*>(v.p) +
           (batch * v.sb + (h / v.rep) * v.sh + static_cast<long long>(u.begin) * v.st) * (A.dtype == PRNN_F32 ? 4 : 2);
  };
  const char *pk = rows(A.k), *pq = rows(A.q);
  Staged<M, 64, 256> rk, rq;
  rk.fetch(pk, A.k.st, n, 0, A.Dk, A.dtype);
  rq.fetch(pq, A.q.st, n, 0, A.Dk, A.dtype);
  float g = 0.0f, rate = 0.0f;
  if (wave == 3 && lane < n) {
    g = la_decay(A.g, batch, u.begin + lane, h);
    rate = dr_rate(A.b, batch, u.begin + lane, h);
  }
  char* sys = A.sys + (static_cast<size_t>(id) * A.H + h) * kDrSys;
  float* weights = reinterpret_cast<float*>(sys + 2 * kDrTiles);
  // ---- products: registers earlier tokens j, lanes later ones i
  if (tid == 0) s_stop = kDrC;
  f16v N, P;
#pragma unroll
  for (int r = 0; r < 16; ++r) N[r] = P[r] = 0.0f;
  if (wave == 3) {
    double G = g;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const double o = __shfl_up(G, k);
      if (lane >= k) G += o;
    }
    const double last = __shfl(G, 63);
    const float hi = static_cast<float>(G), lo = static_cast<float>(G - hi);
    s_hi[lane] = hi;
    s_lo[lane] = lo;
    s_b[lane] = rate;
    weights[kWg * 64 + lane] = fexp(hi);
    weights[kWr * 64 + lane] = fexp(static_cast<float>(last - G));
    weights[kWb * 64 + lane] = rate;
    weights[kWhi * 64 + lane] = hi;
    weights[kWlo * 64 + lane] = lo;
    s_bad[lane] = not_finite(g) | not_finite(rate);
    if (lane == 0) s_whole = fexp(static_cast<float>(last));
  }
  bool bad = false;
  for (int c0 = 0; c0 < A.Dk; c0 += 64) {
    if (c0 > 0) __syncthreads();
    rk.template put<RB>(sK, A.dtype);
    rq.template put<RB>(sQ, A.dtype);
    __syncthreads();
    if (c0 + 64 < A.Dk) {
      rk.fetch(pk, A.k.st, n, c0 + 64, A.Dk, A.dtype);
      rq.fetch(pq, A.q.st, n, c0 + 64, A.Dk, A.dtype);
    }
    if (wave < 3) {
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const auto k0 = row_op<M, 2>(sK + tj * RB, f, half), k1 = row_op<M, 2>(sK + ti * RB, f, half);
        const auto q1 = row_op<M, 2>(sQ + ti * RB, f, half);
        mul<32>(N, k0, k1);
        mul<32>(P, k0, q1);
        float x[8];
        values(k1, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) bad |= not_finite(x[i]);
      }
    }
  }
  if (bad && it == jt && wave < 3) atomicMin(&s_stop, ti);
  if (wave == 3 && s_bad[lane]) atomicMin(&s_stop, lane);
  __syncthreads();
  const int stop = s_stop;
  if (wave == 3)
    weights[kWmeta * 64 + lane] = lane == 0 ? s_whole : lane == 1 ? __int_as_float(stop) : 0.0f;

  // ---- weights; the system's matrix without what is not finite
  if (wave < 3) {
    char* pairs = sys + kDrTiles + wave * (kDrTiles / 3);
    const float Hi = s_hi[ti], Lo = s_lo[ti];
    auto four = [](const float* v) { return *reinterpret_cast<const f4*>(v); };
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = 32 * jt + 8 * q + 4 * half;
      const f4 hj = four(s_hi + j), lj = four(s_lo + j), bj = four(s_b + j);
      f4 m, p;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float w = fexp((Hi - hj[r]) + (Lo - lj[r]));
        m[r] = ((j + r < ti) & (ti < stop)) ? N[4 * q + r] * w * bj[r] : 0.0f;
        p[r] = j + r <= ti ? P[4 * q + r] * w * A.scale : 0.0f;
      }
      *reinterpret_cast<f4*>(&sM[ti * kLd + j]) = m;
      *reinterpret_cast<f4*>(pairs + l32 * 128 + dr_unit_of(l32, 2 * q + half) * 16) = p;
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
  if (wave < 3) {
    char* tiles = sys + wave * (kDrTiles / 3);
    const int row = 32 * it + l32;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int unit = 4 * half + k, col = 32 * jt + 4 * unit;
      const f4 w = *reinterpret_cast<const f4*>(&sT[row * kLd + col]);
      f4 t;
#pragma unroll
      for (int r = 0; r < 4; ++r) t[r] = col + r < row ? w[r] : 0.0f;
      *reinterpret_cast<f4*>(tiles + l32 * 128 + dr_unit_of(l32, unit) * 16) = t;
    }
  }
}

template <class M>
int launch(const DrSystems& a, hipStream_t stream) {
  const long long groups = dr_units(a.seqs, kDrC) * a.H + (a.order ? 1 : 0);
  if (int rc = check_grid("delta_rule", groups, 256)) return rc;
  dr_systems_kernel<M><<<static_cast<unsigned>(groups), 256, 0, stream>>>(a);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

}  // namespace

int dr_systems(const DrSystems& a, bool bf16_walk, hipStream_t stream) {
  return bf16_walk ? launch<InBf16>(a, stream) : launch<InF32>(a, stream);
}

}  // namespace prnn
