// Gated delta rule: the gradients of q, k, the log decays and the rates, a workgroup per chunk and
// head, all chunks at once (the walks leave the states before the chunks and the adjoints behind).
//
// 1. Pairs of tokens, a tile of 32 x 32 of the lower triangle per wave, rows straight from memory:
//    go u^T, dv u^T, q k^T, k k^T; with the decays' weights the first two go to LDS as operands.
// 2. dq and dk in tiles of 32 columns and 32 tokens, formed transposed (lane: token).
// 3. dL/dg_t is the flow through the decay of token t,
//      F_t = sum over sources j < t and uses l >= t of what l reads of j,
//    where a source may also be the state before the chunk and a use the adjoint behind it.  It is
//    summed as that double sum and not as a running difference of gains and losses: behind a strong
//    decay the flow is a tiny part of either.
#include "delta_rule_loads.h"

namespace prnn {
namespace {

constexpr int kSlab = 64;  // columns of k and q in LDS at a time
constexpr int kLf = 65;    // floats of a row of the flow's matrix

template <class M, typename T>
__global__ __launch_bounds__(256) void dr_grad_kernel(DrGrad A) {
  using E = typename M::E;
  using D = std::conditional_t<sizeof(E) == 2, bf16, float>;  // dense arrays
  constexpr bool kNarrow = sizeof(E) == 2;
  constexpr int ES = static_cast<int>(sizeof(E));
  constexpr int RW = dr_row_z(kNarrow, 64), RK = dr_row_k(kNarrow, kSlab), P = M::kParts;
  __shared__ __align__(16) char sW1[P][kDrC * RW], sX[P][kDrC * RW];
  __shared__ __align__(16) char sK[kDrC * RK], sQ[kDrC * RK];
  __shared__ float sF[kDrC * kLf], s_in[8][kDrC], s_out[8][kDrC];
  __shared__ __align__(16) float sw[kDrW * 64];
  __shared__ float s_through;
  const int h = blockIdx.x % A.H, id = blockIdx.x / A.H;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
  const DrUnit u = dr_unit(A.seqs, kDrC, id);
  if (!u.any || u.begin >= u.end) {
    if (A.g_part && tid == 0) A.g_part[static_cast<size_t>(id) * A.H + h] = 0.0f;
    return;
  }
  const int n = u.end - u.begin, batch = dr_batch(A.seqs, u);
  const size_t tok0 = dr_token(A.seqs, u, u.begin);
  const size_t unit = static_cast<size_t>(id) * A.H + h;
  const float* weights = reinterpret_cast<const float*>(A.sys + unit * kDrSys + 2 * kDrTiles);
  for (int i = tid; i < kDrW * 64; i += 256) sw[i] = weights[i];

  auto rows = [&](const LaView& v) {
    return make_rsrc(static_cast<const T*>(v.p) + (batch * v.sb + (h / v.rep) * v.sh +
                                                   static_cast<long long>(u.begin) * v.st), 0x7fffffffu);
  };
  auto dense = [&](const void* p, int width) {
    return make_rsrc(static_cast<const D*>(p) + (tok0 * A.H + h) * width, 0x7fffffffu);
  };
  auto state = [&](const void* p) {
    return make_rsrc(static_cast<const D*>(p) + unit * A.Dk * A.Dv, static_cast<uint32_t>(A.Dk * A.Dv) * ES);
  };
  const rsrc_t rq = rows(A.q), rk = rows(A.k), rg = rows(A.go);
  const rsrc_t re = dense(A.e, A.Dv), rd = dense(A.dv, A.Dv);
  const rsrc_t rS = state(A.before), rR = state(A.behind);
  const int TS = static_cast<int>(sizeof(T)), row_e = A.H * A.Dv * ES;
  const bool flow = A.dg || A.g_part;
  __syncthreads();

  // ---- 1
  if (wave < 3) {
    const int it = wave > 0, jt = wave > 1, i = 32 * it + l32, j = 32 * jt + l32;
    f16v GU, DU, QK, KK;
#pragma unroll
    for (int r = 0; r < 16; ++r) GU[r] = DU[r] = QK[r] = KK[r] = 0.0f;
    for (int c = 8 * half; c < A.Dv + 8 * half; c += 16) {
      const auto ej = global_op<M, D>(re, j < n, j * row_e, c, A.Dv);
      mul<32>(GU, ej, global_op<M, T>(rg, i < n, i * static_cast<int>(A.go.st) * TS, c, A.Dv));
      mul<32>(DU, ej, global_op<M, D>(rd, i < n, i * row_e, c, A.Dv));
    }
    if (flow)
      for (int c = 8 * half; c < A.Dk + 8 * half; c += 16) {
        const auto kj = global_op<M, T>(rk, j < n, j * static_cast<int>(A.k.st) * TS, c, A.Dk);
        mul<32>(QK, kj, global_op<M, T>(rq, i < n, i * static_cast<int>(A.q.st) * TS, c, A.Dk));
        mul<32>(KK, kj, global_op<M, T>(rk, i < n, i * static_cast<int>(A.k.st) * TS, c, A.Dk));
      }
    const float Hi = sw[kWhi * 64 + i], Lo = sw[kWlo * 64 + i];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float w1[4], x[4];
      const int j0 = 32 * jt + 8 * q + 4 * half;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int jj = j0 + r, e = 4 * q + r;
        const float w = fexp((Hi - sw[kWhi * 64 + jj]) + (Lo - sw[kWlo * 64 + jj])) * sw[kWb * 64 + jj];
        w1[r] = jj <= i ? w * A.scale * GU[e] : 0.0f;
        x[r] = jj < i ? w * DU[e] : 0.0f;
        sF[jj * kLf + i] = jj < i ? QK[e] * w1[r] - KK[e] * x[r] : 0.0f;
      }
      if constexpr (kNarrow) {
        const u2 a{pack_bf16x2(w1[0], w1[1]), pack_bf16x2(w1[2], w1[3])};
        const u2 b{pack_bf16x2(w1[0] - lo_bf16(a[0]), w1[1] - hi_bf16(a[0])),
                   pack_bf16x2(w1[2] - lo_bf16(a[1]), w1[3] - hi_bf16(a[1]))};
        *reinterpret_cast<u2*>(sW1[0] + i * RW + j0 * 2) = a;
        *reinterpret_cast<u2*>(sW1[P - 1] + i * RW + j0 * 2) = b;
      } else {
        *reinterpret_cast<f4*>(sW1[0] + i * RW + j0 * 4) = f4{w1[0], w1[1], w1[2], w1[3]};
      }
      // -(X + X^T): either triangle from the one value
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int jj = j0 + r;
        if (jj > i) continue;
        if constexpr (kNarrow) {
          const bf16 a = from_f32<bf16>(-x[r]), b = from_f32<bf16>(-x[r] - to_f32(a));
          *reinterpret_cast<bf16*>(sX[0] + i * RW + jj * 2) = a;
          *reinterpret_cast<bf16*>(sX[0] + jj * RW + i * 2) = a;
          *reinterpret_cast<bf16*>(sX[P - 1] + i * RW + jj * 2) = b;
          *reinterpret_cast<bf16*>(sX[P - 1] + jj * RW + i * 2) = b;
        } else {
          *reinterpret_cast<float*>(sX[0] + i * RW + jj * 4) = -x[r];
          *reinterpret_cast<float*>(sX[0] + jj * RW + i * 4) = -x[r];
        }
      }
    }
  } else {
    // the rates' gradient: the walk's columns in their order
    if (A.dbeta && lane < n) {
      float d = 0.0f;
      for (int t = 0; t < A.db_tiles; ++t) d += A.db[(static_cast<size_t>(t) * A.tokens + tok0 + lane) * A.H + h];
      const size_t at = (tok0 + lane) * A.H + h;
      if (A.b_dtype == PRNN_F32)
        static_cast<float*>(A.dbeta)[at] = d;
      else if (A.b_dtype == PRNN_F16)
        static_cast<f16*>(A.dbeta)[at] = from_f32<f16>(d);
      else
        static_cast<bf16*>(A.dbeta)[at] = from_f32<bf16>(d);
    }
    if (flow) {  // from the state before to the adjoint behind
      float d = 0.0f;
      for (int e = lane * 8; e < A.Dk * A.Dv; e += 512) {
        float a[8], b[8];
        values(global_op<M, D>(rS, true, 0, e, A.Dk * A.Dv), a);
        values(global_op<M, D>(rR, true, 0, e, A.Dk * A.Dv), b);
#pragma unroll
        for (int i = 0; i < 8; ++i) d = fmaf(a[i], b[i], d);
      }
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) d += __shfl_xor(d, m);
      if (lane == 0) s_through = d * sw[kWmeta * 64];
    }
  }

  // ---- 2
  const int kt = wave & 1, it = wave >> 1, i = 32 * it + l32;
  const float wg = sw[kWg * 64 + i], wr = sw[kWr * 64 + i] * sw[kWb * 64 + i];
  for (int c0 = 0; c0 < A.Dk; c0 += kSlab) {
    {
      Staged<M, kSlab, 256> k, q;
      constexpr int kCode = kNarrow ? PRNN_BF16 : std::is_same_v<T, float> ? PRNN_F32
                            : std::is_same_v<T, f16>                       ? PRNN_F16
                                                                           : PRNN_BF16;
      auto at = [&](const LaView& v) {
        return reinterpret_cast<const char*>(static_cast<const T*>(v.p) + (batch * v.sb + (h / v.rep) * v.sh +
                                                                           static_cast<long long>(u.begin) * v.st));
      };
      k.fetch(at(A.k), A.k.st, n, c0, A.Dk, kCode);
      q.fetch(at(A.q), A.q.st, n, c0, A.Dk, kCode);
      __syncthreads();  // the pairs are there; the last slab has been read
      k.template put<RK>(sK, kCode);
      q.template put<RK>(sQ, kCode);
    }
    __syncthreads();
    const int row = c0 + 32 * kt + l32;
    f16v dq, du, ds;
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[r] = du[r] = ds[r] = 0.0f;
    if (c0 + 32 * kt < A.Dk) {
      const bool in = row < A.Dk;
      const uint32_t at = row * A.Dv * ES;
      for (int c = 8 * half; c < A.Dv + 8 * half; c += 16) {
        const auto s = global_op<M, D>(rS, in, at, c, A.Dv), r = global_op<M, D>(rR, in, at, c, A.Dv);
        mul<32>(dq, s, global_op<M, T>(rg, i < n, i * static_cast<int>(A.go.st) * TS, c, A.Dv));
        mul<32>(du, r, global_op<M, D>(re, i < n, i * row_e, c, A.Dv));
        mul<32>(ds, s, global_op<M, D>(rd, i < n, i * row_e, c, A.Dv));
      }
      float in_sum = 0.0f, out_sum = 0.0f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = 32 * kt + 8 * q + 4 * half;
        float qv[4], kv[4];
        if constexpr (kNarrow) {
          const u2 a = *reinterpret_cast<const u2*>(sQ + i * RK + col * 2);
          const u2 b = *reinterpret_cast<const u2*>(sK + i * RK + col * 2);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            qv[r] = r & 1 ? hi_bf16(a[r >> 1]) : lo_bf16(a[r >> 1]);
            kv[r] = r & 1 ? hi_bf16(b[r >> 1]) : lo_bf16(b[r >> 1]);
          }
        } else {
          const f4 a = *reinterpret_cast<const f4*>(sQ + i * RK + col * 4);
          const f4 b = *reinterpret_cast<const f4*>(sK + i * RK + col * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            qv[r] = a[r];
            kv[r] = b[r];
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int e = 4 * q + r;
          dq[e] *= wg * A.scale;
          ds[e] *= wg;
          du[e] *= wr;
          in_sum = fmaf(qv[r], dq[e], fmaf(-kv[r], ds[e], in_sum));
          out_sum = fmaf(kv[r], du[e], out_sum);
          du[e] -= ds[e];
        }
      }
      in_sum += __shfl_xor(in_sum, 32);
      out_sum += __shfl_xor(out_sum, 32);
      if (half == 0) {
        s_in[c0 / 32 + kt][i] = in_sum;
        s_out[c0 / 32 + kt][i] = out_sum;
      }
      const char* kat = sK + 32 * kt * ES + col_share<M, 2, RK>(lane);
      const char* qat = sQ + 32 * kt * ES + col_share<M, 2, RK>(lane);
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int jt = f >> 1;
        const auto kc = col_op<M, 2, RK>(kat, 16 * f, 0);
        Op<M, P> x;
        auto both = [&](auto&& get) {
#pragma unroll
          for (int p = 0; p < P; ++p) {
            const auto one = get(p);
            if constexpr (kNarrow)
              x.p[p] = one.p[0];
            else
              x = one;
          }
        };
        both([&](int p) { return row_op<M, 2>(sX[p] + i * RW, f, half); });
        mul<32>(du, kc, x);
        if (jt <= it) {
          both([&](int p) { return row_op<M, 2>(sW1[p] + i * RW, f, half); });
          mul<32>(dq, kc, x);
        }
        if (jt >= it) {
          both([&](int p) { return col_op<M, 2, RW>(sW1[p] + col_share<M, 2, RW>(lane), 16 * f, 32 * it); });
          mul<32>(du, col_op<M, 2, RK>(qat, 16 * f, 0), x);
        }
      }
      auto out = [&](void* p, int f32, const f16v& v) {
        const int size = f32 ? 4 : TS;
        const rsrc_t r = make_rsrc(static_cast<char*>(p) + (tok0 * A.H + h) * A.Dk * size, 0x7fffffffu);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = c0 + 32 * kt + 8 * q + 4 * half;
          const uint32_t to = (i * A.H * A.Dk + col) * size;
          if (kNarrow && !f32) {
            __builtin_amdgcn_raw_buffer_store_b64(
                u2{pack_bf16x2(v[4 * q], v[4 * q + 1]), pack_bf16x2(v[4 * q + 2], v[4 * q + 3])}, r,
                la_in((i < n) & (col < A.Dk), to), 0, 0);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t one = la_in((i < n) & (col + e < A.Dk), to + e * size);
              if (f32)
                stb<float>(r, one, 0, v[4 * q + e]);
              else
                stb<T>(r, one, 0, v[4 * q + e]);
            }
          }
        }
      };
      out(A.dq, A.q_f32, dq);
      out(A.dk, A.k_f32, du);
    }
  }
  if (!flow) return;
  __syncthreads();

  // ---- 3
  if (wave != 0) return;
  const int tiles = (A.Dk + 31) / 32;
  float into = 0.0f, from = 0.0f;
  for (int t = 0; t < tiles; ++t) {
    into += s_in[t][lane];
    from += s_out[t][lane];
  }
  // row j: sums of its uses from l on
#pragma unroll 8
  for (int l = 63; l > 0; --l) {
    if (l > lane) {
      from += sF[lane * kLf + l];
      sF[lane * kLf + l] = from;
    }
  }
  // the state's uses from token i on
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const float o = __shfl_down(into, m);
    if (lane + m < 64) into += o;
  }
  float F = s_through + into;
#pragma unroll 8
  for (int j = 0; j < 63; ++j)
    if (j < lane) F += sF[j * kLf + lane];
  const bool there = lane < n;
  if (!there || la_decay(A.g, batch, u.begin + (there ? lane : 0), h) <= -104.0f) F = 0.0f;
  if (A.dg && there) {
    const size_t at = (tok0 + lane) * A.H + h;
    if (A.g_dtype == PRNN_F32)
      static_cast<float*>(A.dg)[at] = F;
    else if (A.g_dtype == PRNN_F16)
      static_cast<f16*>(A.dg)[at] = from_f32<f16>(F);
    else
      static_cast<bf16*>(A.dg)[at] = from_f32<bf16>(F);
  }
  if (A.g_part) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) F += __shfl_xor(F, m);
    if (lane == 0) A.g_part[unit] = F;
  }
}

template <class M, typename T>
int launch(const DrGrad& a, hipStream_t stream) {
  const long long groups = dr_units(a.seqs, kDrC) * a.H;
  if (int rc = check_grid("delta_rule backward", groups, 256)) return rc;
  dr_grad_kernel<M, T><<<static_cast<unsigned>(groups), 256, 0, stream>>>(a);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

}  // namespace

int dr_grad(const DrGrad& a, bool bf16_walk, hipStream_t stream) {
  if (bf16_walk) return launch<InBf16, bf16>(a, stream);
  return with_storage(a.dtype, [&](auto z) { return launch<InF32, decltype(z)>(a, stream); });
}

}  // namespace prnn
