// Gated delta rule: the gradients of q, k, the log decays and the rates, a workgroup per chunk and
// head, all chunks at once (the walks leave the states before the chunks and the adjoints behind).
//
// 1. Pairs of tokens, a tile of 32 x 32 of the lower triangle per wave: go e^T, dv e^T, q k^T, k k^T;
//    and the products with the states, tiles of 32 columns and 32 tokens, formed transposed (lane:
//    token).  Tokens' rows come through LDS in slabs of 64 columns, states and e as operands.
// 2. The pairs, weighted, in fp32 in LDS, over the slabs of go and dv: the rest of dq and dk.
// 3. dL/dg_t is the flow through the decay of token t,
//      F_t = sum over sources j < t and uses l >= t of what l reads of j,
//    where a source may also be the state before the chunk and a use the adjoint behind it.  It is
//    summed as that double sum and not as a running difference of gains and losses: behind a strong
//    decay the flow is a tiny part of either.  The rates' gradient is what all read of a unit of what
//    the token writes: the same sums by rows, and the token's own.
//
// Eight waves: four for the pairs and dq, four for dk, each with its own code and the same barriers, so
// that two workgroups a CU (what LDS holds) are four waves a SIMD (four waves that did all took 1.24
// times as long).  4096 chunks of bf16, D = 64: 158 us for 470 MB, of which 324 reach memory (3 TB/s of all).
// Vector instructions take half of the time, most of them the splits of fp32 operands into three bf16 parts
// (125 us with two parts, whose 16 bits showed in the results' last place), the phases' latencies the rest.
#include "delta_rule_loads.h"

namespace prnn {
namespace {

constexpr int kLf = 65;  // floats of a row of the flow's matrix

// KS slabs of 64 columns of dq and dk at a time; WIDE: keys of more than KS, in several passes (the
// pairs then need a place of their own).
template <class M, int KS, bool WIDE>
__global__ __launch_bounds__(512, sizeof(typename M::E) == 2 && KS == 1 ? 4 : 2) void dr_grad_kernel(DrGrad A) {
  using E = typename M::E;
  constexpr bool kNarrow = sizeof(E) == 2;
  constexpr int ES = static_cast<int>(sizeof(E));
  constexpr int kAt = 2;  // steps whose operands are under way
  constexpr int RB = dr_row_k(kNarrow, 64), kSlab = kDrC * RB;
  constexpr int RF = dr_row_k(false, 64), kFloats = kDrC * RF;  // a slab of floats
  // k, q, go, dv; the pairs go u^T and X, in the place of go and dv where those are read once
  constexpr int kPairsAt = WIDE ? 3 * kSlab + kFloats : 2 * kSlab;
  __shared__ __align__(16) char lds[kPairsAt + 2 * kFloats];
  __shared__ float sF[kDrC * kLf], s_in[2][8][kDrC], s_out[8][kDrC];
  __shared__ __align__(16) float sw[kDrW * 64];
  __shared__ float s_through[4], s_own[kDrC], s_into[kDrC], s_waves[8];
  char *const sK = lds, *const sQ = lds + kSlab, *const sG = lds + 2 * kSlab, *const sD = lds + 3 * kSlab;
  char *const sP = lds + kPairsAt, *const s_x = sP + kFloats;
  const int h = blockIdx.x % A.H, id = blockIdx.x / A.H;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
  const int wave = (tid >> 6) & 3;
  const bool lead = __builtin_amdgcn_readfirstlane(tid >> 8) == 0;  // pairs and dq; the other waves dk
  const DrUnit u = dr_unit(A.seqs, kDrC, id);
  if (!u.any || u.begin >= u.end) {
    if (A.g_part && tid == 0) A.g_part[static_cast<size_t>(id) * A.H + h] = 0.0f;
    return;
  }
  const int n = u.end - u.begin, batch = dr_batch(A.seqs, u);
  const size_t tok0 = dr_token(A.seqs, u, u.begin);
  const size_t unit = static_cast<size_t>(id) * A.H + h;
  const int TS = A.dtype == PRNN_F32 ? 4 : 2;
  auto rows = [&](const LaView& v) {
    return static_cast<const char*>(v.p) + (batch * v.sb + (h / v.rep) * v.sh +
                                            static_cast<long long>(u.begin) * v.st) * TS;
  };
  const char *pq = rows(A.q), *pk = rows(A.k), *pg = rows(A.go);
  const float* pd = A.dv + (tok0 * A.H + h) * A.Dv;
  const int d_step = A.H * A.Dv;
  auto operands = [&](const float* p, int r, int c) {
    const size_t elems = dr_operand_elems(r, c);
    return make_rsrc(p + unit * elems, static_cast<uint32_t>(elems) * 4);
  };
  const rsrc_t re = operands(A.e, kDrC, A.Dv), rS = operands(A.before, A.Dk, A.Dv),
               rR = operands(A.behind, A.Dk, A.Dv);
  const int vs = (A.Dv + 15) / 16, last_k = (A.Dk - 1) / 64 * 64;
  Staged<M, 64, 512> ga, ka, kb;
  std::conditional_t<kNarrow, StagedFloats<64, 512>, Staged<M, 64, 512>> gd;
  auto fetch_dv = [&](int v0) {
    if constexpr (kNarrow)
      gd.fetch(pd, d_step, n, v0, A.Dv);
    else
      gd.fetch(reinterpret_cast<const char*>(pd), d_step, n, v0, A.Dv, PRNN_F32);
  };
  auto put_dv = [&](int v0, bool result) {
    if constexpr (kNarrow) {
      gd.template put<RF>(sD);
      if (result && A.dv16) gd.as_bf16(static_cast<uint16_t*>(A.dv16) + (tok0 * A.H + h) * A.Dv, d_step, n, v0, A.Dv);
    } else {
      gd.template put<RF>(sD, PRNN_F32);
    }
  };
  ga.fetch(pg, A.go.st, n, 0, A.Dv, A.dtype);
  fetch_dv(0);
  ka.fetch(pk, A.k.st, n, last_k, A.Dk, A.dtype);
  kb.fetch(pq, A.q.st, n, last_k, A.Dk, A.dtype);
  const float* weights = reinterpret_cast<const float*>(A.sys + unit * kDrSys + 2 * kDrTiles);
  const int kt = wave & 1, it = wave >> 1, t = 32 * it + l32;
  for (int i = tid; i < kDrW * 64; i += 512) sw[i] = weights[i];
  ga.template put<RB>(sG, A.dtype);
  put_dv(0, true);
  ka.template put<RB>(sK, A.dtype);
  kb.template put<RB>(sQ, A.dtype);

  // The first four waves: the pairs go e^T, dv e^T, q k^T, k k^T of their tile and a tile of dq in every
  // slab, the others: e R^T and dv S^T of their tile of dk.  Either way its own code, with the same
  // barriers: in common branches the registers of both were taken.
  const int pi = wave > 0, pj = wave > 1, i = 32 * pi + l32;
  float through = 0.0f;
  auto run = [&](auto role) {
    constexpr bool kLead = decltype(role)::value;
    // operands of a wave's tiles of the states and of its tokens' e; the pairs' earlier tokens are the
    // same ones (waves 0 and 1: the first 32, wave 2: the others)
    Eight ei[kAt], S[KS][kAt], R[KS][kAt];
    auto fetch = [&](int p0, int v0, int f0) {
#pragma unroll
      for (int f = 0; f < kAt; ++f) {
        const int step = v0 / 16 + f0 + f;
        ei[f] = global_op(re, step < vs, it * vs + step);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int tile = p0 / 32 + 2 * s + kt;
          S[s][f] = global_op(rS, (step < vs) & (32 * tile < A.Dk), tile * vs + step);
          if constexpr (!kLead) R[s][f] = global_op(rR, (step < vs) & (32 * tile < A.Dk), tile * vs + step);
        }
      }
    };
    // what lies in LDS as floats, as operands of 24 bits: a token's dv, a pair's row and column
    auto float_row = [&](const char* rows, int token, int f) {
      auto o = row_op<InF32, 2>(rows + token * RF, f, half);
      return parts_of<M, 3>(o.x);
    };
    const int column_at = col_share<InF32, 2, RF>(lane);
    auto float_col = [&](const char* rows, int t0, int c0) {
      auto o = col_op<InF32, 2, RF>(rows + column_at, t0, c0);
      return parts_of<M, 3>(o.x);
    };
    const bool pairs = kLead && wave < 3;

    for (int p0 = 0; p0 < (WIDE ? A.Dk : 1); p0 += 64 * KS) {
      f16v GU, DU;
#pragma unroll
      for (int r = 0; r < 16; ++r) GU[r] = DU[r] = 0.0f;
      f16v main[KS], ds[KS];  // dq, or dk and dv S^T
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int r = 0; r < 16; ++r) main[s][r] = ds[s][r] = 0.0f;
      // ---- 1
      for (int v0 = 0; v0 < A.Dv; v0 += 64) {
        if (p0 > 0 || v0 > 0) {
          ga.fetch(pg, A.go.st, n, v0, A.Dv, A.dtype);
          fetch_dv(v0);
          __syncthreads();
          ga.template put<RB>(sG, A.dtype);
          put_dv(v0, p0 == 0);
        }
        fetch(p0, v0, 0);
        __syncthreads();
#pragma unroll
        for (int f0 = 0; f0 < 4; f0 += kAt) {
          if (f0 > 0) fetch(p0, v0, f0);
          if constexpr (kLead) {
#pragma unroll
            for (int f = 0; f < kAt; ++f) {
              const auto gi = row_op<M, 2>(sG + t * RB, f0 + f, half);
#pragma unroll
              for (int s = 0; s < KS; ++s) mul<32>(main[s], whole<M>(S[s][f]), gi);
              if (p0 == 0 && pairs) {
                const auto e = whole<M>(ei[f]);
                mul<32>(GU, e, row_op<M, 2>(sG + i * RB, f0 + f, half));
                mul<32>(DU, e, float_row(sD, i, f0 + f));
              }
            }
          } else {
#pragma unroll
            for (int f = 0; f < kAt; ++f) {
              const auto di = float_row(sD, t, f0 + f), e = whole<M>(ei[f]);
#pragma unroll
              for (int s = 0; s < KS; ++s) {
                // from the state before to the adjoint behind: two waves have the same operands, a step each
                if (((f0 + f) & 1) == it) {
#pragma unroll
                  for (int x = 0; x < 8; ++x) through = fmaf(S[s][f].x[x], R[s][f].x[x], through);
                }
                mul<32>(main[s], whole<M>(R[s][f]), e);
                mul<32>(ds[s], whole<M>(S[s][f]), di);
              }
            }
          }
        }
      }
      if (p0 == 0) {
        f16v QK, KK;
#pragma unroll
        for (int r = 0; r < 16; ++r) QK[r] = KK[r] = 0.0f;
        auto keys = [&]() {
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const auto kj = row_op<M, 2>(sK + (32 * pj + l32) * RB, f, half);
            mul<32>(QK, kj, row_op<M, 2>(sQ + i * RB, f, half));
            mul<32>(KK, kj, row_op<M, 2>(sK + i * RB, f, half));
          }
        };
        if (pairs) keys();
        for (int c0 = last_k - 64; c0 >= 0; c0 -= 64) {
          ka.fetch(pk, A.k.st, n, c0, A.Dk, A.dtype);
          kb.fetch(pq, A.q.st, n, c0, A.Dk, A.dtype);
          __syncthreads();
          ka.template put<RB>(sK, A.dtype);
          kb.template put<RB>(sQ, A.dtype);
          __syncthreads();
          if (pairs) keys();
        }
        __syncthreads();  // go and dv have been read: the pairs take their place
        if (pairs) {
          const float Hi = sw[kWhi * 64 + i], Lo = sw[kWlo * 64 + i];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float w1[4], x[4];
            const int j0 = 32 * pj + 8 * q + 4 * half;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int jj = j0 + r, e = 4 * q + r;
              const float w = fexp((Hi - sw[kWhi * 64 + jj]) + (Lo - sw[kWlo * 64 + jj]));
              w1[r] = jj <= i ? w * A.scale * GU[e] : 0.0f;
              x[r] = jj < i ? w * DU[e] : 0.0f;
              // what token i reads of a unit of what j writes (its rate is still to come)
              sF[jj * kLf + i] = jj < i ? QK[e] * w1[r] - KK[e] * x[r] : 0.0f;
              if (jj == i) s_own[i] = QK[e] * w1[r];
              w1[r] *= sw[kWb * 64 + jj];
              x[r] *= -sw[kWb * 64 + jj];
            }
            *reinterpret_cast<f4*>(sP + i * RF + j0 * 4) = f4{w1[0], w1[1], w1[2], w1[3]};
            *reinterpret_cast<f4*>(s_x + i * RF + j0 * 4) = f4{x[0], x[1], x[2], x[3]};
          }
        }
        __syncthreads();
      }

      // ---- 2
      auto four = [&](const char* row, int col, float* v) {
        if constexpr (kNarrow) {
          const u2 a = *reinterpret_cast<const u2*>(row + col * 2);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = r & 1 ? hi_bf16(a[r >> 1]) : lo_bf16(a[r >> 1]);
        } else {
          const f4 a = *reinterpret_cast<const f4*>(row + col * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = a[r];
        }
      };
      const int col_at = col_share<M, 2, RB>(lane);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int c0 = p0 + 64 * s;
        if (c0 >= A.Dk) continue;
        if (c0 > 0) {
          ka.fetch(pk, A.k.st, n, c0, A.Dk, A.dtype);
          kb.fetch(pq, A.q.st, n, c0, A.Dk, A.dtype);
          __syncthreads();
          ka.template put<RB>(sK, A.dtype);
          kb.template put<RB>(sQ, A.dtype);
          __syncthreads();
        }
        const bool any = c0 + 32 * kt < A.Dk;
        const char* const kat = sK + 32 * kt * ES + col_at;
        if constexpr (kLead) if (any) {
          f16v& dq = main[s];
          const float w = sw[kWg * 64 + t] * A.scale;
          float in_sum = 0.0f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[4];
            four(sQ + t * RB, 32 * kt + 8 * q + 4 * half, v);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              dq[4 * q + r] *= w;
              in_sum = fmaf(v[r], dq[4 * q + r], in_sum);
            }
          }
          in_sum += __shfl_xor(in_sum, 32);
          if (half == 0) s_in[0][c0 / 32 + kt][t] = in_sum;
#pragma unroll
          for (int f = 0; f < 4; ++f)
            if ((f >> 1) <= it)
              mul<32>(dq, col_op<M, 2, RB>(kat, 16 * f, 0), float_row(sP, t, f));
        }
        if constexpr (!kLead) if (any) {
          f16v &du = main[s], &dS = ds[s];
          const float wg = sw[kWg * 64 + t], wr = sw[kWr * 64 + t], rate = sw[kWb * 64 + t];
          float in_sum = 0.0f, out_sum = 0.0f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[4];
            four(sK + t * RB, 32 * kt + 8 * q + 4 * half, v);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int e = 4 * q + r;
              dS[e] *= wg;
              du[e] *= wr;
              in_sum = fmaf(-v[r], dS[e], in_sum);
              out_sum = fmaf(v[r], du[e], out_sum);
              du[e] = fmaf(rate, du[e], -dS[e]);
            }
          }
          in_sum += __shfl_xor(in_sum, 32);
          out_sum += __shfl_xor(out_sum, 32);
          if (half == 0) {
            s_in[1][c0 / 32 + kt][t] = in_sum;
            s_out[c0 / 32 + kt][t] = out_sum;
          }
          const char* const qat = sQ + 32 * kt * ES + col_at;
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const int jt = f >> 1;
            const auto kc = col_op<M, 2, RB>(kat, 16 * f, 0);
            // -(X + X^T), rows of X before the token and columns behind it
            if (jt <= it) mul<32>(du, kc, float_row(s_x, t, f));
            if (jt >= it) {
              mul<32>(du, kc, float_col(s_x, 16 * f, 32 * it));
              mul<32>(du, col_op<M, 2, RB>(qat, 16 * f, 0), float_col(sP, 16 * f, 32 * it));
            }
          }
        }
        auto out = [&](void* p, int f32, const f16v& v) {
          const int size = f32 ? 4 : TS;
          const rsrc_t r = make_rsrc(static_cast<char*>(p) + (tok0 * A.H + h) * A.Dk * size, 0x7fffffffu);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int col = c0 + 32 * kt + 8 * q + 4 * half;
            const uint32_t to = (t * A.H * A.Dk + col) * size;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t one = la_in((t < n) & (col + e < A.Dk), to + e * size);
              if (f32 || A.dtype == PRNN_F32)
                stb<float>(r, one, 0, v[4 * q + e]);
              else if (A.dtype == PRNN_F16)
                stb<f16>(r, one, 0, v[4 * q + e]);
              else
                stb<bf16>(r, one, 0, v[4 * q + e]);
            }
          }
        };
        if constexpr (kNarrow) {
          // bf16 rows leave by way of LDS, 16 bytes a lane side by side
          auto put = [&](char* to, const f16v& v) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<u2*>(to + t * RB + (32 * kt + 8 * q + 4 * half) * 2) =
                  u2{pack_bf16x2(v[4 * q], v[4 * q + 1]), pack_bf16x2(v[4 * q + 2], v[4 * q + 3])};
          };
          auto rows_out = [&](void* p, const char* from) {
            const rsrc_t r = make_rsrc(static_cast<char*>(p) + (tok0 * A.H + h) * A.Dk * 2, 0x7fffffffu);
            const int row = tid >> 3, unit = tid & 7, col = c0 + 8 * unit;
            __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const u4*>(from + row * RB + unit * 16), r,
                                                   la_in((row < n) & (col < A.Dk), (row * A.H * A.Dk + col) * 2), 0, 0);
          };
          __syncthreads();  // k and q have been read
          const bool f32 = kLead ? A.q_f32 : A.k_f32;
          if (any && !f32) put(kLead ? sQ : sK, main[s]);
          __syncthreads();
          if (!A.q_f32) rows_out(A.dq, sQ);
          if (!A.k_f32) rows_out(A.dk, sK);
          if (any && f32) out(kLead ? A.dq : A.dk, 1, main[s]);
        } else if (any) {
          out(kLead ? A.dq : A.dk, kLead ? A.q_f32 : A.k_f32, main[s]);
        }
      }
    }
  };
  if (lead)
    run(std::true_type{});
  else
    run(std::false_type{});
  if (!A.dg && !A.g_part && !A.dbeta) return;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) through += __shfl_xor(through, m);
  if (lane == 0 && !lead) s_through[wave] = through;
  __syncthreads();

  // ---- 3: eight lanes per token, an eighth of the others' each
  const int tok = tid >> 3, part = tid & 7, tiles = (A.Dk + 31) / 32;
  {
    // row tok: sums of its uses from l on, what the adjoint behind reads among them
    float m[8], sum = 0.0f, after = 0.0f;
#pragma unroll
    for (int x = 7; x >= 0; --x) {
      const int l = 8 * part + x;
      const float flow = sF[tok * kLf + l];
      sum += l > tok ? flow : 0.0f;
      m[x] = sum;
    }
#pragma unroll
    for (int k = 1; k < 8; k <<= 1) {
      const float o = __shfl_down(sum, k);
      if (part + k < 8) sum += o;
    }
    const float later = __shfl_down(sum, 1);
    for (int k = 0; k < tiles; ++k) after += s_out[k][tok];
    after += part < 7 ? later : 0.0f;
    const float rate = sw[kWb * 64 + tok];
#pragma unroll
    for (int x = 0; x < 8; ++x) sF[tok * kLf + 8 * part + x] = rate * (after + m[x]);  // (up to l = tok: not read)
    if (!lead && wave == 3) {  // what the tokens from one on read of the state before
      float into = 0.0f;
      for (int k = 0; k < tiles; ++k) into += s_in[0][k][lane] + s_in[1][k][lane];
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const float o = __shfl_down(into, m);
        if (lane + m < 64) into += o;
      }
      s_into[lane] = into + ((s_through[0] + s_through[1]) + (s_through[2] + s_through[3])) * sw[kWmeta * 64];
    }
    if (A.dbeta && part == 0 && tok < n) {
      const float d = after + m[0] + s_own[tok];
      const size_t at = (tok0 + tok) * A.H + h;
      if (A.b_dtype == PRNN_F32)
        static_cast<float*>(A.dbeta)[at] = d;
      else if (A.b_dtype == PRNN_F16)
        static_cast<f16*>(A.dbeta)[at] = from_f32<f16>(d);
      else
        static_cast<bf16*>(A.dbeta)[at] = from_f32<bf16>(d);
    }
  }
  if (!A.dg && !A.g_part) return;
  __syncthreads();
  // column tok: the sources before it
  float F = 0.0f;
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const int j = 8 * part + x;
    const float flow = sF[j * kLf + tok];
    F += j < tok ? flow : 0.0f;
  }
#pragma unroll
  for (int m = 1; m < 8; m <<= 1) F += __shfl_xor(F, m);
  F += s_into[tok];
  const bool there = tok < n;
  // nothing comes through a factor that is zero
  if (!there || la_decay(A.g, batch, u.begin + (there ? tok : 0), h) <= -104.0f) F = 0.0f;
  if (A.dg && there && part == 0) {
    const size_t at = (tok0 + tok) * A.H + h;
    if (A.g_dtype == PRNN_F32)
      static_cast<float*>(A.dg)[at] = F;
    else if (A.g_dtype == PRNN_F16)
      static_cast<f16*>(A.dg)[at] = from_f32<f16>(F);
    else
      static_cast<bf16*>(A.dg)[at] = from_f32<bf16>(F);
  }
  if (A.g_part) {
    F = part == 0 ? F : 0.0f;
#pragma unroll
    for (int m = 8; m < 64; m <<= 1) F += __shfl_xor(F, m);
    if (lane == 0) s_waves[tid >> 6] = F;
    __syncthreads();
    if (tid == 0)
      A.g_part[unit] = ((s_waves[0] + s_waves[1]) + (s_waves[2] + s_waves[3])) +
                       ((s_waves[4] + s_waves[5]) + (s_waves[6] + s_waves[7]));
  }
}

template <class M, int KS, bool WIDE>
int launch(const DrGrad& a, hipStream_t stream) {
  const long long groups = dr_units(a.seqs, kDrC) * a.H;
  if (int rc = check_grid("delta_rule backward", groups, 512)) return rc;
  dr_grad_kernel<M, KS, WIDE><<<static_cast<unsigned>(groups), 512, 0, stream>>>(a);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}
template <class M>
int launch_width(const DrGrad& a, hipStream_t stream) {
  if (a.Dk <= 64) return launch<M, 1, false>(a, stream);
  if constexpr (sizeof(typename M::E) == 4) return launch<M, 1, true>(a, stream);  // registers
  else return a.Dk <= 128 ? launch<M, 2, false>(a, stream) : launch<M, 2, true>(a, stream);
}

}  // namespace

int dr_grad(const DrGrad& a, bool bf16_walk, hipStream_t stream) {
  return bf16_walk ? launch_width<InBf16>(a, stream) : launch_width<InF32>(a, stream);
}

}  // namespace prnn
