// Gated delta rule: the states before (backwards: the adjoints behind) a cut sequence's pieces.
//
// Unlike a plain decay, what a piece does to the state that it begins with is a matrix: the walk over
// the piece from the unit matrix, without values, leaves it (the transfer M_p, Dk x Dk), from zeros
// the piece's own part U_p.  Then S_{p+1} = M_p S_p + U_p, one after another.
//
// A workgroup takes 32 columns of the state; its four waves take 32 rows each in turn, all operands in
// three bf16 parts (24 bits), the state handed round through LDS in parts.  Transfers lie in memory as
// operands (dr_operand_at).  Bound by the chain from piece to piece, 2.6 us each (D = 128, 16 pieces: 40
// us), of which the next piece's operands, held in registers, and two sums in turn have taken a third.
#include "delta_rule_loads.h"

namespace prnn {
namespace {

struct JoinArgs {
  LaSeqs seqs;
  float* piece;           // in: U_p, out: S_{p+1}  (slot, H, Dk, Dv)
  const uint16_t* transfer;  // (slot, H): operands in three parts
  LaState init;
  int H, Dk, Dv, tiles, back;
};

// R: row tiles of 32 of a wave (4 R of them hold Dk).
template <int R>
__global__ __launch_bounds__(256) void dr_join_kernel(JoinArgs A) {
  constexpr int F = 8 * R;  // steps of the contraction
  __shared__ __align__(16) char lds[F][3][1024];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
  const int tile = blockIdx.x % A.tiles, h = blockIdx.x / A.tiles % A.H, seq = blockIdx.x / A.tiles / A.H;
  const int s0 = A.seqs.cu ? la_offset(A.seqs, seq) : 0;
  const int first = dr_base(A.seqs, A.seqs.len, seq, s0);
  const DrUnit u = dr_unit(A.seqs, A.seqs.len, first);
  if (!u.any || u.seq != seq || u.count < 2) return;
  const int col = 32 * tile + l32;
  const size_t state_floats = static_cast<size_t>(A.Dk) * A.Dv;
  const size_t elems = dr_operand_elems(A.Dk, A.Dk);
  const int steps = (A.Dk + 15) / 16;
  auto at = [&](int r, int e) {  // element of register e of row tile r of this wave
    const int i = 32 * (4 * r + wave) + 8 * (e >> 2) + 4 * half + (e & 3);
    return la_in((i < A.Dk) & (col < A.Dv), (i * A.Dv + col) * 4);
  };
  f16v S[R];
  const float* init = la_row(A.init, seq, A.H * state_floats);
  const rsrc_t ri =
      make_rsrc(init ? init + h * state_floats : A.piece, init ? static_cast<uint32_t>(state_floats) * 4 : 0);
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < 16; ++e) S[r][e] = ldb<float>(ri, at(r, e), 0);
  // A piece's own state and the operands of its transfer.  Where a wave has one tile of rows they are all
  // in registers, each loaded for the next piece as soon as it has been used for this one.
  constexpr bool kAhead = R == 1;
  Op<InBf16, 3> m[8];
  f16v own[R];
  auto unit_of = [&](int k) {
    k = min(k, u.count - 2);
    return dr_slot(A.seqs, u, A.back ? u.count - 2 - k : k) * A.H + h;
  };
  auto transfer_of = [&](int k) {  // (the last piece hands on to none)
    return make_rsrc(A.transfer + unit_of(k) * 3 * elems, k + 1 < u.count ? static_cast<uint32_t>(elems) * 6 : 0u);
  };
  auto operand = [&](rsrc_t rm, int r, int f) {
    Op<InBf16, 3> o;
#pragma unroll
    for (int j = 0; j < 3; ++j)
      o.p[j] = __builtin_bit_cast(
          b8, __builtin_amdgcn_raw_buffer_load_b128(
                  rm, la_in(f < steps, j * static_cast<uint32_t>(elems) * 2 + (((4 * r + wave) * steps + f) * 64 + lane) * 16),
                  0, 0));
    return o;
  };
  auto state = [&](int k) {
    const rsrc_t rp = make_rsrc(A.piece + unit_of(k) * state_floats,
                                k + 1 < u.count ? static_cast<uint32_t>(state_floats) * 4 : 0u);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 16; ++e) own[r][e] = ldb<float>(rp, at(r, e), 0);
  };
  state(0);
  if (kAhead) {
    const rsrc_t rm = transfer_of(0);
#pragma unroll
    for (int f = 0; f < 8; ++f) m[f] = operand(rm, 0, f);
  }
  for (int k = 0; k + 1 < u.count; ++k) {
    const rsrc_t rp = make_rsrc(A.piece + unit_of(k) * state_floats, static_cast<uint32_t>(state_floats) * 4);
    f16v sum[R][2];  // a matrix instruction waits for its own sum's last one
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sum[r][0] = own[r];
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[r][1][e] = 0.0f;
    }
    __syncthreads();  // the last step's operands have been read
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = S[r][8 * f + e];
        const auto o = parts_of<InBf16, 3>(v);
#pragma unroll
        for (int j = 0; j < 3; ++j)
          *reinterpret_cast<b8*>(&lds[2 * (4 * r + wave) + f][j][lane * 16]) = o.p[j];
      }
    state(k + 1);
    __syncthreads();
    const rsrc_t now = transfer_of(k), next = transfer_of(k + 1);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int f = 0; f < F; ++f) {
        Op<InBf16, 3> s;
#pragma unroll
        for (int j = 0; j < 3; ++j) s.p[j] = *reinterpret_cast<const b8*>(&lds[f][j][lane * 16]);
        if constexpr (kAhead) {
          mul<32>(sum[r][f & 1], m[f], s);
          m[f] = operand(next, 0, f);
        } else {
          mul<32>(sum[r][f & 1], operand(now, r, f), s);
        }
      }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        S[r][e] = sum[r][0][e] + sum[r][1][e];
        stb<float>(rp, at(r, e), 0, S[r][e]);  // in the place of the piece's own
      }
  }
}

}  // namespace

int dr_join(const DrWalk& a, bool back, hipStream_t stream) {
  JoinArgs j{a.seqs, a.piece, a.transfer, a.init, a.H, a.Dk, a.Dv, (a.Dv + 31) / 32, back};
  const long long groups = 1ll * a.seqs.n_seq * a.H * j.tiles;
  if (int rc = check_grid("delta_rule", groups, 256)) return rc;
  if (a.Dk <= 128)
    dr_join_kernel<1><<<static_cast<unsigned>(groups), 256, 0, stream>>>(j);
  else
    dr_join_kernel<2><<<static_cast<unsigned>(groups), 256, 0, stream>>>(j);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

}  // namespace prnn
