// Gated delta rule: the states before (backwards: the adjoints behind) a cut sequence's pieces.
//
// Unlike a plain decay, what a piece does to the state that it begins with is a matrix: the walk over
// the piece from the unit matrix, without values, leaves it (the transfer M_p, Dk x Dk), from zeros
// the piece's own part U_p.  Then S_{p+1} = M_p S_p + U_p, one after another.
//
// A workgroup takes 32 columns of the state; its four waves take 32 rows each in turn, all operands in
// three bf16 parts (24 bits), the state handed round through LDS in parts.  Transfers lie in memory as
// operands (dr_operand_at).
#include "delta_rule_loads.h"

namespace prnn {
namespace {

struct JoinArgs {
  LaSeqs seqs;
  float* piece;           // in: U_p, out: S_p  (piece, H, Dk, Dv)
  const float* transfer;  // (piece, H): operands
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
  const size_t transfer_floats = dr_operand_elems(A.Dk, A.Dk);
  const int steps = (A.Dk + 15) / 16;
  auto at = [&](int r, int e) {  // element of register e of row tile r of this wave
    const int i = 32 * (4 * r + wave) + 8 * (e >> 2) + 4 * half + (e & 3);
    return la_in((i < A.Dk) & (col < A.Dv), (i * A.Dv + col) * 4);
  };
  f16v S[R];
  const float* init = la_row(A.init, seq, A.H * state_floats);
  const rsrc_t ri = make_rsrc(init ? init + h * state_floats : A.piece, init ? static_cast<uint32_t>(state_floats) * 4 : 0);
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < 16; ++e) S[r][e] = ldb<float>(ri, at(r, e), 0);
  // a piece's own state and the operands of its transfer (for one row tile a wave all of them, a piece
  // ahead; the last piece hands on to none)
  constexpr int kHeld = R == 1 ? 2 : 1;
  struct Piece {
    u4 m[8][2];
    f16v own[R];
  };
  Piece held[kHeld];
  auto unit_of = [&](int k) { return static_cast<size_t>(first + (A.back ? u.count - 1 - k : k)) * A.H + h; };
  auto operands = [&](Piece& x, int k, int r, int f0) {
    const rsrc_t rm = make_rsrc(A.transfer + unit_of(k) * transfer_floats,
                                k + 1 < u.count ? static_cast<uint32_t>(transfer_floats) * 4 : 0u);
#pragma unroll
    for (int f = 0; f < 8; ++f)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        x.m[f][e] = __builtin_amdgcn_raw_buffer_load_b128(
            rm, la_in(f0 + f < steps, (((4 * r + wave) * steps + f0 + f) * 64 + lane) * 32 + e * 16), 0, 0);
  };
  auto fetch = [&](Piece& x, int k) {
    k = min(k, u.count - 1);
    operands(x, k, 0, 0);
    const rsrc_t rp = make_rsrc(A.piece + unit_of(k) * state_floats,
                                k + 1 < u.count ? static_cast<uint32_t>(state_floats) * 4 : 0u);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 16; ++e) x.own[r][e] = ldb<float>(rp, at(r, e), 0);
  };
  auto step = [&](Piece& x, Piece& other, int k) {
    const rsrc_t rp = make_rsrc(A.piece + unit_of(k) * state_floats, static_cast<uint32_t>(state_floats) * 4);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 16; ++e) stb<float>(rp, at(r, e), 0, S[r][e]);
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
    if (kHeld == 2) fetch(other, k + 1);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      f16v sum = x.own[r];
#pragma unroll
      for (int f0 = 0; f0 < F; f0 += 8) {
        if (r > 0 || f0 > 0) operands(x, k, r, f0);
#pragma unroll
        for (int f = 0; f < 8; ++f) {
          Op<InBf16, 3> s;
#pragma unroll
          for (int j = 0; j < 3; ++j) s.p[j] = *reinterpret_cast<const b8*>(&lds[f0 + f][j][lane * 16]);
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(x.m[f][e >> 2][e & 3]);
          mul<32>(sum, parts_of<InBf16, 3>(v), s);
        }
      }
      S[r] = sum;
    }
    if (kHeld == 1) fetch(x, k + 1);
  };
  fetch(held[0], 0);
  for (int k = 0; k < u.count; k += kHeld) {
    step(held[0], held[kHeld - 1], k);
    if (kHeld == 2 && k + 1 < u.count) step(held[1], held[0], k + 1);
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
