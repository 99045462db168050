// Gated delta rule, the walks from chunk to chunk, forwards and backwards.
//
// A wave keeps NC columns of the state (or of its adjoint) in the result layout of the matrix
// instructions (tiles.h), lane = column, and goes through its piece's chunks.  The three products
// of a chunk's chain, with rows of K read from LDS along and across,
//
//   forwards   x = K S,   e = (1 + T)(v - exp(G) x),          S' = exp(G_last) S + K^T (..u)
//   backwards  x = K R,   dv = (1 + T)^T b (P^T go + .. x),     R' = exp(G_last) R + Q^T (..go) - K^T (..dv)
//
// take what the one before left in registers, so a wave's chain meets no other wave: a chunk's
// barriers only hand K, Q and the system through LDS.  The output is formed transposed from the same
// registers (state and u as first operands), so that a lane holds consecutive columns of a token.
//
// Bound by this chain: one wave a SIMD goes through some 9500 cycles a chunk (bf16, D = 64; matrix
// instructions 2700 of them, the rest splits of results into bf16 parts, LDS reads and waits), so 2048
// tokens of 128 heads take 130 us forwards with what is kept and 115 backwards, and 16384 tokens of 8
// heads, D = 128, in 16 pieces, 74 us.
//
// bf16 operands: K, Q and z as they are given; the state, what the tokens write, the system and its right
// side in three parts (all 24 bits of an fp32 value).  What the gradients read (e, dv, states, adjoints)
// leaves in fp32.
#pragma once

#include "delta_rule_loads.h"

namespace prnn {

// The same in one go, a few loads at a time: where the registers for a chunk ahead are not there.
template <class M, int COLS, int NT, int RB>
__device__ __forceinline__ void fill(char* tile, const char* p, long long st, int n, int width, int dtype) {
  constexpr int kAt = 16;
  const rsrc_t b = make_rsrc(p, 0x7fffffffu);
  for (int e0 = threadIdx.x; e0 < kDrC * COLS; e0 += kAt * NT) {
    float v[kAt];
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      const int e = e0 + k * NT, row = e / COLS, c = e % COLS;
      const uint32_t at = la_in((row < n) & (c < width), (row * static_cast<int>(st) + c) * (dtype == PRNN_F32 ? 4 : 2));
      v[k] = dtype == PRNN_F32 ? ldb<float>(b, at, 0) : dtype == PRNN_F16 ? ldb<f16>(b, at, 0) : ldb<bf16>(b, at, 0);
    }
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      const int e = e0 + k * NT, row = e / COLS, c = e % COLS;
      *reinterpret_cast<float*>(tile + row * RB + c * 4) = v[k];
    }
  }
}
struct NotStaged {};

// Operands of a stored matrix (the system's inverse or the pairs): rows NC rt .. of the 64, step f of
// the contraction over tokens; BACK: of the transposed matrix, read down the stored rows.  On bf16
// instructions it lies in LDS in three parts, one after another.
template <class M, int NC, bool BACK>
struct Stored {
  static constexpr bool kSplit = sizeof(typename M::E) == 2;
  static constexpr int G = 64 / NC;
  static constexpr int ES = kSplit ? 2 : 4, kRow = 32 * ES, kUnit = 4 * ES;
  static constexpr int kTile = kDrTiles / 3 / (kSplit ? 2 : 1);
  // whether there is anything in the 32 x 32 tile
  static constexpr bool any(int rt, int f) {
    const int a = NC * rt / 32, b = 8 * G * f / 32;
    return BACK ? b >= a : b <= a;
  }
  static __device__ __forceinline__ const char* at(const char* tile, int row, int col) {
    return tile + row * kRow + dr_unit_of(row, col >> 2) * kUnit + (col & 3) * ES;
  }
  static __device__ __forceinline__ Op<M, 3> get(const char* m, int rt, int f, int n, int g) {
    const char* t = m + (NC * rt / 32 + 8 * G * f / 32) * kTile;
    const int own = (NC * rt) & 31, other = (8 * G * f) & 31;
    if constexpr (kSplit) {
      Op<M, 3> o;
      const char *x, *y;
      if constexpr (BACK) {
        const int lane = threadIdx.x & 63, i = lane & 15, gg = lane >> 4;
        const int row = other + (G == 2 ? 4 * (gg >> 1) : 4 * gg) + (i >> 2);
        const int col = own + (G == 2 ? 16 * (gg & 1) : 0) + 4 * (i & 3);
        x = at(t, row, col);
        y = at(t, row + 4 * G, col);
      } else {
        x = at(t, own + n, other + 4 * g);
        y = at(t, own + n, other + 4 * G + 4 * g);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        union {
          u2 h[2];
          s4 s[2];
          b8 v;
        } r;
        if constexpr (BACK) {
          r.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(x + p * 3 * kTile));
          r.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(y + p * 3 * kTile));
        } else {
          r.h[0] = *reinterpret_cast<const u2*>(x + p * 3 * kTile);
          r.h[1] = *reinterpret_cast<const u2*>(y + p * 3 * kTile);
        }
        o.p[p] = r.v;
      }
      return o;
    } else {
      float v[8];
      if constexpr (BACK) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = *reinterpret_cast<const float*>(at(t, other + 4 * G * (i >> 2) + 4 * g + (i & 3), own + n));
      } else {
        const f4 x = *reinterpret_cast<const f4*>(at(t, own + n, other + 4 * g));
        const f4 y = *reinterpret_cast<const f4*>(at(t, own + n, other + 4 * G + 4 * g));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = x[i];
          v[4 + i] = y[i];
        }
      }
      return parts_of<M, 3>(v);
    }
  }
};

// Workgroups of one head's column tiles, which read the same rows and systems, are 8 apart: they
// run on one XCD (workgroups go to the 8 XCDs in turn).
__device__ __forceinline__ void dr_place(int tiles, int H, int& tile, int& h, int& piece) {
  const int group = blockIdx.x / (8 * tiles), in = blockIdx.x - group * 8 * tiles;
  tile = in >> 3;
  const int item = group * 8 + (in & 7);
  piece = item / H;
  h = item - piece * H;
}

// Pieces' own states run two workgroups a CU (D = 128: 87 us for 512 of them, 111 at one, a few registers
// over that limit).
template <class M, int NC, int KD, int W, int KIND>
constexpr int dr_pair_waves =
    (KIND == kDrState || KIND == kDrAdjoint) && sizeof(typename M::E) == 2 && NC == 16 && KD <= 128 && W == 4 ? 2 : 1;

// W waves of NC columns each.  L: waves besides that do nothing but bring the next chunk to LDS, into
// one of two buffers, while the others work on this one (bringing it took 4500 of a chunk's 9700 cycles
// of a wave that does both); 0: the same waves do it, and the chunk's LDS is there once.
template <class M, int NC, int KD, int W, int L, int KIND>
__global__ __launch_bounds__(64 * (W + L), (dr_pair_waves<M, NC, KD, W, KIND>)) void dr_walk_kernel(DrWalk A) {
  using E = typename M::E;
  constexpr bool kNarrow = sizeof(E) == 2;
  constexpr bool kBack = KIND == kDrBackward || KIND == kDrAdjoint;
  constexpr bool kOwn = KIND == kDrState || KIND == kDrAdjoint;  // pieces' own states only
  constexpr bool kOut = KIND == kDrForward || KIND == kDrKept, kKeeps = KIND == kDrKept || KIND == kDrBackward;
  constexpr int G = 64 / NC, NT = 64 * (L ? L : W), VT = NC * W;  // NT: threads that bring rows
  constexpr int RT = NC * NC / 64;   // registers of a tile
  constexpr int KT = KD / NC;        // the state's tiles
  constexpr int KF = KD / (8 * G);   // steps of a contraction over its rows
  constexpr int TT = kDrC / NC;      // token tiles
  constexpr int TF = kDrC / (8 * G); // steps of a contraction over tokens
  constexpr int RK = dr_row_k(kNarrow, KD), RZ = dr_row_z(kNarrow, VT, KD);
  constexpr bool kQ = KIND != kDrState;  // Q takes part
  constexpr bool kP = KIND != kDrState;
  constexpr int ES = static_cast<int>(sizeof(E));
  using A_t = Acc<NC>;
  using Mat = Stored<M, NC, kBack>;
  // fp32 widths over 64 have no registers for the next chunk's K and Q, over 128 no LDS for the system
  constexpr bool kAhead = kNarrow || KD <= 64, kSysLds = kNarrow || KD <= 128;
  static_assert(kAhead || kDrC * KD % (16 * NT) == 0, "whole rounds of fill");
  // (the system comes in fp32)
  constexpr int kPart = kDrTiles / (kNarrow ? 2 : 1), kPairsAt = (kNarrow ? 3 : 1) * kPart;
  constexpr int kSysBytes = kPairsAt * (kP ? 2 : 1);
  constexpr int kSysUnits = (kP ? 2 : 1) * kDrTiles / 16 / NT;
  static_assert(kDrTiles % (16 * NT) == 0, "whole units");
  static_assert(L == 0 || (kAhead && kSysLds), "waves that only load hold a chunk");
  // a chunk in LDS: K, Q, z, the system and the pairs, the weights
  constexpr int oQ = kDrC * RK, oZ = oQ + (kQ ? kDrC * RK : 0), oS = oZ + kDrC * RZ,
                oW = oS + (kSysLds ? kSysBytes : 0), kChunk = oW + kDrW * 64 * 4;
  __shared__ __align__(16) char lds[(L ? 2 : 1) * kChunk];

  int tile, h, piece;
  dr_place(A.tiles, A.H, tile, h, piece);
  if (A.order && piece < A.n_pieces) piece = A.order[piece];
  const DrUnit pc = dr_unit(A.seqs, A.seqs.len, piece);
  if (!pc.any || pc.seq >= A.seqs.n_seq) return;
  // the last piece of the walk's direction hands its state to none
  if (kOwn && pc.index == (kBack ? 0 : pc.count - 1)) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int tid = static_cast<int>(threadIdx.x) - (L ? 64 * W : 0);  // of those that bring rows
  const int nn = lane % NC, g = lane / NC;
  const bool transfer = kOwn && tile >= A.own_tiles;
  const int col0 = (transfer ? tile - A.own_tiles : tile) * VT;
  const int col = col0 + NC * wave + nn;
  const int batch = dr_batch(A.seqs, pc);
  const int row0 = dr_base(A.seqs, kDrC, pc.seq, pc.s0) + (pc.begin - pc.s0) / kDrC;
  const int chunks = (pc.end - pc.begin + kDrC - 1) / kDrC;
  const size_t state_floats = static_cast<size_t>(A.Dk) * A.Dv;
  const size_t tok0 = dr_token(A.seqs, pc, 0);

  std::conditional_t<kAhead, Staged<M, KD, NT>, NotStaged> rk, rq;
  Staged<M, VT, NT> rz;
  u4 rs[kSysLds ? kSysUnits : 1], rw[(kDrW * 64 / 4 + NT - 1) / NT];
  const int size = kNarrow || A.dtype != PRNN_F32 ? 2 : 4;
  auto head = [&](const LaView& v, int t) {
    return static_cast<const char*>(v.p) +
           (batch * v.sb + (h / v.rep) * v.sh + static_cast<long long>(t) * v.st) * size;
  };
  auto fetch = [&](int c) {
    const int t = pc.begin + c * kDrC, n = min(pc.end - t, kDrC);
    const char* sys = A.sys + (static_cast<size_t>(row0 + c) * A.H + h) * kDrSys;
#pragma unroll
    for (int k = 0; k < (kSysLds ? kSysUnits : 0); ++k) rs[k] = *reinterpret_cast<const u4*>(sys + (tid + k * NT) * 16);
    const char* w = sys + 2 * kDrTiles;
#pragma unroll
    for (int k = 0; k < (kDrW * 16 + NT - 1) / NT; ++k)
      if (tid + k * NT < kDrW * 16) rw[k] = *reinterpret_cast<const u4*>(w + (tid + k * NT) * 16);
    if constexpr (kAhead) rk.fetch(head(A.k, t), A.k.st, n, 0, A.Dk, A.dtype, tid);
    if constexpr (kAhead && kQ) rq.fetch(head(A.q, t), A.q.st, n, 0, A.Dk, A.dtype, tid);
    rz.fetch(head(A.z, t), A.z.st, transfer ? 0 : n, col0, A.Dv, A.dtype, tid);
  };
  auto chunk_of = [&](int step) { return kBack ? chunks - 1 - step : step; };
  auto put = [&](char* to, int c) {
    if constexpr (kAhead) {
      rk.template put<RK>(to, A.dtype, tid);
      if constexpr (kQ) rq.template put<RK>(to + oQ, A.dtype, tid);
    } else {
      const int t = pc.begin + c * kDrC, n = min(pc.end - t, kDrC);
      fill<M, KD, NT, RK>(to, head(A.k, t), A.k.st, n, A.Dk, A.dtype);
      if constexpr (kQ) fill<M, KD, NT, RK>(to + oQ, head(A.q, t), A.q.st, n, A.Dk, A.dtype);
    }
    rz.template put<RZ>(to + oZ, A.dtype, tid);
#pragma unroll
    for (int k = 0; k < (kSysLds ? kSysUnits : 0); ++k) {
      if constexpr (kNarrow) {
        constexpr int kUnits = kDrTiles / 16 / NT;  // of a matrix
        const bool pairs = k >= kUnits;
        char* const at = to + oS + (pairs ? kPairsAt : 0) + (tid + (pairs ? k - kUnits : k) * NT) * 8;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(rs[k][e]);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          const u2 v{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
          *reinterpret_cast<u2*>(at + p * kPart) = v;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] -= e & 1 ? hi_bf16(v[e >> 1]) : lo_bf16(v[e >> 1]);
        }
      } else {
        *reinterpret_cast<u4*>(to + oS + (tid + k * NT) * 16) = rs[k];
      }
    }
#pragma unroll
    for (int k = 0; k < (kDrW * 16 + NT - 1) / NT; ++k)
      if (tid + k * NT < kDrW * 16) *reinterpret_cast<u4*>(to + oW + (tid + k * NT) * 16) = rw[k];
  };
  if constexpr (L > 0) {
    if (wave >= W) {  // one barrier a chunk, as the others' below
      if (chunks > 0) {
        fetch(chunk_of(0));
        put(lds, 0);
      }
      if (chunks > 1) fetch(chunk_of(1));
      __syncthreads();
      for (int step = 0; step < chunks; ++step) {
        if (step + 1 < chunks) put(lds + (~step & 1) * kChunk, 0);
        if (step + 2 < chunks) fetch(chunk_of(step + 2));
        __syncthreads();
      }
      return;
    }
  }

  // ---- the state that the piece begins with
  A_t S[KT];
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int i = NC * t + 4 * G * (r >> 2) + 4 * g + (r & 3);
      S[t][r] = transfer && i == col && i < A.Dk ? 1.0f : 0.0f;
    }
  if (!kOwn) {
    const float* src = nullptr;
    if (A.piece && pc.index != (kBack ? pc.count - 1 : 0))
      src = A.piece + (dr_slot(A.seqs, pc, kBack ? pc.index : pc.index - 1) * A.H + h) * state_floats;
    else if (const float* row = la_row(A.init, pc.seq, A.H * state_floats))
      src = row + h * state_floats;
    if (src) {
      const rsrc_t rs = make_rsrc(src, static_cast<uint32_t>(state_floats) * 4);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int i = NC * t + 4 * G * (r >> 2) + 4 * g + (r & 3);
          S[t][r] = ldb<float>(rs, la_in((i < A.Dk) & (col < A.Dv), (i * A.Dv + col) * 4), 0);
        }
    }
  }

  // What a chunk leaves is stored after the next one's rows have come: loads and stores come back in
  // order, and a wait for rows behind stores would wait for those too.
  constexpr int kHeld = kNarrow ? NC / 2 : NC;
  uint32_t held_o[kOut ? kHeld : 1];
  float held_k[kKeeps ? NC : 1];  // e or dv
  int held_n = 0, held_c = 0;
  auto at_token = [&](int i) { return NC * (i / RT) + 4 * G * ((i % RT) >> 2) + 4 * g + (i & 3); };
  // Element (row, col) of a matrix of operands (dr_operand_at) with row = NC t + 4 G q + 4 g + r: this
  // lane's share of the address, and the rest, the same for all lanes.
  const int v_steps = (A.Dv + 15) / 16;
  const uint32_t operand_lane = la_in(
      col < v_steps * 16, (((col >> 4) * 64 + 4 * g + 32 * ((col >> 2) & 1)) * 8 + (col & 3) + 4 * ((col >> 3) & 1)) * 4);
  auto operand_rest = [&](int t, int reg) {
    const int q = reg >> 2, r = reg & 3, row = NC == 32 ? 8 * q + r : 16 * (t & 1) + r;
    return std::pair<int, int>{(NC == 32 ? t : t >> 1) * v_steps * 2048, row * 32};
  };
  // bf16: states are turned by products of their three parts with the unit matrix (the sum is the value,
  // exactly), so that a lane has four columns of a row and not a row's place in four of them: 16 bytes a
  // store and not 4.
  Op<M, 1> unit[2];
  if constexpr (kNarrow && kKeeps) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int place = NC == 32 ? nn - 16 * j : nn + 16 * j;  // of the contraction that is this lane's column
      float one[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) one[e] = place == 4 * G * (e >> 2) + 4 * g + (e & 3) ? 1.0f : 0.0f;
      unit[j] = parts_of<M, 1>(one);
    }
  }
  // Step f of a contraction into its tile (NC = 32: of two steps, `d` the sum; 16: of half a step, j which):
  // lane its row, registers columns.
  auto turn = [&](A_t& d, const Op<M, 3>& o, int j) {
    if (NC == 16 || j == 0) {
#pragma unroll
      for (int r = 0; r < RT; ++r) d[r] = 0.0f;
    }
    mul<NC>(d, o, unit[j]);
  };
  // The place of registers 4 q .. of such a tile among operands in memory.
  auto turned_at = [&](int t, int q) {
    const int row = NC * t + nn, step = (col0 + NC * wave + (NC == 32 ? 16 * (q >> 1) : 0)) >> 4;
    return la_in(step < v_steps, (((row >> 5) * v_steps + step) * 64 + (row & 31) + 32 * (g & 1)) * 32 +
                                     16 * (NC == 32 ? q & 1 : g >> 1));
  };
  auto four = [](const float* v) {
    return u4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  };
  auto hold = [&](uint32_t* to, const float* v) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if constexpr (kNarrow)
        to[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      else
        to[i] = __float_as_uint(v[i]);
    }
  };
  // A chunk's e, or dv; NaN for the tokens that `stop` tells (behind the walk's direction of it).
  auto hold_rows = [&](const float* v, int stop) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      held_k[i] = (kBack ? at_token(i) <= stop : at_token(i) >= stop) ? __builtin_nanf("") : v[i];
  };
  auto flush = [&]() {
    const int t0 = pc.begin + held_c * kDrC, n = held_n;  // nothing held: 0 tokens
    if constexpr (kOut) {
      const int step = static_cast<int>(A.o_st) * size, c0 = col0 + NC * wave + 4 * g;
      const rsrc_t ro = make_rsrc(static_cast<char*>(A.out) + (batch * A.o_sb + h * A.o_sh +
                                                               static_cast<long long>(t0) * A.o_st) * size,
                                  !kNarrow ? 0x7fffffffu : n > 0 ? (n - 1) * step + A.Dv * size : 0);
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const int tok = NC * t + nn;
#pragma unroll
        for (int q = 0; q < RT / 4; ++q) {
          const int cc = c0 + 4 * G * q;
          if constexpr (kNarrow) {
            const int i = (RT * t + 4 * q) / 2;
            __builtin_amdgcn_raw_buffer_store_b64(u2{held_o[i], held_o[i + 1]}, ro,
                                                  la_in(cc < A.Dv, tok * step + cc * 2), 0, 0);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const uint32_t to = la_in((tok < n) & (cc + r < A.Dv), tok * step + (cc + r) * size);
              const float v = __uint_as_float(held_o[RT * t + 4 * q + r]);
              if (A.dtype == PRNN_F32)
                stb<float>(ro, to, 0, v);
              else if (A.dtype == PRNN_F16)
                stb<f16>(ro, to, 0, v);
              else
                stb<bf16>(ro, to, 0, v);
            }
          }
        }
      }
    }
    if constexpr (kKeeps) {
      if (n > 0) {
        // backwards dense rows of the tokens that are there (the others lie behind the buffer), forwards
        // operands (zeros behind the sequence)
        const int step = A.H * A.Dv * 4;
        const size_t elems = dr_operand_elems(kDrC, A.Dv);
        const size_t row = ((tok0 + t0) * A.H + h) * A.Dv, unit = static_cast<size_t>(row0 + held_c) * A.H + h;
        const rsrc_t r = kBack ? make_rsrc(A.dv + row, (n - 1) * step + A.Dv * 4)
                               : make_rsrc(A.e + unit * elems, static_cast<uint32_t>(elems) * 4);
        const uint32_t lane_at = kBack ? la_in(col < A.Dv, 4 * g * step + col * 4) : operand_lane;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const auto rest = kBack ? std::pair<int, int>{0, (at_token(i) - 4 * g) * step} : operand_rest(i / RT, i % RT);
          stb<float>(r, lane_at + rest.second, rest.first, held_k[i]);
        }
      }
    }
  };
  if constexpr (L > 0) {
    __syncthreads();
  } else {
    if (chunks > 0) fetch(chunk_of(0));
  }

  for (int step = 0; step < chunks; ++step) {
    const int c = chunk_of(step), t0 = pc.begin + c * kDrC, n = min(pc.end - t0, kDrC);
    char* const at = lds + (L ? (step & 1) * kChunk : 0);
    const char *const sK = at, *const sQ = at + oQ, *const sZ = at + oZ;
    const float* const sW = reinterpret_cast<const float*>(at + oW);
    if constexpr (L == 0) put(at, c);
    if (!kOwn) flush();
    // what the gradients of this chunk need of the state
    if constexpr (kKeeps && !kNarrow) {
      const size_t elems = dr_operand_elems(A.Dk, A.Dv);
      const rsrc_t rs = make_rsrc(A.keep + (static_cast<size_t>(row0 + c) * A.H + h) * elems, static_cast<uint32_t>(elems) * 4);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const auto rest = operand_rest(t, r);
          if (NC * t < (A.Dk + 31) / 32 * 32)  // rows behind the matrix: zeros up to the end of its tile
            stb<float>(rs, operand_lane + rest.second, rest.first, S[t][r]);
        }
    }
    const char* const sS = kSysLds ? at + oS : A.sys + (static_cast<size_t>(row0 + c) * A.H + h) * kDrSys;
    if constexpr (L == 0) {
      __syncthreads();
      if (step + 1 < chunks) fetch(chunk_of(step + 1));
    }

    // ---- x = K S and the state's part of the output, S^T Q^T
    A_t X[TT], O[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int r = 0; r < RT; ++r) X[t][r] = O[t][r] = 0.0f;
    const size_t keep_elems = dr_operand_elems(A.Dk, A.Dv);
    const rsrc_t keep = make_rsrc(A.keep + (static_cast<size_t>(row0 + c) * A.H + h) * keep_elems,
                                  kNarrow && kKeeps ? static_cast<uint32_t>(keep_elems) * 4 : 0);
    A_t kept;
#pragma unroll
    for (int f = 0; f < KF; ++f) {
      float s[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = S[(8 * f + e) / RT][(8 * f + e) % RT];
      const auto sp = parts_of<M, 3>(s);
      if constexpr (kNarrow && kKeeps) {
        // the state before the chunk (backwards the adjoint behind it): zeros up to the end of its tile of 32
        // rows
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int t = NC == 32 ? f >> 1 : 2 * f + j;
          if (NC == 32 && j != (f & 1)) continue;
          turn(kept, sp, j);
          if ((NC == 32 && j == 0) || NC * t / 32 * 32 >= A.Dk) continue;
#pragma unroll
          for (int q = 0; q < RT / 4; ++q) {
            const float v[4] = {kept[4 * q], kept[4 * q + 1], kept[4 * q + 2], kept[4 * q + 3]};
            __builtin_amdgcn_raw_buffer_store_b128(four(v), keep, turned_at(t, q), 0, 0);
          }
        }
      }
      Op<M, 1> ko[TT], qo[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        ko[t] = row_op<M, G>(sK + (NC * t + nn) * RK, f, g);
        if constexpr (kOut) qo[t] = row_op<M, G>(sQ + (NC * t + nn) * RK, f, g);
      }
#pragma unroll
      for (int k = 0; k < kPairs<1, 3>; ++k)
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          mul_one<NC>(X[t], ko[t], sp, k);
          if constexpr (kOut) mul_one<NC>(O[t], sp, qo[t], k);
        }
    }

    const char* zat = sZ + NC * wave * ES + col_share<M, G, RZ>(lane);
    float y[NC];  // the system's right side: token of element i at_token(i)
    auto weight = [&](int which, int i) {  // of elements i .. i + 3
      return *reinterpret_cast<const f4*>(&sW[which * 64 + at_token(i)]);
    };
    A_t Y[TT];
    Op<M, 1> zo[TF];
#pragma unroll
    for (int f = 0; f < TF; ++f) zo[f] = col_op<M, G, RZ>(zat, 8 * G * f, 0);

    // A token that is not finite, in this column or (the system's word) in all of them, must not reach
    // earlier ones, and backwards later ones, through products with zeros: from it on (backwards: up to
    // it) the column's tokens take no part, and get NaN afterwards.
    constexpr int kNone = kBack ? -1 : kDrC;
    int stop = kNone;
    bool poisoned = false;
    auto reached = [&](int token) { return kBack ? token <= stop : token >= stop; };
    auto widen = [&](const float* x, int from) {  // by what is not finite of elements from .. from + 7
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!(x[i] * 0.0f == 0.0f)) stop = kBack ? max(stop, at_token(from + i)) : min(stop, at_token(from + i));
    };
    auto agree = [&]() {  // the lanes of a column
#pragma unroll
      for (int m = NC; m < 64; m <<= 1) stop = kBack ? max(stop, __shfl_xor(stop, m)) : min(stop, __shfl_xor(stop, m));
    };
    if constexpr (kBack) {
      float zero = 0.0f;
#pragma unroll
      for (int f = 0; f < TF; ++f) {
        float v[8];
        values(zo[f], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) zero = fmaf(v[e], 0.0f, zero);
      }
      if (__any(!(zero == 0.0f))) {
        float v[8];
#pragma unroll
        for (int f = 0; f < TF; ++f) {
          values(zo[f], v);
          widen(v, 8 * f);
        }
        agree();
#pragma unroll
        for (int f = 0; f < TF; ++f) {
          values(zo[f], v);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = reached(at_token(8 * f + e)) ? 0.0f : v[e];
          zo[f] = parts_of<M, 1>(v);
        }
      }
    }
    if constexpr (!kBack) {
#pragma unroll
      for (int f = 0; f < TF; ++f) {
        float v[8];
        values(zo[f], v);
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const f4 w = weight(kWg, 8 * f + e);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = 8 * f + e + r;
            y[i] = fmaf(-w[r], X[i / RT][i % RT], v[e + r]);
          }
        }
      }
    } else {
      // P^T go, then the adjoint behind the chunk
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int r = 0; r < RT; ++r) Y[t][r] = 0.0f;
#pragma unroll
      for (int f = 0; f < TF; ++f) {
        Op<M, 3> m[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (Mat::any(t, f)) m[t] = Mat::get(sS + kPairsAt, t, f, nn, g);
#pragma unroll
        for (int k = 0; k < kPairs<3, 1>; ++k)
#pragma unroll
          for (int t = 0; t < TT; ++t)
            if (Mat::any(t, f)) mul_one<NC>(Y[t], m[t], zo[f], k);
      }
#pragma unroll
      for (int i = 0; i < NC; i += 4) {
        const f4 w = weight(kWr, i), b = weight(kWb, i);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          y[i + r] = b[r] * fmaf(w[r], X[(i + r) / RT][(i + r) % RT], Y[(i + r) / RT][(i + r) % RT]);
      }
    }

    {
      float zero = 0.0f;
#pragma unroll
      for (int i = 0; i < NC; ++i) zero = fmaf(y[i], 0.0f, zero);
      const int all = __float_as_int(sW[kWmeta * 64 + 1]);
      poisoned = __any(!(zero == 0.0f) || all < kDrC || stop != kNone);
      if (poisoned) {
        // (backwards what such a token's keys do to the system, which is without them, is not known)
        if (all < kDrC) stop = kBack ? kDrC - 1 : all;
#pragma unroll
        for (int f = 0; f < TF; ++f) widen(y + 8 * f, 8 * f);
        agree();
#pragma unroll
        for (int i = 0; i < NC; ++i)
          if (reached(at_token(i))) y[i] = 0.0f;
      }
    }

    // ---- (1 + T) y
    Op<M, 3> yo[TF];
#pragma unroll
    for (int f = 0; f < TF; ++f) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = y[8 * f + e];
      yo[f] = parts_of<M, 3>(v);
    }
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int r = 0; r < RT; ++r) Y[t][r] = y[RT * t + r];
#pragma unroll
    for (int f = 0; f < TF; ++f) {
      Op<M, 3> m[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t)
        if (Mat::any(t, f)) m[t] = Mat::get(sS, t, f, nn, g);
#pragma unroll
      for (int k = 0; k < kPairs<3, 3>; ++k)
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (Mat::any(t, f)) mul_one<NC>(Y[t], m[t], yo[f], k);
    }

    float u[NC];  // what is written: b e forwards, dv backwards
#pragma unroll
    for (int i = 0; i < NC; i += 4) {
      const f4 b = kBack ? f4{1.0f, 1.0f, 1.0f, 1.0f} : weight(kWb, i);
#pragma unroll
      for (int r = 0; r < 4; ++r) u[i + r] = b[r] * Y[(i + r) / RT][(i + r) % RT];
    }
    if (poisoned) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (reached(at_token(i))) u[i] = 0.0f;
    }

    if constexpr (kOut) {
      // ---- out
      Op<M, 3> uo[TF];
#pragma unroll
      for (int f = 0; f < TF; ++f) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = u[8 * f + e];
        uo[f] = parts_of<M, 3>(v);
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const float w = sW[kWg * 64 + NC * t + nn] * A.scale;
#pragma unroll
        for (int r = 0; r < RT; ++r) O[t][r] *= w;
      }
#pragma unroll
      for (int f = 0; f < TF; ++f) {
        Op<M, 3> m[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (Mat::any(t, f)) m[t] = Mat::get(sS + kPairsAt, t, f, nn, g);
#pragma unroll
        for (int k = 0; k < kPairs<3, 3>; ++k)
#pragma unroll
          for (int t = 0; t < TT; ++t)
            if (Mat::any(t, f)) mul_one<NC>(O[t], uo[f], m[t], k);
      }
      if (poisoned) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
          for (int r = 0; r < RT; ++r)
            if (NC * t + nn >= __shfl(stop, 4 * G * (r >> 2) + 4 * g + (r & 3))) O[t][r] = __int_as_float(0x7fc00000);
      }
      float v[NC];
#pragma unroll
      for (int i = 0; i < NC; ++i) v[i] = O[i / RT][i % RT];
      hold(held_o, v);
      if constexpr (KIND == kDrKept) {
#pragma unroll
        for (int i = 0; i < NC; ++i) v[i] = Y[i / RT][i % RT];
        hold_rows(v, stop);
      }
    }
    if constexpr (KIND == kDrBackward) {
      hold_rows(u, stop);
    }
    held_n = n;
    held_c = c;

    // ---- the state behind (backwards: the adjoint before) the chunk
    const float tot = sW[kWmeta * 64];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < RT; ++r) S[t][r] *= tot;
    const char* kat = sK + col_share<M, G, RK>(lane);
    const char* qat = sQ + col_share<M, G, RK>(lane);
#pragma unroll
    for (int f = 0; f < TF; ++f) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const f4 w = weight(kBack ? kWg : kWr, 8 * f + e);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[e + r] = (kBack ? -w[r] : w[r]) * u[8 * f + e + r];
      }
      const auto uo = parts_of<M, 3>(v);
      auto into = [&](const char* rows, const Op<M, 3>& o) {
        Op<M, 1> c[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) c[t] = col_op<M, G, RK>(rows, 8 * G * f, NC * t);
#pragma unroll
        for (int k = 0; k < kPairs<1, 3>; ++k)
#pragma unroll
          for (int t = 0; t < KT; ++t) mul_one<NC>(S[t], c[t], o, k);
      };
      into(kat, uo);
      if constexpr (kBack) {
        float z[8];
        values(zo[f], z);
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const f4 w = weight(kWg, 8 * f + e);
#pragma unroll
          for (int r = 0; r < 4; ++r) z[e + r] *= w[r] * A.scale;
        }
        const auto go = parts_of<M, 3>(z);
        into(qat, go);
      }
    }
    if (poisoned && stop != kNone) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < RT; ++r) S[t][r] = __int_as_float(0x7fc00000);
    }
    __syncthreads();
  }

  if (!kOwn) flush();

  // ---- the state behind the piece
  const size_t slot = kOwn ? dr_slot(A.seqs, pc, kBack ? pc.index - 1 : pc.index) : 0;
  if (transfer) {
    const size_t elems = dr_operand_elems(A.Dk, A.Dk);
    const rsrc_t rs = make_rsrc(A.transfer + (slot * A.H + h) * 3 * elems,
                                static_cast<uint32_t>(elems) * 6);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int i = NC * t + 4 * G * (r >> 2) + 4 * g + (r & 3);
        const uint32_t at = la_in((i < (A.Dk + 31) / 32 * 32) & (col < (A.Dk + 15) / 16 * 16),
                                  dr_operand_at(A.Dk, i, col) * 2);
        float v = S[t][r];
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          stb<bf16>(rs, at, j * static_cast<uint32_t>(elems) * 2, v);
          v -= round_to<bf16>(v);
        }
      }
    return;
  }
  float* dst = nullptr;
  if (kOwn) {
    dst = A.piece + (slot * A.H + h) * state_floats;
  } else if (pc.index == (kBack ? 0 : pc.count - 1)) {
    if (float* row = la_row(A.last, pc.seq, A.H * state_floats)) dst = row + h * state_floats;
  }
  if (dst) {
    const rsrc_t rs = make_rsrc(dst, static_cast<uint32_t>(state_floats) * 4);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int i = NC * t + 4 * G * (r >> 2) + 4 * g + (r & 3);
        stb<float>(rs, la_in((i < A.Dk) & (col < A.Dv), (i * A.Dv + col) * 4), 0, S[t][r]);
      }
  }
}

template <class M, int NC, int KD, int W, int L, int KIND>
int dr_launch_walk(const DrWalk& a, hipStream_t stream) {
  const long long items = dr_units(a.seqs, a.seqs.len) * a.H;
  const long long groups = (items + 7) / 8 * 8 * a.tiles;
  if (int rc = check_grid("delta_rule", groups, 64 * (W + L))) return rc;
  dr_walk_kernel<M, NC, KD, W, L, KIND><<<static_cast<unsigned>(groups), 64 * (W + L), 0, stream>>>(a);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

// On bf16 matrix instructions.
template <int KIND, int KD>
int dr_launch_cols(const DrWalk& a, int cols, hipStream_t stream) {
  // Waves that only load: not for pieces' own states, of which two workgroups a CU run without (D = 128,
  // 512 of them: 74 us, 87 with, in two parts throughout), nor where two chunks do not fit LDS.
  constexpr int kLoad = KD <= 128 && KIND != kDrState && KIND != kDrAdjoint ? 4 : 0;
  if (cols == 16 && a.group == 4) return dr_launch_walk<InBf16, 16, KD, 4, kLoad, KIND>(a, stream);
  if constexpr (KD <= 128) {
    if (cols == 16) return dr_launch_walk<InBf16, 16, KD, 2, kLoad, KIND>(a, stream);
    if (a.group == 4) return dr_launch_walk<InBf16, 32, KD, 4, 0, KIND>(a, stream);
    if constexpr (KD <= 64) return dr_launch_walk<InBf16, 32, KD, 2, 0, KIND>(a, stream);
  }
  return fail(PRNN_ERR_RUNTIME, "no walk of %d columns a wave for keys of %d", cols, a.Dk);
}
template <int KIND>
int dr_launch_bf16(const DrWalk& a, int cols, hipStream_t stream) {
  if (a.Dk <= 32) return dr_launch_cols<KIND, 32>(a, cols, stream);
  if (a.Dk <= 64) return dr_launch_cols<KIND, 64>(a, cols, stream);
  if (a.Dk <= 128) return dr_launch_cols<KIND, 128>(a, cols, stream);
  return dr_launch_cols<KIND, 256>(a, cols, stream);
}

}  // namespace prnn
