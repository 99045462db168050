// Decayed linear attention, the walk for bf16 storage on v_mfma_f32_32x32x16_bf16: chunks of 64
// tokens, 32 columns of the state per wave.
//
// Everything is formed transposed, so that what one product leaves in registers is the next one's
// operand as it is.  The instruction's result has lane l hold column l % 32 and rows
// 8 b + 4 (l / 32) + r; its operands have lane l hold row (or column) l % 32 and 8 places of the
// contraction.  The order of a contraction is free, so a lane's 8 places are the rows
// {4 (l / 32) + r, 8 + 4 (l / 32) + r} of 16:
//   pairs^T = y x^T    (a tile per wave, handed round through LDS as whole operands)
//   out^T   = S^T x^T + z^T pairs^T
//   S      <- tot S + y^T (w z)
// x lies in LDS with its columns in that order (one 16-byte read per operand), y and z as they
// come, read across tokens by the transposing LDS load.
//
// Operands in bf16 parts: the pairs' weights and the state (S itself stays fp32) in two, 16 bits, so
// that an output is as good as a sum in fp32 that is rounded once (one part each: outputs 2.35e-3 off
// in the 2-norm, for 1.66e-3 of the rounding alone, and 86 us for 91 on 16384 tokens of 8 heads of
// (128, 128)); what enters the state, w z, in three, 24 bits, where the state is an fp32 result, and
// in two where it only goes on to be rounded.  DOTS: roles may have dots with their output (the
// decays' gradient).
//
// An infinity counts as one that is not finite, no more: its parts and their products may be NaN where
// the sum is infinite.
//
// Bound by the chain inside a chunk at the two or three waves a SIMD that the state leaves registers
// for: between the products stand 930 (forward) to 970 (backward) vector instructions a wave and
// chunk of 64 at (64, 64) against 58 and 50 matrix instructions (scaling, splitting, packing); in the
// backward walk they take 28 % of a wave's cycles, waits for LDS, memory and barriers 45 %, and the
// matrix units are busy for 13 % of the time.  16384 tokens of 8 heads of (128, 128): the pieces'
// contributions 28 us (67 MB of k and v, 2.4 TB/s), the walk 47 (134 MB, 2.9 TB/s).  8 x 2048 tokens
// of 16 heads of (64, 64): 22 and 37, backward with all gradients 22 and 120 (115 without the token's
// own pair left out of the dots).  Chunks of 32 (half the work on pairs, twice the scalings of the
// state, two buffers and one barrier) were no faster when these took 34 and 112: 34 and 134.
#include "linear_attention.h"

namespace prnn {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

constexpr int kC = 64;  // tokens per chunk

__device__ __forceinline__ f16v mfma(b8 a, b8 b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// LDS rows.  x is read 16 bytes a lane down 16 rows: its 16-byte units are exchanged by the row's
// number so that these fall into different banks.  y and z are also read 64 bytes along 4 rows,
// for which a pad does (y's four windows overlap by a quarter or a half: two-way conflicts there).
template <int U>
__device__ __forceinline__ int exchange_x(int row) {
  return (U >= 16 ? row & 15 : U == 8 ? (row >> 1) & 7 : (row >> 2) & 3) << 4;
}
constexpr int row_y(int cols) { return cols >= 128 ? cols * 2 + 48 : cols * 2 + 16; }
constexpr int row_z(int cols) { return cols == 32 ? 64 : cols == 64 ? 144 : cols * 2 + 48; }

// Two transposing loads: this lane's column (c0 + lane % 32) at 8 tokens of the 16 from t0.
// `at`: the tile with this lane's share of the address, across_share.
template <int RB>
__device__ __forceinline__ int across_share(int lane) {
  const int i = lane & 15, g = lane >> 4;
  return (4 * (g >> 1) + (i >> 2)) * RB + (16 * (g & 1) + 4 * (i & 3)) * 2;
}
template <int RB>
__device__ __forceinline__ b8 load_across(const char* at, int t0, int c0) {
  union {
    s4 h[2];
    b8 v;
  } r;
  r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + t0 * RB + c0 * 2));
  r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + (t0 + 8) * RB + c0 * 2));
  return r.v;
}

__device__ __forceinline__ b8 pack8(const float* x) {
  union {
    uint32_t w[4];
    b8 v;
  } r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  return r.v;
}
// x as bf16, and what that leaves of it in x.
__device__ __forceinline__ b8 split8(float* x) {
  union {
    uint32_t w[4];
    b8 v;
  } r;
  r.v = pack8(x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] -= lo_bf16(r.w[i]);
    x[2 * i + 1] -= hi_bf16(r.w[i]);
  }
  return r.v;
}

// By value: of two elements of an array the compiler would make one with a variable index.
__device__ __forceinline__ float pick(bool b, float x, float y) { return b ? x : y; }

// Upper half of a's lanes for the lower half of b's; odd rows of 16 lanes for even ones.
__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
__device__ __forceinline__ void swap_rows(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
// A tile of 32 tokens and 32 columns in 16 bits.  As a product leaves it, p: lane l has token l % 32
// and columns 8 q + 4 (l / 32) + {0 .. 3} in p[q].  As rows lie in memory, u: lane l has columns
// 8 (l / 16) + {0 .. 7} of tokens l % 16 in u[0] and 16 + l % 16 in u[1], so that an access of 16
// bytes a lane takes whole 64 bytes of 16 rows, not 16 bytes of 32.
__device__ __forceinline__ void to_rows(u2* p, u4* u) {
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t a = p[q][w], b = p[q + 2][w];
      swap_halves(a, b);
      p[q][w] = a;
      p[q + 2][w] = b;
    }
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t a = p[w & 2][w & 1], b = p[(w & 2) + 1][w & 1];
    swap_rows(a, b);
    u[0][w] = a;
    u[1][w] = b;
  }
}
__device__ __forceinline__ void from_rows(const u4* u, u2* p) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t a = u[0][w], b = u[1][w];
    swap_rows(a, b);
    p[w & 2][w & 1] = a;
    p[(w & 2) + 1][w & 1] = b;
  }
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t a = p[q][w], b = p[q + 2][w];
      swap_halves(a, b);
      p[q][w] = a;
      p[q + 2][w] = b;
    }
}

// Inclusive running sum over the wave's lanes: rows of 16 by shifts, then the rows' last lanes
// handed on.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float scan_up(float v) {
  v = dpp_add<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);  // lane 15 of a row to the next (rows 1 and 3)
  v = dpp_add<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
  return v;
}

template <int KD, int W, bool STATE_ONLY, bool DOTS>
__global__ __launch_bounds__(64 * W, (KD >= 256 || (W < 4 && KD >= 128) || (W == 1 && KD >= 64)) ? 1 : 2)
void la_walk_bf16_kernel(LaParams P) {
  constexpr int NT = 64 * W, VT = 32 * W;
  constexpr int UX = KD / 8, UZ = VT / 8;      // 16-byte units of a row
  constexpr int NX = kC * UX / NT, NZ = kC * UZ / NT;
  constexpr int KT = KD / 32;                  // 32-row tiles of the state
  constexpr int RX = KD * 2, RY = row_y(KD), RZ = row_z(VT);
  constexpr int KX = STATE_ONLY ? 0 : kC * RX;
  constexpr int KP = STATE_ONLY ? 0 : 3 * 2 * 64 * 16 * 2;
  __shared__ __align__(16) char sx[KX ? KX : 16];
  __shared__ __align__(16) char sy[kC * RY];
  __shared__ __align__(16) char sz[kC * RZ];
  __shared__ __align__(16) char sp[KP ? KP : 16];
  __shared__ __align__(16) float sG[kC], se[kC], sw[kC];
  __shared__ float sdot[W][kC], s_own[DOTS ? kC : 1], s_tot, s_sum;
  __shared__ int s_stop[2];

  const LaPlace place = la_place(P);
  if (!place.any) return;
  const LaRole& R = P.role[place.role];
  const int h = place.h, tile = place.tile, piece = place.piece;
  if (tile * VT >= R.vd) return;
  const LaPiece pc = la_piece(P.seqs, piece);
  if (STATE_ONLY) {
    // a part of the piece that the walk ends with hands its state to none
    const int at = pc.begin / P.seqs.span;
    if (pc.alone || at == (R.rev ? pc.s0 : pc.s1 - 1) / P.seqs.span) return;
  } else if (pc.begin >= pc.end && !pc.first) {
    return;  // no piece (an empty sequence is one, it hands its state on)
  }
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int l32 = lane & 31, half = lane >> 5;
  const int b = la_batch(P.seqs, pc);
  const int col0 = tile * VT;
  const int col = col0 + 32 * wave + l32;  // this lane's column of the state
  const size_t row_floats = static_cast<size_t>(P.H) * P.Dk * P.Dv;
  const size_t head_floats = static_cast<size_t>(h) * P.Dk * P.Dv;

  const int n_tok = pc.end - pc.begin;
  float sum_decay = 0.0f;
  auto token = [&](int i) { return R.rev ? pc.end - 1 - i : pc.begin + i; };

  // An array's rows of a chunk are a window of 64 in memory, walked through by one pointer.  A
  // buffer over the window's rows that belong to the piece leaves the others, and columns behind
  // the width, outside: they are read as zero and not written, without a comparison.
  constexpr int DX = NT / UX, DZ = NT / UZ;  // rows between a thread's loads
  const int rowx = tid / UX, cx = (tid % UX) * 8, rowz = tid / UZ, cz = col0 + (tid % UZ) * 8;
  const int ahead = R.rev ? -1 : 1;
  const int low = R.rev ? pc.end - kC : pc.begin;
  auto window = [&](const LaView& v, int size) {
    return static_cast<const char*>(v.p) +
           (b * v.sb + (h / v.rep) * v.sh + static_cast<long long>(low) * v.st) * size;
  };
  const int stx = static_cast<int>(R.x.st) * 2, sty = static_cast<int>(R.y.st) * 2,
            stz = static_cast<int>(R.z.st) * 2;
  const char *px = STATE_ONLY ? nullptr : window(R.x, 2), *py = window(R.y, 2),
             *pz = window(R.z, 2);
  const int fx = R.rev ? kC - 1 - rowx : rowx, fz = R.rev ? kC - 1 - rowz : rowz;
  const uint32_t vx = la_in(cx < R.kd, fx * stx + cx * 2), vy = la_in(cx < R.kd, fx * sty + cx * 2),
                 vz = la_in(cz < R.vd, fz * stz + cz * 2);
  u4 rx[STATE_ONLY ? 1 : NX], ry[NX], rz[NZ];
  LaBits rg{0, 0};
  auto fetch = [&](int base) {
    const int have = max(0, min(n_tok - base, kC)), cut = R.rev ? kC - have : 0;
    rg = la_step_decays<kC>(P.g, R.rev, pc, b, h, base, lane);
    if (!STATE_ONLY) {
      const rsrc_t bx = make_rsrc(px + static_cast<long long>(cut) * stx, have * stx);
#pragma unroll
      for (int k = 0; k < NX; ++k)
        rx[k] = __builtin_amdgcn_raw_buffer_load_b128(bx, vx + (ahead * k * DX - cut) * stx, 0, 0);
      px += ahead * kC * static_cast<long long>(stx);
    }
    const rsrc_t by = make_rsrc(py + static_cast<long long>(cut) * sty, have * sty);
#pragma unroll
    for (int k = 0; k < NX; ++k)
      ry[k] = __builtin_amdgcn_raw_buffer_load_b128(by, vy + (ahead * k * DX - cut) * sty, 0, 0);
    py += ahead * kC * static_cast<long long>(sty);
    const rsrc_t bz = make_rsrc(pz + static_cast<long long>(cut) * stz, have * stz);
#pragma unroll
    for (int k = 0; k < NZ; ++k)
      rz[k] = __builtin_amdgcn_raw_buffer_load_b128(bz, vz + (ahead * k * DZ - cut) * stz, 0, 0);
    pz += ahead * kC * static_cast<long long>(stz);
  };
  auto move_on = [&](int by) {
    if (!STATE_ONLY) px += ahead * by * static_cast<long long>(stx);
    py += ahead * by * static_cast<long long>(sty);
    pz += ahead * by * static_cast<long long>(stz);
  };
  // the output and the rows that it is multiplied with, one window behind
  const int so = R.out_f32 ? 4 : 2, sto = static_cast<int>(R.o_st) * so,
            std_ = static_cast<int>(R.dot.st) * 2;
  const char *po = nullptr, *pd = nullptr;
  if (!STATE_ONLY) po = window(LaView{R.out, R.o_sb, R.o_st, R.o_sh, 1, 1}, so);
  if (DOTS) pd = window(R.dot, 2);
  // Dots leave out a token's pair with itself (linear_attention.hip): its part of the output is added
  // behind them.
  const bool dots = DOTS && R.dots != nullptr;
  // Decays of the chunk's first `n` tokens: running sums from the front for the pairs and the
  // state's part, from the back for what enters the state, so that each weight that counts is the
  // exponential of a short sum.
  auto decays = [&](uint32_t bits, int n) {
    const float g = lane < n ? la_decay_value(P.g, bits) : 0.0f;
    const float G = scan_up(g);
    const float last = __shfl(G, kC - 1);
    const float back = scan_up(__shfl(g, kC - 1 - lane));  // lane l: the sum of the last l + 1
    const float behind = __shfl(back, (kC - 2 - lane) & 63);
    sG[lane] = G * 1.4426950408889634f;
    se[lane] = fexp(G) * R.x_scale;
    sw[lane] = lane == kC - 1 ? R.u_scale : fexp(behind) * R.u_scale;
    if (lane == 0) {
      s_tot = fexp(last);
      s_sum = last;
    }
  };
  const float log_scale = __builtin_amdgcn_logf(fabsf(R.p_scale));  // to base 2; -inf for 0
  if (tid < 2) s_stop[tid] = kC;
  fetch(0);

  // ---- the state before the piece
  f16v S[KT];
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) S[t][r] = 0.0f;
  if (!STATE_ONLY) {
    const float* src = nullptr;
    if (R.piece_state && !pc.alone)
      src = R.piece_state + head_floats +
            la_state_row(P.seqs, pc.seq, R.rev ? pc.end - 1 : pc.begin) * row_floats;
    else if (const float* row = la_row(R.init, pc.seq, row_floats))
      src = row + head_floats;
    if (src) {
      const rsrc_t rs = make_rsrc(src, static_cast<uint32_t>(P.Dk * P.Dv) * 4);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int i = 32 * t + 8 * (r >> 2) + 4 * half + (r & 3);
          const uint32_t o = static_cast<uint32_t>(i * R.sk + col * R.sv) * 4;
          S[t][r] = ldb<float>(rs, la_in((i < R.kd) & (col < R.vd), o), 0);
        }
    }
  }
  __syncthreads();

  int next = 0;
  for (int base = 0, turn = 0; base < n_tok; base = next, turn ^= 1) {
    // x: columns 0-3 | 8-11 and 4-7 | 12-15 of every 16 side by side
#pragma unroll
    for (int k = 0; k < NX; ++k) {
      const int row = rowx + k * DX;
      if (!STATE_ONLY) {
        const int o = row * RX + (tid & 1) * 8, u = (tid % UX >> 1) * 32, f = exchange_x<UX>(row);
        *reinterpret_cast<u2*>(sx + o + (u ^ f)) = u2{rx[k][0], rx[k][1]};
        *reinterpret_cast<u2*>(sx + o + ((u | 16) ^ f)) = u2{rx[k][2], rx[k][3]};
      }
      *reinterpret_cast<u4*>(sy + row * RY + cx * 2) = ry[k];
    }
    int stop_here = kC;
#pragma unroll
    for (int k = NZ - 1; k >= 0; --k) {
      *reinterpret_cast<u4*>(sz + (rowz + k * DZ) * RZ + (tid % UZ) * 16) = rz[k];
      // an exponent of ones: infinity or NaN
      uint32_t bad = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) bad |= (rz[k][q] & 0x7f807f80u) + 0x00800080u;
      if ((bad & 0x80008000u) && rowz + k * DZ > 0) stop_here = rowz + k * DZ;
    }
    if (stop_here < kC) atomicMin(&s_stop[turn], stop_here);
    if (wave == 0) decays(rg.get(), kC);
    next = base + kC;
    __syncthreads();
    if (tid == 0) s_stop[turn ^ 1] = kC;
    const int stop = s_stop[turn];
    if (stop < kC) {
      // A masked pair is an exact zero, but zero times an infinity or NaN of a later token is
      // not: where z holds one behind the chunk's first token (rare), the chunk ends before it
      // and the next one begins there.
      for (int e = tid; e < (kC - stop) * (RY / 16); e += NT)
        *reinterpret_cast<u4*>(sy + stop * RY + e * 16) = u4{0, 0, 0, 0};
      for (int e = tid; e < (kC - stop) * (RZ / 16); e += NT)
        *reinterpret_cast<u4*>(sz + stop * RZ + e * 16) = u4{0, 0, 0, 0};
      if (wave == 0) decays(rg.get(), stop);
      next = base + stop;
      move_on(stop - kC);
      __syncthreads();
    }
    const int n_here = min(n_tok, next) - base;  // tokens of this chunk
    if (STATE_ONLY) fetch(next);

    f16v O[2];
    u4 dv[2][2];
    const int c4 = col0 + 32 * wave + 4 * half;           // first of this lane's columns of out
    const int c8 = col0 + 32 * wave + 8 * (lane >> 4);    // and of its rows in memory
    if (!STATE_ONLY) {
      // ---- the chunk's pairs: tiles (out rows, earlier rows) (0,0), (1,0), (1,1)
      for (int id = wave; id < 3; id += W) {
        const int it = id > 0, jt = id > 1;
        f16v acc;
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
        const int i = 32 * it + l32;
        const char* yr = sy + (32 * jt + l32) * RY + 8 * half;
        const char* xr = sx + i * RX;
        const int f = exchange_x<UX>(i) ^ (16 * half);
#pragma unroll
        for (int k = 0; k < KD / 16; ++k) {
          union {
            uint2 h[2];
            b8 v;
          } y;
          y.h[0] = *reinterpret_cast<const uint2*>(yr + 32 * k);
          y.h[1] = *reinterpret_cast<const uint2*>(yr + 32 * k + 16);
          acc = mfma(y.v, *reinterpret_cast<const b8*>(xr + (f ^ 32 * k)), acc);
        }
        // weights: exponentials to base 2, the scale among them
        if (dots && it == jt) {
          // element 4 q + r with 8 q + 4 half + r = l32
          float a[8], c[4];
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = pick(l32 & 1, acc[2 * e + 1], acc[2 * e]);
#pragma unroll
          for (int e = 0; e < 4; ++e) c[e] = pick(l32 & 2, a[2 * e + 1], a[2 * e]);
          const float d = pick(l32 & 16, pick(l32 & 8, c[3], c[2]), pick(l32 & 8, c[1], c[0]));
          if ((l32 >> 2 & 1) == half) s_own[i] = R.p_scale * d;
        }
        const float Gi = sG[i] + log_scale;
        // Not to be known before: as masks of its own kept over the walk it costs two lane reads
        // an element.
        int before = 32 * jt + 4 * half - i + dots;
        asm volatile("" : "+v"(before));
        float w[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f4 Gj = *reinterpret_cast<const f4*>(&sG[32 * jt + 8 * q + 4 * half]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = acc[4 * q + r] * __builtin_amdgcn_exp2f(Gi - Gj[r]);
            w[4 * q + r] = before <= -(8 * q + r) ? e : 0.0f;
          }
        }
        if (R.p_scale < 0.0f) {
#pragma unroll
          for (int r = 0; r < 16; ++r) w[r] = -w[r];
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          b8* at = reinterpret_cast<b8*>(sp) + (id * 2 + s) * 64 + lane;
          at[0] = split8(w + 8 * s);
          at[3 * 2 * 64] = pack8(w + 8 * s);
        }
      }
      // The rows that the output is multiplied with, then the next chunk's: what is waited for first is
      // loaded first, and nothing before the registers of the pairs are free.  Behind the piece's end
      // nothing is loaded; a branch would be waited at.
      if (DOTS) {
        const int have = dots ? min(n_tok - base, kC) : 0, cut = R.rev ? kC - have : 0;
        const rsrc_t bd = make_rsrc(pd + static_cast<long long>(cut) * std_, have * std_);
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int i = 32 * it + 16 * u + (lane & 15), row = (R.rev ? kC - 1 - i : i) - cut;
            dv[it][u] = __builtin_amdgcn_raw_buffer_load_b128(
                bd, la_in(c8 < R.vd, 0) | (row * std_ + c8 * 2), 0, 0);
          }
      }
      fetch(next);
      // ---- the state's part of the output
#pragma unroll
      for (int it = 0; it < 2; ++it)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[it][r] = 0.0f;
#pragma unroll
      for (int k = 0; k < KD / 16; ++k) {
        float x[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] = S[k / 2][8 * (k & 1) + q];
        const b8 s0 = split8(x), s1 = pack8(x);
#pragma unroll
        for (int it = 0; it < 2; ++it) {
          const b8 xr = *reinterpret_cast<const b8*>(
              sx + (32 * it + l32) * RX + (exchange_x<UX>(l32) ^ (16 * half) ^ (32 * k)));
          O[it] = mfma(s0, xr, O[it]);
          O[it] = mfma(s1, xr, O[it]);
        }
      }
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        const float e = se[32 * it + l32];
#pragma unroll
        for (int r = 0; r < 16; ++r) O[it][r] *= e;
      }
      __syncthreads();
    }

    union Z8 {
      uint32_t w[4];
      b8 v;
    };
    Z8 zf[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) zf[t].v = load_across<RZ>(sz + wave * 64 + across_share<RZ>(lane), 16 * t, 0);

    if (!STATE_ONLY) {
      // ---- the chunk's own part
      auto pairs = [&](int id, int s, int lo) {
        return reinterpret_cast<const b8*>(sp)[((lo * 3 + id) * 2 + s) * 64 + lane];
      };
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        O[1] = mfma(zf[s].v, pairs(1, s, 0), O[1]);
        O[1] = mfma(zf[s].v, pairs(1, s, 1), O[1]);
      }
#pragma unroll
      for (int it = 0; it < 2; ++it)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          O[it] = mfma(zf[2 * it + s].v, pairs(2 * it, s, 0), O[it]);
          O[it] = mfma(zf[2 * it + s].v, pairs(2 * it, s, 1), O[it]);
        }
      // ---- out
      const int cut = R.rev ? kC - n_here : 0;
      const rsrc_t bo = make_rsrc(po + static_cast<long long>(cut) * sto, n_here * sto);
      po += ahead * (next - base) * static_cast<long long>(sto);
      if (DOTS) pd += ahead * (next - base) * static_cast<long long>(std_);
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        if (dots) {
          u2 r[4];
          from_rows(dv[it], r);
          float d = 0.0f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            d = fmaf(O[it][4 * q], lo_bf16(r[q][0]), d);
            d = fmaf(O[it][4 * q + 1], hi_bf16(r[q][0]), d);
            d = fmaf(O[it][4 * q + 2], lo_bf16(r[q][1]), d);
            d = fmaf(O[it][4 * q + 3], hi_bf16(r[q][1]), d);
          }
          d += __shfl_xor(d, 32);
          if (half == 0) sdot[wave][32 * it + l32] = d;
          const float own = s_own[32 * it + l32];
          const char* zr = sz + (32 * it + l32) * RZ + wave * 64 + 8 * half;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const u2 z = *reinterpret_cast<const u2*>(zr + 16 * q);
            O[it][4 * q] = fmaf(own, lo_bf16(z[0]), O[it][4 * q]);
            O[it][4 * q + 1] = fmaf(own, hi_bf16(z[0]), O[it][4 * q + 1]);
            O[it][4 * q + 2] = fmaf(own, lo_bf16(z[1]), O[it][4 * q + 2]);
            O[it][4 * q + 3] = fmaf(own, hi_bf16(z[1]), O[it][4 * q + 3]);
          }
        }
        if (R.out_f32) {
          const int i = 32 * it + l32, row = (R.rev ? kC - 1 - i : i) - cut;
          const uint32_t at = row * sto + c4 * 4;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            __builtin_amdgcn_raw_buffer_store_b128(
                u4{__float_as_uint(O[it][4 * q]), __float_as_uint(O[it][4 * q + 1]),
                   __float_as_uint(O[it][4 * q + 2]), __float_as_uint(O[it][4 * q + 3])},
                bo, la_in(c4 + 8 * q < R.vd, 0) | (at + 32 * q), 0, 0);
        } else {
          u2 p[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            p[q] = u2{pack_bf16x2(O[it][4 * q], O[it][4 * q + 1]),
                      pack_bf16x2(O[it][4 * q + 2], O[it][4 * q + 3])};
          u4 u[2];
          to_rows(p, u);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int i = 32 * it + 16 * k + (lane & 15), row = (R.rev ? kC - 1 - i : i) - cut;
            __builtin_amdgcn_raw_buffer_store_b128(
                u[k], bo, la_in(c8 < R.vd, 0) | (row * sto + c8 * 2), 0, 0);
          }
        }
      }
    }

    // ---- the state behind the chunk
    const float tot = s_tot;
    sum_decay += s_sum;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[t][r] *= tot;
#pragma unroll
    for (int ts = 0; ts < 4; ++ts) {
      float x[8];
      const f4 w0 = *reinterpret_cast<const f4*>(&sw[16 * ts + 4 * half]);
      const f4 w1 = *reinterpret_cast<const f4*>(&sw[16 * ts + 8 + 4 * half]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        x[q] = (q & 1 ? hi_bf16(zf[ts].w[q / 2]) : lo_bf16(zf[ts].w[q / 2])) * w0[q];
        x[4 + q] = (q & 1 ? hi_bf16(zf[ts].w[2 + q / 2]) : lo_bf16(zf[ts].w[2 + q / 2])) * w1[q];
      }
      const b8 z0 = split8(x);
      if ((!DOTS && !STATE_ONLY) || R.exact) {
        const b8 z1 = split8(x), z2 = pack8(x);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const b8 y = load_across<RY>(sy + across_share<RY>(lane), 16 * ts, 32 * t);
          S[t] = mfma(y, z0, S[t]);
          S[t] = mfma(y, z1, S[t]);
          S[t] = mfma(y, z2, S[t]);
        }
      } else {
        const b8 z1 = pack8(x);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const b8 y = load_across<RY>(sy + across_share<RY>(lane), 16 * ts, 32 * t);
          S[t] = mfma(y, z0, S[t]);
          S[t] = mfma(y, z1, S[t]);
        }
      }
    }
    __syncthreads();
    if (dots && tid < n_here) {
      float d = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) d += sdot[w][tid];
      const size_t at = P.seqs.cu ? token(base + tid)
                                  : static_cast<size_t>(b) * P.seqs.T + token(base + tid);
      R.dots[(static_cast<size_t>(tile) * P.H + h) * P.batch_tokens + at] = d;
    }
  }

  // ---- the state behind the piece
  float* dst = nullptr;
  float f = 1.0f;
  if (STATE_ONLY) {
    dst = R.piece_state + static_cast<size_t>(piece) * row_floats + head_floats;
    if (tile == 0 && tid == 0) R.piece_decay[static_cast<size_t>(piece) * P.H + h] = sum_decay;
  } else if (R.rev ? pc.first : pc.last) {
    if (float* row = la_row(R.last, pc.seq, row_floats)) dst = row + head_floats;
    // backwards the first token's decay lies between its R and the initial state's gradient
    if (R.rev && pc.s1 > pc.s0) f = fexp(la_decay(P.g, b, pc.s0, h));
  }
  if (dst) {
    const rsrc_t rs = make_rsrc(dst, static_cast<uint32_t>(P.Dk * P.Dv) * 4);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = 32 * t + 8 * (r >> 2) + 4 * half + (r & 3);
        const uint32_t o = static_cast<uint32_t>(i * R.sk + col * R.sv) * 4;
        stb<float>(rs, la_in((i < R.kd) & (col < R.vd), o), 0, S[t][r] * f);
      }
  }
}

template <int KD, int W>
int launch(const LaParams& p, bool state_only, bool dots, hipStream_t stream) {
  const int block = 64 * W;
  if (int rc = check_grid("linear_attention", la_grid(p), block)) return rc;
  const unsigned grid = la_grid(p);
  if (state_only)
    la_walk_bf16_kernel<KD, W, true, false><<<grid, block, 0, stream>>>(p);
  else if (dots)
    la_walk_bf16_kernel<KD, W, false, true><<<grid, block, 0, stream>>>(p);
  else
    la_walk_bf16_kernel<KD, W, false, false><<<grid, block, 0, stream>>>(p);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

template <int KD>
int launch_kd(const LaParams& p, int roles, bool state_only, bool dots, hipStream_t stream) {
  const int cols = la_bf16_tile_cols(la_widest(p, roles));
  if (cols == 32) return launch<KD, 1>(p, state_only, dots, stream);
  if (cols == 64) return launch<KD, 2>(p, state_only, dots, stream);
  return launch<KD, 4>(p, state_only, dots, stream);
}

}  // namespace

// A wave per 32 columns, as many as the head has, up to four: a workgroup forms the pairs once for
// all of them.  Tiles of 32, 64 and 128 columns, forward in us: 8 x 2048 tokens of 16 heads of
// (64, 64) 85, 63, 79; 4 x 2048 of (96, 96) 119, 97, 71; of (128, 128) 149, 104, 80; 8 x 2048 of
// (32, 32) 49, 47, 66.
int la_bf16_tile_cols(int vd) { return vd <= 32 ? 32 : vd <= 64 ? 64 : 128; }

int la_walk_bf16(LaParams p, int roles, bool state_only, bool dots, hipStream_t stream) {
  const int vd = la_widest(p, roles), cols = la_bf16_tile_cols(vd);
  p.tiles = (vd + cols - 1) / cols;
  p.roles = roles;
  int kd = 0;
  for (int i = 0; i < roles; ++i) kd = std::max(kd, p.role[i].kd);
  if (kd <= 32) return launch_kd<32>(p, roles, state_only, dots, stream);
  if (kd <= 64) return launch_kd<64>(p, roles, state_only, dots, stream);
  if (kd <= 128) return launch_kd<128>(p, roles, state_only, dots, stream);
  return launch_kd<256>(p, roles, state_only, dots, stream);
}

}  // namespace prnn
