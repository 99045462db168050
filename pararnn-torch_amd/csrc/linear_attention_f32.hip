// Decayed linear attention, the walk in fp32 arithmetic (fp32 and fp16 storage, and bf16 where
// the bf16 kernel does not apply): v_mfma_f32_16x16x4_f32, chunks of 32 tokens.
//
// A workgroup walks one piece of one head for 16 columns of the state per wave.  The state's
// 16-row tiles stay in the matrix instruction's result layout (lane: column l % 16, rows
// 4 (l / 16) + r) and are its second operand as they are: the order of a contraction is free,
// so instruction r takes rows {r, 4 + r, 8 + r, 12 + r} and the other operand is read to match,
// four instructions' worth in one 16-byte LDS read.
//
// fp16 storage comes here too: its values are exact in fp32, while a state rounded to fp16 for
// a 16-bit matrix product could pass 65504.
//
// Bound by the chain from chunk to chunk (LDS, products of 16 x 16 x 4, decays in fp64), which the
// waves of a CU do not hide: 8 x 2048 tokens of 16 heads of (64, 64) in fp32 138 us with the
// pieces' contributions, 62 TFLOP/s of the 154 of a large product.  Training on 3 x 1001 tokens of
// 6 heads of (48, 72): contributions 13 us, walk 18; backward 13 and 45.
#include "linear_attention.h"

namespace prnn {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kC = 32;  // tokens per chunk

// 2^x of a difference formed in fp64
__device__ __forceinline__ float exp2_diff(double a, double b) {
  return __builtin_amdgcn_exp2f(static_cast<float>(a - b));
}

// Lane i of a row of 16 gets lane i's neighbour's value by a DPP control (0 where there is none).
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROWS, 0xf, false);
  return v + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Inclusive running sum over lanes 0 .. 31.
__device__ __forceinline__ double scan_up(double v) {
  v = dpp_add<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  return dpp_add<0x142, 0xa>(v);  // lane 15 to the next row
}
// Sum over a row of 16 lanes, in every lane: rotations by 8, 4, 2, 1.
template <int CTRL>
__device__ __forceinline__ float rot_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float row_sum(float v) {
  return rot_add<0x121>(rot_add<0x122>(rot_add<0x124>(rot_add<0x128>(v))));
}

// Four elements of a row as they are stored (raw), from a buffer or one by one; zeros outside.
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
template <typename T>
struct Raw {
  using type = u2;
  template <bool VEC>
  static __device__ __forceinline__ u2 load(rsrc_t r, uint32_t o, int left) {
    if (VEC) return __builtin_amdgcn_raw_buffer_load_b64(r, la_in(left >= 4, o), 0, 0);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_amdgcn_raw_buffer_load_b16(r, la_in(i < left, o + 2 * i), 0, 0);
    return u2{(w[0] & 0xffffu) | w[1] << 16, (w[2] & 0xffffu) | w[3] << 16};
  }
  static __device__ __forceinline__ float one(rsrc_t r, uint32_t o) { return ldb<T>(r, o, 0); }
  static __device__ __forceinline__ bool bad(u2 w) {
    constexpr uint32_t kOnes = std::is_same_v<T, f16> ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t kStep = std::is_same_v<T, f16> ? 0x04000400u : 0x00800080u;
    return ((((w[0] & kOnes) + kStep) | ((w[1] & kOnes) + kStep)) & 0x80008000u) != 0;
  }
  static __device__ __forceinline__ f4 value(u2 w) {
    return f4{Narrow<T>::lo(w[0]), Narrow<T>::hi(w[0]), Narrow<T>::lo(w[1]), Narrow<T>::hi(w[1])};
  }
};
template <>
struct Raw<float> {
  using type = u4;
  template <bool VEC>
  static __device__ __forceinline__ u4 load(rsrc_t r, uint32_t o, int left) {
    if (VEC) return __builtin_amdgcn_raw_buffer_load_b128(r, la_in(left >= 4, o), 0, 0);
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_amdgcn_raw_buffer_load_b32(r, la_in(i < left, o + 4 * i), 0, 0);
    return w;
  }
  static __device__ __forceinline__ float one(rsrc_t r, uint32_t o) { return ldb<float>(r, o, 0); }
  static __device__ __forceinline__ bool bad(u4 w) {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) b |= (w[i] & 0x7f800000u) + 0x00800000u;
    return (b & 0x80000000u) != 0;
  }
  static __device__ __forceinline__ f4 value(u4 w) {
    return f4{__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]),
              __uint_as_float(w[3])};
  }
};

constexpr int low_power(int n) { return n < 2 ? 1 : 2 * low_power(n / 2); }

// KT: 32-column blocks of x and y (padded with zeros); W: waves, 16 columns of z each; VEC: rows
// of x, y and z admit accesses of four elements.
template <typename T, int KT, int W, bool VEC, bool STATE_ONLY>
__global__ __launch_bounds__(64 * W) void la_walk_f32_kernel(LaParams P) {
  constexpr int KD = 32 * KT;
  constexpr int NT = 64 * W;
  constexpr int XS = KD + 4;       // row strides in floats: 16 rows of 16-byte reads and
  constexpr int ZS = 16 * W + 4;   // 4 rows, 4 apart, of 16 words each fall into different banks
  constexpr int PS = kC + 4;
  constexpr int UX = KD / 4, UZ = 4 * W;                     // units of four in a row
  constexpr int DX = std::min(kC, low_power(NT / UX)), DZ = NT / UZ;  // rows that a round takes
  constexpr int NX = kC / DX, NZ = kC / DZ;
  __shared__ __align__(16) float sx[STATE_ONLY ? 4 : kC * XS];
  __shared__ __align__(16) float sy[kC * XS];
  __shared__ __align__(16) float sz[kC * ZS];
  __shared__ __align__(16) float sp[STATE_ONLY ? 4 : kC * PS];
  __shared__ __align__(16) double sG[kC];
  __shared__ __align__(16) float se[kC], sw[kC], s_own[STATE_ONLY ? 4 : kC];
  __shared__ float sdot[W][kC], s_tot, s_sum;
  __shared__ int s_stop[2];

  const LaPlace place = la_place(P);
  if (!place.any) return;
  const LaRole& R = P.role[place.role];
  const int h = place.h, tile = place.tile, piece = place.piece;
  const int col0 = tile * 16 * W;            // first column of the workgroup
  if (col0 >= R.vd) return;
  const LaPiece pc = la_piece(P.seqs, piece);
  if (STATE_ONLY) {
    // a part of the piece that the walk ends with hands its state to none
    const int at = pc.begin / P.seqs.span;
    if (pc.alone || at == (R.rev ? pc.s0 : pc.s1 - 1) / P.seqs.span) return;
  } else if (pc.begin >= pc.end && !pc.first) {
    return;  // no piece (an empty sequence is one, it hands its state on)
  }
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int l16 = lane & 15, q4 = lane >> 4;
  const int b = la_batch(P.seqs, pc);
  const int col = col0 + 16 * wave + l16;    // this lane's column of the state and of out
  const size_t row_floats = static_cast<size_t>(P.H) * P.Dk * P.Dv;
  const size_t head_floats = static_cast<size_t>(h) * P.Dk * P.Dv;
  const int n_tok = pc.end - pc.begin;
  float sum_decay = 0.0f;
  // token of local index i of the walk
  auto token = [&](int i) { return R.rev ? pc.end - 1 - i : pc.begin + i; };

  // A thread's loads of an array are rows apart by a constant number; what lies outside the
  // piece or the width is read as zero (an offset outside the resource).
  using raw = typename Raw<T>::type;
  constexpr int SZ = sizeof(T);
  const int rowx = tid / UX, cx = (tid % UX) * 4, rowz = tid / UZ, cz = (tid % UZ) * 4;
  const bool loads_x = rowx < DX;  // all threads but where a row's units are no power of two
  const int widthx = loads_x ? R.kd - cx : 0, widthz = R.vd - col0 - cz;
  const int fx = R.rev ? kC - 1 - rowx : rowx, fz = R.rev ? kC - 1 - rowz : rowz;
  const int ahead = R.rev ? -1 : 1;
  const int stx = static_cast<int>(R.x.st) * SZ, sty = static_cast<int>(R.y.st) * SZ,
            stz = static_cast<int>(R.z.st) * SZ;
  raw rx[STATE_ONLY ? 1 : NX], ry[NX], rz[NZ];
  LaBits rg{0, 0};
  auto fetch = [&](int base) {
    const int left = n_tok - base;
    rg = la_step_decays<kC>(P.g, R.rev, pc, b, h, base, lane);
    if (!STATE_ONLY) {
      const rsrc_t bx = la_rows<kC>(R.x, SZ, b, h, R.rev, pc.begin, pc.end, base);
#pragma unroll
      for (int k = 0; k < NX; ++k)
        rx[k] = Raw<T>::template load<VEC>(bx, (fx + ahead * k * DX) * stx + cx * SZ,
                                           rowx + k * DX < left ? widthx : 0);
    }
    const rsrc_t by = la_rows<kC>(R.y, SZ, b, h, R.rev, pc.begin, pc.end, base);
#pragma unroll
    for (int k = 0; k < NX; ++k)
      ry[k] = Raw<T>::template load<VEC>(by, (fx + ahead * k * DX) * sty + cx * SZ,
                                         rowx + k * DX < left ? widthx : 0);
    const rsrc_t bz = la_rows<kC>(R.z, SZ, b, h, R.rev, pc.begin, pc.end, base);
#pragma unroll
    for (int k = 0; k < NZ; ++k)
      rz[k] = Raw<T>::template load<VEC>(bz, (fz + ahead * k * DZ) * stz + (col0 + cz) * SZ,
                                         rowz + k * DZ < left ? widthz : 0);
  };
  // Decays of the chunk's first n tokens, to base 2: running sums in fp64, so that differences of
  // nearby ones keep their digits.
  auto decays = [&](uint32_t bits, int n) {
    const float g = lane < n ? la_decay_value(P.g, bits) : 0.0f;
    const double G = scan_up(g * 1.4426950408889634);
    const double last = __shfl(G, kC - 1);
    if (lane < kC) {
      sG[lane] = G;
      se[lane] = exp2_diff(G, 0.0) * R.x_scale;
      sw[lane] = exp2_diff(last, G) * R.u_scale;
    }
    if (lane == 0) {
      s_tot = exp2_diff(last, 0.0);
      s_sum = static_cast<float>(last * 0.6931471805599453);
    }
  };
  if (tid < 2) s_stop[tid] = kC;
  fetch(0);

  // ---- the state before the piece
  f4 S[2 * KT];
#pragma unroll
  for (int t = 0; t < 2 * KT; ++t) S[t] = f4{0, 0, 0, 0};
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
      for (int t = 0; t < 2 * KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * t + 4 * q4 + r;
          const uint32_t o = static_cast<uint32_t>(i * R.sk + col * R.sv) * 4;
          S[t][r] = ldb<float>(rs, la_in((i < R.kd) & (col < R.vd), o), 0);
        }
    }
  }
  __syncthreads();

  int next = 0;
  for (int base = 0, turn = 0; base < n_tok; base = next, turn ^= 1) {
#pragma unroll
    for (int k = 0; k < NX; ++k) {
      const int o = (rowx + k * DX) * XS + cx;
      if (loads_x) {
        if (!STATE_ONLY) *reinterpret_cast<f4*>(&sx[o]) = Raw<T>::value(rx[k]);
        *reinterpret_cast<f4*>(&sy[o]) = Raw<T>::value(ry[k]);
      }
    }
    int stop_here = kC;
#pragma unroll
    for (int k = NZ - 1; k >= 0; --k) {
      *reinterpret_cast<f4*>(&sz[(rowz + k * DZ) * ZS + cz]) = Raw<T>::value(rz[k]);
      if (Raw<T>::bad(rz[k]) && rowz + k * DZ > 0) stop_here = rowz + k * DZ;
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
      for (int e = stop * XS + tid; e < kC * XS; e += NT) sy[e] = 0.0f;
      for (int e = stop * ZS + tid; e < kC * ZS; e += NT) sz[e] = 0.0f;
      if (wave == 0) decays(rg.get(), stop);
      next = base + stop;
      __syncthreads();
    }
    const int n_here = min(n_tok, next) - base;  // tokens of this chunk

    // ---- the chunk's pairs, masked and decayed: quadrants (0,0), (1,0), (1,1).  Dots leave out a
    // token's pair with itself (linear_attention.hip): its part of the output is added behind them.
    float dv[2][4];
    if (!STATE_ONLY) {
      for (int id = wave; id < 3; id += W) {
        const int mi = id > 0, ni = id > 1;
        f4 acc[2] = {f4{0, 0, 0, 0}, f4{0, 0, 0, 0}};
        const float* xr = &sx[(16 * mi + l16) * XS + 4 * q4];
        const float* yr = &sy[(16 * ni + l16) * XS + 4 * q4];
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) {
          const f4 a = *reinterpret_cast<const f4*>(xr + 16 * t);
          const f4 bb = *reinterpret_cast<const f4*>(yr + 16 * t);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[r & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], bb[r], acc[r & 1], 0, 0, 0);
        }
        const int n = 16 * ni + l16;
        const double Gn = sG[n];
        // not to be known before, or its masks are kept over the walk
        int after = n - 16 * mi - 4 * q4;
        asm volatile("" : "+v"(after));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int m = 16 * mi + 4 * q4 + r;
          acc[0][r] = (acc[0][r] + acc[1][r]) * (R.p_scale * exp2_diff(sG[m], Gn));
          sp[m * PS + n] = after <= r ? acc[0][r] : 0.0f;
        }
        if (R.dots) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (after == r) {
              const int m = 16 * mi + 4 * q4 + r;
              s_own[m] = acc[0][r];
              sp[m * PS + n] = 0.0f;
            }
        }
      }
      // The rows that the output is multiplied with, then the next chunk's: what is waited for
      // first is loaded first.  Behind the piece's end nothing is loaded; a branch would be
      // waited at.
      const rsrc_t bd = la_rows<kC>(R.dot, SZ, b, h, R.rev, pc.begin, pc.end, base);
#pragma unroll
      for (int mi = 0; mi < 2; ++mi)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * mi + 4 * q4 + r, row = R.rev ? kC - 1 - i : i;
          dv[mi][r] = Raw<T>::one(bd, la_in((R.dots != nullptr) & (i < n_here) & (col < R.vd),
                                            (row * static_cast<int>(R.dot.st) + col) * SZ));
        }
    }
    fetch(next);
    if (!STATE_ONLY) __syncthreads();

    float zr[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int s = 0; s < 4; ++s) zr[u][s] = sz[(16 * u + 4 * q4 + s) * ZS + 16 * wave + l16];

    // ---- the output: the state's part, then the chunk's own
    if (!STATE_ONLY) {
      f4 O[2] = {f4{0, 0, 0, 0}, f4{0, 0, 0, 0}};
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t) {
        const f4 a0 = *reinterpret_cast<const f4*>(&sx[l16 * XS + 16 * t + 4 * q4]);
        const f4 a1 = *reinterpret_cast<const f4*>(&sx[(16 + l16) * XS + 16 * t + 4 * q4]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          O[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(a0[r], S[t][r], O[0], 0, 0, 0);
          O[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(a1[r], S[t][r], O[1], 0, 0, 0);
        }
      }
#pragma unroll
      for (int mi = 0; mi < 2; ++mi) {
        const f4 e = *reinterpret_cast<const f4*>(&se[16 * mi + 4 * q4]);
        O[mi] *= e;
      }
      const f4 p0 = *reinterpret_cast<const f4*>(&sp[l16 * PS + 4 * q4]);
      const f4 p1 = *reinterpret_cast<const f4*>(&sp[(16 + l16) * PS + 4 * q4]);
      const f4 p2 = *reinterpret_cast<const f4*>(&sp[(16 + l16) * PS + 16 + 4 * q4]);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        O[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(p0[s], zr[0][s], O[0], 0, 0, 0);
        O[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(p1[s], zr[0][s], O[1], 0, 0, 0);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s)
        O[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(p2[s], zr[1][s], O[1], 0, 0, 0);
      const int so = R.out_f32 ? 4 : SZ;
      const rsrc_t bo = la_rows<kC>(LaView{R.out, R.o_sb, R.o_st, R.o_sh, 1, 1}, so, b, h, R.rev,
                                    pc.begin, pc.end, base);
#pragma unroll
      for (int mi = 0; mi < 2; ++mi) {
        if (R.dots) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float d = row_sum(O[mi][r] * dv[mi][r]);
            if (l16 == 0) sdot[wave][16 * mi + 4 * q4 + r] = d;
          }
          const f4 own = *reinterpret_cast<const f4*>(&s_own[16 * mi + 4 * q4]);
#pragma unroll
          for (int r = 0; r < 4; ++r) O[mi][r] = fmaf(own[r], zr[mi][r], O[mi][r]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * mi + 4 * q4 + r, row = R.rev ? kC - 1 - i : i;
          const uint32_t o = la_in((i < n_here) & (col < R.vd),
                                   (row * static_cast<int>(R.o_st) + col) * so);
          if (R.out_f32)
            stb<float>(bo, o, 0, O[mi][r]);
          else
            stb<T>(bo, o, 0, O[mi][r]);
        }
      }
    }

    // ---- the state behind the chunk
    const float tot = s_tot;
    sum_decay += s_sum;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const f4 w = *reinterpret_cast<const f4*>(&sw[16 * u + 4 * q4]);
#pragma unroll
      for (int s = 0; s < 4; ++s) zr[u][s] *= w[s];
    }
#pragma unroll
    for (int t = 0; t < 2 * KT; ++t) S[t] *= tot;
    // two tiles at a time: their chains of products run side by side
#pragma unroll
    for (int t = 0; t < 2 * KT; t += 2)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const float* y = &sy[(16 * u + 4 * q4 + s) * XS + 16 * t + l16];
          S[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[0], zr[u][s], S[t], 0, 0, 0);
          S[t + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[16], zr[u][s], S[t + 1], 0, 0, 0);
        }
    __syncthreads();
    if (!STATE_ONLY && R.dots && tid < n_here) {
      float d = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) d += sdot[w][tid];
      const size_t row = P.seqs.cu ? token(base + tid)
                                   : static_cast<size_t>(b) * P.seqs.T + token(base + tid);
      R.dots[(static_cast<size_t>(tile) * P.H + h) * P.batch_tokens + row] = d;
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
    for (int t = 0; t < 2 * KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * t + 4 * q4 + r;
        const uint32_t o = static_cast<uint32_t>(i * R.sk + col * R.sv) * 4;
        stb<float>(rs, la_in((i < R.kd) & (col < R.vd), o), 0, S[t][r] * f);
      }
  }
}

template <typename T, int KT, int W, bool VEC>
int launch(const LaParams& p, bool state_only, hipStream_t stream) {
  const int block = 64 * W;
  if (int rc = check_grid("linear_attention", la_grid(p), block)) return rc;
  const unsigned grid = la_grid(p);
  if (state_only)
    la_walk_f32_kernel<T, KT, W, VEC, true><<<grid, block, 0, stream>>>(p);
  else
    la_walk_f32_kernel<T, KT, W, VEC, false><<<grid, block, 0, stream>>>(p);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

template <typename T, int KT>
int launch_kt(const LaParams& p, int roles, bool state_only, hipStream_t stream) {
  bool vec = true;
  for (int i = 0; i < roles; ++i) {
    const LaRole& r = p.role[i];
    vec = vec && (state_only || r.x.vec) && r.y.vec && r.z.vec && r.kd % 4 == 0 && r.vd % 4 == 0;
  }
  if (la_f32_tile_cols(la_widest(p, roles)) == 32)
    return vec ? launch<T, KT, 2, true>(p, state_only, stream)
               : launch<T, KT, 2, false>(p, state_only, stream);
  return vec ? launch<T, KT, 4, true>(p, state_only, stream)
             : launch<T, KT, 4, false>(p, state_only, stream);
}

}  // namespace

// Four waves, or two where four would leave half of them without columns.  Tiles of 32 and 64
// columns, forward in us: 8 x 2048 tokens of 16 heads of (64, 64) 184 and 137, 4 x 2048 of (96, 96)
// 185 and 174 (on the edge of the rule), of (128, 128) 297 and 209; a training step on widths (48, 72)
// 113 and 140.
int la_f32_tile_cols(int vd) { return (vd + 63) / 64 * 64 - vd >= 32 ? 32 : 64; }

int la_walk_f32(LaParams p, int roles, bool state_only, int dtype, hipStream_t stream) {
  const int vd = la_widest(p, roles), cols = la_f32_tile_cols(vd);
  p.tiles = (vd + cols - 1) / cols;
  p.roles = roles;
  int kd = 0;
  for (int i = 0; i < roles; ++i) kd = std::max(kd, p.role[i].kd);
  return with_storage(dtype, [&](auto z) {
    using T = decltype(z);
    if (kd <= 32) return launch_kt<T, 1>(p, roles, state_only, stream);
    if (kd <= 64) return launch_kt<T, 2>(p, roles, state_only, stream);
    if (kd <= 96) return launch_kt<T, 3>(p, roles, state_only, stream);
    if (kd <= 128) return launch_kt<T, 4>(p, roles, state_only, stream);
    return launch_kt<T, 8>(p, roles, state_only, stream);
  });
}

}  // namespace prnn
