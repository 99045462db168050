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
#include "linear_attention.h"

namespace prnn {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kC = 32;  // tokens per chunk

// exp(x) of a difference formed in fp64
__device__ __forceinline__ float exp_diff(double a, double b) {
  return fexp(static_cast<float>(a - b));
}

// Four elements of a row as they are stored (raw), from a buffer or one by one; zeros outside.
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
template <typename T>
struct Raw {
  using type = u2;
  static __device__ __forceinline__ u2 load(rsrc_t r, uint32_t o, int left, bool vec) {
    if (vec) return __builtin_amdgcn_raw_buffer_load_b64(r, la_in(left >= 4, o), 0, 0);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_amdgcn_raw_buffer_load_b16(r, la_in(i < left, o + 2 * i), 0, 0);
    return u2{(w[0] & 0xffffu) | w[1] << 16, (w[2] & 0xffffu) | w[3] << 16};
  }
  static __device__ __forceinline__ f4 value(u2 w) {
    return f4{Narrow<T>::lo(w[0]), Narrow<T>::hi(w[0]), Narrow<T>::lo(w[1]), Narrow<T>::hi(w[1])};
  }
};
template <>
struct Raw<float> {
  using type = u4;
  static __device__ __forceinline__ u4 load(rsrc_t r, uint32_t o, int left, bool vec) {
    if (vec) return __builtin_amdgcn_raw_buffer_load_b128(r, la_in(left >= 4, o), 0, 0);
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_amdgcn_raw_buffer_load_b32(r, la_in(i < left, o + 4 * i), 0, 0);
    return w;
  }
  static __device__ __forceinline__ f4 value(u4 w) {
    return f4{__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]),
              __uint_as_float(w[3])};
  }
};

// KT: 32-column blocks of x and y (padded with zeros); W: waves, 16 columns of z each.
template <typename T, int KT, int W, bool STATE_ONLY>
__global__ __launch_bounds__(64 * W) void la_walk_f32_kernel(LaParams P) {
  constexpr int KD = 32 * KT;
  constexpr int NT = 64 * W;
  constexpr int XS = KD + 4;       // row strides in floats: 16 rows of 16-byte reads and
  constexpr int ZS = 16 * W + 4;   // 4 rows, 4 apart, of 16 words each fall into different banks
  constexpr int PS = kC + 4;
  constexpr int NX = kC * KD / 4 / NT;       // 16-byte loads of x (and y) per thread
  constexpr int NZ = kC * 16 * W / 4 / NT;   // of z: 2
  __shared__ __align__(16) float sx[STATE_ONLY ? 4 : kC * XS];
  __shared__ __align__(16) float sy[kC * XS];
  __shared__ __align__(16) float sz[kC * ZS];
  __shared__ __align__(16) float sp[STATE_ONLY ? 4 : kC * PS];
  __shared__ double sG[kC];
  __shared__ float se[kC], sw[kC], sdot[W][kC];
  __shared__ float s_tot, s_sum;

  const LaPlace at = la_place(P);
  if (!at.any) return;
  const LaRole& R = P.role[at.role];
  const int h = at.h, tile = at.tile, piece = at.piece;
  const int tiles = (R.vd + 16 * W - 1) / (16 * W);
  if (tile >= tiles) return;
  const LaPiece pc = la_piece(P.seqs, piece);
  if (STATE_ONLY) {
    // the piece that a walk ends with hands its state to none
    if (pc.alone || (R.rev ? pc.first : pc.last)) return;
  } else if (pc.begin >= pc.end && !pc.first) {
    return;  // no piece (an empty sequence is one, it hands its state on)
  }
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int l16 = lane & 15, q4 = lane >> 4;
  const int b = la_batch(P.seqs, pc);
  const int col0 = tile * 16 * W;            // first column of the workgroup
  const int col = col0 + 16 * wave + l16;    // this lane's column of the state and of out
  const size_t row_floats = static_cast<size_t>(P.H) * P.Dk * P.Dv;
  const size_t head_floats = static_cast<size_t>(h) * P.Dk * P.Dv;

  // ---- the state before the piece
  f4 S[2 * KT];
#pragma unroll
  for (int t = 0; t < 2 * KT; ++t) S[t] = f4{0, 0, 0, 0};
  if (!STATE_ONLY) {
    const float* src = nullptr;
    if (R.piece_state && !pc.alone)
      src = R.piece_state + static_cast<size_t>(piece) * row_floats + head_floats;
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

  const int n_tok = pc.end - pc.begin;
  const int chunks = (n_tok + kC - 1) / kC;
  float sum_decay = 0.0f;

  // A thread's loads of an array are rows apart by a constant number; what lies outside the
  // piece or the width is read as zero (an offset outside the resource).
  using raw = typename Raw<T>::type;
  constexpr int SZ = sizeof(T);
  constexpr int UX = KD / 4, UZ = 4 * W, DX = NT / UX, DZ = NT / UZ;
  const int rowx = tid / UX, cx = (tid % UX) * 4, rowz = tid / UZ, cz = col0 + (tid % UZ) * 4;
  const int fx = R.rev ? kC - 1 - rowx : rowx, fz = R.rev ? kC - 1 - rowz : rowz;
  const int ahead = R.rev ? -1 : 1;
  const int stx = static_cast<int>(R.x.st) * SZ, sty = static_cast<int>(R.y.st) * SZ,
            stz = static_cast<int>(R.z.st) * SZ;
  raw rx[STATE_ONLY ? 1 : NX], ry[NX], rz[NZ];
  LaBits rg{0, 0};
  // token of local index i of the walk
  auto token = [&](int i) { return R.rev ? pc.end - 1 - i : pc.begin + i; };
  auto fetch = [&](int c) {
    const int base = c * kC, left = n_tok - base;
    rg = la_step_decays<kC>(P.g, R.rev, pc, b, h, base, lane);
    if (!STATE_ONLY) {
      const rsrc_t bx = la_rows<kC>(R.x, SZ, b, h, R.rev, pc.begin, pc.end, base);
#pragma unroll
      for (int k = 0; k < NX; ++k)
        rx[k] = Raw<T>::load(bx, (fx + ahead * k * DX) * stx + cx * SZ,
                             rowx + k * DX < left ? R.kd - cx : 0, R.x.vec && R.kd % 4 == 0);
    }
    const rsrc_t by = la_rows<kC>(R.y, SZ, b, h, R.rev, pc.begin, pc.end, base);
#pragma unroll
    for (int k = 0; k < NX; ++k)
      ry[k] = Raw<T>::load(by, (fx + ahead * k * DX) * sty + cx * SZ,
                           rowx + k * DX < left ? R.kd - cx : 0, R.y.vec && R.kd % 4 == 0);
    const rsrc_t bz = la_rows<kC>(R.z, SZ, b, h, R.rev, pc.begin, pc.end, base);
#pragma unroll
    for (int k = 0; k < NZ; ++k)
      rz[k] = Raw<T>::load(bz, (fz + ahead * k * DZ) * stz + cz * SZ,
                           rowz + k * DZ < left ? R.vd - cz : 0, R.z.vec && R.vd % 4 == 0);
  };
  fetch(0);

  for (int c = 0; c < chunks; ++c) {
    const int base = c * kC;
#pragma unroll
    for (int k = 0; k < NX; ++k) {
      const int o = (rowx + k * DX) * XS + cx;
      if (!STATE_ONLY) *reinterpret_cast<f4*>(&sx[o]) = Raw<T>::value(rx[k]);
      *reinterpret_cast<f4*>(&sy[o]) = Raw<T>::value(ry[k]);
    }
#pragma unroll
    for (int k = 0; k < NZ; ++k)
      *reinterpret_cast<f4*>(&sz[(rowz + k * DZ) * ZS + (tid % UZ) * 4]) = Raw<T>::value(rz[k]);
    if (wave == 0) {
      // running sums of the decays in fp64: differences of nearby ones keep their digits
      double G = la_decay_value(P.g, rg.get());
#pragma unroll
      for (int d = 1; d < kC; d <<= 1) {
        const double o = __shfl_up(G, d);
        if (lane >= d) G += o;
      }
      const double last = __shfl(G, kC - 1);
      if (lane < kC) {
        sG[lane] = G;
        se[lane] = fexp(static_cast<float>(G));
        sw[lane] = exp_diff(last, G) * R.u_scale;
      }
      if (lane == 0) {
        s_tot = fexp(static_cast<float>(last));
        s_sum = static_cast<float>(last);
      }
    }
    fetch(c + 1);  // behind the piece's end nothing is loaded; a branch would be waited at
    __syncthreads();

    // ---- the chunk's pairs, masked and decayed: quadrants (0,0), (1,0), (1,1)
    if (!STATE_ONLY) {
      for (int id = wave; id < 3; id += W) {
        const int mi = id > 0, ni = id > 1;
        f4 acc = {0, 0, 0, 0};
        const float* xr = &sx[(16 * mi + l16) * XS + 4 * q4];
        const float* yr = &sy[(16 * ni + l16) * XS + 4 * q4];
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) {
          const f4 a = *reinterpret_cast<const f4*>(xr + 16 * t);
          const f4 bb = *reinterpret_cast<const f4*>(yr + 16 * t);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], bb[r], acc, 0, 0, 0);
        }
        const int n = 16 * ni + l16;
        const double Gn = sG[n];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int m = 16 * mi + 4 * q4 + r;
          sp[m * PS + n] = n <= m ? acc[r] * (R.p_scale * exp_diff(sG[m], Gn)) : 0.0f;
        }
      }
      __syncthreads();
    }

    float zr[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int s = 0; s < 4; ++s) zr[u][s] = sz[(16 * u + 4 * q4 + s) * ZS + 16 * wave + l16];

    // ---- the output: the state's part, then the chunk's own
    if (!STATE_ONLY) {
      f4 O[2] = {f4{0, 0, 0, 0}, f4{0, 0, 0, 0}};
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t)
#pragma unroll
        for (int mi = 0; mi < 2; ++mi) {
          const f4 a = *reinterpret_cast<const f4*>(&sx[(16 * mi + l16) * XS + 16 * t + 4 * q4]);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            O[mi] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], S[t][r], O[mi], 0, 0, 0);
        }
#pragma unroll
      for (int mi = 0; mi < 2; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) O[mi][r] *= R.x_scale * se[16 * mi + 4 * q4 + r];
      }
      // A masked pair is an exact zero, but zero times an infinity or NaN of a later token is
      // not: rows before a column's first such value (rare) are formed without it.
      f4 clean[2] = {O[0], O[1]};
      float bad = 0.0f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < 4; ++s) bad = fmaf(zr[u][s], 0.0f, bad);
      const bool rare = __any(bad != 0.0f);
      int first = kC;
      if (rare) {
#pragma unroll
        for (int u = 1; u >= 0; --u)
#pragma unroll
          for (int s = 3; s >= 0; --s)
            if (zr[u][s] * 0.0f != 0.0f) first = 16 * u + 4 * q4 + s;
        first = min(first, __shfl_xor(first, 16));
        first = min(first, __shfl_xor(first, 32));
      }
#pragma unroll
      for (int mi = 0; mi < 2; ++mi)
#pragma unroll
        for (int u = 0; u <= mi; ++u) {
          const f4 a = *reinterpret_cast<const f4*>(&sp[(16 * mi + l16) * PS + 16 * u + 4 * q4]);
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            O[mi] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], zr[u][s], O[mi], 0, 0, 0);
            if (rare)
              clean[mi] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  a[s], 16 * u + 4 * q4 + s < first ? zr[u][s] : 0.0f, clean[mi], 0, 0, 0);
          }
        }
      if (rare)
#pragma unroll
        for (int mi = 0; mi < 2; ++mi)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * mi + 4 * q4 + r < first) O[mi][r] = clean[mi][r];
#pragma unroll
      for (int mi = 0; mi < 2; ++mi)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * mi + 4 * q4 + r;
          const bool in = base + i < n_tok && col < R.vd;
          const long long t = token(base + i);
          if (in) {
            const long long o = b * R.o_sb + t * R.o_st + h * R.o_sh + col;
            if (R.out_f32)
              static_cast<float*>(R.out)[o] = O[mi][r];
            else
              static_cast<T*>(R.out)[o] = from_f32<T>(O[mi][r]);
          }
          if (R.dots) {
            float d = 0.0f;
            if (in)
              d = O[mi][r] * to_f32(static_cast<const T*>(R.dot.p)[b * R.dot.sb + t * R.dot.st +
                                                                   (h / R.dot.rep) * R.dot.sh + col]);
#pragma unroll
            for (int k = 1; k < 16; k <<= 1) d += __shfl_xor(d, k);
            if (l16 == 0) sdot[wave][i] = d;
          }
        }
    }

    // ---- the state behind the chunk
    const float tot = s_tot;
    sum_decay += s_sum;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int s = 0; s < 4; ++s) zr[u][s] *= sw[16 * u + 4 * q4 + s];
#pragma unroll
    for (int t = 0; t < 2 * KT; ++t) {
      S[t] *= tot;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < 4; ++s)
          S[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(sy[(16 * u + 4 * q4 + s) * XS + 16 * t + l16],
                                                      zr[u][s], S[t], 0, 0, 0);
    }
    __syncthreads();
    if (!STATE_ONLY && R.dots && tid < kC && base + tid < n_tok) {
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

template <typename T, int KT, int W>
int launch(const LaParams& p, bool state_only, hipStream_t stream) {
  const unsigned grid = la_grid(p), block = 64 * W;
  if (state_only)
    la_walk_f32_kernel<T, KT, W, true><<<grid, block, 0, stream>>>(p);
  else
    la_walk_f32_kernel<T, KT, W, false><<<grid, block, 0, stream>>>(p);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

template <typename T, int KT>
int launch_kt(const LaParams& p, int roles, bool state_only, hipStream_t stream) {
  return la_f32_tile_cols(la_widest(p, roles)) == 32
             ? launch<T, KT, 2>(p, state_only, stream)
             : launch<T, KT, 4>(p, state_only, stream);
}

}  // namespace

// two waves where all columns fit in 32, else four
int la_f32_tile_cols(int vd) { return vd <= 32 ? 32 : 64; }

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
    if (kd <= 128) return launch_kt<T, 4>(p, roles, state_only, stream);
    return launch_kt<T, 8>(p, roles, state_only, stream);
  });
}

}  // namespace prnn
