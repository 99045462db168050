// Gated delta rule: what its kernels and their host code share.
//
// One head holds a state S (Dk x Dv) in fp32; a token with log decay g_t and rate b_t writes what
// the decayed state lacks of v_t at k_t:
//
//   e_t = v_t - exp(g_t) S_{t-1}^T k_t,   u_t = b_t e_t,
//   S_t = exp(g_t) S_{t-1} + k_t u_t^T,   o_t = scale S_t^T q_t.
//
// Chunks of 64 tokens, G_i the running sum of g inside a chunk (its first token included), S the
// state before it, and the strictly lower N_ij = exp(G_i - G_j) k_i . k_j:
//
//   (1 + N diag(b)) e = v - exp(G) K S             a unit triangular system
//   o  = scale [ exp(G) Q S + P u ],               P_ij = exp(G_i - G_j) q_i . k_j  (j <= i)
//   S' = exp(G_last) S + (exp(G_last - G) K)^T u.
//
// Its gradients, with R = dL/dS behind the chunk:
//
//   (1 + N diag(b))^T dv = diag(b) [ scale P^T go + exp(G_last - G) K R ]     the same system
//   R' = exp(G_last) R + (scale exp(G) Q)^T go - (exp(G) K)^T dv
//   dq = scale [ exp(G) go S^T + (go u^T . lower) K ]
//   dk = exp(G_last - G) u R^T + scale (go u^T . lower)^T Q - exp(G) dv S^T - (X + X^T) K,
//   X_ij = exp(G_i - G_j) dv_i . u_j (j < i).
//
// The inverses of the systems, the pairs P and the decays' exponentials do not depend on the state:
// a kernel of their own forms them for all chunks at once (delta_rule_systems.hip).  What is left
// goes from chunk to chunk: three products forwards (delta_rule_walk.h), the same three backwards.
// With the states before and the adjoints behind the chunks, all other gradients are formed for all
// chunks at once (delta_rule_grad.hip).
//
// Two arithmetics: bf16 storage of widths in eights on bf16 matrix instructions, operands that are
// not given in bf16 in three bf16 parts, all of an fp32 value's 24 bits; everything else (fp32, fp16, odd
// widths) on fp32 ones.  Whatever goes through memory (systems, kept errors, states and adjoints) is fp32.
#pragma once

#include "linear_attention.h"

namespace prnn {

constexpr int kDrC = 64;  // tokens of a chunk

// ---- where chunks and pieces lie ---------------------------------------------------------
//
// Units of `len` tokens counted from every sequence's own start.  (How long pieces are goes by the whole
// batch, and with it the last bits of a result.)  Unit i of sequence s of a packed stream is number
// s + floor(cu[s] / len) + i: numbers are distinct and below n_seq + ceil(T / len).
struct DrUnit {
  int seq, index, count;  // index of `count` in its sequence
  int s0, s1;             // the sequence's tokens
  int begin, end;         // the unit's
  bool any;               // false: no unit has this number
};

__device__ __forceinline__ int dr_base(const LaSeqs& q, int len, int s, int s0) {
  return q.cu ? s + s0 / len : s * (q.T > len ? (q.T + len - 1) / len : 1);
}

__device__ __forceinline__ DrUnit dr_unit(const LaSeqs& q, int len, int id) {
  DrUnit r;
  if (q.cu == nullptr) {
    r.count = q.T > len ? (q.T + len - 1) / len : 1;
    r.seq = id / r.count;
    r.index = id - r.seq * r.count;
    r.s0 = 0;
    r.s1 = q.T;
    r.any = r.seq < q.n_seq;
  } else {
    int lo = 0, hi = q.n_seq;  // the last s with s + cu[s] / len <= id
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (mid + la_offset(q, mid) / len <= id) lo = mid; else hi = mid;
    }
    r.seq = lo;
    r.s0 = la_offset(q, lo);
    r.s1 = la_offset(q, lo + 1);
    if (r.s1 < r.s0) r.s1 = r.s0;
    r.count = r.s1 - r.s0 > len ? (r.s1 - r.s0 + len - 1) / len : 1;
    r.index = id - lo - r.s0 / len;
    r.any = r.index >= 0 && r.index < r.count;
  }
  const long long b = r.s0 + static_cast<long long>(r.index) * len;
  r.begin = b < r.s1 ? static_cast<int>(b) : r.s1;
  r.end = r.s1 - r.begin > len ? r.begin + len : r.s1;
  return r;
}
inline long long dr_units(const LaSeqs& q, long long len) {
  if (q.cu) return q.n_seq + (q.T + len - 1) / len;
  return static_cast<long long>(q.n_seq) * (q.T > len ? (q.T + len - 1) / len : 1);
}

// Between a cut sequence's pieces i and i + 1 lies slot i of its own, for a state and a transfer.  Of a
// packed stream it is number floor(cu[s] / len) + i: the last of a sequence's, with n = ceil(L / len) pieces,
// is below floor((cu[s] + L) / len), where the next one's begin, and all are below T / len.
__device__ __forceinline__ size_t dr_slot(const LaSeqs& q, const DrUnit& piece, int i) {
  return static_cast<size_t>(q.cu ? piece.s0 / q.len : piece.seq * (piece.count - 1)) + i;
}
inline long long dr_slots(const LaSeqs& q) { return q.cu ? q.T / q.len : dr_units(q, q.len) - q.n_seq; }

// Token 0 of a unit among all tokens of the batch (rows of dense arrays).
__device__ __forceinline__ size_t dr_token(const LaSeqs& q, const DrUnit& u, int t) {
  return q.cu ? static_cast<size_t>(t) : static_cast<size_t>(u.seq) * q.T + t;
}
__device__ __forceinline__ int dr_batch(const LaSeqs& q, const DrUnit& u) { return q.cu ? 0 : u.seq; }

// ---- a chunk's system --------------------------------------------------------------------
//
// Per chunk and head: the strictly lower part of the inverse, then the pairs, each as the tiles
// (0, 0), (1, 0), (1, 1) of 32 x 32, rows of 32 elements whose units of four are exchanged by the row
// (dr_unit_of), fp32; then kDrW rows of 64 floats.
constexpr int kDrTiles = 3 * 32 * 32 * 4;  // bytes of a matrix
enum { kWg, kWr, kWb, kWhi, kWlo, kWmeta, kDrW };  // exp(G), exp(G_last - G), b, G in two parts
constexpr int kDrSys = 2 * kDrTiles + kDrW * 64 * 4;
static_assert(kDrSys % 256 == 0, "blocks stay aligned");
// kWmeta: [0] exp(G_last), [1] the first token that is not finite (64: none), as an integer

// (so that 16 or 32 rows of a step fall into all banks, two words each)
__device__ __forceinline__ int dr_unit_of(int row, int unit) { return unit ^ ((row >> 1) & 7); }

// A token's rate.
__device__ __forceinline__ float dr_rate(const LaDecay& b, int batch, int t, int h) {
  const uint32_t bits = la_decay_bits(b, batch, t, h);
  return b.dtype == PRNN_F32   ? __uint_as_float(bits)
         : b.dtype == PRNN_F16 ? Narrow<f16>::val(bits)
                               : Narrow<bf16>::val(bits);
}

struct DrSystems {
  LaSeqs seqs;
  LaView q, k;
  LaDecay g, b;
  char* sys;
  int H, Dk, dtype;
  // Of a packed batch also the order in which a walk takes its pieces, longest first (37 sequences of 130
  // to 1500 tokens, 16 heads: the walk 126 us in the order given, 82 so).
  LaSeqs pieces;
  int* order;  // NULL: none
  int n_pieces;
  float scale;
};

// Matrices that are only read as operands lie in memory as such, in fp32: tiles of 32 rows, steps of 16 columns,
// lane by lane the 8 places that it has of a row (tiles.h); what is behind the matrix holds zeros.
inline __host__ __device__ size_t dr_operand_elems(int rows, int cols) {
  return static_cast<size_t>((rows + 31) / 32) * ((cols + 15) / 16) * 512;
}
__device__ __forceinline__ uint32_t dr_operand_at(int cols, int i, int j) {
  const int lane = (i & 31) + 32 * ((j >> 2) & 1), e = (j & 3) + 4 * ((j >> 3) & 1);
  return (((i >> 5) * ((cols + 15) / 16) + (j >> 4)) * 64 + lane) * 8 + e;
}

struct DrWalk {
  LaSeqs seqs;               // len: tokens of a piece, a multiple of 64
  LaView q, k, z;            // z: v, backwards go
  const char* sys;
  void* out;                 // forwards: o by the strides below, storage type
  long long o_sb, o_st, o_sh;
  float* e;                  // forwards: (chunk, H), 64 x Dv as operands
  float* keep;               // (chunk, H), Dk x Dv likewise: states before the chunks, adjoints behind them
  float* dv;                 // backwards, dense (token, H, Dv)
  LaState init, last;
  float* piece;              // (slot, H, Dk, Dv): the pieces' own states, then those that they begin with
  uint16_t* transfer;        // (slot, H): their transfers, as operands in three bf16 parts
  int H, Dk, Dv, dtype;
  const int* order;          // of the pieces (DrSystems), NULL: as they are
  int n_pieces;
  int group;                 // waves of a workgroup (dr_walk_group)
  int tiles, own_tiles;      // column tiles of a launch; of them of the state (the rest: transfers)
  float scale;
};

struct DrGrad {
  LaSeqs seqs;
  LaView q, k, go;
  LaDecay g;
  const char* sys;           // only its decays and rates are read
  const float *e, *before, *behind;  // as operands: (chunk, H), 64 x Dv and Dk x Dv
  const float* dv;           // (token, H, Dv)
  void* dv16;                // on bf16 instructions: where it goes as the result (NULL: heads are summed)
  void *dq, *dk;             // (token, H, Dk): the storage type, or floats (q_f32, k_f32)
  int q_f32, k_f32;
  void *dg, *dbeta;          // (token, H); dg NULL: not wanted, or sums per chunk:
  float* g_part;             // (chunk, H)
  int H, Dk, Dv, dtype, g_dtype, b_dtype;
  float scale;
};

// kDrKept: forwards, and what the backward pass reads is kept; kDrState, kDrAdjoint: pieces' own
enum DrKind { kDrForward, kDrKept, kDrState, kDrBackward, kDrAdjoint };

int dr_systems(const DrSystems& a, bool bf16, hipStream_t stream);
int dr_walk_bf16(const DrWalk& a, DrKind kind, int cols, hipStream_t stream);
int dr_walk_bf16_out(const DrWalk& a, bool kept, int cols, hipStream_t stream);
int dr_walk_bf16_back(const DrWalk& a, DrKind kind, int cols, hipStream_t stream);
int dr_walk_f32(const DrWalk& a, DrKind kind, hipStream_t stream);
// The pieces' own states and transfers to the states that the pieces begin with.
int dr_join(const DrWalk& a, bool back, hipStream_t stream);
int dr_grad(const DrGrad& a, bool bf16, hipStream_t stream);

// Waves of a walk's workgroup, `cols` columns each.  items: (piece, head) pairs.  Narrow values have two
// column tiles' waves at most; and where there is a CU for each half of a workgroup, halves (D = 64, 128
// sequences' heads: 99 us forwards, 112 whole; 350 pieces: 155 us, 117 whole; with operands of two parts).
inline int dr_walk_group(int Dk, int Dv, int cols, bool bf16, long long items) {
  if (!bf16) return Dk <= 128 ? 4 : 2;
  if (Dk > 128) return 4;
  if (cols == 32) return Dv <= 64 ? 2 : 4;
  return Dv <= 32 || (Dk <= 64 && items * ((Dv + 31) / 32) <= 256) ? 2 : 4;
}

}  // namespace prnn
