// Decayed linear attention: what the walk kernels and their host code share.
//
// One head holds a state S (Dk x Dv) in fp32 and a log decay g_t per token:
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,      o_t = scale q_t^T S_t.
//
// The kernels walk a sequence in chunks with S in registers.  With G_i the running sum of g
// inside a chunk (the chunk's first token included) and S the state before the chunk,
//
//   o_i = scale [ sum_{j <= i} exp(G_i - G_j) (q_i . k_j) v_j  +  exp(G_i) q_i^T S ]
//   S'  = exp(G_last) S + sum_j exp(G_last - G_j) k_j v_j^T:
//
// four matrix products a chunk.  All three gradients are walks of the same form with the
// arrays in other roles (x: the rows of the output, y and z: what the state is made of):
//
//             x   y   z    state            direction
//   o     =   q   k   v    S                forward
//   dq    =   go  v   k    S^T              forward
//   dk    =   v   go  q    R^T              backward
//   dv    =   k   q   go   R                backward
//
// where R_t = exp(g_{t+1}) R_{t+1} + scale q_t go_t^T is dL/dS_t; backwards the decay between
// a token and the one walked before it is the later one's.  A sequence may be cut into pieces
// that run side by side: a first pass forms every piece's own contribution to the state, a
// small one joins them into the states at the pieces' starts.
#pragma once

#include <algorithm>

#include "prnn_host.h"

namespace prnn {

constexpr int kLaMaxDim = 256;  // widest head (keys or values)

struct LaView {
  const void* p;
  long long sb, st, sh;  // elements between batches, tokens, heads
  int rep = 1;           // consecutive heads that share one of this array
  int vec = 0;           // rows and base admit 16-byte accesses
};

// Chunks' rows are read by unsigned 32-bit offsets from the lowest token's.
constexpr bool la_stride_fits(long long st, int size) { return st >= 0 && st <= (1 << 24) / size; }

// The decays: (B, T, H) by strides, or one per head (sb = st = 0); fp32 or the storage type.
struct LaDecay {
  const void* p;
  long long sb, st, sh;
  int dtype;
};

// How the tokens lie: B sequences of T tokens, or one packed stream with offsets cu.
struct LaSeqs {
  const int* cu;    // NULL: rectangular
  int n_seq;
  int T;            // tokens of a sequence (rectangular) or of the stream
  int len;          // tokens of a piece at most
  int pieces;       // upper bound of the pieces (the grid's)
  int sub;          // tokens between the states that are formed first: divides len
  int span;         // tokens of a walk's piece: len, or where those states are formed more
};

// States at the ends of the walks: rows of H x Dk x Dv floats.
struct LaState {
  float* p;
  const int* table;  // row of sequence s (NULL: s); outside [0, rows): none
  int rows;
};

struct LaRole {
  LaView x, y, z;
  void* out;            // (batch, token, head, vd) by the strides below
  long long o_sb, o_st, o_sh;
  int out_f32;          // out holds floats (heads that are summed afterwards)
  LaView dot;           // dots[token] = (out without the token's own pair) . dot, where given
  float* dots;          // [column tile][head][token of the whole batch]
  int kd, vd;           // columns of x, y and of z, out
  int sk, sv;           // strides of the state's kd and vd axes
  int rev;
  int exact;            // the final state is a result: all of its 24 bits count
  float p_scale, x_scale, u_scale;  // of the pairs, of the state's part, of what enters it
  float* piece_state;   // [la_state_row][head][Dk][Dv]: states before the pieces (NULL: not cut)
  float* piece_decay;   // [piece][head]: a piece's whole log decay in the walk's direction
  LaState init, last;   // given state; where the final one goes (p = NULL: none)
};

struct LaParams {
  LaRole role[3];
  LaDecay g;
  LaSeqs seqs;
  int H, Dk, Dv;
  int tiles;            // column tiles of the widest role (the grid's)
  int roles, near;      // near: consecutive heads that share arrays
  int batch_tokens;     // tokens of the whole batch (dots' rows)
};

// A piece of a sequence: tokens [begin, end) of sequence [s0, s1).
struct LaPiece {
  int seq, begin, end, s0, s1;
  bool first, last, alone;
};

// Sequence s of a packed stream starts at cu[s]; whatever the offsets hold, nothing outside
// the stream is touched.
__device__ __forceinline__ int la_offset(const LaSeqs& q, int s) {
  const int v = q.cu[s];
  return v < 0 ? 0 : v > q.T ? q.T : v;
}

// Piece p.  Rectangular: every sequence has ceil(T / len) of them.  Packed: the stream is cut
// at multiples of len and at sequence heads, so sequence s starts with piece
// s + floor(cu[s] / len); its last piece may be empty.
__device__ __forceinline__ LaPiece la_piece(const LaSeqs& q, int p) {
  LaPiece r;
  if (q.cu == nullptr) {
    const int n = q.T > q.len ? (q.T + q.len - 1) / q.len : 1;
    r.seq = p / n;
    const int i = p - r.seq * n;
    r.s0 = 0;
    r.s1 = q.T;
    r.begin = i * q.len;
    r.end = r.begin + q.len < q.T ? r.begin + q.len : q.T;
    r.first = i == 0;
    r.last = i == n - 1;
  } else {
    int lo = 0, hi = q.n_seq;  // the last s with s + cu[s] / len <= p
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (mid + la_offset(q, mid) / q.len <= p) lo = mid; else hi = mid;
    }
    r.seq = lo;
    r.s0 = la_offset(q, lo);
    r.s1 = la_offset(q, lo + 1);
    if (r.s1 < r.s0) r.s1 = r.s0;
    const int q0 = r.s0 / q.len;
    const int i = p - lo - q0;
    // the piece that holds the last token is the last one; behind it nothing is done
    const int n = r.s1 > r.s0 ? (r.s1 - 1) / q.len - q0 + 1 : 1;
    if (i < 0 || i >= n) {
      r.begin = r.end = r.s1;
      r.first = r.last = false;
      r.alone = true;
      return r;
    }
    const int b = (q0 + i) * q.len, e = b + q.len;
    r.begin = b > r.s0 ? b : r.s0;
    r.end = e < r.s1 ? e : r.s1;
    r.first = i == 0;
    r.last = i == n - 1;
  }
  r.alone = r.first && r.last;
  return r;
}

// Row of the states (one every `sub` tokens, numbered like pieces of that length) before, and
// backwards behind, the part of sequence s that token t lies in.
__device__ __forceinline__ int la_state_row(const LaSeqs& q, int s, int t) {
  return (q.cu ? s : s * ((q.T + q.sub - 1) / q.sub)) + t / q.sub;
}

// Row of sequence s, or NULL where there is none.
__device__ __forceinline__ float* la_row(const LaState& st, int s, size_t row_floats) {
  if (st.p == nullptr) return nullptr;
  const int r = st.table ? st.table[s] : s;
  return r < 0 || r >= st.rows ? nullptr : st.p + static_cast<size_t>(r) * row_floats;
}

// Log decay as it is used: below -104 the factor is zero in fp32 whatever the value (a -inf
// that resets the state included), and sums stay finite; NaN stays NaN.
__device__ __forceinline__ float la_clamp(float g) { return g < -104.0f ? -104.0f : g; }

// A decay as it is stored, and its value: a load's bits are looked at only when they are used,
// or the wave would wait for everything that it loaded before.
__device__ __forceinline__ uint32_t la_decay_bits(const LaDecay& d, int b, int t, int h) {
  const long long at = static_cast<long long>(b) * d.sb + static_cast<long long>(t) * d.st +
                       static_cast<long long>(h) * d.sh;
  return d.dtype == PRNN_F32 ? static_cast<const uint32_t*>(d.p)[at]
                             : static_cast<const uint16_t*>(d.p)[at];
}
__device__ __forceinline__ float la_decay_value(const LaDecay& d, uint32_t bits) {
  return la_clamp(d.dtype == PRNN_F32   ? __uint_as_float(bits)
                  : d.dtype == PRNN_F16 ? Narrow<f16>::val(bits)
                                        : Narrow<bf16>::val(bits));
}
__device__ __forceinline__ float la_decay(const LaDecay& d, int b, int t, int h) {
  return la_decay_value(d, la_decay_bits(d, b, t, h));
}

// Batch of a piece: rectangular sequences are batches of their own.
__device__ __forceinline__ int la_batch(const LaSeqs& q, const LaPiece& pc) {
  return q.cu ? 0 : pc.seq;
}

// A byte offset in a buffer, or one outside it.  Arithmetic and not a choice: the compiler turns
// `in ? offset : kOOB` around a load into two branches with a load each.
__device__ __forceinline__ uint32_t la_in(bool in, uint32_t offset) {
  return offset | (static_cast<uint32_t>(!in) << 31);
}

// A head's rows of an array: a buffer resource at the lowest row of a chunk of C tokens of the
// walk, and byte offsets in it (la_stride_fits).
template <int C>
__device__ __forceinline__ rsrc_t la_rows(const LaView& v, int size, int b, int h, int rev,
                                          int begin, int end, int base) {
  const long long t = rev ? static_cast<long long>(end) - base - C : static_cast<long long>(begin) + base;
  return make_rsrc(static_cast<const char*>(v.p) + (b * v.sb + (h / v.rep) * v.sh + t * v.st) * size,
                   0x7fffffffu);
}

// The decays of C tokens of the walk from local index base, lane i's in place: forwards g of the
// token that a step reaches, backwards the next token's (none, and zero bits are a zero of every
// type, behind the sequence's last token and outside the piece).  Nothing here is a branch, and
// either width is loaded, one of them from an empty buffer: behind a branch the wave would wait
// for the load as soon as the ways meet, and with it for all loads before.
struct LaBits {
  uint32_t wide, narrow;
  __device__ __forceinline__ uint32_t get() const { return wide | narrow; }
};
template <int C>
__device__ __forceinline__ LaBits la_step_decays(const LaDecay& d, int rev, const LaPiece& pc,
                                                   int b, int h, int base, int lane) {
  const int size = d.dtype == PRNN_F32 ? 4 : 2;
  const int left = pc.end - pc.begin - base;
  // lowest token of the C (backwards: behind the lowest that is walked)
  const int low = rev ? pc.end - base - C + 1 : pc.begin + base;
  const int row = rev ? C - 1 - lane : lane;
  const bool in = (lane < left) & (lane < C) & (low + row < pc.s1);
  const char* p = static_cast<const char*>(d.p) +
                  (b * d.sb + static_cast<long long>(low) * d.st + h * d.sh) * size;
  const uint32_t o = la_in(in, static_cast<uint32_t>(row * static_cast<int>(d.st)) * size);
  LaBits bits;
  bits.wide = __builtin_amdgcn_raw_buffer_load_b32(make_rsrc(p, size == 4 ? 0x7fffffffu : 0u), o, 0, 0);
  bits.narrow = __builtin_amdgcn_raw_buffer_load_b16(make_rsrc(p, size == 4 ? 0u : 0x7fffffffu), o, 0, 0);
  return bits;
}

// First piece of sequence s and their number.
__device__ __forceinline__ void la_pieces_of(const LaSeqs& q, int s, int& p0, int& n) {
  if (q.cu == nullptr) {
    n = q.T > q.len ? (q.T + q.len - 1) / q.len : 1;
    p0 = s * n;
  } else {
    const int s0 = la_offset(q, s), s1 = la_offset(q, s + 1);
    p0 = s + s0 / q.len;
    n = s1 > s0 ? (s1 - 1) / q.len - s0 / q.len + 1 : 1;
  }
}

// Where a workgroup of the walks works.  Workgroups go to the 8 XCDs in turn, each with an L2 of
// its own, so those that read the same rows (the roles and column tiles of a piece, and the heads
// that share arrays) are 8 apart and next to each other on one XCD.
struct LaPlace {
  int role, tile, piece, h;
  bool any;
};
__device__ __forceinline__ LaPlace la_place(const LaParams& p) {
  const int same = p.roles * p.tiles * p.near;
  const int group = blockIdx.x / (8 * same), in = blockIdx.x - group * 8 * same;
  int sub = in >> 3;
  const int item = group * 8 + (in & 7);  // piece and the first of `near` heads
  const int heads = p.H / p.near;
  LaPlace r;
  r.piece = item / heads;
  r.h = (item - r.piece * heads) * p.near;
  const int k = sub / p.near;
  r.h += sub - k * p.near;
  r.role = k / p.tiles;
  r.tile = k - r.role * p.tiles;
  r.any = r.piece < p.seqs.pieces;
  return r;
}
inline long long la_grid(const LaParams& p) {
  const long long items = 1ll * p.seqs.pieces * (p.H / p.near);
  return (items + 7) / 8 * 8 * p.roles * p.tiles * p.near;
}

inline int la_widest(const LaParams& p, int roles) {
  int vd = 0;
  for (int i = 0; i < roles; ++i) vd = std::max(vd, p.role[i].vd);
  return vd;
}

// The walks of `roles` roles of `p`, or (state_only) their pieces' own contributions to the
// states.  *_tile_cols: columns of z that a workgroup takes where the widest role has vd.
int la_walk_f32(LaParams p, int roles, bool state_only, int dtype, hipStream_t stream);
int la_f32_tile_cols(int vd);
// bf16 storage with widths in multiples of 8, rows that admit 16-byte accesses (x, y, z, dot, out),
// and tokens at least a row apart.  dots: some role has dots.
int la_walk_bf16(LaParams p, int roles, bool state_only, bool dots, hipStream_t stream);
int la_bf16_tile_cols(int vd);

// What the entry points check of a problem, and an array of it as the kernels read it (D: its width).
int la_check(const prnn_linear_attention_problem* a);
LaView la_view(const prnn_la_view& v, const prnn_linear_attention_problem& a, int D);

// Gradients of shared heads: dst (token, H / rep, D) of the storage type, the sums of src (token, H,
// D) over heads that share an array, in their order.  src NULL: nothing to do.
struct LaHeadSums {
  const float* src[3];
  void* dst[3];
  int rep[3], D[3];
  int H;
  size_t tokens;
};
int la_head_sums(const LaHeadSums& a, int dtype, hipStream_t stream);
// dg (H) = the sums of per_part (parts, H), in a fixed order.
int la_decay_sums(const float* per_part, void* dg, int g_dtype, int parts, int H, hipStream_t stream);

}  // namespace prnn
