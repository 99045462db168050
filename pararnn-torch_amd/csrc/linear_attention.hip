// Decayed linear attention: the small kernels around the walks and the C entry points.
//
// * la_join_kernel: states before a cut sequence's pieces from the pieces' own contributions;
// * la_decay_grad_kernel: the log decays' gradient.  dL/dg_t = exp(g_t)
//   <S_{t-1}, R_t> is the flow from all earlier tokens to t and later ones; from one token to the
//   next it gains what token t hands on and loses what it receives, so it is a running sum of
//   k_t . dk_t - q_t . dq_t (both formed in fp32 by the walks).  What a token hands to itself,
//   scale (q_t . k_t)(v_t . go_t), is in both and in neither here: behind a strong decay the flow is a
//   small part of it (exp(-12) of it and less, which fp32 differences of the whole would lose).  The
//   flow itself stays bounded while the sum's roundings add up, so the sum is tied at both ends of a
//   sequence (<S_0, dL/dS_0> and <S_T, dL/dS_T>, zero without states) and of every piece, whose
//   states are there; what it misses the end by is taken back along the way, by the squares of its
//   terms;
// * la_head_sum_kernel: gradients of shared heads, summed in a fixed order.
#include "linear_attention.h"

namespace prnn {
namespace {

// ---- states before the pieces ------------------------------------------------------------

struct JoinArgs {
  LaSeqs seqs;
  float* state[2];
  const float* decay[2];
  LaState init[2];
  int rev[2];
  int H, DD;
};

// V floats of the state a thread; the contributions of kAhead pieces are under way before the
// first is added (from empty buffers behind the last: a branch would be waited at).  Bound by
// memory where there are many states (52 pieces of 8 heads of (128, 128): 12.7 us, 4.3 TB/s), by
// the chain of pieces, 0.12 us each, where there are few.
template <int V>
__global__ __launch_bounds__(256) void la_join_kernel(JoinArgs A, int seq_blocks) {
  typedef uint32_t vec __attribute__((ext_vector_type(V)));
  constexpr int kAhead = 8;
  const int role = blockIdx.z, h = blockIdx.y;
  const int seq = blockIdx.x / seq_blocks;
  const int e = ((blockIdx.x - seq * seq_blocks) * 256 + threadIdx.x) * V;
  int p0, n;
  la_pieces_of(A.seqs, seq, p0, n);
  if (n < 2 || e >= A.DD) return;
  // parts in the walk's order up to the one that its last piece starts with
  const int s0 = A.seqs.cu ? la_offset(A.seqs, seq) : 0;
  const int s1 = A.seqs.cu ? la_offset(A.seqs, seq + 1) : A.seqs.T;
  const int per = A.seqs.span / A.seqs.sub, behind = n, c0 = s0 / A.seqs.sub;
  n = A.rev[role] ? n - ((s0 / A.seqs.span + 1) * per - 1 - c0)
                  : (s1 - 1) / A.seqs.span * per - c0 + 1;
  if (n < 2) return;  // the walk has one piece
  const size_t row = static_cast<size_t>(A.H) * A.DD;
  const size_t at = static_cast<size_t>(h) * A.DD;
  const float* init = la_row(A.init[role], seq, row);
  const int dir = A.rev[role] ? -1 : 1, from = A.rev[role] ? p0 + behind - 1 : p0;
  float S[V];
#pragma unroll
  for (int v = 0; v < V; ++v) S[v] = init ? init[at + e + v] : 0.0f;
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    vec U[kAhead];
    float d[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const bool more = i0 + i + 1 < n;  // the last piece hands on to none
      const size_t p = from + dir * min(i0 + i, n - 1);
      const rsrc_t r = make_rsrc(A.state[role] + p * row + at, more ? A.DD * 4u : 0u);
      if constexpr (V == 4)
        U[i] = __builtin_amdgcn_raw_buffer_load_b128(r, e * 4, 0, 0);
      else
        U[i] = __builtin_amdgcn_raw_buffer_load_b32(r, e * 4, 0, 0);
      d[i] = A.decay[role][p * A.H + h];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i >= n) break;
      const size_t p = from + dir * (i0 + i);
      float* w = A.state[role] + p * row + at + e;
      const float f = fexp(d[i]);
      vec s;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        s[v] = __float_as_uint(S[v]);
        S[v] = fmaf(f, S[v], __uint_as_float(U[i][v]));
      }
      *reinterpret_cast<vec*>(w) = s;
    }
  }
}

// ---- gradient of the log decays --------------------------------------------------------

struct DecayGradArgs {
  LaSeqs seqs;          // the parts that are tied at their ends: pieces, or whole sequences
  LaDecay g;
  const float* q_dots;  // [tile][head][token]
  const float* k_dots;
  int tiles, H, DD, batch_tokens;
  LaState h0;
  const float *dh0, *last, *gs;          // rows of sequences: dL/dS_0, S_T, dL/dS_T
  const float *state, *adjoint;          // the walks' states, either direction
  int g_dtype;
  void* dg;             // (token, H) of g's type, or NULL
  float* per_part;      // (piece, H) sums for decays per head, or NULL
};

// Sum over a workgroup of 256, in every thread.
__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) v += __shfl_xor(v, k);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}
__device__ __forceinline__ double block_dot(const float* a, const float* b, int n, double* lds) {
  constexpr int kAhead = 8;  // loads under way, from empty places behind the end
  const rsrc_t ra = make_rsrc(a, n * 4u), rb = make_rsrc(b, n * 4u);
  double d = 0.0;
  for (int e = threadIdx.x; e < n; e += 256 * kAhead) {
    float x[kAhead], y[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      x[i] = ldb<float>(ra, (e + 256 * i) * 4u, 0);
      y[i] = ldb<float>(rb, (e + 256 * i) * 4u, 0);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) d += static_cast<double>(x[i]) * y[i];
  }
  return block_sum(d, lds);
}

// The flow at the first token of a part: its state with the adjoint of that token, which is the one
// behind the part before.
__device__ __forceinline__ double flow_at(const DecayGradArgs& A, const LaPiece& pc, int begin,
                                          int h, double* lds) {
  const size_t row = static_cast<size_t>(A.H) * A.DD, head = static_cast<size_t>(h) * A.DD;
  return block_dot(A.state + la_state_row(A.seqs, pc.seq, begin) * row + head,
                   A.adjoint + la_state_row(A.seqs, pc.seq, begin - 1) * row + head, A.DD, lds) *
         fexp(la_decay(A.g, la_batch(A.seqs, pc), begin, h));
}

// A workgroup per part and head.  The dots are read twice (their sum first, to tie the end), the
// second time from the L2; 8 x 2048 tokens of 16 heads take 9.1 us, a chain of reductions in fp64
// behind two products of states a part, 1001 tokens x 3 of 6 heads of (48, 72) 9.3.
__global__ __launch_bounds__(256) void la_decay_grad_kernel(DecayGradArgs A) {
  __shared__ double s_wave[4], s_weight[4];
  constexpr int kEach = 4;
  const int h = blockIdx.y, p = blockIdx.x, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  const LaPiece pc = la_piece(A.seqs, p);
  const size_t ph = static_cast<size_t>(p) * A.H + h;
  const int n = pc.end - pc.begin;
  if (n <= 0) {
    if (A.per_part && tid == 0) A.per_part[ph] = 0.0f;
    return;
  }
  const size_t t0 = A.seqs.cu ? pc.begin : static_cast<size_t>(pc.seq) * A.seqs.T + pc.begin;
  // what the flow gains behind tokens base + t, base + t + stride, .., and the weight of its error:
  // all loads before the first sum, zeros behind the part's end
  auto steps = [&](double* x, double* w, int base, int t, int stride) {
    const uint32_t bytes = min(n - base, 256 * kEach) * 4u;
    double in[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) x[i] = in[i] = 0.0;
    for (int k = 0; k < A.tiles; ++k) {
      const size_t at = (static_cast<size_t>(k) * A.H + h) * A.batch_tokens + t0 + base;
      const rsrc_t rk = make_rsrc(A.k_dots + at, bytes), rq = make_rsrc(A.q_dots + at, bytes);
      float u[kEach], v[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        u[i] = ldb<float>(rk, (t + i * stride) * 4u, 0);
        v[i] = ldb<float>(rq, (t + i * stride) * 4u, 0);
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        x[i] += u[i];
        in[i] += v[i];
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      w[i] = x[i] * x[i] + in[i] * in[i];
      x[i] -= in[i];
    }
  };
  const size_t row = static_cast<size_t>(A.H) * A.DD;
  const size_t head = pc.seq * row + static_cast<size_t>(h) * A.DD;
  double begin = 0.0, end = 0.0;
  if (!pc.first)
    begin = flow_at(A, pc, pc.begin, h, s_wave);
  else if (const float* s0 = la_row(A.h0, pc.seq, row))
    begin = block_dot(s0 + static_cast<size_t>(h) * A.DD, A.dh0 + head, A.DD, s_wave);
  if (!pc.last)
    end = flow_at(A, pc, pc.end, h, s_wave);
  else if (A.gs)
    end = block_dot(A.last + head, A.gs + head, A.DD, s_wave);
  double all = 0.0, weight = 0.0;
  for (int base = 0; base < n; base += 256 * kEach) {
    double x[kEach], w[kEach];
    steps(x, w, base, tid, 256);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      all += x[i];
      weight += w[i];
    }
  }
  all = block_sum(all, s_wave);
  weight = block_sum(weight, s_weight) + begin * begin + end * end;
  // What is missed at the end, a unit of weight: every term of the sum is off by a like part of itself,
  // so the squares say how much of it came from where.  (The last token alone may hand more to the
  // final state than ever flows through a strong decay: what that is off by is not the others'.)
  const double miss = weight > 0.0 ? (begin + all - end) / weight : weight;
  double flow = begin, known = begin * begin, total = 0.0;
  for (int base = 0; base < n; base += 256 * kEach) {
    double x[kEach], w[kEach], d[kEach], c[kEach], sum = 0.0, squares = 0.0;
    uint32_t g[kEach];  // decays, loaded ahead too (the last token's behind the end)
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      g[i] = la_decay_bits(A.g, la_batch(A.seqs, pc), min(pc.begin + base + tid * kEach + i, pc.end - 1), h);
    steps(x, w, base, tid * kEach, 1);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      d[i] = sum;  // what came before within the thread's tokens
      c[i] = squares;
      sum += x[i];
      squares += w[i];
    }
    double run = sum, run_c = squares;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const double o = __shfl_up(run, k), p = __shfl_up(run_c, k);
      if (lane >= k) {
        run += o;
        run_c += p;
      }
    }
    __syncthreads();
    if (lane == 63) {
      s_wave[wave] = run;
      s_weight[wave] = run_c;
    }
    __syncthreads();
    double before = flow + run - sum, before_c = known + run_c - squares;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < wave) {
        before += s_wave[i];
        before_c += s_weight[i];
      }
      flow += s_wave[i];
      known += s_weight[i];
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int t = base + tid * kEach + i;
      if (t >= n) continue;
      // nothing comes through a factor that is zero
      const float v = la_decay_value(A.g, g[i]) <= -104.0f ? 0.0f
                          : static_cast<float>(before + d[i] - miss * (before_c + c[i]));
      total += v;
      if (A.dg) {
        const size_t at = (t0 + t) * A.H + h;
        if (A.g_dtype == PRNN_F32)
          static_cast<float*>(A.dg)[at] = v;
        else if (A.g_dtype == PRNN_F16)
          static_cast<f16*>(A.dg)[at] = from_f32<f16>(v);
        else
          static_cast<bf16*>(A.dg)[at] = from_f32<bf16>(v);
      }
    }
  }
  if (A.per_part) {
    total = block_sum(total, s_wave);
    if (tid == 0) A.per_part[ph] = static_cast<float>(total);
  }
}

// One wave per head: the parts' sums in a fixed order.
__global__ __launch_bounds__(64) void la_decay_sum_kernel(const float* __restrict__ per_part,
                                                          void* dg, int g_dtype, int parts, int H) {
  const int h = blockIdx.x;
  double d = 0.0;
  for (int s = threadIdx.x; s < parts; s += 64) d += per_part[static_cast<size_t>(s) * H + h];
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) d += __shfl_xor(d, k);
  if (threadIdx.x) return;
  const float v = static_cast<float>(d);
  if (g_dtype == PRNN_F32)
    static_cast<float*>(dg)[h] = v;
  else if (g_dtype == PRNN_F16)
    static_cast<f16*>(dg)[h] = from_f32<f16>(v);
  else
    static_cast<bf16*>(dg)[h] = from_f32<bf16>(v);
}

// ---- gradients of shared heads ---------------------------------------------------------

struct HeadSumArgs {
  const float* src[3];  // (token, H, D)
  void* dst[3];         // (token, H / rep, D)
  int rep[3], D[3];
  int H;
  size_t tokens;
};

// Bound by memory: 3003 tokens, 6 heads to 3 in fp32, (48, 72): 6.6 us.
template <typename T>
__global__ __launch_bounds__(256) void la_head_sum_kernel(HeadSumArgs A) {
  const int k = blockIdx.y;
  if (A.src[k] == nullptr) return;
  const int D = A.D[k], rep = A.rep[k], heads = A.H / rep;
  const size_t n = A.tokens * heads * D, stride = static_cast<size_t>(gridDim.x) * 256;
  for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += stride) {
    const size_t d = i % D, th = i / D, hh = th % heads, t = th / heads;
    const float* s = A.src[k] + (t * A.H + hh * rep) * D + d;
    float v = 0.0f;
    for (int r = 0; r < rep; ++r) v += s[static_cast<size_t>(r) * D];
    static_cast<T*>(A.dst[k])[i] = from_f32<T>(v);
  }
}

// ---- host ------------------------------------------------------------------------------

using Problem = prnn_linear_attention_problem;

// D: the array's width.  A lone token's stride is what suits the walks.
LaView view(const prnn_la_view& v, const Problem& a, int D) {
  const int H = a.H, dtype = a.dtype;
  LaView r{v.p, v.sb, a.T > 1 ? v.st : D, v.sh, 1, 0};
  if (v.heads > 0) r.rep = H / v.heads;
  const long long size = dtype == PRNN_F32 ? 4 : 2;
  const long long bytes = static_cast<long long>(reinterpret_cast<uintptr_t>(v.p)) |
                          r.sb * size | r.st * size | r.sh * size;
  r.vec = (bytes & 15) == 0 && r.st >= D;
  return r;
}

// The stride of an only token is never used.
int check_tokens(const Problem& a, long long st) {
  if (a.T > 1 && !la_stride_fits(st, a.dtype == PRNN_F32 ? 4 : 2))
    return fail(PRNN_ERR_VALUE, "tokens %lld elements apart do not lie 0 bytes to 16 MiB apart", st);
  return PRNN_OK;
}

int check(const Problem* a) {
  if (a == nullptr) return fail(PRNN_ERR_VALUE, "the problem must be non-null");
  if (int rc = check_dtype(a->dtype)) return rc;
  if (a->g_dtype != PRNN_F32 && a->g_dtype != a->dtype)
    return fail(PRNN_ERR_TYPE, "log_decay must be float32 or of the storage type");
  if (a->H < 1 || a->H > 65535) return fail(PRNN_ERR_VALUE, "H=%d is not in 1 .. 65535", a->H);
  if (a->Dk < 1 || a->Dk > kLaMaxDim || a->Dv < 1 || a->Dv > kLaMaxDim)
    return fail(PRNN_ERR_VALUE, "head widths (%d, %d) are not in 1 .. %d", a->Dk, a->Dv, kLaMaxDim);
  if (a->B < 0 || a->T < 0 || (a->cu_seqlens ? a->n_seq < 1 || a->B != 1 : a->n_seq != 0))
    return fail(PRNN_ERR_VALUE, "B=%d, T=%d, n_seq=%d do not describe a batch", a->B, a->T,
                a->n_seq);
  if (static_cast<long long>(a->B) * a->T > (1ll << 30))
    return fail(PRNN_ERR_VALUE, "%lld tokens are more than 2^30", 1ll * a->B * a->T);
  for (const prnn_la_view* v : {&a->q, &a->k, &a->v})
    if (v->heads < 1 || a->H % v->heads)
      return fail(PRNN_ERR_VALUE, "%d heads do not divide H=%d", v->heads, a->H);
  if (static_cast<long long>(a->B) * a->T > 0)
    for (const void* p : {a->q.p, a->k.p, a->v.p, a->g})
      if (p == nullptr) return fail(PRNN_ERR_VALUE, "q, k, v and log_decay must be non-null");
  for (const prnn_la_view* v : {&a->q, &a->k, &a->v})
    if (int rc = check_tokens(*a, v->st)) return rc;
  if (a->T > 1 && !la_stride_fits(a->g_st, 4))
    return fail(PRNN_ERR_VALUE, "decays %lld elements apart do not lie 0 bytes to 16 MiB apart", a->g_st);
  if (!la_stride_fits(1ll * a->H * std::max(a->Dk, a->Dv), 4))
    return fail(PRNN_ERR_VALUE, "H=%d heads of (%d, %d) are too wide", a->H, a->Dk, a->Dv);
  if (a->h0 && a->h0_rows < 0) return fail(PRNN_ERR_VALUE, "h0_rows=%d", a->h0_rows);
  return PRNN_OK;
}

int sequences(const Problem& a) { return a.cu_seqlens ? a.n_seq : a.B; }

bool is_cut(const LaSeqs& s) { return s.len <= s.T; }

LaDecay decay_of(const Problem& a) { return LaDecay{a.g, a.g_sb, a.g_st, a.g_sh, a.g_dtype}; }

// Scratch of either direction.  `roles`: states that are kept per piece (forward 1,
// backward 2).
struct Scratch {
  float* state[2];
  float* decay[2];
  float* dots[2];
  float* heads[3];
  float *last, *per_part;
  size_t bytes;
};

// Whether the walks run on the bf16 matrix instructions: bf16 storage whose widths and rows admit
// 16-byte accesses.  What is odd takes the fp32 walk: 8 x 2048 tokens of 16 heads of (64, 64) 63 us
// on bf16 instructions and 138 in fp32, a training step 235 and 464, 4 x 2048 of (128, 128) 80 and
// 207, 8 x 2048 of (32, 32) 49 and 77.
bool on_bf16(const Problem& a, const prnn_la_view* other) {
  if (a.dtype != PRNN_BF16 || a.Dk % 8 || a.Dv % 8) return false;
  return view(a.q, a, a.Dk).vec && view(a.k, a, a.Dk).vec && view(a.v, a, a.Dv).vec &&
         view(*other, a, a.Dv).vec;
}

// The walks of a call and the columns of z that one of their workgroups takes.
struct Walks {
  bool bf16;
  int dtype;
  int cols(int vd) const { return bf16 ? la_bf16_tile_cols(vd) : la_f32_tile_cols(vd); }
  int tiles(int vd) const { return (vd + cols(vd) - 1) / cols(vd); }
  int run(const LaParams& p, int roles, bool state_only, bool dots, hipStream_t st) const {
    return bf16 ? la_walk_bf16(p, roles, state_only, dots, st)
                : la_walk_f32(p, roles, state_only, dtype, st);
  }
};

// How long the pieces are, a multiple of 64 tokens.  Time in microseconds, measured on single
// sequences of 2048 and 8192 tokens in pieces of 64 .. 1024:
// * a piece's tokens come one after another, twice (its own contribution, then the walk): 0.085 a
//   token on bf16 instructions, 0.17 in fp32; two thirds of that for a sequence that is not cut;
// * the join takes a sequence's pieces one after another: 0.12 a piece;
// * a state per piece and direction is written, read, written and read: 16 bytes an element at
//   5.3 MB per us;
// * two launches more than without a cut: 8.
// So pieces are as long as makes the first equal to what falls with their length, unless the
// chip has workgroups enough with longer ones: about 8 waves a CU on bf16 instructions, 16 in
// fp32, run at a time.  Lengths of 64, 256 and 1024 and this rule's, us, heads of (64, 64) in bf16:
// 2 x 512 tokens of 4 heads 20, 35, 34 and 20; 2048 of 4 heads 24, 36, 99 and 24, their training
// step 63, 87, 233 and 63; 16384 of 8 heads 88, 58, 104 and 56, their training step 263, 171, 265
// and 161; 8 x 2048 of 16 heads 94, 63, 106 and 63; 32 x 300 of 4 heads 31, 39, 25 and 25 (whole).
//
// Pieces that are longer for that get their states from the contributions of shorter parts, of the
// length above: a training step of 8 x 2048 tokens of 16 heads 234 us, with parts as long as the
// pieces 249.  A piece that a walk ends with has no contribution formed.
LaSeqs pieces(const Problem& a, long long len, long long sub, long long span) {
  LaSeqs s{a.cu_seqlens, sequences(a), a.T, a.T + 1, sequences(a), a.T + 1, a.T + 1};
  if (len < a.T) {
    s.len = static_cast<int>(len);
    s.sub = static_cast<int>(sub);
    s.span = static_cast<int>(span);
    s.pieces = a.cu_seqlens ? s.n_seq + a.T / s.len : a.B * ((a.T + s.len - 1) / s.len);
  }
  return s;
}

LaSeqs cut(const Problem& a, const Walks& w, int widest, int roles, int states) {
  const double serial = w.bf16 ? 0.085 : 0.17, per_piece = 0.12, bytes_us = 5.3e6, launches = 8.0;
  const double tokens = 1.0 * a.B * a.T;
  // packed sequences of unknown lengths: one may be all there is (100 of 60 tokens, 8 heads of (64,
  // 64): 12 us where that is known, 43 where not)
  const double longest = a.cu_seqlens && a.longest > 0 ? std::min(a.longest, a.T) : a.T;
  const double falls = per_piece * longest + 16.0 * states * a.Dk * a.Dv * a.H * tokens / bytes_us;
  const long long best = std::max(1ll, std::llround(std::sqrt(falls / serial) / 64)) * 64;
  long long len = best;
  if (serial * longest * 2 / 3 <= serial * len + falls / len + launches) len = 1ll + a.T;
  const long long waves = w.cols(widest) / (w.bf16 ? 32 : 16);
  const long long most = (w.bf16 ? 2048 : 4096) / waves;  // workgroups that run at a time
  const long long fill = (1ll * a.B * a.T * a.H * roles * w.tiles(widest) + most - 1) / most;
  if (len < fill) {
    // a batch's sequences in equal pieces, no more than run at a time
    const long long n = a.cu_seqlens ? 1 : std::max(1ll, a.T / fill);
    len = std::max(fill, a.cu_seqlens ? 0ll : (a.T + n - 1) / n);
    len = (len + 63) / 64 * 64;
  }
  if (len >= longest) return pieces(a, 1ll + a.T, 0, 0);  // every sequence whole
  long long n = std::max(1ll, len / best);
  while (len % (64 * n)) --n;
  return pieces(a, len, len / n, len);
}

// The parts whose contributions to the states are formed.
LaSeqs parts_of(const Problem& a, const LaSeqs& s) {
  return is_cut(s) ? pieces(a, s.sub, s.sub, s.span) : s;
}

LaSeqs forward_cut(const Problem& a, const Walks& w) { return cut(a, w, a.Dv, 1, 1); }
LaSeqs backward_cut(const Problem& a, const Walks& w) {
  return cut(a, w, std::max(a.Dk, a.Dv), 3, 2);
}

Scratch carve(void* ws, const Problem& a, const Walks& w, bool backward, bool decay_grad) {
  Carver c(ws);
  Scratch s{};
  const LaSeqs q = backward ? backward_cut(a, w) : forward_cut(a, w);
  const size_t dd = static_cast<size_t>(a.Dk) * a.Dv;
  const size_t tokens = static_cast<size_t>(a.B) * a.T;
  for (int i = 0; i < (backward ? 2 : 1); ++i)
    if (is_cut(q)) {
      const size_t rows = parts_of(a, q).pieces;
      s.state[i] = static_cast<float*>(c.take(4 * dd * a.H * rows));
      s.decay[i] = static_cast<float*>(c.take(4 * a.H * rows));
    }
  if (backward) {
    if (decay_grad) {
      const size_t tiles = w.tiles(std::max(a.Dk, a.Dv));
      for (float*& d : s.dots) d = static_cast<float*>(c.take(4 * tiles * a.H * tokens));
      const size_t seqs = sequences(a);
      s.last = static_cast<float*>(c.take(4 * dd * a.H * seqs));
      s.per_part = static_cast<float*>(c.take(4 * static_cast<size_t>(a.H) * q.pieces));
    }
    const int heads[3] = {a.q.heads, a.k.heads, a.v.heads}, D[3] = {a.Dk, a.Dk, a.Dv};
    for (int i = 0; i < 3; ++i)
      if (heads[i] != a.H)
        s.heads[i] = static_cast<float*>(c.take(4 * tokens * a.H * D[i]));
  }
  s.bytes = c.used;
  return s;
}

// Enough for either walk: which one runs also depends on the other arrays' rows.
size_t need(const Problem& a, bool backward, bool decay_grad) {
  return std::max(carve(nullptr, a, Walks{true, a.dtype}, backward, decay_grad).bytes,
                  carve(nullptr, a, Walks{false, a.dtype}, backward, decay_grad).bytes);
}

int check_ws(size_t need, const void* ws, size_t bytes) {
  if (need && (ws == nullptr || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255)))
    return fail(PRNN_ERR_VALUE, "the workspace must hold %zu bytes, 256-byte aligned (got %zu)",
                need, bytes);
  return PRNN_OK;
}

int join(const LaParams& p, const Scratch& s, const LaState* init, const int* rev, int roles,
         hipStream_t st) {
  JoinArgs j{};
  j.seqs = p.seqs;
  j.H = p.H;
  j.DD = p.Dk * p.Dv;
  for (int i = 0; i < roles; ++i) {
    j.state[i] = s.state[i];
    j.decay[i] = s.decay[i];
    j.init[i] = init[i];
    j.rev[i] = rev[i];
  }
  const bool vec = j.DD % 4 == 0;
  const int blocks = (j.DD / (vec ? 4 : 1) + 255) / 256;
  if (int rc = check_grid("linear_attention", 1ll * p.seqs.n_seq * blocks, 256)) return rc;
  const dim3 grid(static_cast<unsigned>(p.seqs.n_seq) * blocks, p.H, roles);
  if (vec)
    la_join_kernel<4><<<grid, 256, 0, st>>>(j, blocks);
  else
    la_join_kernel<1><<<grid, 256, 0, st>>>(j, blocks);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

LaParams params(const Problem& a, const LaSeqs& q) {
  LaParams p{};
  p.g = decay_of(a);
  p.seqs = q;
  p.H = a.H;
  p.Dk = a.Dk;
  p.Dv = a.Dv;
  p.batch_tokens = a.B * a.T;
  // heads that share q, k or v: up to 8 of them side by side
  const int shared = a.H / std::min({a.q.heads, a.k.heads, a.v.heads});
  p.near = 1;
  for (int n = 2; n <= 8; ++n)
    if (shared % n == 0) p.near = n;
  return p;
}

LaState initial(const Problem& a) {
  return LaState{const_cast<float*>(a.h0), a.h0_table, a.h0_rows};
}

int forward(const Problem& a, const prnn_la_view& out, float* state_out, const int* out_table,
            int out_rows, void* ws, hipStream_t st) {
  const Walks w{on_bf16(a, &out), a.dtype};
  const Scratch s = carve(ws, a, w, false, false);
  LaParams p = params(a, forward_cut(a, w));
  LaRole& r = p.role[0];
  r.x = view(a.q, a, a.Dk);
  r.y = view(a.k, a, a.Dk);
  r.z = view(a.v, a, a.Dv);
  r.out = const_cast<void*>(out.p);
  r.o_sb = out.sb;
  r.o_st = a.T > 1 ? out.st : a.Dv;
  r.o_sh = out.sh;
  r.exact = 1;  // asked for or not: the output has the same bits
  r.kd = a.Dk;
  r.vd = a.Dv;
  r.sk = a.Dv;
  r.sv = 1;
  r.p_scale = r.x_scale = a.scale;
  r.u_scale = 1.0f;
  r.piece_state = s.state[0];
  r.piece_decay = s.decay[0];
  r.init = initial(a);
  r.last = LaState{state_out, out_table, out_rows};
  if (is_cut(p.seqs)) {
    const LaSeqs walked = p.seqs;
    p.seqs = parts_of(a, walked);
    if (int rc = w.run(p, 1, true, false, st)) return rc;
    const int rev = 0;
    if (int rc = join(p, s, &r.init, &rev, 1, st)) return rc;
    p.seqs = walked;
  }
  return w.run(p, 1, false, false, st);
}

int backward(const Problem& a, const prnn_la_view& go, const float* gs, void* dq, void* dk,
             void* dv, void* dg, float* dh0, void* ws, hipStream_t st) {
  // the bf16 walk writes 16 bytes at a time: dense rows of widths in eights, from such a boundary
  const uintptr_t bases = reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) |
                          reinterpret_cast<uintptr_t>(dv);
  const Walks w{on_bf16(a, &go) && (bases & 15) == 0, a.dtype};
  const Scratch s = carve(ws, a, w, true, dg != nullptr);
  LaParams p = params(a, backward_cut(a, w));
  const LaView q = view(a.q, a, a.Dk), k = view(a.k, a, a.Dk), v = view(a.v, a, a.Dv),
               o = view(go, a, a.Dv);
  const LaState init = initial(a), fin{const_cast<float*>(gs), nullptr, sequences(a)};
  const LaView none{nullptr, 0, 0, 0, 1, 1};
  auto role = [&](LaView x, LaView y, LaView z, int kd, int vd, bool transposed, int rev) {
    LaRole r{};
    r.x = x;
    r.y = y;
    r.z = z;
    r.kd = kd;
    r.vd = vd;
    r.sk = transposed ? 1 : a.Dv;
    r.sv = transposed ? a.Dv : 1;
    r.rev = rev;
    r.exact = rev && dh0 != nullptr;
    r.p_scale = a.scale;
    r.x_scale = rev ? 1.0f : a.scale;
    r.u_scale = rev ? a.scale : 1.0f;
    r.piece_state = s.state[rev];
    r.piece_decay = s.decay[rev];
    r.init = rev ? fin : init;
    r.dot = none;
    return r;
  };
  if (is_cut(p.seqs)) {
    const LaSeqs walked = p.seqs;
    p.seqs = parts_of(a, walked);
    p.role[0] = role(none, k, v, a.Dk, a.Dv, false, 0);
    p.role[1] = role(none, q, o, a.Dk, a.Dv, false, 1);
    if (int rc = w.run(p, 2, true, false, st)) return rc;
    const LaState inits[2] = {init, fin};
    const int rev[2] = {0, 1};
    if (int rc = join(p, s, inits, rev, 2, st)) return rc;
    p.seqs = walked;
  }
  p.role[0] = role(o, v, k, a.Dv, a.Dk, true, 0);
  p.role[1] = role(v, o, q, a.Dv, a.Dk, true, 1);
  p.role[2] = role(k, q, o, a.Dk, a.Dv, false, 1);
  void* outs[3] = {dq, dk, dv};
  const int D[3] = {a.Dk, a.Dk, a.Dv}, heads[3] = {a.q.heads, a.k.heads, a.v.heads};
  HeadSumArgs hs{};
  bool sums = false;
  for (int i = 0; i < 3; ++i) {
    LaRole& r = p.role[i];
    r.out_f32 = s.heads[i] != nullptr;
    r.out = r.out_f32 ? s.heads[i] : outs[i];
    r.o_sh = D[i];
    r.o_st = static_cast<long long>(a.H) * D[i];
    r.o_sb = r.o_st * a.T;
    hs.src[i] = s.heads[i];
    hs.dst[i] = outs[i];
    hs.rep[i] = a.H / heads[i];
    hs.D[i] = D[i];
    sums = sums || s.heads[i];
  }
  p.role[2].last = LaState{dh0, nullptr, sequences(a)};
  if (dg) {
    // the final state, for the flow into it
    if (gs) p.role[0].last = LaState{s.last, nullptr, sequences(a)};
    p.role[0].dot = q;
    p.role[0].dots = s.dots[0];
    p.role[1].dot = k;
    p.role[1].dots = s.dots[1];
  }
  if (int rc = w.run(p, 3, false, dg != nullptr, st)) return rc;
  const size_t tokens = static_cast<size_t>(a.B) * a.T;
  if (sums && tokens) {
    hs.H = a.H;
    hs.tokens = tokens;
    const size_t most = tokens * a.H * std::max(a.Dk, a.Dv);
    const unsigned blocks = static_cast<unsigned>(std::min<size_t>((most + 1023) / 1024, 4096));
    if (int rc = with_storage(a.dtype, [&](auto z) {
          la_head_sum_kernel<decltype(z)><<<dim3(blocks, 3), 256, 0, st>>>(hs);
          PRNN_HIP(hipGetLastError());
          return static_cast<int>(PRNN_OK);
        }))
      return rc;
  }
  if (dg) {
    DecayGradArgs d{};
    d.seqs = p.seqs;
    d.g = p.g;
    d.q_dots = s.dots[0];
    d.k_dots = s.dots[1];
    const int cols = w.cols(std::max(a.Dk, a.Dv));
    d.tiles = (a.Dk + cols - 1) / cols;
    d.H = a.H;
    d.DD = a.Dk * a.Dv;
    d.batch_tokens = static_cast<int>(tokens);
    d.h0 = init;
    d.dh0 = dh0;
    d.last = s.last;
    d.gs = gs;
    d.state = s.state[0];
    d.adjoint = s.state[1];
    d.g_dtype = a.g_dtype;
    const bool per_head = a.g_sb == 0 && a.g_st == 0;
    d.dg = per_head ? nullptr : dg;
    d.per_part = per_head ? s.per_part : nullptr;
    if (int rc = check_grid("linear_attention", d.seqs.pieces, 256)) return rc;
    const dim3 grid(d.seqs.pieces, a.H);
    la_decay_grad_kernel<<<grid, 256, 0, st>>>(d);
    PRNN_HIP(hipGetLastError());
    if (per_head) {
      la_decay_sum_kernel<<<a.H, 64, 0, st>>>(s.per_part, dg, a.g_dtype, d.seqs.pieces, a.H);
      PRNN_HIP(hipGetLastError());
    }
  }
  return PRNN_OK;
}

}  // namespace
}  // namespace prnn

using namespace prnn;

extern "C" PRNN_API size_t
prnn_linear_attention_workspace_size(const prnn_linear_attention_problem* a) {
  if (check(a)) return 0;
  return need(*a, false, false);
}

extern "C" PRNN_API int prnn_linear_attention(const prnn_linear_attention_problem* a,
                                              const prnn_la_view* out, float* state_out,
                                              const int* out_table, int out_rows, void* workspace,
                                              size_t bytes, void* stream) {
  if (int rc = check(a)) return rc;
  if (out == nullptr || (out->p == nullptr && 1ll * a->B * a->T > 0))
    return fail(PRNN_ERR_VALUE, "out must be non-null");
  if (int rc = check_tokens(*a, out->st)) return rc;
  if (sequences(*a) == 0) return PRNN_OK;
  if (int rc = check_ws(need(*a, false, false), workspace, bytes)) return rc;
  return forward(*a, *out, state_out, out_table, out_rows, workspace,
                 static_cast<hipStream_t>(stream));
}

extern "C" PRNN_API size_t prnn_linear_attention_backward_workspace_size(
    const prnn_linear_attention_problem* a, int decay_grad) {
  if (check(a)) return 0;
  return need(*a, true, decay_grad != 0);
}

extern "C" PRNN_API int prnn_linear_attention_backward(
    const prnn_linear_attention_problem* a, const prnn_la_view* go, const float* gs, void* dq,
    void* dk, void* dv, void* dg, float* dh0, void* workspace, size_t bytes, void* stream) {
  if (int rc = check(a)) return rc;
  const bool any = 1ll * a->B * a->T > 0;
  if (go == nullptr || (any && (!go->p || !dq || !dk || !dv)))
    return fail(PRNN_ERR_VALUE, "go, dq, dk and dv must be non-null");
  if (int rc = check_tokens(*a, go->st)) return rc;
  if (a->h0_table) return fail(PRNN_ERR_VALUE, "a block table has no gradient");
  if (a->h0 && a->h0_rows < sequences(*a))
    return fail(PRNN_ERR_VALUE, "h0 has %d rows for %d sequences", a->h0_rows, sequences(*a));
  if (dg && a->h0 && !dh0)
    return fail(PRNN_ERR_VALUE, "the decays' gradient with an initial state needs dh0");
  if (sequences(*a) == 0) return PRNN_OK;  // (an empty batch's decays per head: the caller's zeros)
  if (int rc = check_ws(need(*a, true, dg != nullptr), workspace, bytes)) return rc;
  return backward(*a, *go, gs, dq, dk, dv, dg, dh0, workspace, static_cast<hipStream_t>(stream));
}
