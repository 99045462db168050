// Gated delta rule: the C entry points and how a call is laid out.
#include "delta_rule.h"

namespace prnn {
namespace {

using Problem = prnn_delta_rule_problem;

int check(const Problem* a) {
  if (a == nullptr) return fail(PRNN_ERR_VALUE, "the problem must be non-null");
  if (int rc = la_check(&a->la)) return rc;
  if (a->b_dtype != PRNN_F32 && a->b_dtype != a->la.dtype)
    return fail(PRNN_ERR_TYPE, "beta must be float32 or of the storage type");
  if (1ll * a->la.B * a->la.T > 0 && a->b == nullptr)
    return fail(PRNN_ERR_VALUE, "beta must be non-null");
  return PRNN_OK;
}

// bf16 storage of widths in eights runs on bf16 matrix instructions; its rows are read 16 bytes at a
// time.
bool on_bf16(const Problem& a) {
  return a.la.dtype == PRNN_BF16 && a.la.Dk % 8 == 0 && a.la.Dv % 8 == 0;
}
int check_rows(const Problem& a, const prnn_la_view& other) {
  if (1ll * a.la.B * a.la.T == 0 || !on_bf16(a)) return PRNN_OK;
  if (la_view(a.la.q, a.la, a.la.Dk).vec && la_view(a.la.k, a.la, a.la.Dk).vec &&
      la_view(a.la.v, a.la, a.la.Dv).vec && la_view(other, a.la, a.la.Dv).vec)
    return PRNN_OK;
  return fail(PRNN_ERR_VALUE, "bfloat16 rows of widths in eights must start on 16-byte boundaries and "
                              "lie at least a row apart");
}
int check_strides(const Problem& a, const prnn_la_view& other) {
  if (a.la.T > 1 && !la_stride_fits(other.st, a.la.dtype == PRNN_F32 ? 4 : 2))
    return fail(PRNN_ERR_VALUE, "tokens %lld elements apart do not lie 0 bytes to 16 MiB apart", other.st);
  return PRNN_OK;
}

int sequences(const Problem& a) { return a.la.cu_seqlens ? a.la.n_seq : a.la.B; }
size_t tokens_of(const Problem& a) { return static_cast<size_t>(a.la.B) * a.la.T; }

LaSeqs sequences_of(const Problem& a) {
  LaSeqs q{};
  q.cu = a.la.cu_seqlens;
  q.n_seq = sequences(a);
  q.T = a.la.T;
  q.len = 1 << 30;  // whole
  return q;
}

// What the backward pass reads of the forward one: as operands e and the states before the chunks, and
// the chunks' systems.
struct Kept {
  float *e, *before;
  char* sys;
  int* order;  // of a packed batch's pieces
  size_t bytes;
};
int pieces_of(const Problem& a);  // (of a plan; 0: not packed)
Kept kept_of(void* p, const Problem& a) {
  Carver c(p);
  const size_t heads = a.la.H;
  Kept k{};
  const size_t units = dr_units(sequences_of(a), kDrC);
  k.e = static_cast<float*>(c.take(4 * units * heads * dr_operand_elems(kDrC, a.la.Dv)));
  k.before = static_cast<float*>(c.take(4 * units * heads * dr_operand_elems(a.la.Dk, a.la.Dv)));
  k.sys = static_cast<char*>(c.take(units * heads * kDrSys));
  k.order = static_cast<int*>(c.take(4 * static_cast<size_t>(pieces_of(a))));
  k.bytes = c.used;
  return k;
}

struct Scratch {
  char* sys;
  int* order;
  float *behind, *dv;
  float* piece;
  uint16_t* transfer;
  float *dq32, *dk32, *g_part;
  size_t bytes;
};

// How a walk is laid out: columns of a wave, tokens of a piece (more than T: whole sequences).
struct Plan {
  int cols;
  LaSeqs seqs;
  bool cut;
};

// Columns of a wave: 32, or 16 where there are not enough waves of 32 for two of the chip's 1024 SIMDs (and
// where 32 columns of wide keys do not fit the registers).
int wave_cols(const Problem& a, const LaSeqs& q) {
  if (!on_bf16(a)) return 16;
  if (a.la.Dk > 128 || (a.la.Dk > 64 && a.la.Dv <= 64)) return 16;
  return dr_units(q, q.len) * a.la.H * ((a.la.Dv + 31) / 32) >= 2048 ? 32 : 16;
}

// A sequence's chunks come one after another.  Cut into n pieces they go side by side, but every piece
// but the last walks a second time, without outputs and over Dv + Dk columns, and the join takes the
// pieces one after another.  In units of a chunk of the full walk (4.2 us): 0.6 for one of the state
// alone, 0.4 for a piece's step of the join, 4 for the two launches more.  A CU's second workgroup
// makes both slower by half, further ones wait.
Plan plan(const Problem& a) {
  Plan p{16, sequences_of(a), false};
  const long long longest = a.la.cu_seqlens && a.la.longest > 0 ? std::min(a.la.longest, a.la.T) : a.la.T;
  const long long chunks = (longest + kDrC - 1) / kDrC, tokens = 1ll * a.la.B * a.la.T;
  const int group_cols = dr_walk_group(a.la.Dk, a.la.Dv, 16, on_bf16(a), 1 << 20) * 16;
  const double tiles = (a.la.Dv + group_cols - 1) / group_cols;
  // of a packed batch half the tokens are taken to be in sequences that are cut
  const double own = (tiles + (a.la.Dk + group_cols - 1) / group_cols) * (a.la.cu_seqlens ? 0.5 : 1.0);
  const double work = static_cast<double>(tokens) / kDrC * a.la.H / 256.0;  // chunks a CU and column tile
  auto time = [&](double each, double tiles) {
    const double x = work * tiles / each;
    return each * (x <= 1.0 ? 1.0 : std::max(0.5 + 0.5 * x, 0.75 * x));
  };
  double best = 0.0;
  long long pieces = 1;
  for (long long n = 1; n <= 64 && n <= chunks; ++n) {
    const double each = static_cast<double>((chunks + n - 1) / n);
    double t = time(each, tiles);
    if (n > 1) t += 0.6 * time(each, own) + 0.4 * n + 4.0;
    if (n == 1 || t < best) {
      best = t;
      pieces = n;
    }
  }
  if (pieces > 1) {
    p.seqs.len = static_cast<int>((chunks + pieces - 1) / pieces * kDrC);
    p.cut = p.seqs.len < longest;
    if (!p.cut) p.seqs.len = 1 << 30;
  }
  p.cols = wave_cols(a, p.seqs);
  return p;
}

int pieces_of(const Problem& a) {
  if (a.la.cu_seqlens == nullptr) return 0;
  const Plan p = plan(a);
  return static_cast<int>(std::min<long long>(dr_units(p.seqs, p.seqs.len), 1 << 30));
}

Scratch carve(void* ws, const Problem& a, const Plan& plan, bool systems, bool backward, bool decay_grad) {
  Carver c(ws);
  Scratch s{};
  const size_t heads = a.la.H, tokens = tokens_of(a);
  const size_t units = dr_units(plan.seqs, kDrC);
  if (systems) {
    s.sys = static_cast<char*>(c.take(units * heads * kDrSys));
    s.order = static_cast<int*>(c.take(4 * static_cast<size_t>(pieces_of(a))));
  }
  if (plan.cut) {
    const size_t slots = dr_slots(plan.seqs) * heads;
    s.piece = static_cast<float*>(c.take(4 * slots * a.la.Dk * a.la.Dv));
    s.transfer = static_cast<uint16_t*>(c.take(6 * slots * dr_operand_elems(a.la.Dk, a.la.Dk)));
  }
  if (backward) {
    s.behind = static_cast<float*>(c.take(4 * units * heads * dr_operand_elems(a.la.Dk, a.la.Dv)));
    // fp32 dv is written where it is wanted, unless its heads are summed or it is stored in another type
    if (a.la.v.heads != a.la.H || a.la.dtype != PRNN_F32)
      s.dv = static_cast<float*>(c.take(4 * tokens * heads * a.la.Dv));
    if (a.la.q.heads != a.la.H) s.dq32 = static_cast<float*>(c.take(4 * tokens * heads * a.la.Dk));
    if (a.la.k.heads != a.la.H) s.dk32 = static_cast<float*>(c.take(4 * tokens * heads * a.la.Dk));
    if (decay_grad) s.g_part = static_cast<float*>(c.take(4 * units * heads));
  }
  s.bytes = c.used;
  return s;
}
size_t need(const Problem& a, bool systems, bool backward, bool decay_grad) {
  return carve(nullptr, a, plan(a), systems, backward, decay_grad).bytes;
}

int check_ws(const char* what, size_t need, const void* ws, size_t bytes) {
  if (need && (ws == nullptr || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255)))
    return fail(PRNN_ERR_VALUE, "the %s must hold %zu bytes, 256-byte aligned (got %zu)", what, need, bytes);
  return PRNN_OK;
}

LaDecay decay_of(const Problem& a) {
  return LaDecay{a.la.g, a.la.g_sb, a.la.g_st, a.la.g_sh, a.la.g_dtype};
}
LaDecay rate_of(const Problem& a) { return LaDecay{a.b, a.b_sb, a.b_st, a.b_sh, a.b_dtype}; }

int systems(const Problem& a, const Plan& plan, char* sys, int* order, hipStream_t st) {
  DrSystems y{};
  y.seqs = sequences_of(a);
  y.q = la_view(a.la.q, a.la, a.la.Dk);
  y.k = la_view(a.la.k, a.la, a.la.Dk);
  y.g = decay_of(a);
  y.b = rate_of(a);
  y.sys = sys;
  y.H = a.la.H;
  y.Dk = a.la.Dk;
  y.dtype = a.la.dtype;
  y.pieces = plan.seqs;
  y.n_pieces = pieces_of(a);
  y.order = y.n_pieces ? order : nullptr;
  y.scale = a.la.scale;
  return dr_systems(y, on_bf16(a), st);
}

DrWalk walk_of(const Problem& a, const Plan& plan, const Scratch& s, const char* sys, const int* order) {
  DrWalk w{};
  w.seqs = plan.seqs;
  w.q = la_view(a.la.q, a.la, a.la.Dk);
  w.k = la_view(a.la.k, a.la, a.la.Dk);
  w.sys = sys;
  w.n_pieces = pieces_of(a);
  w.order = w.n_pieces ? order : nullptr;
  w.piece = s.piece;
  w.transfer = s.transfer;
  w.H = a.la.H;
  w.Dk = a.la.Dk;
  w.Dv = a.la.Dv;
  w.dtype = a.la.dtype;
  w.scale = a.la.scale;
  return w;
}
int run(DrWalk w, DrKind kind, const Problem& a, const Plan& plan, hipStream_t st) {
  const bool own = kind == kDrState || kind == kDrAdjoint;
  // (pieces' own states have the transfers' columns besides)
  const long long items = dr_units(plan.seqs, plan.seqs.len) * a.la.H * (own ? 2 : 1);
  w.group = dr_walk_group(a.la.Dk, a.la.Dv, plan.cols, on_bf16(a), items);
  const int cols = w.group * plan.cols;
  w.own_tiles = (a.la.Dv + cols - 1) / cols;
  w.tiles = w.own_tiles + (own ? (a.la.Dk + cols - 1) / cols : 0);
  return on_bf16(a) ? dr_walk_bf16(w, kind, plan.cols, st) : dr_walk_f32(w, kind, st);
}
// The walk of a direction; of a cut sequence the pieces' own states and the join before it.
int walk(const DrWalk& w, bool back, const Problem& a, const Plan& plan, hipStream_t st) {
  if (plan.cut) {
    DrWalk own = w;
    if (int rc = run(own, back ? kDrAdjoint : kDrState, a, plan, st)) return rc;
    if (int rc = dr_join(w, back, st)) return rc;
  }
  return run(w, back ? kDrBackward : w.keep ? kDrKept : kDrForward, a, plan, st);
}

int forward(const Problem& a, const prnn_la_view& out, float* state_out, const int* out_table, int out_rows,
            void* kept, void* ws, hipStream_t st) {
  const Plan p = plan(a);
  const Scratch s = carve(ws, a, p, kept == nullptr, false, false);
  const Kept k = kept_of(kept, a);
  char* sys = kept ? k.sys : s.sys;
  int* order = kept ? k.order : s.order;
  if (int rc = systems(a, p, sys, order, st)) return rc;
  DrWalk w = walk_of(a, p, s, sys, order);
  w.z = la_view(a.la.v, a.la, a.la.Dv);
  w.out = const_cast<void*>(out.p);
  w.o_sb = out.sb;
  w.o_st = a.la.T > 1 ? out.st : a.la.Dv;
  w.o_sh = out.sh;
  if (kept) {
    w.e = k.e;
    w.keep = k.before;
  }
  w.init = LaState{const_cast<float*>(a.la.h0), a.la.h0_table, a.la.h0_rows};
  w.last = LaState{state_out, out_table, out_rows};
  return walk(w, false, a, p, st);
}

int backward(const Problem& a, const prnn_la_view& go, const float* gs, const void* kept, void* dq, void* dk,
             void* dv, void* dg, void* db, float* dh0, void* ws, hipStream_t st) {
  const bool per_head = a.la.g_sb == 0 && a.la.g_st == 0;
  const Plan p = plan(a);
  const Scratch s = carve(ws, a, p, false, true, dg != nullptr);
  const Kept k = kept_of(const_cast<void*>(kept), a);
  DrWalk w = walk_of(a, p, s, k.sys, k.order);
  w.z = la_view(go, a.la, a.la.Dv);
  w.keep = s.behind;
  w.dv = s.dv ? s.dv : static_cast<float*>(dv);
  w.init = LaState{const_cast<float*>(gs), nullptr, sequences(a)};
  w.last = LaState{dh0, nullptr, sequences(a)};
  if (int rc = walk(w, true, a, p, st)) return rc;
  DrGrad g{};
  g.seqs = w.seqs;
  g.q = w.q;
  g.k = w.k;
  g.go = w.z;
  g.g = decay_of(a);
  g.sys = k.sys;
  g.e = k.e;
  g.dv = w.dv;
  g.dv16 = on_bf16(a) && a.la.v.heads == a.la.H ? dv : nullptr;
  g.before = k.before;
  g.behind = s.behind;
  g.q_f32 = s.dq32 != nullptr;
  g.k_f32 = s.dk32 != nullptr;
  g.dq = g.q_f32 ? s.dq32 : dq;
  g.dk = g.k_f32 ? s.dk32 : dk;
  g.dg = per_head ? nullptr : dg;
  g.g_part = per_head && dg ? s.g_part : nullptr;
  g.dbeta = db;
  g.H = a.la.H;
  g.Dk = a.la.Dk;
  g.Dv = a.la.Dv;
  g.dtype = a.la.dtype;
  g.g_dtype = a.la.g_dtype;
  g.b_dtype = a.b_dtype;
  g.scale = a.la.scale;
  if (int rc = dr_grad(g, on_bf16(a), st)) return rc;
  LaHeadSums hs{};
  const float* from[3] = {s.dq32, s.dk32, g.dv16 ? nullptr : s.dv};
  void* to[3] = {dq, dk, dv};
  const int D[3] = {a.la.Dk, a.la.Dk, a.la.Dv}, heads[3] = {a.la.q.heads, a.la.k.heads, a.la.v.heads};
  bool sums = false;
  for (int i = 0; i < 3; ++i) {
    hs.src[i] = from[i];
    hs.dst[i] = to[i];
    hs.rep[i] = a.la.H / heads[i];
    hs.D[i] = D[i];
    sums = sums || from[i];
  }
  hs.H = a.la.H;
  hs.tokens = tokens_of(a);
  if (sums)
    if (int rc = la_head_sums(hs, a.la.dtype, st)) return rc;
  if (g.g_part) {
    const int parts = static_cast<int>(dr_units(w.seqs, kDrC));
    if (int rc = la_decay_sums(s.g_part, dg, a.la.g_dtype, parts, a.la.H, st)) return rc;
  }
  return PRNN_OK;
}

}  // namespace
}  // namespace prnn

using namespace prnn;

extern "C" PRNN_API size_t prnn_delta_rule_workspace_size(const prnn_delta_rule_problem* a, int kept) {
  if (check(a)) return 0;
  return need(*a, kept == 0, false, false);
}

extern "C" PRNN_API size_t prnn_delta_rule_kept_size(const prnn_delta_rule_problem* a) {
  if (check(a)) return 0;
  return kept_of(nullptr, *a).bytes;
}

extern "C" PRNN_API int prnn_delta_rule(const prnn_delta_rule_problem* a, const prnn_la_view* out,
                                        float* state_out, const int* out_table, int out_rows, void* kept,
                                        void* workspace, size_t bytes, void* stream) {
  if (int rc = check(a)) return rc;
  if (out == nullptr || (out->p == nullptr && tokens_of(*a) > 0))
    return fail(PRNN_ERR_VALUE, "out must be non-null");
  if (int rc = check_strides(*a, *out)) return rc;
  if (int rc = check_rows(*a, *out)) return rc;
  if (sequences(*a) == 0) return PRNN_OK;
  if (kept && (reinterpret_cast<uintptr_t>(kept) & 255))
    return fail(PRNN_ERR_VALUE, "what is kept must lie on a 256-byte boundary");
  if (int rc = check_ws("workspace", need(*a, kept == nullptr, false, false), workspace, bytes)) return rc;
  return forward(*a, *out, state_out, out_table, out_rows, kept, workspace, static_cast<hipStream_t>(stream));
}

extern "C" PRNN_API size_t prnn_delta_rule_backward_workspace_size(const prnn_delta_rule_problem* a,
                                                                   int decay_grad) {
  if (check(a)) return 0;
  return need(*a, false, true, decay_grad != 0);
}

extern "C" PRNN_API int prnn_delta_rule_backward(const prnn_delta_rule_problem* a, const prnn_la_view* go,
                                                 const float* gs, const void* kept, void* dq, void* dk,
                                                 void* dv, void* dg, void* db, float* dh0, void* workspace,
                                                 size_t bytes, void* stream) {
  if (int rc = check(a)) return rc;
  const bool any = tokens_of(*a) > 0;
  if (go == nullptr || (any && (!go->p || !kept || !dq || !dk || !dv)))
    return fail(PRNN_ERR_VALUE, "go, kept, dq, dk and dv must be non-null");
  if (int rc = check_strides(*a, *go)) return rc;
  if (int rc = check_rows(*a, *go)) return rc;
  if (on_bf16(*a) && ((reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) |
                       reinterpret_cast<uintptr_t>(dv)) & 15))
    return fail(PRNN_ERR_VALUE, "dq, dk and dv must start on 16-byte boundaries");
  if (a->la.h0_table) return fail(PRNN_ERR_VALUE, "a block table has no gradient");
  if (a->la.h0 && a->la.h0_rows < sequences(*a))
    return fail(PRNN_ERR_VALUE, "h0 has %d rows for %d sequences", a->la.h0_rows, sequences(*a));
  if (sequences(*a) == 0) return PRNN_OK;
  if (int rc = check_ws("workspace", need(*a, false, true, dg != nullptr), workspace, bytes)) return rc;
  return backward(*a, *go, gs, kept, dq, dk, dv, dg, db, dh0, workspace, static_cast<hipStream_t>(stream));
}
