// Beam search: the best continuations over beams and vocabulary.
//
//   total(k, t) = score_k + logits_kt - logsumexp_t(logits_kt),  the M largest of a search's K V,
//   ties to the lowest beam, in a beam to the larger logit (a score far from zero makes totals of
//   different logits equal), then to the lowest token.
//
// Two launches.  The first reads the logits once: a workgroup per beam and slice of 8176 tokens, 32
// values a thread in registers, gives the slice's largest value, its sum of exponentials and its M
// best.  The second, a workgroup per search, joins the slices' sums in fp64 and chooses among the
// slices' best.
//
// Candidates of two beams may lie next to each other, and equal beams tie: which one goes on must not
// hang on where a row lies in memory.  So slices are of fixed tokens, the exponentials are formed in fp64
// and added as whole multiples of 2^-50 of the slice's largest: the sum is the same in any order (which
// thread holds a token goes by the row's address), and off by 2^-51 a token at most.
//
// The M best of some thousand values: the M-th largest of the threads' own largest is a bound that at
// least M values reach, and only values of those M threads can; what reaches it (a few more than M of
// ordinary logits) is ranked by counting, so the order of arrival does not matter.  Up to 32 best the
// bound is the largest of the four waves' own, found by a quarter of the comparisons.
//
// 32 searches of 8 beams over 50257 bf16 logits: 26 us (26 MB; the exponentials' instructions, some twenty
// of fp64 each, bound it: 15 us with exponentials and sums of fp32, which told equal beams apart) and 11
// us (latency: a wave per beam's sum, then three rounds through LDS); one search of 4 beams over 32000:
// 8.2 and 8.8 us, latency.
#include <algorithm>

#include "prnn_host.h"

namespace prnn {
namespace {

constexpr int kMost = 128;     // candidates that are wanted
constexpr int kEach = 32;      // tokens of a thread
constexpr int kSlice = 256 * kEach;
// Tokens of a slice: its values' places but those that a row's start inside a 16-byte unit may take.
// Whole units, so that all slices of a row start at the same place in one.
constexpr int kTokens = kSlice - 16;
constexpr int kFew = 32;       // up to which a bound is a wave's
constexpr int kRound = 2;     // candidates of a thread and round of the second launch

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Order of floats as of unsigned numbers, zeros of either sign alike; -infinity and NaN are 0: never
// chosen.
__device__ __forceinline__ uint32_t order(float v) {
  const uint32_t b = v == 0.0f ? 0u : __float_as_uint(v);
  if (!(v > -INFINITY)) return 0u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order(double v) {
  const uint64_t b = v == 0.0 ? 0ull : __builtin_bit_cast(uint64_t, v);
  if (!(v > -static_cast<double>(INFINITY))) return 0ull;
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double value(uint64_t o) {
  return __builtin_bit_cast(double, o >> 63 ? o & ~(1ull << 63) : ~o);
}

// exp(x) for x <= 0 as a whole number of 2^-50: 2^n 2^f with |f| <= 1/2, 2^f = sum (f ln 2)^i / i! to i = 12.
// Off by half of one, and by (|x| + 2) 2^-53 of itself (the reduction and what the sum leaves out).
constexpr int kUnit = 50;
struct Taylor {
  double c[13] = {1.0};
  constexpr Taylor() {
    for (int i = 1; i < 13; ++i) c[i] = c[i - 1] * 0.69314718055994530942 / i;
  }
};
__device__ __forceinline__ uint64_t exp_units(double x) {
  // below -48 it is nothing of a unit, and a -infinity would leave NaN
  const double t = fmax(x, -48.0) * 1.4426950408889634074, n = rint(t), f = t - n;
  constexpr Taylor y;
  double p = y.c[12];
#pragma unroll
  for (int i = 11; i >= 0; --i) p = fma(p, f, y.c[i]);
  // p 2^n in units, rounded at the last place of a number in 2^52 .. 2^53
  const double scale = __builtin_bit_cast(double, static_cast<uint64_t>(1023 + kUnit + static_cast<int>(n)) << 52);
  return __builtin_bit_cast(uint64_t, fma(p, scale, 0x1p52)) & ((1ull << 52) - 1);
}

struct Slice {
  double sum;  // of exp(logit - most)
  float most;  // NaN: the beam has no finite probabilities
  int count;
};

struct BeamArgs {
  const void* logits;
  long long sb, sk;
  const float* scores;
  const uint8_t* ended;
  Slice* slices;          // (B K, S)
  uint2* best;            // (B K, S, M): order and token
  float* out_scores;
  int *out_parents, *out_tokens;
  int B, K, V, M, S, pad;
};

// MOST: candidates that are wanted at most.
template <typename T, int MOST>
__global__ __launch_bounds__(256) void beam_slice_kernel(BeamArgs A) {
  constexpr int V = 16 / sizeof(T);
  __shared__ __align__(16) uint64_t s_top[256];
  __shared__ uint64_t s_list[(MOST <= kFew ? 4 : 1) * MOST * kEach];
  __shared__ uint64_t s_sum[4];
  __shared__ float s_most[4];
  __shared__ bool s_bad[4];
  __shared__ uint64_t s_bound[4];
  __shared__ int s_count;
  const int tid = threadIdx.x, slice = blockIdx.x % A.S, row = blockIdx.x / A.S;
  const int b = row / A.K, k = row - b * A.K;
  if (A.ended && A.ended[row]) return;
  const T* p = static_cast<const T*>(A.logits) + b * A.sb + k * A.sk;
  // units of 16 bytes as memory has them; the row starts `skip` values into the first.  All loads go out
  // together (in branches they came one after another): units behind the row lie behind the buffer, and
  // what else is in its first and last one is taken out afterwards.
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  const int first_token = slice * kTokens, there = min(A.V - first_token, kTokens);
  const rsrc_t row_part =
      make_rsrc(p + first_token - skip, ((there + skip) * static_cast<uint32_t>(sizeof(T)) + 15) & ~15u);
  u4 raw[kEach / V];
#pragma unroll
  for (int u = 0; u < kEach / V; ++u)
    raw[u] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(row_part, (u * 256 + tid) * 16, 0, 0));
  float v[kEach];
#pragma unroll
  for (int u = 0; u < kEach / V; ++u)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (sizeof(T) == 4)
        v[u * V + i] = __uint_as_float(raw[u][i]);
      else
        v[u * V + i] = i & 1 ? Narrow<T>::hi(raw[u][i / 2]) : Narrow<T>::lo(raw[u][i / 2]);
    }
  auto place_of = [&](int i) { return ((i / V) * 256 + tid) * V + i % V - skip; };  // in the slice
  auto token = [&](int i) { return first_token + place_of(i); };
  // (of a whole slice the first wave's first unit and the last wave's last ones)
  if (there < kTokens || (tid < 64 && skip) || tid >= 192) {
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (place_of(i) < 0 || place_of(i) >= there) v[i] = -INFINITY;
  }
  // this thread's largest, the lowest token of equals
  float most = v[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) most = fmaxf(most, v[i]);
  int place = 0;
#pragma unroll
  for (int i = kEach - 1; i >= 0; --i) place = v[i] == most ? i : place;
  const uint32_t first = order(most);
  const uint64_t top = first ? static_cast<uint64_t>(first) << 32 | static_cast<uint32_t>(~token(place)) : 0ull;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) most = fmaxf(most, __shfl_xor(most, m));
  s_top[tid] = top;
  if ((tid & 63) == 0) s_most[tid >> 6] = most;
  if (tid < 4) s_bound[tid] = 1;
  if (tid == 0) s_count = 0;
  __syncthreads();
  most = fmaxf(fmaxf(s_most[0], s_most[1]), fmaxf(s_most[2], s_most[3]));
  const bool none = !(most > -INFINITY);
  uint64_t sum = 0;
  bool bad = false;  // NaN or an infinity: no finite probabilities
  {
    const double from = none ? 0.0 : most;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      sum += exp_units(v[i] - from);
      bad |= !(v[i] < INFINITY);
    }
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
  bad = __any(bad);
  if ((tid & 63) == 0) {
    s_sum[tid >> 6] = sum;
    s_bad[tid >> 6] = bad;
  }
  // this thread's place among the threads' largest
  int above = 0;
  if (top) {
    constexpr int kAmong = MOST <= kFew ? 64 : 256;
    const int first = MOST <= kFew ? tid & ~63 : 0;
#pragma unroll 8
    for (int i = 0; i < kAmong; i += 2) {
      const ulong2 o = *reinterpret_cast<const ulong2*>(&s_top[first + i]);
      above += (o.x > top) + (o.y > top);
    }
    if (above == A.M - 1) s_bound[first >> 6] = top;
  }
  __syncthreads();
  uint64_t bound = s_bound[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) bound = s_bound[w] > bound ? s_bound[w] : bound;
  const uint32_t lowest = static_cast<uint32_t>(bound >> 32);
  const float least = lowest == 0 ? -INFINITY : __uint_as_float(lowest & 0x80000000u ? lowest & 0x7fffffffu : ~lowest);
  if (top >= bound) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (!(v[i] >= least)) continue;
      const uint32_t o = order(v[i]);
      if (o == 0) continue;
      const uint64_t key = static_cast<uint64_t>(o) << 32 | static_cast<uint32_t>(~token(i));
      if (key >= bound) s_list[atomicAdd(&s_count, 1)] = key;
    }
  }
  __syncthreads();
  const int n = s_count;
  const size_t at = static_cast<size_t>(row) * A.S + slice;
  for (int i = tid; i < n; i += 256) {
    const uint64_t o = s_list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s_list[j] > o;
    if (rank < A.M)
      A.best[at * A.M + rank] = make_uint2(static_cast<uint32_t>(o >> 32), ~static_cast<uint32_t>(o));
  }
  if (tid == 0) {
    const uint64_t all = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    const bool any_bad = s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3];
    A.slices[at] = Slice{static_cast<double>(all) * 0x1p-50, any_bad ? NAN : most, min(n, A.M)};
  }
}

// A candidate of the second launch: the order of its total; its beam and, turned, its logit's order; its
// token.  Compared without branches (with them 32 choices among 448 took 21 us, 11 without).
struct Total {
  uint64_t o, place;
  uint32_t t;
};
__device__ __forceinline__ Total total(double v, int k, uint32_t low, uint32_t t) {
  return Total{order(v), static_cast<uint64_t>(static_cast<uint32_t>(k)) << 32 | low, t};
}
__device__ __forceinline__ bool before(const Total& a, const Total& b) {
  return (a.o > b.o) | ((a.o == b.o) & ((a.place < b.place) | ((a.place == b.place) & (a.t < b.t))));
}
constexpr Total kNoTotal{0, ~0ull, ~0u};

__global__ __launch_bounds__(256) void beam_choose_kernel(BeamArgs A) {
  __shared__ Total s_top[256], s_list[kMost * kRound + kMost], s_carry[kMost], s_bound[4];
  __shared__ int s_count, s_held;
  // A total is ((logit - most) + score) - log(sum): the first two sums are exact for logits and scores of like
  // size, so that what is equal in a row's candidates, or in equal rows', stays equal.
  __shared__ double s_most[kMost], s_score[kMost], s_log[kMost];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, b = blockIdx.x;
  const int per = A.S * A.M;  // candidates of a beam; all of kMost beams' are below 2^26
  const bool few = A.M <= kFew;
  if (tid == 0) s_held = 0;
  // What the beams' totals are made of, beams in blocks of kMost, a beam a wave; the largest logit stays
  // apart (masks of the type's lowest value would swallow the logarithm)
  for (int k0 = 0; k0 < A.K; k0 += kMost) {
    __syncthreads();
    const int end = min(A.K - k0, kMost) * per;
    // a round's candidates, the first ones under way while the totals' shares are formed
    uint2 best[kRound];
    int beam[kRound];  // -1: none
    bool over[kRound]; // goes on as it is, with one token
    auto load = [&](int base) {
      int count[kRound], rank[kRound];
#pragma unroll
      for (int i = 0; i < kRound; ++i) {
        const int at = min(base + i * 256 + tid, end - 1);
        const int k = at / per, in = at - k * per, s = in / A.M;
        const int row = b * A.K + k0 + k;
        const size_t slice = static_cast<size_t>(row) * A.S + s;
        rank[i] = in - s * A.M;
        over[i] = A.ended && A.ended[row];
        best[i] = A.best[slice * A.M + rank[i]];
        count[i] = A.slices[slice].count;
        if (over[i]) {
          rank[i] = in;
          count[i] = 1;
        }
        beam[i] = k;
      }
#pragma unroll
      for (int i = 0; i < kRound; ++i)
        if (base + i * 256 + tid >= end || rank[i] >= count[i]) beam[i] = -1;
    };
    for (int base = 0; base < end; base += 256 * kRound) {
      load(base);
      if (base == 0) {
        for (int k = k0 + wave; k < min(A.K, k0 + kMost); k += 4) {
          const int row = b * A.K + k;
          double score = A.scores[row], most = -static_cast<double>(INFINITY), log_sum = 0.0;
          if (!(A.ended && A.ended[row])) {
            const Slice* x = A.slices + static_cast<size_t>(row) * A.S;
            Slice own = lane < A.S ? x[lane] : Slice{0.0, -INFINITY, 0};
            float top = own.most;
            bool bad = top != top;
            double sum = 0.0;
            for (int s = lane + 64; s < A.S; s += 64) {
              bad |= x[s].most != x[s].most;
              top = fmaxf(top, x[s].most);
            }
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
            for (int s = lane;; own = x[s]) {
              if (own.sum > 0.0) sum += own.sum * exp(static_cast<double>(own.most) - top);
              if ((s += 64) >= A.S) break;
            }
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
            most = top;
            if (__any(bad)) score = -static_cast<double>(INFINITY);
            log_sum = log(sum);
          }
          if (lane == 0) {
            s_most[k - k0] = most;
            s_score[k - k0] = score;
            s_log[k - k0] = log_sum;
          }
        }
        __syncthreads();
      }
      Total c[kRound], top = kNoTotal;
#pragma unroll
      for (int i = 0; i < kRound; ++i) {
        c[i] = kNoTotal;
        const int k = beam[i];
        if (k < 0) continue;
        if (over[i]) {
          c[i] = total(s_score[k], k0 + k, 0, A.pad);
        } else {
          const float logit = __uint_as_float(best[i].x & 0x80000000u ? best[i].x & 0x7fffffffu : ~best[i].x);
          const double t = ((static_cast<double>(logit) - s_most[k]) + s_score[k]) - s_log[k];
          c[i] = total(t, k0 + k, ~best[i].x, best[i].y);
        }
        if (c[i].o && before(c[i], top)) top = c[i];
      }
      s_top[tid] = top;
      if (tid < 4) s_bound[tid] = Total{1, ~0ull, ~0u};
      const int held = s_held;
      for (int i = tid; i < held; i += 256) s_list[i] = s_carry[i];
      if (tid == 0) s_count = held;
      __syncthreads();
      // where candidates are few, all are ranked
      if (end - base > 128 && top.o) {
        const int first = few ? tid & ~63 : 0, among = few ? 64 : 256;
        int above = 0;
#pragma unroll 8
        for (int i = 0; i < among; ++i) above += before(s_top[first + i], top);
        if (above == A.M - 1) s_bound[first >> 6] = top;
      }
      __syncthreads();
      Total bound = s_bound[0];
#pragma unroll
      for (int w = 1; w < 4; ++w) bound = before(s_bound[w], bound) ? s_bound[w] : bound;
#pragma unroll
      for (int i = 0; i < kRound; ++i)
        if (c[i].o && !before(bound, c[i])) s_list[atomicAdd(&s_count, 1)] = c[i];
      __syncthreads();
      const int n = s_count;
      for (int i = tid; i < n; i += 256) {
        const Total own = s_list[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += before(s_list[j], own);
        if (rank < A.M) s_carry[rank] = own;
      }
      if (tid == 0) s_held = min(n, A.M);
      __syncthreads();
    }
  }
  __syncthreads();
  const int held = s_held;
  for (int i = tid; i < A.M; i += 256) {
    const bool any = i < held;
    const size_t at = static_cast<size_t>(b) * A.M + i;
    A.out_scores[at] = any ? static_cast<float>(value(s_carry[i].o)) : -INFINITY;
    A.out_parents[at] = any ? static_cast<int>(s_carry[i].place >> 32) : -1;
    A.out_tokens[at] = any ? static_cast<int>(s_carry[i].t) : -1;
  }
}

int slices_of(int V) { return (V - 1) / kTokens + 1; }

struct Scratch {
  Slice* slices;
  uint2* best;
  size_t bytes;
};
Scratch carve(void* ws, int B, int K, int V, int M) {
  Carver c(ws);
  Scratch s{};
  const size_t n = static_cast<size_t>(B) * K * slices_of(V);
  s.slices = static_cast<Slice*>(c.take(n * sizeof(Slice)));
  s.best = static_cast<uint2*>(c.take(n * M * sizeof(uint2)));
  s.bytes = c.used;
  return s;
}

int check(int B, int K, int V, int M) {
  if (B < 0 || K < 1 || V < 1 || M < 1 || M > kMost)
    return fail(PRNN_ERR_VALUE, "B=%d, K=%d, V=%d, M=%d: M must be in 1 .. %d", B, K, V, M, kMost);
  if (static_cast<long long>(K) * V >= 1ll << 31 || static_cast<long long>(B) * K >= 1ll << 31)
    return fail(PRNN_ERR_VALUE, "K=%d beams of V=%d tokens are more than 2^31 - 1", K, V);
  return PRNN_OK;
}

}  // namespace
}  // namespace prnn

using namespace prnn;

extern "C" PRNN_API size_t prnn_beam_select_workspace_size(int B, int K, int V, int M) {
  return check(B, K, V, M) ? 0 : carve(nullptr, B, K, V, M).bytes;
}

extern "C" PRNN_API int prnn_beam_select(const void* logits, long long l_sb, long long l_sk,
                                         const float* scores, const void* ended, int pad,
                                         float* out_scores, int* out_parents, int* out_tokens, int B,
                                         int K, int V, int M, int dtype, void* workspace, size_t bytes,
                                         void* stream) {
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check(B, K, V, M)) return rc;
  if (ended && (pad < 0 || pad >= V)) return fail(PRNN_ERR_VALUE, "pad=%d is no token of %d", pad, V);
  if (B == 0) return PRNN_OK;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens)
    return fail(PRNN_ERR_VALUE, "logits, scores and the outputs must be non-null");
  const Scratch s = carve(workspace, B, K, V, M);
  if (workspace == nullptr || bytes < s.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(PRNN_ERR_VALUE, "the workspace must hold %zu bytes, 256-byte aligned (got %zu)", s.bytes, bytes);
  const BeamArgs a{logits, l_sb, l_sk, scores, static_cast<const uint8_t*>(ended), s.slices, s.best,
                   out_scores, out_parents, out_tokens, B, K, V, M, slices_of(V), pad};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const long long groups = static_cast<long long>(B) * K * a.S;
  if (int rc = check_grid("beam_select", groups, 256)) return rc;
  return with_storage(dtype, [&](auto z) {
    using T = decltype(z);
    if (M <= 16)
      beam_slice_kernel<T, 16><<<static_cast<unsigned>(groups), 256, 0, st>>>(a);
    else if (M <= kFew)
      beam_slice_kernel<T, kFew><<<static_cast<unsigned>(groups), 256, 0, st>>>(a);
    else
      beam_slice_kernel<T, kMost><<<static_cast<unsigned>(groups), 256, 0, st>>>(a);
    PRNN_HIP(hipGetLastError());
    beam_choose_kernel<<<B, 256, 0, st>>>(a);
    PRNN_HIP(hipGetLastError());
    return static_cast<int>(PRNN_OK);
  });
}
