// Group norm, channels last, with an activation or a gate:
//
//   h = (x - mean) rstd,  z = w h + b,   y = act(z)   or   y = z act(gate)
//
// with mean and rstd = (var + eps)^(-1/2) over a group of channels of one token, or over all
// tokens of a sample.  Backward, with dz = dy act'(z) (gate: dy act(gate)), dh = w dz and the
// means m1 = <dh>, m2 = <dh h> over the same elements:
//
//   dx = rstd (dh - m1 - h m2),  dw = sum dz h,  db = sum dz,  dgate = dy z act'(gate).
//
// Bound by memory: a token's group sits in a few lanes' registers, so the statistics, the
// normalisation and in the backward pass all sums over the group come from one read of the
// arrays.  The parameters' sums are kept per thread (a thread's channels stay the same from row
// to row), then per workgroup, and are added up in a fixed order by a second kernel.
//
// Statistics and sums are fp32: two passes over registers for a token, running means and squared
// deviations (joined by their exact combination rule) for a sample.
#include <algorithm>

#include "prnn_host.h"

namespace prnn {
namespace {

enum { kActNone = 0, kActSilu = 1, kActSigmoid = 2 };

struct NormArgs {
  const void *x, *w, *b, *gate, *gy;
  void *y, *dx, *dgate;
  float* stats;      // (N, G) mean, rstd (tokens: where wanted)
  float* part;       // partial sums, see the kernels
  float* part2;
  size_t rows;       // tokens (token kernels)
  int N, L, C, G, Cg;
  int act, w_f32;    // w and b are float32
  int w_vec;         // and lie on 16-byte boundaries
  int lanes;         // lanes of a group: a power of two
  int strips, strip_rows;
  float eps;
};

__device__ __forceinline__ float act_of(int act, float z) {
  if (act == kActNone) return z;
  const float s = fsigmoid(z);
  return act == kActSilu ? z * s : s;
}
// act(z) and act'(z)
__device__ __forceinline__ void act_grad(int act, float z, float& f, float& d) {
  if (act == kActNone) {
    f = z;
    d = 1.0f;
    return;
  }
  const float s = fsigmoid(z);
  // 1 - s as a sigmoid of its own: no cancellation for large z
  const float c = fsigmoid(-z);
  if (act == kActSilu) {
    f = z * s;
    d = s * fmaf(z, c, 1.0f);
  } else {
    f = s;
    d = s * c;
  }
}

// V consecutive elements (V * sizeof(T) bytes, aligned) as floats.
template <typename T, int V>
__device__ __forceinline__ void loadv(const T* p, float* v) {
  if constexpr (V == 1) {
    v[0] = to_f32(*p);
  } else if constexpr (sizeof(T) == 4) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    static_assert(V == 4, "");
    const f4 q = *reinterpret_cast<const f4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q[i];
  } else if constexpr (V == 2) {
    const uint32_t q = *reinterpret_cast<const uint32_t*>(p);
    v[0] = Narrow<T>::lo(q);
    v[1] = Narrow<T>::hi(q);
  } else {
    static_assert(V == 8, "");
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = Narrow<T>::lo(w[i]);
      v[2 * i + 1] = Narrow<T>::hi(w[i]);
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void storev(T* p, const float* v) {
  if constexpr (V == 1) {
    *p = from_f32<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<f4*>(p) = f4{v[0], v[1], v[2], v[3]};
  } else if constexpr (V == 2) {
    *reinterpret_cast<uint32_t*>(p) = Narrow<T>::pack(v[0], v[1]);
  } else {
    *reinterpret_cast<uint4*>(p) = uint4{Narrow<T>::pack(v[0], v[1]), Narrow<T>::pack(v[2], v[3]),
                                         Narrow<T>::pack(v[4], v[5]), Narrow<T>::pack(v[6], v[7])};
  }
}

template <typename T>
__device__ __forceinline__ float param(const void* p, int f32, int c, float none) {
  if (p == nullptr) return none;
  return f32 ? static_cast<const float*>(p)[c] : to_f32(static_cast<const T*>(p)[c]);
}

// V consecutive parameters; c is a multiple of V, so where x's channels admit vectors and the
// parameters' rows lie alike (vec) these do too.
template <typename T, int V>
__device__ __forceinline__ void params(const void* p, int f32, int vec, int c, float none,
                                       float* v) {
  if (p != nullptr && vec) {
    if (!f32) {
      loadv<T, V>(static_cast<const T*>(p) + c, v);
      return;
    }
    if constexpr (V >= 4) {
#pragma unroll
      for (int i = 0; i < V; i += 4) loadv<float, 4>(static_cast<const float*>(p) + c + i, v + i);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = param<T>(p, f32, c + i, none);
}

// Sum over the `lanes` lanes of a group (a power of two; every lane gets it).
__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int k = 1; k < lanes; k <<= 1) v += __shfl_xor(v, k);
  return v;
}

// ---- statistics per token ----------------------------------------------------------------
// Lanes are laid over a row's groups, `lanes` to a group, K vectors of V channels to a lane
// (vector k of lane l: channels (k lanes + l) V); lanes behind a group's end idle.  Where a row
// takes fewer than 256 lanes a workgroup works on several rows at a time.

struct TokenPlace {
  int row, rows_per, group, l;
  bool on;
};
__device__ __forceinline__ TokenPlace token_place(const NormArgs& A) {
  const int per_row = A.G * A.lanes;
  TokenPlace p;
  int u;
  if (per_row <= 256) {
    p.rows_per = 256 / per_row;
    p.row = threadIdx.x / per_row;
    u = threadIdx.x - p.row * per_row;
    p.on = p.row < p.rows_per;
  } else {
    p.rows_per = 1;
    p.row = 0;
    u = blockIdx.y * 256 + threadIdx.x;
    p.on = u < per_row;
  }
  p.group = u / A.lanes;
  p.l = u - p.group * A.lanes;
  return p;
}

// 16384 tokens of 1024 bf16 channels in 16 groups with a gate: 20.3 us, 4.96 TB/s (a large copy:
// 5.14); 32 tokens 4.0 us, a launch's own time.
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void norm_token_kernel(NormArgs A) {
  const TokenPlace p = token_place(A);
  const float inv = 1.0f / A.Cg;
  float w[K][V], b[K][V];
  bool in[K];
  int ch[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * A.lanes + p.l) * V;
    in[k] = p.on && c < A.Cg;
    ch[k] = in[k] ? p.group * A.Cg + c : 0;
    params<T, V>(A.w, A.w_f32, A.w_vec, ch[k], 1.0f, w[k]);
    params<T, V>(A.b, A.w_f32, A.w_vec, ch[k], 0.0f, b[k]);
  }
  // all lanes of a wave stay in the loop: the sums are shuffles
  for (size_t r0 = static_cast<size_t>(blockIdx.x) * p.rows_per; r0 < A.rows;
       r0 += static_cast<size_t>(gridDim.x) * p.rows_per) {
    const size_t row = r0 + p.row;
    const bool live = p.on && row < A.rows;
    const size_t at = row * A.C;
    float x[K][V], g[K][V], s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool go = live && in[k];
      if (go) {
        loadv<T, V>(static_cast<const T*>(A.x) + at + ch[k], x[k]);
        if (A.gate) loadv<T, V>(static_cast<const T*>(A.gate) + at + ch[k], g[k]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!go) x[k][i] = g[k][i] = 0.0f;
        s += x[k][i];
      }
    }
    const float mean = group_sum(s, A.lanes) * inv;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = in[k] ? x[k][i] - mean : 0.0f;
        s = fmaf(d, d, s);
      }
    const float rstd = 1.0f / sqrtf(fmaf(group_sum(s, A.lanes), inv, A.eps));
    if (A.stats && live && p.l == 0) {
      float* st = A.stats + 2 * (row * A.G + p.group);
      st[0] = mean;
      st[1] = rstd;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!(live && in[k])) continue;
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = fmaf(w[k][i], (x[k][i] - mean) * rstd, b[k][i]);
        y[i] = A.gate ? z * act_of(A.act, g[k][i]) : act_of(A.act, z);
      }
      storev<T, V>(static_cast<T*>(A.y) + at + ch[k], y);
    }
  }
}

// part: [gridDim.x][2][C] sums of dz h and dz.  The same 16384 tokens: 38.4 us, 4.4 TB/s, and 4.1 us
// for the parameters' sums.
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void norm_token_bwd_kernel(NormArgs A) {
  __shared__ float red[256];
  const TokenPlace p = token_place(A);
  const float inv = 1.0f / A.Cg;
  float w[K][V], b[K][V], dw[K][V], db[K][V];
  bool in[K];
  int ch[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * A.lanes + p.l) * V;
    in[k] = p.on && c < A.Cg;
    ch[k] = in[k] ? p.group * A.Cg + c : 0;
    params<T, V>(A.w, A.w_f32, A.w_vec, ch[k], 1.0f, w[k]);
    params<T, V>(A.b, A.w_f32, A.w_vec, ch[k], 0.0f, b[k]);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.0f;
  }
  for (size_t r0 = static_cast<size_t>(blockIdx.x) * p.rows_per; r0 < A.rows;
       r0 += static_cast<size_t>(gridDim.x) * p.rows_per) {
    const size_t row = r0 + p.row;
    const bool live = p.on && row < A.rows;
    const size_t at = row * A.C;
    float x[K][V], g[K][V], dz[K][V], s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool go = live && in[k];
      if (go) {
        loadv<T, V>(static_cast<const T*>(A.x) + at + ch[k], x[k]);
        loadv<T, V>(static_cast<const T*>(A.gy) + at + ch[k], dz[k]);
        if (A.gate) loadv<T, V>(static_cast<const T*>(A.gate) + at + ch[k], g[k]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!go) x[k][i] = g[k][i] = dz[k][i] = 0.0f;
        s += x[k][i];
      }
    }
    const float mean = group_sum(s, A.lanes) * inv;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = in[k] ? x[k][i] - mean : 0.0f;
        s = fmaf(d, d, s);
      }
    const float rstd = 1.0f / sqrtf(fmaf(group_sum(s, A.lanes), inv, A.eps));
    float m1 = 0.0f, m2 = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool go = live && in[k];
      float dg[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float h = go ? (x[k][i] - mean) * rstd : 0.0f;
        const float z = fmaf(w[k][i], h, b[k][i]);
        float f, d;
        act_grad(A.act, A.gate ? g[k][i] : z, f, d);
        if (A.gate) {
          dg[i] = dz[k][i] * z * d;
          dz[k][i] *= f;
        } else {
          dz[k][i] *= d;
        }
        x[k][i] = h;
        if (go) {  // an idle lane adds nothing, whatever act gives there
          dw[k][i] = fmaf(dz[k][i], h, dw[k][i]);
          db[k][i] += dz[k][i];
          const float dh = w[k][i] * dz[k][i];
          m1 += dh;
          m2 = fmaf(dh, h, m2);
        }
      }
      if (go && A.gate) storev<T, V>(static_cast<T*>(A.dgate) + at + ch[k], dg);
    }
    m1 = group_sum(m1, A.lanes) * inv;
    m2 = group_sum(m2, A.lanes) * inv;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!(live && in[k])) continue;
      float dx[V];
#pragma unroll
      for (int i = 0; i < V; ++i)
        dx[i] = rstd * (fmaf(w[k][i], dz[k][i], -m1) - x[k][i] * m2);
      storev<T, V>(static_cast<T*>(A.dx) + at + ch[k], dx);
    }
  }
  // the workgroup's rows, in their order
  const int per_row = A.G * A.lanes;
  float* out = A.part + static_cast<size_t>(blockIdx.x) * 2 * A.C;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const float mine = which ? db[k][i] : dw[k][i];
        float sum = mine;
        if (p.rows_per > 1) {
          __syncthreads();
          red[threadIdx.x] = mine;
          __syncthreads();
          if (p.row == 0)
            for (int r = 1; r < p.rows_per; ++r) sum += red[r * per_row + threadIdx.x];
        }
        if (p.row == 0 && in[k]) out[which * A.C + ch[k] + i] = sum;
      }
}

// dw and db from partial sums [parts][2][C]: 32 channels a workgroup, 32 lanes to a channel, each
// with 8 loads under way.  A thousand partial sums of 1024 channels: 4.1 us, 8 MB.
template <typename T>
__global__ __launch_bounds__(1024) void norm_param_kernel(const float* __restrict__ part, int parts,
                                                          int C, void* dw, void* db, int f32) {
  __shared__ float red[32][33];
  const int l = threadIdx.x & 31, sub = threadIdx.x >> 5, c = blockIdx.x * 32 + l;
  const int which = blockIdx.y;
  float s = 0.0f;
  if (c < C) {
    const float* p = part + static_cast<size_t>(which) * C + c;
    for (int k = sub; k < parts; k += 256) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = k + 32 * i < parts ? p[static_cast<size_t>(k + 32 * i) * 2 * C] : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
  }
  red[sub][l] = s;
  __syncthreads();
  void* out = which ? db : dw;
  if (sub == 0 && c < C && out) {
    for (int k = 1; k < 32; ++k) s += red[k][l];
    if (f32)
      static_cast<float*>(out)[c] = s;
    else
      static_cast<T*>(out)[c] = from_f32<T>(s);
  }
}

// ---- statistics per sample ---------------------------------------------------------------
// A sample (L tokens) is cut into strips of rows, one workgroup each.  Threads lie over the
// channels, V to a thread, and over as many rows at a time as fit.  8 x 2047 tokens of 256 fp32
// channels in 32 groups (16.8 MB an array): statistics 7.7 us, y 9.2, sums 9.9, dx 14.1,
// parameters 4.0: each a few dependent rounds of rows behind a launch, 2.2 to 3.6 TB/s.  Samples of
// 16384 tokens: 35 for the statistics (one array), y 45 (two), sums 54 (two), dx 68 (three), 3.9 to
// 6.0 TB/s with what the last-level cache still holds.

// Groups of a sample whose sums every workgroup forms itself.  A training step of 8 x 2047 tokens of
// 256 fp32 channels: 42 us against 45 with launches of their own for 32 groups, 40 against 48 for 16, and with 64 groups
// (before both got faster) 61 against 56.
constexpr int kJoinGroups = 32;
constexpr int kRows = 4;         // rows of a thread under way at a time

struct SamplePlace {
  int slots, rows_per, row, slot;
  bool on;
};
template <int V>
__device__ __forceinline__ SamplePlace sample_place(const NormArgs& A) {
  SamplePlace p;
  p.slots = A.C / V;
  if (p.slots <= 256) {
    p.rows_per = 256 / p.slots;
    p.row = threadIdx.x / p.slots;
    p.slot = threadIdx.x - p.row * p.slots;
    p.on = p.row < p.rows_per;
  } else {
    p.rows_per = 1;
    p.row = 0;
    p.slot = threadIdx.x;
    p.on = true;
  }
  return p;
}

// Rows of a strip: unsigned, so that a step behind the last of 2^31 - 1 does not wrap.
__device__ __forceinline__ unsigned strip_begin(const NormArgs& A, int strip) {
  return static_cast<unsigned>(strip) * A.strip_rows;
}
__device__ __forceinline__ unsigned strip_end(const NormArgs& A, unsigned begin) {
  return min(static_cast<unsigned>(A.L), begin + A.strip_rows);
}

// Sum over a workgroup of 256 (every thread gets it).
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) v += __shfl_xor(v, k);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// Lanes of a sum over `items` values: a power of two.
__device__ __forceinline__ int lanes_for(int items) {
  int lanes = 1;
  while (lanes < 64 && lanes < items) lanes <<= 1;
  return lanes;
}

// Statistics of strip `strip` of sample n, one group after another of those in the workgroup's
// share: mean and squared deviations per thread and channel, then joined per group.
// part: [N][strips][G][2].
template <typename T, int V>
__global__ __launch_bounds__(256) void norm_sample_stats_kernel(NormArgs A) {
  extern __shared__ float lds[];  // [256][2 V] mean and squared deviations per thread
  const int n = blockIdx.x / A.strips, strip = blockIdx.x - n * A.strips;
  const SamplePlace p = sample_place<V>(A);
  const unsigned l0 = strip_begin(A, strip), l1 = strip_end(A, l0);
  const T* x = static_cast<const T*>(A.x) + static_cast<size_t>(n) * A.L * A.C;
  float* out = A.part + (static_cast<size_t>(n) * A.strips + strip) * A.G * 2;
  // slots beyond 256 in rounds, a whole number of groups each
  const int per_group = A.Cg / V;
  const int groups_round = p.slots <= 256 ? A.G : max(1, 256 / per_group);
  for (int g0 = 0; g0 < A.G; g0 += groups_round) {
    const int gn = min(groups_round, A.G - g0);
    if (p.slots > 256 && per_group > 256) {
      // a group wider than the workgroup: its channels in turns, two passes over the strip
      const size_t c0 = static_cast<size_t>(g0) * A.Cg;
      float s = 0.0f;
      for (unsigned l = l0; l < l1; ++l)
        for (int u = threadIdx.x; u < per_group; u += 256) {
          float v[V];
          loadv<T, V>(x + static_cast<size_t>(l) * A.C + c0 + u * V, v);
#pragma unroll
          for (int i = 0; i < V; ++i) s += v[i];
        }
      const float cnt = static_cast<float>(l1 - l0) * A.Cg;
      const float mean = block_sum(s, lds) / cnt;
      s = 0.0f;
      for (unsigned l = l0; l < l1; ++l)
        for (int u = threadIdx.x; u < per_group; u += 256) {
          float v[V];
          loadv<T, V>(x + static_cast<size_t>(l) * A.C + c0 + u * V, v);
#pragma unroll
          for (int i = 0; i < V; ++i) s = fmaf(v[i] - mean, v[i] - mean, s);
        }
      s = block_sum(s, lds);
      if (threadIdx.x == 0) {
        out[2 * g0] = mean;
        out[2 * g0 + 1] = s;
      }
      __syncthreads();
      continue;
    }
    const int slot = p.slots <= 256 ? p.slot : g0 * per_group + threadIdx.x;
    const bool on = p.slots <= 256 ? p.on : threadIdx.x < static_cast<unsigned>(gn * per_group);
    float mean[V], m2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.0f;
    float cnt = 0.0f;
    if (on)
      for (unsigned l = l0 + p.row; l < l1; l += 2 * kRows * p.rows_per) {
        // one array alone: twice the rows for as many bytes under way
        float v[2 * kRows][V];
#pragma unroll
        for (int k = 0; k < 2 * kRows; ++k)
          loadv<T, V>(x + static_cast<size_t>(min(l + k * p.rows_per, l1 - 1)) * A.C + slot * V, v[k]);
#pragma unroll
        for (int k = 0; k < 2 * kRows; ++k) {
          if (l + k * p.rows_per >= l1) break;
          cnt += 1.0f;
          const float inv = frcp(cnt);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float d = v[k][i] - mean[i];
            mean[i] = fmaf(d, inv, mean[i]);
            m2[i] = fmaf(d, v[k][i] - mean[i], m2[i]);
          }
        }
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      lds[threadIdx.x * 2 * V + 2 * i] = mean[i];
      lds[threadIdx.x * 2 * V + 2 * i + 1] = m2[i];
    }
    __syncthreads();
    // some lanes per group: the mean of the means, then the deviations from it
    const int items = per_group * p.rows_per, lanes = lanes_for(items);
    const int lane = threadIdx.x & (lanes - 1);
    const int n_rows = l1 - l0;
    const float total = static_cast<float>(n_rows) * A.Cg;
    for (int at = 0; at < gn; at += 256 / lanes) {
      const int g = at + threadIdx.x / lanes, n_items = g < gn ? items : 0;
      float s = 0.0f;
      for (int it = lane; it < n_items; it += lanes) {
        const int r = it / per_group, u = g * per_group + it - r * per_group;
        const float c = static_cast<float>((n_rows - r + p.rows_per - 1) / p.rows_per);
        const float* e = &lds[(r * (p.slots <= 256 ? p.slots : 0) + u) * 2 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) s = fmaf(c, e[2 * i], s);
      }
      for (int k = 1; k < lanes; k <<= 1) s += __shfl_xor(s, k);
      const float gm = s / total;
      s = 0.0f;
      for (int it = lane; it < n_items; it += lanes) {
        const int r = it / per_group, u = g * per_group + it - r * per_group;
        const float c = static_cast<float>((n_rows - r + p.rows_per - 1) / p.rows_per);
        const float* e = &lds[(r * (p.slots <= 256 ? p.slots : 0) + u) * 2 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = e[2 * i] - gm;
          s += fmaf(c * d, d, e[2 * i + 1]);
        }
      }
      for (int k = 1; k < lanes; k <<= 1) s += __shfl_xor(s, k);
      if (lane == 0 && g < gn) {
        out[2 * (g0 + g)] = gm;
        out[2 * (g0 + g) + 1] = s;
      }
    }
  }
}

// Mean and rstd of a (sample, group) from its strips, by the 8 lanes of a thread's share.
__device__ __forceinline__ double sum_8(double v) {
#pragma unroll
  for (int k = 1; k < 8; k <<= 1) v += __shfl_xor(v, k);
  return v;
}
__device__ __forceinline__ void join_group(const NormArgs& A, int n, int g, bool on,
                                           float& mean_out, float& rstd_out) {
  const float2* e = reinterpret_cast<const float2*>(A.part) + static_cast<size_t>(n) * A.strips * A.G + g;
  const int strips = on ? A.strips : 0, sub = threadIdx.x & 7;
  // sums of means and of squares in fp64: one pass, 8 strips a lane under way
  double s1 = 0.0, s2 = 0.0;
  for (int k0 = sub; k0 < strips; k0 += 64) {
    float2 v[8];  // mean, squared deviations
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = k0 + 8 * i;
      v[i] = float2{0.0f, 0.0f};
      if (k < strips) v[i] = e[static_cast<size_t>(k) * A.G];
      c[i] = k < strips ? static_cast<float>(min(A.strip_rows, A.L - k * A.strip_rows)) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double m = v[i].x, cm = c[i] * m;
      s1 += cm;
      s2 += v[i].y + cm * m * A.Cg;
    }
  }
  const double mean = sum_8(s1) / A.L;
  const double var = sum_8(s2) / (static_cast<double>(A.L) * A.Cg) - mean * mean;
  mean_out = static_cast<float>(mean);
  rstd_out = static_cast<float>(1.0 / sqrt((var > 0.0 ? var : var == var ? 0.0 : var) + A.eps));
}

// The same for every (sample, group): 32 a workgroup.
__global__ __launch_bounds__(256) void norm_sample_join_kernel(NormArgs A) {
  const long long id = static_cast<long long>(blockIdx.x) * 32 + (threadIdx.x >> 3);
  const bool on = id < static_cast<long long>(A.N) * A.G;
  const int n = on ? static_cast<int>(id / A.G) : 0;
  const int g = on ? static_cast<int>(id - static_cast<long long>(n) * A.G) : 0;
  float mean, rstd;
  join_group(A, n, g, on, mean, rstd);
  if (on && (threadIdx.x & 7) == 0) {
    A.stats[2 * id] = mean;
    A.stats[2 * id + 1] = rstd;
  }
}

// y of a strip.  JOIN: every workgroup forms its sample's statistics from the strips' itself (the
// first one keeps them for the backward pass): with few groups that is cheaper than a launch.
template <typename T, int V, bool JOIN>
__global__ __launch_bounds__(256) void norm_sample_apply_kernel(NormArgs A) {
  __shared__ float s_stats[JOIN ? 2 * kJoinGroups : 2];
  const int n = blockIdx.x / A.strips, strip = blockIdx.x - n * A.strips;
  const SamplePlace p = sample_place<V>(A);
  if (JOIN) {
    for (int g0 = 0; g0 < A.G; g0 += 32) {
      const int g = g0 + (threadIdx.x >> 3);
      const bool on = g < A.G;
      float mean, rstd;
      join_group(A, n, on ? g : 0, on, mean, rstd);
      if (on && (threadIdx.x & 7) == 0) {
        s_stats[2 * g] = mean;
        s_stats[2 * g + 1] = rstd;
        if (strip == 0) {
          A.stats[2 * (static_cast<size_t>(n) * A.G + g)] = mean;
          A.stats[2 * (static_cast<size_t>(n) * A.G + g) + 1] = rstd;
        }
      }
    }
    __syncthreads();
  }
  const unsigned l0 = strip_begin(A, strip), l1 = strip_end(A, l0);
  const size_t base = static_cast<size_t>(n) * A.L * A.C;
  if (!p.on) return;
  for (int slot = p.slot; slot < p.slots; slot += 256) {
    const int c = slot * V, g = c / A.Cg;
    const float* st = JOIN ? &s_stats[2 * g] : &A.stats[2 * (static_cast<size_t>(n) * A.G + g)];
    const float mean = st[0], rstd = st[1];
    float w[V], b[V];
    params<T, V>(A.w, A.w_f32, A.w_vec, c, 1.0f, w);
    params<T, V>(A.b, A.w_f32, A.w_vec, c, 0.0f, b);
    // kRows rows under way at a time
    for (unsigned l = l0 + p.row; l < l1; l += kRows * p.rows_per) {
      float x[kRows][V], gt[kRows][V];
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const unsigned r = min(l + k * p.rows_per, l1 - 1);
        const size_t at = base + static_cast<size_t>(r) * A.C + c;
        loadv<T, V>(static_cast<const T*>(A.x) + at, x[k]);
        if (A.gate) loadv<T, V>(static_cast<const T*>(A.gate) + at, gt[k]);
      }
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        if (l + k * p.rows_per >= l1) break;
        const size_t at = base + static_cast<size_t>(l + k * p.rows_per) * A.C + c;
        float y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float z = fmaf(w[i], (x[k][i] - mean) * rstd, b[i]);
          y[i] = A.gate ? z * act_of(A.act, gt[k][i]) : act_of(A.act, z);
        }
        storev<T, V>(static_cast<T*>(A.y) + at, y);
      }
    }
    if (p.slots <= 256) break;
  }
}

// Sums of dz h and dz of a strip per channel: part [N * strips][2][C]; dgate on the way.  JOIN
// (all channels in the workgroup at once): also those of dh h and dh per group, part2
// [N * strips][2][G].
template <typename T, int V, bool JOIN>
__global__ __launch_bounds__(256) void norm_sample_bwd_sums_kernel(NormArgs A) {
  __shared__ float red[2 * V][256];
  __shared__ float s_ch[JOIN ? 2 * 256 * V : 2];
  const int n = blockIdx.x / A.strips, strip = blockIdx.x - n * A.strips;
  const SamplePlace p = sample_place<V>(A);
  const unsigned l0 = strip_begin(A, strip), l1 = strip_end(A, l0);
  const size_t base = static_cast<size_t>(n) * A.L * A.C;
  float* out = A.part + (static_cast<size_t>(n) * A.strips + strip) * 2 * A.C;
  for (int s0 = 0; s0 < p.slots; s0 += 256) {
    const int slot = p.slot + s0;
    const bool on = p.on && slot < p.slots;
    const int c = on ? slot * V : 0, g = c / A.Cg;
    const float mean = A.stats[2 * (static_cast<size_t>(n) * A.G + g)];
    const float rstd = A.stats[2 * (static_cast<size_t>(n) * A.G + g) + 1];
    float w[V], b[V], dw[V], db[V];
    params<T, V>(A.w, A.w_f32, A.w_vec, c, 1.0f, w);
    params<T, V>(A.b, A.w_f32, A.w_vec, c, 0.0f, b);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[i] = db[i] = 0.0f;
    if (on)
      for (unsigned l = l0 + p.row; l < l1; l += kRows * p.rows_per) {
        float xs[kRows][V], gs[kRows][V], ys[kRows][V];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
          const unsigned r = min(l + k * p.rows_per, l1 - 1);
          const size_t at = base + static_cast<size_t>(r) * A.C + c;
          loadv<T, V>(static_cast<const T*>(A.x) + at, xs[k]);
          loadv<T, V>(static_cast<const T*>(A.gy) + at, ys[k]);
          if (A.gate) loadv<T, V>(static_cast<const T*>(A.gate) + at, gs[k]);
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
          if (l + k * p.rows_per >= l1) break;
          const size_t at = base + static_cast<size_t>(l + k * p.rows_per) * A.C + c;
          float *x = xs[k], *gt = gs[k], *dz = ys[k];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float h = (x[i] - mean) * rstd, z = fmaf(w[i], h, b[i]);
            float f, d;
            act_grad(A.act, A.gate ? gt[i] : z, f, d);
            if (A.gate) {
              gt[i] = dz[i] * z * d;
              dz[i] *= f;
            } else {
              dz[i] *= d;
            }
            dw[i] = fmaf(dz[i], h, dw[i]);
            db[i] += dz[i];
          }
          if (A.gate) storev<T, V>(static_cast<T*>(A.dgate) + at, gt);
        }
      }
    if (p.rows_per > 1) {  // all slots at once: one round
#pragma unroll
      for (int i = 0; i < V; ++i) {
        red[i][threadIdx.x] = dw[i];
        red[V + i][threadIdx.x] = db[i];
      }
      __syncthreads();
      if (p.row == 0)
        for (int r = 1; r < p.rows_per; ++r)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            dw[i] += red[i][r * p.slots + threadIdx.x];
            db[i] += red[V + i][r * p.slots + threadIdx.x];
          }
    }
    if (p.row == 0 && on)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        out[c + i] = dw[i];
        out[A.C + c + i] = db[i];
        if (JOIN) {
          s_ch[c + i] = w[i] * dw[i];
          s_ch[256 * V + c + i] = w[i] * db[i];
        }
      }
    if (JOIN) {
      __syncthreads();
      const int lanes = lanes_for(A.Cg), lane = threadIdx.x & (lanes - 1);
      for (int at = 0; at < 2 * A.G; at += 256 / lanes) {
        const int k = at + threadIdx.x / lanes, which = k / A.G, gg = k - which * A.G;
        float sum = 0.0f;
        if (k < 2 * A.G)
          for (int i = lane; i < A.Cg; i += lanes) sum += s_ch[which * 256 * V + gg * A.Cg + i];
        for (int s = 1; s < lanes; s <<= 1) sum += __shfl_xor(sum, s);
        if (k < 2 * A.G && lane == 0)
          A.part2[(static_cast<size_t>(n) * A.strips + strip) * 2 * A.G + k] = sum;
      }
    }
  }
}

// m1 and m2 of a (sample, group), part2 [N][G][2], from the strips' sums per channel: lanes over
// the group's channels and as many strips at a time as fit, 4 of them under way.
template <typename T>
__global__ __launch_bounds__(1024) void norm_sample_means_kernel(NormArgs A) {
  __shared__ double red[2][16];
  const int id = blockIdx.x, n = id / A.G, g = id - n * A.G;
  const float* e = A.part + static_cast<size_t>(n) * A.strips * 2 * A.C + g * A.Cg;
  int lanes = 1;
  while (lanes < static_cast<int>(blockDim.x) && lanes < A.Cg) lanes <<= 1;
  const int k0 = threadIdx.x / lanes, step = blockDim.x / lanes;
  double m1 = 0.0, m2 = 0.0;
  for (int c = threadIdx.x - k0 * lanes; c < A.Cg; c += lanes) {
    const float w = param<T>(A.w, A.w_f32, g * A.Cg + c, 1.0f);
    double s1 = 0.0, s2 = 0.0;
    for (int k = k0; k < A.strips; k += 4 * step) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kk = min(k + i * step, A.strips - 1);
        a[i] = e[static_cast<size_t>(kk) * 2 * A.C + c];
        b[i] = e[static_cast<size_t>(kk) * 2 * A.C + A.C + c];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k + i * step < A.strips) {
          s2 += a[i];
          s1 += b[i];
        }
    }
    m2 += w * s2;
    m1 += w * s1;
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    m1 += __shfl_xor(m1, k);
    m2 += __shfl_xor(m2, k);
  }
  if ((threadIdx.x & 63) == 0) {
    red[0][threadIdx.x >> 6] = m1;
    red[1][threadIdx.x >> 6] = m2;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < static_cast<int>(blockDim.x) / 64; ++k) {
      m1 += red[0][k];
      m2 += red[1][k];
    }
    const double inv = 1.0 / (static_cast<double>(A.L) * A.Cg);
    A.part2[2 * static_cast<size_t>(id)] = static_cast<float>(m1 * inv);
    A.part2[2 * static_cast<size_t>(id) + 1] = static_cast<float>(m2 * inv);
  }
}

// dx of a strip.  JOIN: m1 and m2 of the sample's groups from the strips' sums, in every workgroup.
template <typename T, int V, bool JOIN>
__global__ __launch_bounds__(256) void norm_sample_dx_kernel(NormArgs A) {
  __shared__ float s_m[JOIN ? 2 * kJoinGroups : 2];
  const int n = blockIdx.x / A.strips, strip = blockIdx.x - n * A.strips;
  const SamplePlace p = sample_place<V>(A);
  if (JOIN) {
    for (int k0 = 0; k0 < 2 * A.G; k0 += 32) {
      const int k = k0 + (threadIdx.x >> 3);
      const int strips = k < 2 * A.G ? A.strips : 0;
      double s = 0.0;
      for (int i0 = threadIdx.x & 7; i0 < strips; i0 += 64) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = i0 + 8 * j;
          v[j] = i < strips ? A.part2[(static_cast<size_t>(n) * A.strips + i) * 2 * A.G + k] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
      }
      s = sum_8(s);
      if (strips && (threadIdx.x & 7) == 0)
        s_m[k] = static_cast<float>(s / (static_cast<double>(A.L) * A.Cg));
    }
    __syncthreads();
  }
  const unsigned l0 = strip_begin(A, strip), l1 = strip_end(A, l0);
  const size_t base = static_cast<size_t>(n) * A.L * A.C;
  if (!p.on) return;
  for (int slot = p.slot; slot < p.slots; slot += 256) {
    const int c = slot * V, g = c / A.Cg;
    const size_t ng = static_cast<size_t>(n) * A.G + g;
    const float mean = A.stats[2 * ng], rstd = A.stats[2 * ng + 1];
    const float m1 = JOIN ? s_m[A.G + g] : A.part2[2 * ng], m2 = JOIN ? s_m[g] : A.part2[2 * ng + 1];
    float w[V], b[V];
    params<T, V>(A.w, A.w_f32, A.w_vec, c, 1.0f, w);
    params<T, V>(A.b, A.w_f32, A.w_vec, c, 0.0f, b);
    for (unsigned l = l0 + p.row; l < l1; l += kRows * p.rows_per) {
      float xs[kRows][V], gs[kRows][V], ys[kRows][V];
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const unsigned r = min(l + k * p.rows_per, l1 - 1);
        const size_t at = base + static_cast<size_t>(r) * A.C + c;
        loadv<T, V>(static_cast<const T*>(A.x) + at, xs[k]);
        loadv<T, V>(static_cast<const T*>(A.gy) + at, ys[k]);
        if (A.gate) loadv<T, V>(static_cast<const T*>(A.gate) + at, gs[k]);
      }
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        if (l + k * p.rows_per >= l1) break;
        const size_t at = base + static_cast<size_t>(l + k * p.rows_per) * A.C + c;
        float *x = xs[k], *gt = gs[k], *dz = ys[k];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float h = (x[i] - mean) * rstd, z = fmaf(w[i], h, b[i]);
          if (A.gate) {
            dz[i] *= act_of(A.act, gt[i]);
          } else {
            float f, d;
            act_grad(A.act, z, f, d);
            dz[i] *= d;
          }
          x[i] = rstd * (fmaf(w[i], dz[i], -m1) - h * m2);
        }
        storev<T, V>(static_cast<T*>(A.dx) + at, x);
      }
    }
    if (p.slots <= 256) break;
  }
}

// ---- host ----------------------------------------------------------------------------------

struct Plan {
  bool token;
  int V, K, lanes;       // token kernels
  int blocks_x, blocks_y;
  int strips, strip_rows;
};

// Elements of a 16-byte access; 2 where 16-bit channels come in pairs only; else 1.
int vector_of(int dtype, int Cg, uintptr_t bits) {
  const int size = dtype == PRNN_F32 ? 4 : 2;
  const int v = 16 / size;
  if (Cg % v == 0 && (bits & 15) == 0) return v;
  if (size == 2 && Cg % 2 == 0 && (bits & 3) == 0) return 2;
  return 1;
}

Plan plan(int N, int L, int Cg, int G, int dtype, uintptr_t bits, bool backward) {
  Plan p{};
  p.V = vector_of(dtype, Cg, bits);
  // A token's group in one wave's registers: up to 64 lanes, 4 vectors each.
  if (L == 1 && Cg <= 256 * p.V) {
    p.token = true;
    const int vecs = (Cg + p.V - 1) / p.V;
    p.K = vecs <= 64 ? 1 : 4;
    p.lanes = 1;
    while (p.lanes * p.K < vecs) p.lanes <<= 1;
    const int per_row = G * p.lanes;
    const int rows_per = per_row <= 256 ? 256 / per_row : 1;
    p.blocks_y = (per_row + 255) / 256;
    const int need = static_cast<int>((1ll * N + rows_per - 1) / rows_per);
    // A workgroup reads its parameters once (backward: keeps their sums) and goes on from row to
    // row: about eight a CU forward, four backward, where a partial sum each is written.  A training
    // step of 16384 tokens of 1024 channels: 63 us, with half as many 70, with twice as many 67.
    const int most = std::max(1, (backward ? 1024 : 2048) / p.blocks_y);
    p.blocks_x = std::max(1, std::min(need, most));
    return p;
  }
  // strips: enough workgroups for the chip, each of at least kRows rounds of rows.  512 of them:
  // 42 us for a training step of 8 x 2047 tokens of 256 channels; 256: 45; 1024: 52.
  const int slots = G * Cg / p.V, rows_per = slots <= 256 ? 256 / slots : 1;
  const int want = std::max(1, 512 / std::max(1, N));
  p.strip_rows = std::max(static_cast<int>((1ll * L + want - 1) / want), kRows * rows_per);
  p.strips = static_cast<int>((1ll * L + p.strip_rows - 1) / p.strip_rows);
  return p;
}

template <typename F>
int with_vector(int V, F&& f) {
  if (V == 8) return f(std::integral_constant<int, 8>{});
  if (V == 4) return f(std::integral_constant<int, 4>{});
  if (V == 2) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 1>{});
}

// f(T, V) for the vectors that exist: 16 bytes, a pair of 16-bit elements, one element.
template <typename F>
int with_types(int dtype, int V, F&& f) {
  return with_storage(dtype, [&](auto z) {
    using T = decltype(z);
    return with_vector(V, [&](auto v) -> int {
      constexpr int n = decltype(v)::value;
      if constexpr (n == 1 || (sizeof(T) == 4 ? n == 4 : n == 8 || n == 2))
        return f(z, v);
      else
        return fail(PRNN_ERR_RUNTIME, "no vector of %d elements", n);
    });
  });
}

int check(const char* what, int N, int L, int C, int G, int act, int w_dtype, int dtype) {
  if (int rc = check_dtype(dtype)) return rc;
  if (w_dtype != PRNN_F32 && w_dtype != dtype)
    return fail(PRNN_ERR_TYPE, "%s: weight and bias must be float32 or of x's type", what);
  if (N < 0 || L < 0 || C < 1 || G < 1 || C % G)
    return fail(PRNN_ERR_VALUE, "%s: N=%d, L=%d, C=%d, groups=%d", what, N, L, C, G);
  if (act < 0 || act > 2) return fail(PRNN_ERR_VALUE, "%s: activation code %d", what, act);
  return PRNN_OK;
}

// The launches of statistics per sample.
int check_strips(const Plan& p, int N, int G) {
  if (p.token) return PRNN_OK;
  if (int rc = check_grid("group_norm", 1ll * p.strips * N, 256)) return rc;
  return check_grid("group_norm", 1ll * N * G, 64);  // (sample, group): a wave at least
}

uintptr_t bits_of(std::initializer_list<const void*> ps) {
  uintptr_t b = 0;
  for (const void* p : ps) b |= reinterpret_cast<uintptr_t>(p);
  return b;
}

}  // namespace
}  // namespace prnn

using namespace prnn;

extern "C" PRNN_API size_t prnn_group_norm_workspace_size(int N, int L, int C, int G, int dtype,
                                                          int backward) {
  if (N < 1 || L < 1 || C < 1 || G < 1 || C % G) return 0;
  const bool aligned = backward & 2;
  backward &= 1;
  // the largest over the alignments that a call may turn out to have
  size_t most = 0;
  for (uintptr_t bits : {uintptr_t{0}, uintptr_t{4}, uintptr_t{2}}) {
    if (bits && aligned) break;
    const Plan p = plan(N, L, C / G, G, dtype, bits, backward != 0);
    Carver c(nullptr);
    if (p.token) {
      if (backward) c.take(sizeof(float) * 2 * C * p.blocks_x);
    } else if (!backward) {
      c.take(sizeof(float) * 2 * G * p.strips * static_cast<size_t>(N));
    } else {
      c.take(sizeof(float) * 2 * C * p.strips * static_cast<size_t>(N));
      c.take(sizeof(float) * 2 * G * p.strips * static_cast<size_t>(N));
    }
    most = std::max(most, c.used);
  }
  return most;
}

extern "C" PRNN_API int prnn_group_norm(const void* x, const void* w, const void* b,
                                        const void* gate, void* y, float* stats, int N, int L,
                                        int C, int G, float eps, int act, int w_dtype, int dtype,
                                        void* workspace, size_t bytes, void* stream) {
  if (int rc = check("group_norm", N, L, C, G, act, w_dtype, dtype)) return rc;
  if (N == 0 || L == 0) return PRNN_OK;
  if (!x || !y) return fail(PRNN_ERR_VALUE, "group_norm: x and y must be non-null");
  const Plan p = plan(N, L, C / G, G, dtype, bits_of({x, y, gate}), false);
  if (int rc = check_strips(p, N, G)) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  NormArgs a{};
  a.x = x;
  a.w = w;
  a.b = b;
  a.gate = gate;
  a.y = y;
  a.stats = stats;
  a.rows = N;
  a.N = N;
  a.L = L;
  a.C = C;
  a.G = G;
  a.Cg = C / G;
  a.act = act;
  a.w_f32 = w_dtype == PRNN_F32;
  a.w_vec = (bits_of({w, b}) & 15) == 0;
  a.lanes = p.lanes;
  a.strips = p.strips;
  a.strip_rows = p.strip_rows;
  a.eps = eps;
  if (p.token)
    return with_types(dtype, p.V, [&](auto z, auto v) {
      using T = decltype(z);
      constexpr int V = decltype(v)::value;
      const dim3 grid(p.blocks_x, p.blocks_y);
      if (p.K == 1)
        norm_token_kernel<T, V, 1><<<grid, 256, 0, st>>>(a);
      else
        norm_token_kernel<T, V, 4><<<grid, 256, 0, st>>>(a);
      PRNN_HIP(hipGetLastError());
      return static_cast<int>(PRNN_OK);
    });
  if (!stats) return fail(PRNN_ERR_VALUE, "group_norm: statistics per sample need stats");
  const size_t need = sizeof(float) * 2 * G * p.strips * static_cast<size_t>(N);
  if (!workspace || bytes < need)
    return fail(PRNN_ERR_VALUE, "group_norm: the workspace must hold %zu bytes", need);
  a.part = static_cast<float*>(workspace);
  return with_types(dtype, p.V, [&](auto z, auto v) {
    using T = decltype(z);
    constexpr int V = decltype(v)::value;
    const dim3 grid(static_cast<unsigned>(p.strips) * N);
    norm_sample_stats_kernel<T, V><<<grid, 256, 256 * 2 * V * sizeof(float), st>>>(a);
    PRNN_HIP(hipGetLastError());
    if (G <= kJoinGroups) {
      norm_sample_apply_kernel<T, V, true><<<grid, 256, 0, st>>>(a);
    } else {
      norm_sample_join_kernel<<<static_cast<unsigned>((1ll * N * G + 31) / 32), 256, 0, st>>>(a);
      PRNN_HIP(hipGetLastError());
      norm_sample_apply_kernel<T, V, false><<<grid, 256, 0, st>>>(a);
    }
    PRNN_HIP(hipGetLastError());
    return static_cast<int>(PRNN_OK);
  });
}

extern "C" PRNN_API int prnn_group_norm_backward(
    const void* gy, const void* x, const void* w, const void* b, const void* gate,
    const float* stats, void* dx, void* dw, void* db, void* dgate, int N, int L, int C, int G,
    float eps, int act, int w_dtype, int dtype, void* workspace, size_t bytes, void* stream) {
  if (int rc = check("group_norm backward", N, L, C, G, act, w_dtype, dtype)) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool any = N > 0 && L > 0;
  if (any && (!gy || !x || !dx || (gate && !dgate)))
    return fail(PRNN_ERR_VALUE, "group_norm backward: gy, x, dx (and dgate) must be non-null");
  const Plan p = plan(std::max(N, 1), std::max(L, 1), C / G, G, dtype,
                      bits_of({gy, x, gate, dx, dgate}), true);
  if (int rc = check_strips(p, N, G)) return rc;
  Carver c(workspace);
  float *part, *part2 = nullptr;
  int parts;
  if (p.token) {
    parts = p.blocks_x;
    part = static_cast<float*>(c.take(sizeof(float) * 2 * C * parts));
  } else {
    parts = p.strips * N;
    part = static_cast<float*>(c.take(sizeof(float) * 2 * C * static_cast<size_t>(parts)));
    part2 = static_cast<float*>(c.take(sizeof(float) * 2 * G * static_cast<size_t>(parts)));
  }
  if (any && (!workspace || bytes < c.used))
    return fail(PRNN_ERR_VALUE, "group_norm backward: the workspace must hold %zu bytes", c.used);
  NormArgs a{};
  a.x = x;
  a.w = w;
  a.b = b;
  a.gate = gate;
  a.gy = gy;
  a.dx = dx;
  a.dgate = dgate;
  a.stats = const_cast<float*>(stats);
  a.part = part;
  a.part2 = part2;
  a.rows = N;
  a.N = N;
  a.L = L;
  a.C = C;
  a.G = G;
  a.Cg = C / G;
  a.act = act;
  a.w_f32 = w_dtype == PRNN_F32;
  a.w_vec = (bits_of({w, b}) & 15) == 0;
  a.lanes = p.lanes;
  a.strips = p.strips;
  a.strip_rows = p.strip_rows;
  a.eps = eps;
  if (!any) parts = 0;
  if (any && !p.token && !stats)
    return fail(PRNN_ERR_VALUE, "group_norm backward: statistics per sample need stats");
  return with_types(dtype, p.V, [&](auto z, auto v) {
    using T = decltype(z);
    constexpr int V = decltype(v)::value;
    if (any && p.token) {
      const dim3 grid(p.blocks_x, p.blocks_y);
      if (p.K == 1)
        norm_token_bwd_kernel<T, V, 1><<<grid, 256, 0, st>>>(a);
      else
        norm_token_bwd_kernel<T, V, 4><<<grid, 256, 0, st>>>(a);
      PRNN_HIP(hipGetLastError());
    } else if (any) {
      const dim3 grid(static_cast<unsigned>(p.strips) * N);
      if (G <= kJoinGroups && C / V <= 256) {
        norm_sample_bwd_sums_kernel<T, V, true><<<grid, 256, 0, st>>>(a);
        PRNN_HIP(hipGetLastError());
        norm_sample_dx_kernel<T, V, true><<<grid, 256, 0, st>>>(a);
      } else {
        norm_sample_bwd_sums_kernel<T, V, false><<<grid, 256, 0, st>>>(a);
        PRNN_HIP(hipGetLastError());
        // A thread per 16 sums.  8 samples of one group of 2048 channels, 131072 sums each: 26 us;
        // in 32 groups 4.8.  A wave each took some 140 us for one group of 256 channels.
        int block = 64;
        while (block < 1024 && block * 16ll < 1ll * p.strips * (C / G)) block *= 2;
        if (int rc = check_grid("group_norm backward", 1ll * N * G, block)) return rc;
        norm_sample_means_kernel<T><<<N * G, block, 0, st>>>(a);
        PRNN_HIP(hipGetLastError());
        norm_sample_dx_kernel<T, V, false><<<grid, 256, 0, st>>>(a);
      }
      PRNN_HIP(hipGetLastError());
    }
    if (dw || db) {
      norm_param_kernel<T><<<dim3((C + 31) / 32, 2), 1024, 0, st>>>(part, parts, C, dw, db,
                                                                   a.w_f32);
      PRNN_HIP(hipGetLastError());
    }
    return static_cast<int>(PRNN_OK);
  });
}
