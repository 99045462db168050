// Pages of a state cache: taking, forking, freeing and compacting slots of one or several pools.
//
// Which slot goes where is one workgroup's work: a running count over the `used` flags (4 a
// thread, 4096 a round), so that the k-th wanted slot is the k-th lowest free one whatever the
// timing: two launches would cost more than one workgroup's rounds (2048 slots: taking 300 of them
// 4.7 us, planning a compaction 6.0, most of it the launch).  The pools' data then moves in a launch
// of its own, a workgroup per 16 KB, bound by memory: every byte is read once and written once, 252
// MB of slots of 512 KB in 55 us, 4.5 TB/s (a large copy: 5.1); 8 slots of 128 KB take 8.3 us.
#include <algorithm>

#include "prnn_host.h"

namespace prnn {
namespace {

constexpr int kPagesPools = 16;    // pools of a launch
constexpr int kPagesTables = 16;   // tables of a launch
constexpr int kPlan = 1024;        // threads of the one workgroup
constexpr int kPart = 16384;       // bytes of a slot that a workgroup copies

// Exclusive running count over the workgroup's threads; total gets the sum.
__device__ __forceinline__ int block_rank(int v, int* lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int run = v;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const int o = __shfl_up(run, k);
    if (lane >= k) run += o;
  }
  __syncthreads();  // the last round's counts have been read
  if (lane == 63) lds[wave] = run;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlan / 64; ++w) {
    if (w < wave) before += lds[w];
    total += lds[w];
  }
  return before + run - v;
}

// The `want` lowest free slots, in order, into list; they become used.  Returns how many.
__device__ __forceinline__ int take_lowest(int* used, int slots, int* list, int want, int* lds) {
  int found = 0;
  for (int base = 0; base < slots && found < want; base += 4 * kPlan) {
    bool free[4];
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = base + threadIdx.x * 4 + i;
      free[i] = s < slots && used[s] == 0;
      n += free[i];
    }
    int total, rank = block_rank(n, lds, total) + found;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (free[i]) {
        if (rank < want) {
          list[rank] = base + threadIdx.x * 4 + i;
          used[base + threadIdx.x * 4 + i] = 1;
        }
        ++rank;
      }
    found += total;
  }
  return min(found, want);
}

__global__ __launch_bounds__(kPlan) void pages_take_kernel(int* used, int slots, int* out, int n) {
  __shared__ int lds[kPlan / 64];
  const int got = take_lowest(used, slots, out, n, lds);
  for (int i = got + threadIdx.x; i < n; i += kPlan) out[i] = -1;
}

// scratch: the slots taken, in order.  A parent is a slot in use before the call: a free one could be
// handed out as another entry's child and be read and written by one launch.
__global__ __launch_bounds__(kPlan) void pages_fork_kernel(int* used, int slots,
                                                           const int* __restrict__ parents,
                                                           int* out, int n, int* scratch) {
  __shared__ int lds[kPlan / 64];
  // how many entries have a parent (0 in out until they are told their child)
  int want = 0;
  for (int base = 0; base < n; base += kPlan) {
    const int i = base + threadIdx.x;
    const int p = i < n ? parents[i] : -1;
    const bool has = p >= 0 && p < slots && used[p] != 0;
    if (i < n) out[i] = has ? 0 : -1;
    int total;
    block_rank(has, lds, total);
    want += total;
  }
  const int got = take_lowest(used, slots, scratch, want, lds);
  __syncthreads();
  int first = 0;
  for (int base = 0; base < n; base += kPlan) {
    const int i = base + threadIdx.x;
    const bool has = i < n && out[i] == 0;
    int total;
    const int rank = block_rank(has, lds, total) + first;
    if (has) out[i] = rank < got ? scratch[rank] : -1;
    first += total;
  }
}

__global__ void pages_free_kernel(int* used, int slots, const int* __restrict__ list, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n && list[i] >= 0 && list[i] < slots) used[list[i]] = 0;
}

struct Pools {
  prnn_pool pool[kPagesPools];
  int parts[kPagesPools];  // workgroups per slot, summed up to and including the pool
  int n;
};

// Bytes [at, at + kPart) of slot src into slot dst.
__device__ __forceinline__ void copy_part(const prnn_pool& pool, int src, int dst, long long at) {
  const long long left = min(pool.row_bytes - at, static_cast<long long>(kPart));
  const char* s = static_cast<const char*>(pool.p) + src * pool.row_bytes + at;
  char* d = static_cast<char*>(pool.p) + dst * pool.row_bytes + at;
  if (((reinterpret_cast<uintptr_t>(pool.p) | pool.row_bytes) & 15) == 0) {
    // buffers of what is left: behind it nothing is read or written, without a branch
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    constexpr int kEach = kPart / 16 / 256;
    const rsrc_t rs = make_rsrc(s, static_cast<uint32_t>(left)), rd = make_rsrc(d, static_cast<uint32_t>(left));
    u4 v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      v[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (i * 256 + threadIdx.x) * 16, 0, 0);
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      __builtin_amdgcn_raw_buffer_store_b128(v[i], rd, (i * 256 + threadIdx.x) * 16, 0, 0);
  } else if (((reinterpret_cast<uintptr_t>(pool.p) | pool.row_bytes) & 3) == 0) {
    for (int o = threadIdx.x * 4; o < left; o += 1024)
      *reinterpret_cast<uint32_t*>(d + o) = *reinterpret_cast<const uint32_t*>(s + o);
  } else {
    for (int o = threadIdx.x; o < left; o += 256) d[o] = s[o];
  }
}

// Part `id` of entry i (all pools' parts of a slot side by side).
__device__ __forceinline__ void copy_entry(const Pools& P, int src, int dst, int part) {
  int k = 0;
  while (part >= P.parts[k]) ++k;
  copy_part(P.pool[k], src, dst, static_cast<long long>(part - (k ? P.parts[k - 1] : 0)) * kPart);
}

__global__ __launch_bounds__(256) void pages_copy_kernel(Pools P, int slots,
                                                         const int* __restrict__ src,
                                                         const int* __restrict__ dst, int n) {
  const int per = P.parts[P.n - 1];
  const int i = blockIdx.x / per;
  const int s = src[i], d = dst[i];
  if (s < 0 || s >= slots || d < 0 || d >= slots || s == d) return;
  copy_entry(P, s, d, blockIdx.x - i * per);
}

// A beam's first child keeps its slot; the other children, in order, take the slots of the beams
// without children, in order, and get a copy.  A workgroup per search; src, dst: the copies, -1 where
// there is none.  No copy's source is another's destination: one has a child, the other none.
// Latency: 32 searches of 8 beams 3.8 us, the copies (of 128 KB a slot) 7.5.
constexpr int kBeams = kPlan;
__global__ __launch_bounds__(kPlan) void pages_reorder_kernel(int* table, const int* __restrict__ parents,
                                                              int K, int slots, int* src, int* dst) {
  __shared__ int lds[kPlan / 64], first[kBeams], old[kBeams], spare[kBeams];
  const int i = threadIdx.x;
  const size_t at = static_cast<size_t>(blockIdx.x) * K + i;
  const bool in = i < K;
  int p = in ? parents[at] : -1;
  if (p >= K) p = -1;
  if (in) {
    first[i] = kBeams;
    old[i] = table[at];
  }
  __syncthreads();
  if (p >= 0) atomicMin(&first[p], i);
  __syncthreads();
  const bool barren = in && first[i] == kBeams, other = in && (p < 0 || first[p] != i);
  int total;
  const int free = block_rank(barren, lds, total);
  if (barren) spare[free] = old[i];
  const int rank = block_rank(other, lds, total);
  __syncthreads();
  if (!in) return;
  const int from = p >= 0 ? old[p] : -1, to = other ? spare[rank] : from;
  table[at] = to;
  const bool copy = other && from >= 0 && from < slots && to >= 0 && to < slots;
  src[at] = copy ? from : -1;
  dst[at] = copy ? to : -1;
}

// scratch: [0] moves, [1 .. slots] new place of every slot, then the movers (slots / 2 at most)
// and the holes below them, as many.
__global__ __launch_bounds__(kPlan) void pages_plan_kernel(int* used, int slots, int* live,
                                                           int* scratch) {
  __shared__ int lds[kPlan / 64];
  int* place = scratch + 1;
  int* movers = place + slots;
  int* holes = movers + slots / 2;
  int n = 0;
  for (int s = threadIdx.x; s < slots; s += kPlan) n += used[s] != 0;
  int L;
  block_rank(n, lds, L);
  int moved = 0, hollow = 0;
  for (int base = 0; base < slots; base += kPlan) {
    const int s = base + threadIdx.x;
    const bool on = s < slots && used[s] != 0;
    int total;
    const bool mover = on && s >= L, hole = s < L && !on;
    const int rm = block_rank(mover, lds, total) + moved;
    moved += total;
    const int rh = block_rank(hole, lds, total) + hollow;
    hollow += total;
    if (mover) movers[rm] = s;
    if (hole) holes[rh] = s;
    if (s < slots) place[s] = on ? s : -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moved; i += kPlan) place[movers[i]] = holes[i];
  for (int s = threadIdx.x; s < slots; s += kPlan) used[s] = s < L;
  if (threadIdx.x == 0) {
    scratch[0] = moved;
    *live = L;
  }
}

struct Tables {
  int* p[kPagesTables];
  int len[kPagesTables];
  int n;
};

// The first `table_blocks` workgroups rename the tables' entries, the others move the slots.
__global__ __launch_bounds__(256) void pages_move_kernel(Pools P, Tables T, int slots,
                                                         const int* __restrict__ scratch,
                                                         int table_blocks) {
  const int* place = scratch + 1;
  if (static_cast<int>(blockIdx.x) < table_blocks) {
    for (int k = 0; k < T.n; ++k)
      for (int i = blockIdx.x * 256 + threadIdx.x; i < T.len[k]; i += table_blocks * 256) {
        const int s = T.p[k][i];
        if (s >= 0 && s < slots) T.p[k][i] = place[s];
      }
    return;
  }
  if (P.n == 0) return;
  const int* movers = place + slots;
  const int* holes = movers + slots / 2;
  const int per = P.parts[P.n - 1];
  const long long items = static_cast<long long>(scratch[0]) * per;
  for (long long it = static_cast<int>(blockIdx.x) - table_blocks; it < items;
       it += static_cast<int>(gridDim.x) - table_blocks) {
    const int i = static_cast<int>(it / per);
    copy_entry(P, movers[i], holes[i], static_cast<int>(it - static_cast<long long>(i) * per));
  }
}

// Entries of lists, as of slots: a workgroup's step past the last does not wrap.
bool list_fits(int n) { return n >= 0 && n <= (1 << 30); }

int check_cache(const char* what, const int* used, int slots, const prnn_pool* pools,
                int n_pools) {
  if (slots < 0 || slots > (1 << 30))
    return fail(PRNN_ERR_VALUE, "%s: %d slots are not in 0 .. 2^30", what, slots);
  if (slots > 0 && used == nullptr) return fail(PRNN_ERR_VALUE, "%s: used must be non-null", what);
  if (n_pools < 0 || (n_pools > 0 && pools == nullptr))
    return fail(PRNN_ERR_VALUE, "%s: %d pools", what, n_pools);
  for (int i = 0; i < n_pools; ++i)
    if (pools[i].row_bytes < 0 || (slots > 0 && pools[i].row_bytes > 0 && !pools[i].p) ||
        pools[i].row_bytes > (1ll << 40))
      return fail(PRNN_ERR_VALUE, "%s: pool %d", what, i);
  return PRNN_OK;
}

// Pools [first, first + kPagesPools) that hold anything.
Pools some_pools(const prnn_pool* pools, int n_pools, int first) {
  Pools P{};
  int parts = 0;
  for (int i = first; i < n_pools && i < first + kPagesPools; ++i) {
    if (pools[i].row_bytes == 0) continue;
    parts += static_cast<int>((pools[i].row_bytes + kPart - 1) / kPart);
    P.pool[P.n] = pools[i];
    P.parts[P.n++] = parts;
  }
  return P;
}

int copy(const prnn_pool* pools, int n_pools, int slots, const int* src, const int* dst, int n,
         hipStream_t st) {
  for (int first = 0; first < n_pools; first += kPagesPools) {
    const Pools P = some_pools(pools, n_pools, first);
    if (P.n == 0) continue;
    const long long per = P.parts[P.n - 1];
    // a launch holds fewer than 2^32 threads
    if (int rc = check_grid("copy of pages", per, 256)) return rc;
    const int most = static_cast<int>(std::min<long long>(n, 0xffffffffll / 256 / per));
    for (int i = 0; i < n; i += most) {
      const int m = std::min(most, n - i);
      pages_copy_kernel<<<static_cast<unsigned>(m * per), 256, 0, st>>>(P, slots, src + i, dst + i,
                                                                       m);
      PRNN_HIP(hipGetLastError());
    }
  }
  return PRNN_OK;
}

}  // namespace
}  // namespace prnn

using namespace prnn;

extern "C" PRNN_API int prnn_pages_take(int* used, int slots, int* out, int n, void* stream) {
  if (int rc = check_cache("pages_take", used, slots, nullptr, 0)) return rc;
  if (!list_fits(n) || (n > 0 && out == nullptr)) return fail(PRNN_ERR_VALUE, "pages_take: n=%d", n);
  if (n == 0) return PRNN_OK;
  pages_take_kernel<<<1, kPlan, 0, static_cast<hipStream_t>(stream)>>>(used, slots, out, n);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

extern "C" PRNN_API int prnn_pages_fork(int* used, int slots, const prnn_pool* pools, int n_pools,
                                        const int* parents, int* out, int n, int* scratch,
                                        void* stream) {
  if (int rc = check_cache("pages_fork", used, slots, pools, n_pools)) return rc;
  if (!list_fits(n) || (n > 0 && (!parents || !out || !scratch)))
    return fail(PRNN_ERR_VALUE, "pages_fork: n=%d, parents, out and scratch must be non-null", n);
  if (n == 0) return PRNN_OK;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  pages_fork_kernel<<<1, kPlan, 0, st>>>(used, slots, parents, out, n, scratch);
  PRNN_HIP(hipGetLastError());
  return copy(pools, n_pools, slots, parents, out, n, st);
}

extern "C" PRNN_API int prnn_pages_free(int* used, int slots, const int* list, int n,
                                        void* stream) {
  if (int rc = check_cache("pages_free", used, slots, nullptr, 0)) return rc;
  if (!list_fits(n) || (n > 0 && list == nullptr)) return fail(PRNN_ERR_VALUE, "pages_free: n=%d", n);
  if (n == 0) return PRNN_OK;
  pages_free_kernel<<<(n + 255) / 256, 256, 0, static_cast<hipStream_t>(stream)>>>(used, slots,
                                                                                  list, n);
  PRNN_HIP(hipGetLastError());
  return PRNN_OK;
}

extern "C" PRNN_API int prnn_pages_copy(int slots, const prnn_pool* pools, int n_pools,
                                        const int* src, const int* dst, int n, void* stream) {
  int none = 0;
  if (int rc = check_cache("pages_copy", &none, slots, pools, n_pools)) return rc;
  if (!list_fits(n) || (n > 0 && (!src || !dst)))
    return fail(PRNN_ERR_VALUE, "pages_copy: n=%d, src and dst must be non-null", n);
  if (n == 0 || slots == 0) return PRNN_OK;
  return copy(pools, n_pools, slots, src, dst, n, static_cast<hipStream_t>(stream));
}

extern "C" PRNN_API int prnn_pages_reorder(int slots, const prnn_pool* pools, int n_pools, int* table,
                                           const int* parents, int B, int K, int* scratch,
                                           void* stream) {
  int none = 0;
  if (int rc = check_cache("pages_reorder", &none, slots, pools, n_pools)) return rc;
  if (B < 0 || K < 1 || K > kBeams || static_cast<long long>(B) * K > 1ll << 30)
    return fail(PRNN_ERR_VALUE, "pages_reorder: B=%d, K=%d: K must be in 1 .. %d", B, K, kBeams);
  if (int rc = check_grid("pages_reorder", B, kPlan)) return rc;
  if (B == 0) return PRNN_OK;
  if (!table || !parents || !scratch)
    return fail(PRNN_ERR_VALUE, "pages_reorder: table, parents and scratch must be non-null");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int n = B * K;
  pages_reorder_kernel<<<B, kPlan, 0, st>>>(table, parents, K, slots, scratch, scratch + n);
  PRNN_HIP(hipGetLastError());
  return slots == 0 ? PRNN_OK : copy(pools, n_pools, slots, scratch, scratch + n, n, st);
}

extern "C" PRNN_API int prnn_pages_compact(int* used, int slots, const prnn_pool* pools,
                                           int n_pools, int* const* tables, const int* lens,
                                           int n_tables, int* live, int* scratch, void* stream) {
  if (int rc = check_cache("pages_compact", used, slots, pools, n_pools)) return rc;
  if (n_tables < 0 || (n_tables > 0 && (!tables || !lens)) || !live || !scratch)
    return fail(PRNN_ERR_VALUE, "pages_compact: tables, live and scratch must be non-null");
  for (int i = 0; i < n_tables; ++i)
    if (!list_fits(lens[i]) || (lens[i] > 0 && !tables[i]))
      return fail(PRNN_ERR_VALUE, "pages_compact: table %d", i);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  pages_plan_kernel<<<1, kPlan, 0, st>>>(used, slots, live, scratch);
  PRNN_HIP(hipGetLastError());
  for (int fp = 0, ft = 0; fp < n_pools || ft < n_tables; fp += kPagesPools, ft += kPagesTables) {
    const Pools P = fp < n_pools ? some_pools(pools, n_pools, fp) : Pools{};
    Tables T{};
    int longest = 0;
    for (int i = ft; i < n_tables && i < ft + kPagesTables; ++i)
      if (lens[i] > 0) {
        T.p[T.n] = tables[i];
        T.len[T.n++] = lens[i];
        longest = std::max(longest, lens[i]);
      }
    const int table_blocks = std::min((longest + 255) / 256, 64);
    // at most half the slots move
    const long long items = P.n ? static_cast<long long>(slots / 2) * P.parts[P.n - 1] : 0;
    const int movers = static_cast<int>(std::min<long long>(items, 4096));
    if (table_blocks + movers == 0) continue;
    pages_move_kernel<<<table_blocks + movers, 256, 0, st>>>(P, T, slots, scratch, table_blocks);
    PRNN_HIP(hipGetLastError());
  }
  return PRNN_OK;
}
