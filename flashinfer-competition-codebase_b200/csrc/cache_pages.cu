// cache_pages.cu — the pages of a cache: slots of a pooled recurrent state, pages of a
// paged key-value cache.  A pool is [num_pages, page bytes] with any pitch between pages;
// several pools (layers, keys and values) that share one page numbering go through one call.
//
//   copy      pools[dst[i]] = pools[src[i]] for all i at once: every source is read as it
//             was before the call, of equal dst the last pair wins
//   fork      rows of a block table become children of rows, with reference counts; a
//             partly filled last page is copied for every child but the first
//   compact   live pages behind the first num_live move into the holes before it
//   alloc     the lowest free pages; free: one reference less per listed page
//
// A page is free when its reference count is <= 0.  All results are defined by order of
// index (lowest page first, lowest row first), so they do not depend on scheduling.

#include <string.h>

#include <algorithm>

#include "serving_common.cuh"

namespace {

using namespace gdn_serving;

constexpr int kMaxPools = 32;
constexpr int kMaxPairs = 4096;
constexpr int kMaxPages = 1 << 30;
constexpr int kThreads = 256;
constexpr int kVecs = 16;          // 16-byte vectors a thread holds: 64 KB per CTA

struct Pools {
  char* base[kMaxPools];
  long long bytes[kMaxPools];      // of one page
  long long pitch[kMaxPools];      // from page to page
  int count;
  int num_pages;
};

// ------------------------------------------------------------------ simultaneous copy
//
// A CTA takes one column (the same bytes of every page), reads it from all sources into
// registers, waits for all its threads, and writes it to all destinations.  No other CTA
// touches that column, so sources that are destinations too (a permutation of beams, a
// cycle) are read before they are overwritten, without a second buffer; a source with several
// destinations is read from HBM once, since its readers are in one CTA.
//
// Bound: HBM.  256 pairs of 2 MB, 161 of the sources different: 157 us (875 MB, 5.6 TB/s; a
// plain copy, which writes as much as it reads, 6.57).  4 pairs of 512 KB: 3.5 us, latency.

struct CopyArgs {
  Pools pools;
  const int32_t* src;
  const int32_t* dst;
  int32_t* bad;
  int n;
  int hash;                        // entries of the hash table, a power of two >= 2 n
};

// Pairs that write: both indices valid, different, and no later valid pair with the same
// destination.  Up to 32 pairs live in every warp's registers (lane i: the i-th of them);
// more go through a hash table of destinations into a list in shared memory.
template <bool kFew> struct Pairs;

template <> struct Pairs<true> {
  int s, d, n;
  __device__ Pairs(const CopyArgs& p, int32_t*) {
    const int lane = threadIdx.x % 32, P = p.pools.num_pages;
    s = lane < p.n ? p.src[lane] : -1;
    d = lane < p.n ? p.dst[lane] : -1;
    const bool valid = s >= 0 && d >= 0 && s < P && d < P;
    const bool beyond = s >= 0 && d >= 0 && !valid;
    const uint32_t same = __match_any_sync(0xffffffffu, valid ? d : -1 - lane);
    const uint32_t on = __ballot_sync(0xffffffffu, valid && s != d && (same >> lane) == 1);
    const int bad = __popc(__ballot_sync(0xffffffffu, beyond));
    if (bad && p.bad && blockIdx.x == 0 && threadIdx.x == 0) atomicAdd(p.bad, bad);
    n = __popc(on);
    const int from = lane < n ? __fns(on, 0, lane + 1) : 0;
    s = __shfl_sync(0xffffffffu, s, from);
    d = __shfl_sync(0xffffffffu, d, from);
  }
  __device__ int src(int i) const { return __shfl_sync(0xffffffffu, s, i & 31); }
  __device__ int dst(int i) const { return __shfl_sync(0xffffffffu, d, i & 31); }
};

template <> struct Pairs<false> {
  const int32_t* list;             // [2 n]: source, destination
  int n;
  __device__ Pairs(const CopyArgs& p, int32_t* smem) {
    int32_t* key = smem;           // [hash] destination of an entry
    int32_t* last = smem + p.hash; // [hash] its last pair
    int32_t* out = smem + 2 * p.hash;
    __shared__ int active, bad;
    const int tid = threadIdx.x, P = p.pools.num_pages;
    for (int i = tid; i < p.hash; i += kThreads) {
      key[i] = -1;
      last[i] = -1;
    }
    if (tid == 0) active = bad = 0;
    __syncthreads();
    auto slot_of = [&](int d) {
      uint32_t at = static_cast<uint32_t>(d) * 2654435761u & (p.hash - 1);
      while (true) {               // at most n of >= 2 n entries are taken
        const int k = atomicCAS(&key[at], -1, d);
        if (k == -1 || k == d) return at;
        at = (at + 1) & (p.hash - 1);
      }
    };
    for (int i = tid; i < p.n; i += kThreads) {
      const int s = p.src[i], d = p.dst[i];
      if (s < 0 || d < 0) continue;
      if (s >= P || d >= P) {
        atomicAdd(&bad, 1);
        continue;
      }
      atomicMax(&last[slot_of(d)], i);
    }
    __syncthreads();
    for (int i = tid; i < p.n; i += kThreads) {
      const int s = p.src[i], d = p.dst[i];
      if (s < 0 || d < 0 || s >= P || d >= P || s == d) continue;
      if (last[slot_of(d)] != i) continue;
      const int at = atomicAdd(&active, 1);
      out[2 * at] = s;
      out[2 * at + 1] = d;
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0 && p.bad && bad) atomicAdd(p.bad, bad);
    list = out;
    n = active;
  }
  __device__ int src(int i) const { return list[2 * min(i, n - 1)]; }
  __device__ int dst(int i) const { return list[2 * min(i, n - 1) + 1]; }
};

template <typename U, bool kFew>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ CopyArgs p) {
  extern __shared__ int32_t smem[];
  const Pairs<kFew> pairs(p, smem);
  const int n = pairs.n, tid = threadIdx.x;
  if (n == 0) return;
  // vectors of one page per column: as many as the registers hold, fewer when that would
  // leave CTAs without a column
  int shift = 0;
  while ((2 << shift) * n <= kThreads * kVecs) ++shift;
  long long total = 0;
  for (int i = 0; i < p.pools.count; ++i) total += p.pools.bytes[i] / static_cast<int>(sizeof(U));
  while (shift > 5 && (total >> shift) * 2 <= gridDim.x) --shift;
  const int held = ((n << shift) + kThreads - 1) / kThreads;   // vectors of a thread, <= kVecs
  long long item = blockIdx.x;
  for (int pool = 0; pool < p.pools.count; ++pool) {
    const long long vecs = p.pools.bytes[pool] / static_cast<int>(sizeof(U));
    const long long cols = (vecs + (1ll << shift) - 1) >> shift, pitch = p.pools.pitch[pool];
    char* base = p.pools.base[pool];
    for (; item < cols; item += gridDim.x) {
      U v[kVecs];
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        if (k >= held) break;
        const int f = tid + k * kThreads, i = f >> shift;
        const long long at = (item << shift) + (f & ((1 << shift) - 1));
        const int page = pairs.src(i);
        if (i < n && at < vecs) v[k] = reinterpret_cast<const U*>(base + page * pitch)[at];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        if (k >= held) break;
        const int f = tid + k * kThreads, i = f >> shift;
        const long long at = (item << shift) + (f & ((1 << shift) - 1));
        const int page = pairs.dst(i);
        if (i < n && at < vecs) reinterpret_cast<U*>(base + page * pitch)[at] = v[k];
      }
    }
    item -= cols;
  }
}

// ------------------------------------------------------------------ disjoint moves
//
// Pairs whose destinations are no other pair's source (fork, compact): a work item is a
// segment of one pair's page, and any CTA may take it at any time.
//
// Bound: HBM for compaction (8191 pages of 32 KB in two pools, half of them live: 48 us with its
// plan, 269 MB, 5.6 TB/s); for forks the latency of three launches of which two overlap (512
// rows, up to 4000 tokens: 14.5 us, 22 MB).

struct MoveArgs {
  Pools pools;
  const int32_t* src;              // < 0: no pair
  const int32_t* dst;
  const int32_t* count;            // device count of pairs, or null: n
  int n;
  // compaction's last steps, or remap null
  int32_t* tables;                 // entries to rewrite through remap, or null
  int32_t* remap;                  // [num_pages], the k-th mover's as -2 - k
  int32_t* refcounts;              // [num_pages]
  long long entries;
};

template <typename U>
__global__ void __launch_bounds__(kThreads) move_pages_kernel(const __grid_constant__ MoveArgs p) {
  grid_wait();                     // the plan is the kernel before
  const long long n = p.count ? *p.count : p.n;
  if (p.remap) {
    // a mover's entry is read by the tables' threads while its own thread replaces it: both
    // values lead to the same page
    const long long step = static_cast<long long>(gridDim.x) * kThreads;
    const long long me = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x;
    for (long long k = me; k < n; k += step) {
      const int s = p.src[k], d = p.dst[k];
      p.refcounts[d] = p.refcounts[s];
      p.refcounts[s] = 0;
      __stcg(p.remap + s, d);
    }
    for (long long i = me; i < p.entries; i += step) {
      const int page = p.tables[i];
      if (page < 0 || page >= p.pools.num_pages) continue;
      const int to = __ldcg(p.remap + page);
      p.tables[i] = to <= -2 ? p.dst[-2 - to] : to;
    }
  }
  long long item = blockIdx.x;
  for (int pool = 0; pool < p.pools.count; ++pool) {
    const long long vecs = p.pools.bytes[pool] / static_cast<int>(sizeof(U));
    const long long segs = (vecs + kThreads * kVecs - 1) / (kThreads * kVecs);
    for (; item < n * segs; item += gridDim.x) {
      const long long pair = item / segs, seg = item % segs;
      const int s = p.src[pair], d = p.dst[pair];
      if (s < 0 || d < 0) continue;
      const U* from = reinterpret_cast<const U*>(p.pools.base[pool] + s * p.pools.pitch[pool]);
      U* to = reinterpret_cast<U*>(p.pools.base[pool] + d * p.pools.pitch[pool]);
      U v[kVecs];
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        const long long at = (seg * kVecs + k) * kThreads + threadIdx.x;
        if (at < vecs) v[k] = from[at];
      }
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        const long long at = (seg * kVecs + k) * kThreads + threadIdx.x;
        if (at < vecs) to[at] = v[k];
      }
    }
    item -= n * segs;
  }
}

// ------------------------------------------------------------------ plans (one CTA)

constexpr int kPlanThreads = 1024;

// Exclusive prefix sum over the CTA; `total` gets the sum.  Every thread calls it.
template <typename T> __device__ T block_scan(T x, T& total) {
  __shared__ T part[32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  T y = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();                 // the last call's readers of part are done
  if (lane == 31) part[warp] = y;
  __syncthreads();
  if (warp == 0) {
    T w = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T z = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += z;
    }
    part[lane] = w;
  }
  __syncthreads();
  total = part[31];
  return y - x + (warp ? part[warp - 1] : T(0));
}

// Pages are looked through in rounds: a thread has four neighbours from each of kSets sets of
// 4 kPlanThreads, so loads are coalesced and one scan of packed counts does a round.  One / two /
// four sets: 65536 pages without a free one 13.7 / 10.5 / 11.4 us, compacted half full 33 / 28 / 27
// us; 4096 pages 2.9 / 3.2 / 4.9 and 4.7 / 5.3 / 6.9 us (more code to fetch).
constexpr int kSets = 2, kSet = 4 * kPlanThreads, kRound = kSets * kSet;
static_assert(kSets * 16 <= 32, "packed counts");

struct Counts {
  int c[kSets][4];
  // the counts from page p0 on, `fill` behind the last
  __device__ void load(const int32_t* refcounts, int P, int p0, int fill) {
    const bool wide = (reinterpret_cast<uintptr_t>(refcounts) & 15) == 0;
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
      const int page = p0 + u * kSet + 4 * static_cast<int>(threadIdx.x);
      if (wide && page + 4 <= P) {
        const int4 x = *reinterpret_cast<const int4*>(refcounts + page);
        c[u][0] = x.x; c[u][1] = x.y; c[u][2] = x.z; c[u][3] = x.w;
      } else {
#pragma unroll
        for (int v = 0; v < 4; ++v) c[u][v] = page + v < P ? refcounts[page + v] : fill;
      }
    }
  }
  __device__ int live() const {
    int n = 0;
#pragma unroll
    for (int u = 0; u < kSets; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v) n += c[u][v] > 0;
    return n;
  }
  // live pages of each set, 16 bits each
  __device__ uint32_t packed() const {
    uint32_t n = 0;
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
      int m = 0;
#pragma unroll
      for (int v = 0; v < 4; ++v) m += c[u][v] > 0;
      n |= static_cast<uint32_t>(m) << (16 * u);
    }
    return n;
  }
};
__device__ __forceinline__ int of_set(uint32_t packed, int u) {
  return static_cast<int>(packed >> (16 * u)) & 0xffff;
}

// Gives the k-th wanting row (ascending) the k-th free page (ascending), with reference
// count 1; calls give(row, page) for each wanting row, page -1 when there are too few.
template <typename Wants, typename Give>
__device__ void assign_free(int32_t* refcounts, int P, int n, int32_t* row_of, Wants wants, Give give) {
  int needed = 0;
  uint32_t total;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    const uint32_t w = i < n && wants(i);
    const int at = needed + static_cast<int>(block_scan(w, total));
    if (w) row_of[at] = i;
    needed += static_cast<int>(total);
  }
  __syncthreads();
  // the next round's counts on their way
  int found = 0;
  Counts now, next;
  now.load(refcounts, P, 0, 1);
  for (int p0 = 0; p0 < P && found < needed; p0 += kRound) {
    next.load(refcounts, P, p0 + kRound, 1);
    uint32_t all;
    const uint32_t live = block_scan(now.packed(), all);
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
      int at = found + 4 * static_cast<int>(threadIdx.x) - of_set(live, u);   // free ones before
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (now.c[u][v] <= 0) {
          if (at < needed) {
            const int page = p0 + u * kSet + 4 * threadIdx.x + v;
            refcounts[page] = 1;
            give(row_of[at], page);
          }
          ++at;
        }
      found += kSet - of_set(all, u);
    }
    now = next;
  }
  for (int k = found + threadIdx.x; k < needed; k += kPlanThreads) give(row_of[k], -1);
}

__global__ void __launch_bounds__(kPlanThreads)
alloc_pages_kernel(int32_t* refcounts, int P, const uint8_t* need, int n, int32_t* pages,
                   int32_t* row_of) {
  for (int i = threadIdx.x; i < n; i += kPlanThreads) pages[i] = -1;
  __syncthreads();
  assign_free(refcounts, P, n, row_of, [&](int i) { return need[i] != 0; },
              [&](int i, int page) { pages[i] = page; });
}

__global__ void free_pages_kernel(int32_t* refcounts, int P, const int32_t* pages, long long n,
                                  int32_t* bad) {
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < n; i += step) {
    const int page = pages[i];
    if (page < 0) continue;
    // one reference less; a page that has none keeps its count (the sum of the decrements
    // and of the ones taken back is the same in every order)
    if (page >= P || atomicSub(&refcounts[page], 1) <= 0) {
      if (page < P) atomicAdd(&refcounts[page], 1);
      if (bad) atomicAdd(bad, 1);
    }
  }
}

struct ForkArgs {
  const int32_t* tables;           // [rows_in, width], row stride
  const int32_t* lens;             // [rows_in]
  const int32_t* parents;          // [rows_out]
  int32_t* refcounts;              // [P]
  int32_t* new_tables;             // [rows_out, width]
  int32_t* new_lens;               // [rows_out]
  int32_t* src;                    // workspace [rows_out]: page to copy, or -1
  int32_t* dst;                    // workspace [rows_out]: its copy
  int32_t* row_of;                 // workspace [rows_out]
  int32_t* bad;
  long long stride;
  int rows_in, rows_out, width, P, page_size;
};

// CTA r: the references of input row r, and output row r.
__global__ void __launch_bounds__(kThreads) fork_rows_kernel(const __grid_constant__ ForkArgs p) {
  grid_trigger();
  const int r = blockIdx.x, tid = threadIdx.x;
  __shared__ int count, earlier;
  if (tid == 0) count = earlier = 0;
  __syncthreads();
  const int parent = r < p.rows_out ? p.parents[r] : -1;
  const bool child = parent >= 0 && parent < p.rows_in;
  int c = 0, e = 0;
  for (int i = tid; i < p.rows_out; i += kThreads) {
    const int q = p.parents[i];
    c += q == r;
    e |= i < r && q == parent;
  }
  if (c) atomicAdd(&count, c);
  if (e) earlier = 1;
  __syncthreads();
  auto tokens = [&](int row) {
    const int n = p.lens[row], cap = p.width * p.page_size;
    return n < 0 ? 0 : n > cap ? cap : n;
  };
  if (r < p.rows_in && count != 1) {
    const int n = tokens(r), full = n / p.page_size, part = n % p.page_size != 0;
    const int32_t* row = p.tables + r * p.stride;
    for (int j = tid; j < full + part; j += kThreads) {
      const int page = row[j], delta = j < full ? count - 1 : (count ? 0 : -1);
      if (page >= 0 && page < p.P && delta) atomicAdd(&p.refcounts[page], delta);
    }
  }
  if (r < p.rows_out) {
    const int n = child ? tokens(parent) : 0, full = n / p.page_size, part = n % p.page_size != 0;
    const int32_t* row = p.tables + (child ? parent : 0) * p.stride;
    int32_t* out = p.new_tables + static_cast<long long>(r) * p.width;
    for (int j = tid; j < p.width; j += kThreads) out[j] = j < full + part ? row[j] : -1;
    if (tid == 0) {
      p.new_lens[r] = n;
      const int page = part ? row[full] : -1;
      p.src[r] = (earlier && page >= 0 && page < p.P) ? page : -1;
      p.dst[r] = -1;
      if (parent >= p.rows_in && p.bad) atomicAdd(p.bad, 1);
    }
  }
}

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const __grid_constant__ ForkArgs p) {
  grid_trigger();
  grid_wait();                     // the rows' references are counted
  assign_free(p.refcounts, p.P, p.rows_out, p.row_of, [&](int i) { return p.src[i] >= 0; },
              [&](int i, int page) {
                p.dst[i] = page;
                p.new_tables[static_cast<long long>(i) * p.width + p.new_lens[i] / p.page_size] = page;
                if (page < 0 && p.bad) atomicAdd(p.bad, 1);
              });
}

struct CompactArgs {
  int32_t* refcounts;              // [P]
  int32_t* remap;                  // [P]
  int32_t* live;                   // [1]
  int32_t* src;                    // workspace [P / 2 + 1]
  int32_t* dst;
  int32_t* count;                  // workspace [1]
  int P;
};

// With before(i) the live pages before page i and L all of them, a free page i < L is hole
// number i - before(i), and a live page i >= L is mover number before(i) - before(L); there are
// L - before(L) of either.  So: L, then before(L), then each page's place; a pool of one round
// stays in registers.  Pairing the k-th of each, with its scattered writes, is left to the
// moving kernel's many CTAs (it cost this one CTA 4.5 us of 9).
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const __grid_constant__ CompactArgs p) {
  grid_trigger();
  const bool one = p.P <= kRound;
  Counts c;
  uint32_t mine = 0, live_pages, kept_pages;
  for (int p0 = 0; p0 < p.P; p0 += kRound) {
    c.load(p.refcounts, p.P, p0, 0);
    mine += c.live();
  }
  block_scan(mine, live_pages);
  const int live = static_cast<int>(live_pages);
  mine = 0;
  for (int p0 = 0; p0 < live; p0 += kRound) {
    if (!one) c.load(p.refcounts, p.P, p0, 0);
#pragma unroll
    for (int u = 0; u < kSets; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        mine += c.c[u][v] > 0 && p0 + u * kSet + 4 * static_cast<int>(threadIdx.x) + v < live;
  }
  block_scan(mine, kept_pages);
  const int kept = static_cast<int>(kept_pages);
  int seen = 0;                    // live pages before this set
  for (int p0 = 0; p0 < p.P; p0 += kRound) {
    if (!one) c.load(p.refcounts, p.P, p0, 0);
    uint32_t all;
    const uint32_t scan = block_scan(c.packed(), all);
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
      const int page = p0 + u * kSet + 4 * static_cast<int>(threadIdx.x);
      int before = seen + of_set(scan, u), to[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int i = page + v;
        const bool on = c.c[u][v] > 0;
        to[v] = on ? i : -1;
        if (on && i >= live) {
          to[v] = -2 - (before - kept);
          p.src[before - kept] = i;
        }
        if (!on && i < live) p.dst[i - before] = i;   // live <= P: what is behind is no hole
        before += on;
      }
      if (page + 4 <= p.P && (reinterpret_cast<uintptr_t>(p.remap) & 15) == 0) {
        *reinterpret_cast<int4*>(p.remap + page) = make_int4(to[0], to[1], to[2], to[3]);
      } else {
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (page + v < p.P) p.remap[page + v] = to[v];
      }
      seen += of_set(all, u);
    }
  }
  if (threadIdx.x == 0) {
    *p.live = live;
    *p.count = live - kept;
  }
}

// ------------------------------------------------------------------ host

int check_pools(void* const* pools, const int64_t* bytes, const int64_t* pitch, int num_pools,
                int num_pages, Pools& out, int& unit) {
  if (num_pools < 0 || num_pages < 1 || num_pages > kMaxPages) return GDN_ERR_SHAPE;
  if (num_pools > kMaxPools) return GDN_ERR_LIMIT;
  if (num_pools > 0 && (!pools || !bytes || !pitch)) return GDN_ERR_NULL;
  memset(&out, 0, sizeof(out));
  out.count = num_pools;
  out.num_pages = num_pages;
  unit = 16;
  for (int i = 0; i < num_pools; ++i) {
    if (!pools[i]) return GDN_ERR_NULL;
    if (bytes[i] < 1) return GDN_ERR_SHAPE;
    if (pitch[i] < bytes[i]) return GDN_ERR_ALIAS;     // pages of one pool overlap
    out.base[i] = static_cast<char*>(pools[i]);
    out.bytes[i] = bytes[i];
    out.pitch[i] = pitch[i];
    const uintptr_t all = reinterpret_cast<uintptr_t>(pools[i]) | static_cast<uintptr_t>(bytes[i]) |
                          static_cast<uintptr_t>(pitch[i]);
    while (all % unit) unit /= 4;
    // two pools may interleave (key and value halves of one buffer) but not share a byte
    for (int j = 0; j < i; ++j) {
      if (!overlaps(out.base[i], (num_pages - 1) * pitch[i] + bytes[i], out.base[j],
                    (num_pages - 1) * pitch[j] + bytes[j]))
        continue;
      if (pitch[i] != pitch[j]) return GDN_ERR_ALIAS;
      int64_t off = (out.base[i] - out.base[j]) % pitch[i];
      if (off < 0) off += pitch[i];
      if (off < bytes[j] || off + bytes[i] > pitch[i]) return GDN_ERR_ALIAS;
    }
  }
  return GDN_OK;
}

// CTAs for `pairs` pages to move: two per SM with as few vectors per thread as that leaves,
// and past full registers one per kVecs vectors of its threads, up to `most` per SM.
unsigned grid_for(const Pools& pools, int unit, long long pairs, int most) {
  long long vecs = 0;
  for (int i = 0; i < pools.count; ++i) vecs += pools.bytes[i] / unit;
  const long long thin = (vecs * pairs + kThreads - 1) / kThreads;
  const long long full = (thin + kVecs - 1) / kVecs;
  const long long two = 2 * kSMs, ctas = full > two ? full : thin < two ? thin : two;
  return static_cast<unsigned>(ctas < 1 ? 1 : ctas > 1ll * most * kSMs ? most * kSMs : ctas);
}

cudaError_t launch_moves(const MoveArgs& a, int unit, unsigned grid, cudaStream_t st) {
  if (unit == 16) return launch_after(move_pages_kernel<uint4>, dim3(grid), dim3(kThreads), 0, st, a);
  if (unit == 4) return launch_after(move_pages_kernel<uint32_t>, dim3(grid), dim3(kThreads), 0, st, a);
  return launch_after(move_pages_kernel<uint8_t>, dim3(grid), dim3(kThreads), 0, st, a);
}

}  // namespace

extern "C" {

int gdn_copy_pages(void* const* pools, const int64_t* page_bytes, const int64_t* page_pitch,
                   int num_pools, int num_pages, const int32_t* src, const int32_t* dst, int n,
                   int32_t* bad_index_count, void* stream) {
  CopyArgs a{};
  int unit = 16;
  const int rc = check_pools(pools, page_bytes, page_pitch, num_pools, num_pages, a.pools, unit);
  if (rc != GDN_OK) return rc;
  if (n < 0) return GDN_ERR_SHAPE;
  if (n > kMaxPairs) return GDN_ERR_LIMIT;
  if (n == 0 || num_pools == 0) return GDN_OK;
  if (!src || !dst) return GDN_ERR_NULL;
  if (!aligned(src, 4) || !aligned(dst, 4) || !aligned(bad_index_count, 4)) return GDN_ERR_ALIGN;
  a.src = src;
  a.dst = dst;
  a.bad = bad_index_count;
  a.n = n;
  const bool few = n <= 32;
  a.hash = few ? 0 : 64;
  while (a.hash && a.hash < 2 * n) a.hash *= 2;
  const size_t smem = few ? 0 : (2 * static_cast<size_t>(a.hash) + 2 * static_cast<size_t>(n)) * 4;
  const unsigned grid = grid_for(a.pools, unit, n, 32);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel) {
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem)) != cudaSuccess)
      return GDN_ERR_LAUNCH;
    kernel<<<grid, kThreads, smem, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
  };
  if (unit == 16) return few ? go(copy_pages_kernel<uint4, true>) : go(copy_pages_kernel<uint4, false>);
  if (unit == 4) return few ? go(copy_pages_kernel<uint32_t, true>) : go(copy_pages_kernel<uint32_t, false>);
  return few ? go(copy_pages_kernel<uint8_t, true>) : go(copy_pages_kernel<uint8_t, false>);
}

int gdn_alloc_pages(int32_t* refcounts, int num_pages, const uint8_t* need, int n, int32_t* pages,
                    void* workspace, size_t workspace_bytes, void* stream) {
  if (num_pages < 1 || num_pages > kMaxPages || n < 0) return GDN_ERR_SHAPE;
  if (n == 0) return GDN_OK;
  if (!refcounts || !need || !pages || !workspace) return GDN_ERR_NULL;
  if (!aligned(refcounts, 4) || !aligned(pages, 4) || !aligned(workspace, 4)) return GDN_ERR_ALIGN;
  if (workspace_bytes < static_cast<size_t>(n) * 4) return GDN_ERR_SHAPE;
  alloc_pages_kernel<<<1, kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      refcounts, num_pages, need, n, pages, static_cast<int32_t*>(workspace));
  return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

int gdn_free_pages(int32_t* refcounts, int num_pages, const int32_t* pages, int64_t n,
                   int32_t* bad_index_count, void* stream) {
  if (num_pages < 1 || num_pages > kMaxPages || n < 0) return GDN_ERR_SHAPE;
  if (n == 0) return GDN_OK;
  if (!refcounts || !pages) return GDN_ERR_NULL;
  if (!aligned(refcounts, 4) || !aligned(pages, 4) || !aligned(bad_index_count, 4))
    return GDN_ERR_ALIGN;
  const int64_t ctas = (n + kThreads - 1) / kThreads;
  free_pages_kernel<<<static_cast<unsigned>(ctas > kSMs * 8 ? kSMs * 8 : ctas), kThreads, 0,
                      static_cast<cudaStream_t>(stream)>>>(refcounts, num_pages, pages, n,
                                                           bad_index_count);
  return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

int gdn_fork_pages(const int32_t* block_tables, int64_t table_stride, const int32_t* seq_lens,
                   const int32_t* parents, int32_t* refcounts, int32_t* new_tables,
                   int32_t* new_lens, int rows_in, int rows_out, int table_width, int num_pages,
                   int page_size, void* const* pools, const int64_t* page_bytes,
                   const int64_t* page_pitch, int num_pools, void* workspace,
                   size_t workspace_bytes, int32_t* bad_index_count, void* stream) {
  MoveArgs m{};
  int unit = 16;
  const int rc = check_pools(pools, page_bytes, page_pitch, num_pools, num_pages, m.pools, unit);
  if (rc != GDN_OK) return rc;
  if (rows_in < 0 || rows_out < 0 || table_width < 0 || page_size < 1) return GDN_ERR_SHAPE;
  if (static_cast<long long>(table_width) * page_size > 0x7fffffffLL || table_stride < 0)
    return GDN_ERR_SHAPE;
  if (rows_in == 0 && rows_out == 0) return GDN_OK;
  if (!refcounts || (rows_in > 0 && !seq_lens) || (rows_out > 0 && (!parents || !new_lens || !workspace)))
    return GDN_ERR_NULL;
  if (table_width > 0 && ((rows_in > 0 && !block_tables) || (rows_out > 0 && !new_tables)))
    return GDN_ERR_NULL;
  if (!aligned(block_tables, 4) || !aligned(seq_lens, 4) || !aligned(parents, 4) ||
      !aligned(refcounts, 4) || !aligned(new_tables, 4) || !aligned(new_lens, 4) ||
      !aligned(workspace, 4) || !aligned(bad_index_count, 4))
    return GDN_ERR_ALIGN;
  if (workspace_bytes < 12 * static_cast<size_t>(rows_out)) return GDN_ERR_SHAPE;
  if (table_width > 0 && rows_in > 0 && rows_out > 0 &&
      overlaps(block_tables, ((rows_in - 1) * table_stride + table_width) * 4, new_tables,
               static_cast<size_t>(rows_out) * table_width * 4))
    return GDN_ERR_ALIAS;
  if (rows_in > 0 && rows_out > 0 &&
      overlaps(seq_lens, static_cast<size_t>(rows_in) * 4, new_lens, static_cast<size_t>(rows_out) * 4))
    return GDN_ERR_ALIAS;
  ForkArgs p{};
  p.tables = block_tables; p.lens = seq_lens; p.parents = parents; p.refcounts = refcounts;
  p.new_tables = new_tables; p.new_lens = new_lens;
  p.src = static_cast<int32_t*>(workspace);
  p.dst = p.src + rows_out;
  p.row_of = p.dst + rows_out;
  p.bad = bad_index_count; p.stride = table_stride;
  p.rows_in = rows_in; p.rows_out = rows_out; p.width = table_width; p.P = num_pages;
  p.page_size = page_size;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  fork_rows_kernel<<<rows_in > rows_out ? rows_in : rows_out, kThreads, 0, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return GDN_ERR_LAUNCH;
  if (rows_out == 0) return GDN_OK;
  if (launch_after(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p) != cudaSuccess)
    return GDN_ERR_LAUNCH;
  if (num_pools == 0) return GDN_OK;
  m.src = p.src;
  m.dst = p.dst;
  m.n = rows_out;
  return launch_moves(m, unit, grid_for(m.pools, unit, rows_out, 8), st) == cudaSuccess ? GDN_OK
                                                                                     : GDN_ERR_LAUNCH;
}

int gdn_compact_pages(int32_t* refcounts, int num_pages, int32_t* block_tables,
                      int64_t table_entries, int32_t* remap, int32_t* num_live,
                      void* const* pools, const int64_t* page_bytes, const int64_t* page_pitch,
                      int num_pools, void* workspace, size_t workspace_bytes, void* stream) {
  MoveArgs m{};
  int unit = 16;
  const int rc = check_pools(pools, page_bytes, page_pitch, num_pools, num_pages, m.pools, unit);
  if (rc != GDN_OK) return rc;
  if (table_entries < 0) return GDN_ERR_SHAPE;
  if (!refcounts || !remap || !num_live || !workspace || (table_entries > 0 && !block_tables))
    return GDN_ERR_NULL;
  if (!aligned(refcounts, 4) || !aligned(block_tables, 4) || !aligned(remap, 4) ||
      !aligned(num_live, 4) || !aligned(workspace, 4))
    return GDN_ERR_ALIGN;
  const size_t half = static_cast<size_t>(num_pages) / 2 + 1;
  if (workspace_bytes < (2 * half + 1) * 4) return GDN_ERR_SHAPE;
  CompactArgs p{};
  p.refcounts = refcounts; p.remap = remap; p.live = num_live; p.P = num_pages;
  p.src = static_cast<int32_t*>(workspace);
  p.dst = p.src + half;
  p.count = p.dst + half;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  compact_plan_kernel<<<1, kPlanThreads, 0, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return GDN_ERR_LAUNCH;
  m.tables = block_tables;
  m.entries = table_entries;
  m.remap = remap;
  m.refcounts = refcounts;
  m.src = p.src;
  m.dst = p.dst;
  m.count = p.count;
  const long long small = std::max(static_cast<long long>(table_entries), static_cast<long long>(half));
  const unsigned grid = num_pools > 0
                            ? grid_for(m.pools, unit, static_cast<long long>(half), 8)
                            : static_cast<unsigned>(std::min((small + kThreads - 1) / kThreads, 2ll * kSMs));
  return launch_moves(m, unit, grid, st) == cudaSuccess
             ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // extern "C"
