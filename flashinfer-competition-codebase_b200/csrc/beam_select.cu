// beam_select.cu — beam search's selection over beams and vocabulary.
//
// For each request, the candidates (beam i, token t) with
//   score(i, t) = scores[i] + (logits[i, t] - lse_i),   lse_i = ln(sum_t exp(logits[i, t]))
// and, for a finished beam, the one candidate (i, eos) with score scores[i].  The n best are
// returned in descending order; candidates of one beam are ordered by logit, equal ones by
// token, and beams' candidates are merged by score in 64 bits, equal ones by beam.  What
// has no finite score (masked tokens at -inf, dead beams at -inf, rows with a NaN) is never
// chosen; places left over get token -1, parent -1, score -inf.

#include <float.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "serving_common.cuh"

namespace {

using namespace gdn_serving;

constexpr int kMaxBeams = 64, kMaxSelected = 64;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kSlice = 3072;     // 16-byte vectors of logits a CTA holds: 48 KB, four CTAs per SM
constexpr int kList = 512;       // candidates of a slice that are ranked
constexpr int kMergeThreads = 512;
constexpr int kHeadItems = 1024; // of the merge's bound
constexpr float kLog2e = 1.44269504088896340736f;

struct BeamArgs {
  const void* logits;
  const float* scores;
  const uint8_t* finished;
  int32_t* tokens;
  int32_t* parents;
  float* out_scores;
  unsigned long long* keys;   // workspace [rows, slices, n]: keys, descending, 0 = none
  float2* sums;               // workspace [rows, slices]: m, sum exp(x - m)
  long long stride_batch, stride_beam;
  int B, K, V, n, eos, slices;
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(float x) { return x; }

// Order-preserving key of a candidate of one beam: larger logit first, then lower token.
// 0 is below every finite logit's key and means "none".
__device__ __forceinline__ unsigned long long make_key(float x, int t) {
  const uint32_t u = __float_as_uint(x + 0.f);   // -0 and +0 are equal
  const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (static_cast<unsigned long long>(o) << 32) | (0xffffffffu - static_cast<uint32_t>(t));
}
__device__ __forceinline__ float key_logit(unsigned long long k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ int key_token(unsigned long long k) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k));
}

// A 16-byte vector of logits.
template <typename T> struct Vec {
  static constexpr int kN = 16 / sizeof(T);
  uint4 u;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w = (&u.x)[i / (kN / 4)];
    if constexpr (std::is_same_v<T, float>) {
      return __uint_as_float(w);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      return __uint_as_float(i % 2 ? (w & 0xffff0000u) : (w << 16));
    } else {
      return __half2float(__ushort_as_half(static_cast<unsigned short>(i % 2 ? w >> 16 : w)));
    }
  }
  // its largest value; NaNs do not count
  __device__ __forceinline__ float largest() const {
    if constexpr (std::is_same_v<T, float>) {
      return fmaxf(fmaxf(get(0), get(1)), fmaxf(get(2), get(3)));
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
      const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(__low2float(m), __high2float(m));
    } else {
      const __half2* h = reinterpret_cast<const __half2*>(&u);
      const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(__low2float(m), __high2float(m));
    }
  }
};

// ------------------------------------------------------------------ one slice of a row
//
// A CTA copies its slice of a row to shared memory, all copies in flight at once; from there
// it takes the maximum, then the sum of exponentials and the n best, so the logits cross HBM
// once.  The n-th largest of the threads' maxima, T, is a lower bound of the slice's n-th
// best; what is >= T, rarely more than a few n values, is gathered and ranked.
//
// Bound: HBM for fp32; for 16-bit logits the exponentials come near it (12.3 logits a clock
// and SM at the measured copy rate, of 16 exponentials), so an element costs one unpack,
// one fused multiply-add, one exponential, one addition and 1/8 of a packed maximum,
// compare and two 16-byte loads.

struct SliceShared {
  unsigned long long list[kList];
  float lane_max[kThreads];      // each warp's lane maxima, descending
  float red[kWarps];
  double sum[kWarps];
  int scan[kWarps];
  unsigned long long best[kWarps];
  int count;
  float bound;
};

// Descending bitonic sort of one value per lane.
__device__ __forceinline__ float sort_lanes(float x, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size / 2; step > 0; step >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, x, step);
      const bool up = (lane & size) != 0;            // this run ascends (the last never does)
      const bool low = (lane & step) == 0;
      x = (low != up) ? fmaxf(x, y) : fminf(x, y);
    }
  return x;
}

// Writes the largest n of c <= kList keys, descending, 0 where there are fewer.
__device__ void write_ranked(const unsigned long long* list, int c, int n, unsigned long long* out) {
  for (int i = threadIdx.x; i < c; i += kThreads) {
    const unsigned long long k = list[i];
    int rank = 0;
    for (int j = 0; j < c; ++j) rank += list[j] > k;
    if (rank < n) out[rank] = k;
  }
  for (int i = c + threadIdx.x; i < n; i += kThreads) out[i] = 0;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) beam_slice_kernel(const BeamArgs p) {
  using V = Vec<T>;
  constexpr int E = V::kN;
  extern __shared__ __align__(16) unsigned char smem[];
  V* held = reinterpret_cast<V*>(smem);
  __shared__ SliceShared sh;
  const int slice = blockIdx.x % p.slices, row = blockIdx.x / p.slices, b = row / p.K, i = row % p.K;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  grid_trigger();                // the merge may take its place once the last slices run
  // a finished or dead beam's logits decide nothing
  if ((p.finished && p.finished[row]) || !isfinite(p.scores[row])) return;
  const T* x = reinterpret_cast<const T*>(p.logits) + b * p.stride_batch + i * p.stride_beam;
  // the row as aligned 16-byte vectors; vector c holds tokens c E - mis ...; the first and the
  // last may be partial
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int vecs = (p.V + mis + E - 1) / E;
  const int v0 = static_cast<int>(static_cast<long long>(vecs) * slice / p.slices);
  const int v1 = static_cast<int>(static_cast<long long>(vecs) * (slice + 1) / p.slices);
  const uint4* base = reinterpret_cast<const uint4*>(x - mis);
  const int nv = v1 - v0;
  for (int c = tid; c < nv; c += kThreads) {
    const int t0 = (v0 + c) * E - mis;
    if (t0 >= 0 && t0 + E <= p.V) {
      copy16_async(smem_addr(held + c), base + v0 + c, true);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        reinterpret_cast<T*>(held + c)[e] = (t0 + e >= 0 && t0 + e < p.V) ? x[t0 + e] : T(-INFINITY);
    }
  }
  copy_commit();
  if (tid == 0) {
    sh.count = 0;
    sh.bound = -INFINITY;
  }
  copy_wait<0>();                // a thread looks at its own vectors only: no barrier
  float m = -INFINITY;
#pragma unroll 4
  for (int c = tid; c < nv; c += kThreads) m = fmaxf(m, held[c].largest());
  const float mine = sort_lanes(m, lane);
  sh.lane_max[tid] = mine;
  if (lane == 0) sh.red[warp] = mine;
  __syncthreads();
  m = sh.red[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, sh.red[w]);
  unsigned long long* out = p.keys + (static_cast<long long>(row) * p.slices + slice) * p.n;
  // rank of this thread's entry among all lane maxima: its place in its own warp's list and,
  // by binary search, the entries before it in the others (equal ones: lower warp first)
  if (lane < p.n) {
    int rank = lane;
#pragma unroll
    for (int o = 1; o < kWarps; ++o) {
      const int w = (warp + o) % kWarps;
      const float* other = sh.lane_max + w * 32;
      int lo = 0;
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) {
        const float y = other[lo + s - 1];
        if (w < warp ? y >= mine : y > mine) lo += s;
      }
      const float y = other[lo];
      rank += lo + (w < warp ? y >= mine : y > mine);
    }
    if (rank == p.n - 1) sh.bound = mine;
  }
  __syncthreads();
  // sum of 2^(x f - c) with f = log2 e and c = m f as rounded; what the rounding of c took is
  // put back once at the end.  Four chains of additions per thread.  Where m f could
  // overflow (a slice masked with the type's lowest value) two different logits are so far
  // apart that any small f gives the same sum.
  const float base_m = isfinite(m) ? m : 0.f, f = fabsf(base_m) < 1e30f ? kLog2e : 0x1p-64f;
  const float c0 = base_m * f;
  const float bound = sh.bound;
  float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int c = tid; c < nv; c += kThreads) {
    const V v = held[c];
#pragma unroll
    for (int e = 0; e < E; ++e) s4[e % 4] += exp2_fast(fmaf(v.get(e), f, -c0));
    if (v.largest() >= bound) {
      const int t0 = (v0 + c) * E - mis;
      for (int e = 0; e < E; ++e) {
        const float y = to_f(reinterpret_cast<const T*>(held + c)[e]);
        if (y >= bound && y > -INFINITY) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kList) sh.list[at] = make_key(y, t0 + e);
        }
      }
    }
  }
  double s = static_cast<double>(s4[0] + s4[1]) + static_cast<double>(s4[2] + s4[3]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sh.sum[warp] = s;
  __syncthreads();
  if (tid == 0) {
    s = sh.sum[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) s += sh.sum[w];
    s *= static_cast<double>(exp2f(-fmaf(base_m, f, -c0)));
    p.sums[static_cast<long long>(row) * p.slices + slice] = make_float2(m, static_cast<float>(s));
  }
  if (sh.count <= kList) {
    write_ranked(sh.list, sh.count, p.n, out);
    return;
  }
  // Rare: many values equal to the bound (a mask of the type's lowest value, coarse logits).
  // Those above it, then the first n equal ones in order of tokens, read again from memory.
  const int e0 = max(0, v0 * E - mis), e1 = min(p.V, v1 * E - mis);
  __syncthreads();
  if (tid == 0) sh.count = 0;
  __syncthreads();
  for (int t = e0 + tid; t < e1; t += kThreads) {
    const float y = to_f(x[t]);
    if (y > bound) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kList) sh.list[at] = make_key(y, t);
    }
  }
  __syncthreads();
  const int above = sh.count;
  if (above + p.n <= kList) {
    int have = 0;
    for (int t1 = e0; t1 < e1 && have < p.n; t1 += kThreads) {
      const int t = t1 + tid;
      const bool hit = t < e1 && to_f(x[t]) == bound && bound > -INFINITY;
      const uint32_t hits = __ballot_sync(0xffffffffu, hit);
      if (lane == 0) sh.scan[warp] = __popc(hits);
      __syncthreads();
      int at = have + __popc(hits & ((1u << lane) - 1)), total = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        at += w < warp ? sh.scan[w] : 0;
        total += sh.scan[w];
      }
      if (hit && at < p.n) sh.list[above + at] = make_key(bound, t);
      have += total;
      __syncthreads();
    }
    write_ranked(sh.list, above + min(have, p.n), p.n, out);
    return;
  }
  // Hundreds of values above the bound in fewer than n threads: one after another.
  unsigned long long below = ~0ull;
  for (int r = 0; r < p.n; ++r) {
    unsigned long long top = 0;
    if (below != 0)
      for (int t = e0 + tid; t < e1; t += kThreads) {
        const float y = to_f(x[t]);
        const unsigned long long key = make_key(y, t);
        if (y > -INFINITY && key < below && key > top) top = key;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long y = __shfl_xor_sync(0xffffffffu, top, o);
      top = y > top ? y : top;
    }
    if (lane == 0) sh.best[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = sh.best[w] > top ? sh.best[w] : top;
    __syncthreads();
    below = top;
    if (tid == 0) out[r] = top;
  }
}

// ------------------------------------------------------------------ the merge
//
// One CTA per request.  The n-th best of the slices' first candidates is a lower bound of the
// result's n-th best.  What reaches it gets its rank, among its beam's slices and then among
// all beams, by binary searches in the sorted lists; whoever has a rank below n writes
// itself to that place, so nothing depends on the order in which threads run.

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  double* score = reinterpret_cast<double*>(smem);                   // [K, n] descending
  int* token = reinterpret_cast<int*>(score + p.K * p.n);            // [K, n]
  double* lse = reinterpret_cast<double*>(token + p.K * p.n + (p.K * p.n & 1));   // [K]
  __shared__ int alive;
  __shared__ double head[kHeadItems], bound;
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int per_beam = p.slices * p.n;
  for (int f = tid; f < p.K * p.n; f += kMergeThreads) score[f] = -INFINITY;
  if (tid == 0) {
    alive = 0;
    bound = -INFINITY;
  }
  grid_wait();
  for (int i = warp; i < p.K; i += kMergeThreads / 32) {
    const int row = b * p.K + i;
    const bool skip = (p.finished && p.finished[row]) || !isfinite(p.scores[row]);
    double l = NAN;
    if (!skip) {
      const float2* sums = p.sums + static_cast<long long>(row) * p.slices;
      float m = -INFINITY;
      for (int s = lane; s < p.slices; s += 32) m = fmaxf(m, sums[s].x);
      m = warp_max(m);
      double t = 0.0;
      for (int s = lane; s < p.slices; s += 32) {
        const float2 ms = sums[s];
        if (ms.x > -INFINITY || isnan(ms.y)) t += ms.y * exp(static_cast<double>(ms.x) - m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      l = m + log(t);
    }
    if (lane == 0) lse[i] = l;          // not finite: a row that holds no candidate
  }
  __syncthreads();
  // the first `depth` candidates of every slice (of as many slices as fit), at least n where
  // there are as many
  const unsigned long long* all = p.keys + static_cast<long long>(b) * p.K * per_beam;
  const int lists = p.K * p.slices, depth = (p.n + lists - 1) / lists;
  const int items = min(lists * depth, kHeadItems);
  for (int f = tid; f < items; f += kMergeThreads) {
    const int list = f % lists, i = list / p.slices, r = f / lists;
    double sc = -INFINITY;
    if (isfinite(lse[i])) {
      const unsigned long long k = all[list * p.n + r];
      if (k) sc = static_cast<double>(p.scores[b * p.K + i]) + (static_cast<double>(key_logit(k)) - lse[i]);
    }
    head[f] = sc;
  }
  __syncthreads();
  for (int f = tid; f < items; f += kMergeThreads) {
    const double sc = head[f];
    int rank = 0;
    for (int o = 0; o < items; ++o) rank += head[o] > sc || (head[o] == sc && o < f);
    if (rank == p.n - 1) bound = sc;
  }
  __syncthreads();
  // each beam's candidates at or above the bound, in order
  for (int f = tid; f < p.K * per_beam; f += kMergeThreads) {
    const int i = f / per_beam, at = f % per_beam, s = at / p.n, r = at % p.n;
    if (!isfinite(lse[i])) continue;
    const unsigned long long* keys = all + i * per_beam;
    const unsigned long long k = keys[at];
    if (k == 0) continue;
    const double sc =
        static_cast<double>(p.scores[b * p.K + i]) + (static_cast<double>(key_logit(k)) - lse[i]);
    if (!(sc >= bound)) continue;
    int rank = r;
    for (int o = 0; o < p.slices && rank < p.n; ++o) {
      if (o == s) continue;
      int lo = 0, hi = p.n;              // keys of a beam are all different
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (keys[o * p.n + mid] > k) lo = mid + 1;
        else hi = mid;
      }
      rank += lo;
    }
    if (rank < p.n) {
      score[i * p.n + rank] = sc;
      token[i * p.n + rank] = key_token(k);
    }
  }
  for (int i = tid; i < p.K; i += kMergeThreads)
    if (p.finished && p.finished[b * p.K + i] && isfinite(p.scores[b * p.K + i])) {
      score[i * p.n] = p.scores[b * p.K + i];
      token[i * p.n] = p.eos;
    }
  __syncthreads();
  // the n best of all beams
  int valid = 0;
  for (int f = tid; f < p.K * p.n; f += kMergeThreads) {
    const int i = f / p.n;
    const double sc = score[f];
    if (!(sc > -INFINITY)) continue;
    ++valid;
    int rank = f % p.n;
    for (int o = 0; o < p.K && rank < p.n; ++o) {
      if (o == i) continue;
      int lo = 0, hi = p.n;
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        const double y = score[o * p.n + mid];
        if (o < i ? y >= sc : y > sc) lo = mid + 1;
        else hi = mid;
      }
      rank += lo;
    }
    if (rank < p.n) {
      const long long at = static_cast<long long>(b) * p.n + rank;
      p.tokens[at] = token[f];
      p.parents[at] = i;
      p.out_scores[at] = static_cast<float>(sc);
    }
  }
  if (valid) atomicAdd(&alive, valid);
  __syncthreads();
  for (int r = alive + tid; r < p.n; r += kMergeThreads) {
    const long long at = static_cast<long long>(b) * p.n + r;
    p.tokens[at] = -1;
    p.parents[at] = -1;
    p.out_scores[at] = -INFINITY;
  }
}

// ------------------------------------------------------------------ host

// Slices of a row of 16-byte vectors with `per` logits: as few as a CTA holds, more while
// the rows alone do not give every SM two CTAs and a slice keeps a vector for each thread.
int slices_of(long long rows, int V, int per) {
  const int vecs = V / per + 2;              // of an unaligned row
  int s = (vecs + kSlice - 1) / kSlice;
  while (rows * s < 2 * kSMs && vecs / (2 * s) >= kThreads) s *= 2;
  return s;
}

template <typename T>
int launch(const BeamArgs& p, cudaStream_t st) {
  const int vecs = p.V / Vec<T>::kN + 2;
  const size_t held = static_cast<size_t>(vecs / p.slices + 1) * 16;   // of the largest slice
  if (held > 40 * 1024 &&
      cudaFuncSetAttribute(beam_slice_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (kSlice + 1) * 16) != cudaSuccess)
    return GDN_ERR_LAUNCH;
  beam_slice_kernel<T><<<p.slices * p.B * p.K, kThreads, held, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return GDN_ERR_LAUNCH;
  const size_t smem = static_cast<size_t>(p.K) * (p.n * 12 + 8) + 8;
  if (smem > 32 * 1024 &&
      cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem)) != cudaSuccess)
    return GDN_ERR_LAUNCH;
  return launch_after(beam_merge_kernel, dim3(p.B), dim3(kMergeThreads), smem, st, p) == cudaSuccess
             ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // namespace

extern "C" {

size_t gdn_beam_select_workspace_bytes(int B, int K, int V, int n) {
  if (B < 1 || K < 1 || V < 1 || n < 1) return 0;
  const long long rows = static_cast<long long>(B) * K;
  return static_cast<size_t>(rows) * std::max(slices_of(rows, V, 4), slices_of(rows, V, 8)) * (static_cast<size_t>(n) * 8 + 8);
}

int gdn_beam_select(const void* logits, int dtype, int64_t stride_batch, int64_t stride_beam,
                    const float* scores, const uint8_t* finished, int eos_token, int B, int K,
                    int V, int n, int32_t* tokens, int32_t* parents, float* new_scores,
                    void* workspace, size_t workspace_bytes, void* stream) {
  if (B < 0 || K < 1 || V < 1 || n < 1) return GDN_ERR_SHAPE;
  if (K > kMaxBeams || n > kMaxSelected) return GDN_ERR_LIMIT;
  if (static_cast<long long>(B) * K > 0x7fffffffLL / kMaxSelected) return GDN_ERR_SHAPE;
  if (dtype != GDN_DTYPE_BF16 && dtype != GDN_DTYPE_FP16 && dtype != GDN_DTYPE_FP32) return GDN_ERR_ARG;
  if (stride_batch < 0 || stride_beam < 0) return GDN_ERR_ARG;
  if (finished && (eos_token < 0 || eos_token >= V)) return GDN_ERR_ARG;
  if (B == 0) return GDN_OK;
  if (!logits || !scores || !tokens || !parents || !new_scores || !workspace) return GDN_ERR_NULL;
  if (!aligned(logits, dtype == GDN_DTYPE_FP32 ? 4 : 2) || !aligned(scores, 4) || !aligned(tokens, 4) ||
      !aligned(parents, 4) || !aligned(new_scores, 4) || !aligned(workspace, 16))
    return GDN_ERR_ALIGN;
  if (static_cast<long long>(B) * K * std::max(slices_of(1LL * B * K, V, 4), slices_of(1LL * B * K, V, 8)) >
      0x7fffffffLL)
    return GDN_ERR_SHAPE;
  if (workspace_bytes < gdn_beam_select_workspace_bytes(B, K, V, n)) return GDN_ERR_SHAPE;
  BeamArgs p{};
  p.logits = logits; p.scores = scores; p.finished = finished; p.tokens = tokens;
  p.parents = parents; p.out_scores = new_scores;
  p.slices = slices_of(static_cast<long long>(B) * K, V, dtype == GDN_DTYPE_FP32 ? 4 : 8);
  p.keys = static_cast<unsigned long long*>(workspace);
  p.sums = reinterpret_cast<float2*>(p.keys + static_cast<size_t>(B) * K * p.slices * n);
  p.stride_batch = stride_batch; p.stride_beam = stride_beam;
  p.B = B; p.K = K; p.V = V; p.n = n; p.eos = eos_token;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == GDN_DTYPE_BF16) return launch<__nv_bfloat16>(p, st);
  if (dtype == GDN_DTYPE_FP16) return launch<__half>(p, st);
  return launch<float>(p, st);
}

}  // extern "C"
