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
constexpr int kBatch = 4;        // 16-byte vectors of logits a thread takes at a time
constexpr int kTop = 32 / kWarps;  // lane maxima of each warp, up to kSharp-th largest of all of them
// is a bound; for larger n the warps' own ones are about as sharp, and cheaper.  The one / the other:
// 18 x 10 rows of 151936 logits, n = 20: 23.8 / 26.1 us; 8 x 12 of 116858, n = 24: 18.1 / 17.5 us.
constexpr int kSharp = 20;
constexpr int kList = 1024;      // vectors, then candidates, that a slice gathers
constexpr int kMergeThreads = 512;
constexpr int kHeadItems = 256;  // of the merge's bound, at most 256
constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLn2 = 0.69314718055994530942;

struct BeamArgs {
  const void* logits;
  const float* scores;
  const uint8_t* finished;
  int32_t* tokens;
  int32_t* parents;
  float* out_scores;
  unsigned long long* keys;   // workspace [rows, slices, n]: keys, descending, 0 = none
  float2* sums;               // workspace [rows, slices]: m, sum 2^(x log2 e - reference(m)), or, of
                              // |m| > kHuge, how many logits are m
  long long stride_batch, stride_beam;
  int B, K, V, n, eos, slices;
  uint32_t per_mul, per_shift;   // division by slices n
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
// A row's slices are counted in vectors of 16 bytes from its first token, and a row that need
// not begin on a 16-byte boundary is read in words of 32 bits (64 x 8 rows of 151937 bf16
// logits: 48 us, of 151936 43.5): equal rows get equal sums, bit for bit, wherever they lie, so
// that equal beams tie.
//
// One pass over the slice.  Every thread keeps its own running maximum and its sum of
// exponentials relative to it, so the loop has no barrier; its next batch of vectors is in
// flight while it works on one.  The first batch is a sample spread over the slice, which gives a
// bound T that n logits reach: the n-th largest of the warps' four largest lane maxima, or
// for larger n the smallest of the warps' ceil(n / warps)-th largest.  Vectors that reach T are set
// aside as they are; at the end the n-th largest of their maxima is a sharper bound, and what
// reaches that is ranked.  Raising T on the way takes barriers, which cost more than it saves
// (64 x 8 rows of 151936 logits: 47 us with, 43 without).
//
// Bound: of 16-bit logits no one unit, but two near each other: 90 warp instructions are issued for a vector of
// eight (counted, with sampling, what is set aside and ranking in them; the sums take 24), and one exponential a
// logit, of which an SM does 16 a clock.  64 x 8 rows of 151936 bf16 logits, a tenth finished: 39 us (140 MB,
// 3.6 TB/s; a copy's rate would read them in 21), in which the SMs work 81% of the time (906 slices on 592
// places) and then issue in 62% and have the exponential pipe busy in 60% of the cycles, 26 of 64 warps
// resident.  8 x 32 rows of 50257 fp32, a quarter finished: 16 us (39 MB, 2.4 TB/s) in one wave of 576 slices: the life
// of one, sample, five batches, gathering and ranking, 113 instructions for a vector of four; issue
// 56%, exponentials 38% of the cycles.
// Tried there without gain: three to eight CTAs an SM (41 to 72 us), batches of 2 and 8, a ring
// of asynchronous copies through shared memory (50), places by ballots (55).

struct SliceShared {
  uint4 vec[kList];                // vectors that reach T
  int at[kList];                   // their places in the row
  unsigned long long list[kList];  // keys of candidates
  float red[kWarps];
  float top[32];                   // its own place: red is written again without a barrier between
  double sum[kWarps];
  double folded[kThreads];         // each thread's sum but for its chains
  int scan[kWarps];
  unsigned long long best[kWarps];
  float sample[kThreads];        // of the keys, where they overflow
  int count, keys;
  float bound;
};

// Sums of 2^(x log2 e - c) in two packed chains; one fused multiply-add and one addition do
// two elements.
struct ExpSum {
  unsigned long long s[2] = {0ull, 0ull};
  static __device__ __forceinline__ unsigned long long pack(float lo, float hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
  }
  static __device__ __forceinline__ void unpack(unsigned long long x, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
  }
  __device__ __forceinline__ void add(int chain, float x0, float x1, unsigned long long minus_c) {
    unsigned long long t;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t) : "l"(pack(x0, x1)), "l"(pack(kLog2e, kLog2e)), "l"(minus_c));
    float a, b;
    unpack(t, a, b);
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(s[chain]) : "l"(pack(exp2_fast(a), exp2_fast(b))));
  }
  __device__ __forceinline__ void scale(float f) {     // f a power of two: exact
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(s[i]) : "l"(pack(f, f)));
  }
  __device__ __forceinline__ void clear() { s[0] = s[1] = 0ull; }
  __device__ __forceinline__ float total() const {
    float a, b, c, d;
    unpack(s[0], a, b);
    unpack(s[1], c, d);
    return (a + b) + (c + d);
  }
};

// Two different logits from here on are 64 or more apart, so only the largest counts; below, m log2 e
// as rounded is off by 32 at most, so that sums relative to it stay within fp32.
constexpr float kHuge = 536870912.f;   // 2^29

// The whole number c that a maximum m's exponentials are taken relative to, as 2^(x log2 e - c):
// changing it, as the maximum grows or slices meet, scales a sum by a power of two, without an error.
__device__ __forceinline__ float reference(float m) {
  return rintf(fminf(fmaxf(m, -kHuge), kHuge) * kLog2e);
}
// 2^d for a whole d <= 0, 0 below the normal numbers
__device__ __forceinline__ float power_of_two(float d) {
  return __int_as_float((static_cast<int>(fmaxf(d, -127.f)) + 127) << 23);
}

// One place of a list.  Few lanes of a warp ask at a time, so each asks for itself.
__device__ __forceinline__ int next_place(int* count) {
  int at;
  asm volatile("atom.shared.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(smem_addr(count)) : "memory");
  return at;
}

// The warp's largest x, by one reduction; NaNs do not count.
__device__ __forceinline__ float warp_largest(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// The warp's r-th largest x, equal ones counted one by one.
__device__ __forceinline__ float warp_nth(float x, int r) {
  float y = warp_largest(x);
  for (int i = 1; i < r; ++i) {
    const uint32_t same = __ballot_sync(0xffffffffu, x == y);
    if (same == 0u) return -INFINITY;                  // only NaNs are left
    if (threadIdx.x % 32 == __ffs(same) - 1) x = -INFINITY;
    y = warp_largest(x);
  }
  return y;
}

// Writes the largest n of c <= kList keys, descending, 0 where there are fewer.
__device__ void write_ranked(const unsigned long long* list, int c, int n, unsigned long long* out) {
  for (int i = threadIdx.x; i < c; i += kThreads) {
    const unsigned long long k = list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < c; ++j) rank += list[j] > k;
    if (rank < n) out[rank] = k;
  }
  for (int i = c + threadIdx.x; i < n; i += kThreads) out[i] = 0;
}

// kShift: rows need not begin on a 16-byte boundary.
template <typename T, bool kShift>
__global__ void __launch_bounds__(kThreads, 4) beam_slice_kernel(const BeamArgs p) {
  using V = Vec<T>;
  constexpr int E = V::kN;
  __shared__ SliceShared sh;
  const int slice = blockIdx.y, row = blockIdx.x, b = row / p.K, i = row - b * p.K;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  grid_trigger();                // the merge may take its place once the last slices run
  // a finished or dead beam's logits decide nothing
  const bool done = p.finished != nullptr && p.finished[row];
  if (done | !isfinite(p.scores[row])) return;
  const T* x = reinterpret_cast<const T*>(p.logits) + b * p.stride_batch + i * p.stride_beam;
  // vector c holds tokens c E ...; the row's end is read token by token
  const int vecs = (p.V + E - 1) / E, whole = p.V / E;
  const int each = vecs / p.slices, more = vecs - each * p.slices;   // the first `more` get one more
  const int v0 = slice * each + min(slice, more), v1 = v0 + each + (slice < more ? 1 : 0);
  // kShift with 16-bit tokens: the row begins in the middle of a word, so that the first and
  // the last word read hold a token outside the row beside one of its own
  const bool half = sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(x) & 2);
  const uint32_t* words = reinterpret_cast<const uint32_t*>(x - (half ? 1 : 0));
  // batch j of thread tid: vectors v0 + (j + k batches) 256 + tid, k < kBatch
  const int batches = (v1 - v0 + kThreads * kBatch - 1) / (kThreads * kBatch);
  // what is in flight: words as they lie, put in place when their turn comes
  struct Raw {
    uint32_t w[kShift && E == 8 ? 5 : 4];
  };
  // -inf throughout
  constexpr uint32_t none = std::is_same_v<T, float> ? 0xff800000u
                            : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;
  auto load = [&](Raw (&raw)[kBatch], int j) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int c = v0 + (j + k * batches) * kThreads + tid;
      uint32_t (&w)[sizeof(Raw) / 4] = raw[k].w;
#pragma unroll
      for (int i = 0; i < sizeof(Raw) / 4; ++i) w[i] = none;
      if (c < min(v1, whole)) {
        if constexpr (!kShift) {
          const uint4 u = __ldcs(reinterpret_cast<const uint4*>(x) + c);
          w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = __ldg(words + 4 * c + i);
          if constexpr (E == 8)
            if (half) w[4] = __ldg(words + 4 * c + 4);
        }
      } else if (c < v1) {
        T end[sizeof(Raw) / sizeof(T)];
        const int first = c * E - (half ? 1 : 0);
#pragma unroll 1
        for (int e = 0; e < sizeof(Raw) / sizeof(T); ++e)
          end[e] = first + e >= c * E && first + e < p.V ? x[first + e] : T(-INFINITY);
#pragma unroll
        for (int i = 0; i < sizeof(Raw) / 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(end)[i];
      }
    }
  };
  auto vector = [&](const Raw& raw) {
    uint4 u = make_uint4(raw.w[0], raw.w[1], raw.w[2], raw.w[3]);
    if constexpr (kShift && E == 8)
#pragma unroll
      for (int i = 0; i < 4; ++i) (&u.x)[i] = __funnelshift_r(raw.w[i], raw.w[i + 1], half ? 16 : 0);
    return V{u};
  };
  V v[kBatch];
  Raw next[kBatch];
  load(next, 0);
  if (tid == 0) {
    sh.count = sh.keys = 0;
    sh.bound = -INFINITY;
  }
  float m = -INFINITY;           // this thread's largest logit
#pragma unroll
  for (int k = 0; k < kBatch; ++k) v[k] = vector(next[k]);
#pragma unroll
  for (int k = 0; k < kBatch; ++k) m = fmaxf(m, v[k].largest());
  float bound;
  if (p.n <= kSharp) {
    // the n-th largest of the warps' kTop largest lane maxima
    float x = m, mine = -INFINITY;
#pragma unroll
    for (int i = 0; i < kTop; ++i) {
      const float y = warp_largest(x);
      if (lane == i) mine = y;
      const uint32_t same = __ballot_sync(0xffffffffu, x == y);
      if (same && lane == __ffs(same) - 1) x = -INFINITY;
    }
    if (lane < kTop) sh.top[warp * kTop + lane] = fmaxf(mine, -FLT_MAX);
    __syncthreads();
    const float y = sh.top[lane];
    int reach = 0;               // of the 32 are at least y
#pragma unroll
    for (int i = 0; i < 32; ++i) reach += sh.top[i] >= y;
    bound = warp_largest(reach >= p.n ? y : -INFINITY);
  } else {
    const float nth = warp_nth(m, (p.n + kWarps - 1) / kWarps);
    if (lane == 0) sh.top[warp] = nth;
    __syncthreads();
    bound = sh.top[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) bound = fminf(bound, sh.top[w]);
  }
  unsigned long long* out = p.keys + (static_cast<long long>(row) * p.slices + slice) * p.n;
  // The sum of 2^(x log2 e - c0), in four chains of at most 32 additions (kFold batches), then in 64 bits in
  // shared memory, where it takes no registers from the loop (with it there 44.8 us instead of
  // 43.5 for 64 x 8 rows of 151936 bf16 logits; with chains as long as the slice, whose error grows with it, 43.1).
  constexpr int kFold = 4;
  float c0 = reference(m);
  ExpSum sums;
  sh.folded[tid] = 0.0;
  auto fold = [&]() {
    sh.folded[tid] += sums.total();
    sums.clear();
  };
  bound = fmaxf(bound, -FLT_MAX);   // vectors of -inf alone never count
  auto set_aside = [&](const V& w, int c) {
    const int at = next_place(&sh.count);
    if (at < kList) {
      sh.vec[at] = w.u;
      sh.at[at] = c;
    }
  };
  // A thread keeps its reference until a logit is 7.5 binades above it (4 binades: 44.8 us), since some
  // lane's maximum grows in nearly every batch.
  auto raise = [&](float top) {
    const float c1 = reference(top), f = power_of_two(c0 - c1);
    sums.scale(f);
    sh.folded[tid] *= f;
    c0 = c1;
  };
  for (int j = 0;; ++j) {
    if (j + 1 < batches) load(next, j + 1);
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float t = v[k].largest();
      if (t >= bound) set_aside(v[k], v0 + (j + k * batches) * kThreads + tid);
      top = fmaxf(top, t);
    }
    m = fmaxf(m, top);
    if (top > (c0 + 7.5f) * static_cast<float>(kLn2)) raise(top);
    const unsigned long long minus_c = ExpSum::pack(-c0, -c0);
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
#pragma unroll
      for (int e = 0; e < E; e += 2) sums.add(e / 2 % 2, v[k].get(e), v[k].get(e + 1), minus_c);
    if (j + 1 >= batches) break;
    if (j % kFold == kFold - 1) fold();
#pragma unroll
    for (int k = 0; k < kBatch; ++k) v[k] = vector(next[k]);
  }
  // the CTA's maximum and sum
  const float wm = warp_largest(m);
  if (lane == 0) sh.red[warp] = wm;
  __syncthreads();
  m = sh.red[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, sh.red[w]);
  fold();
  double part = sh.folded[tid] * power_of_two(c0 - reference(m));
  const int e0 = v0 * E, e1 = min(p.V, v1 * E);   // the slice's tokens
  if (fabsf(m) > kHuge && isfinite(m)) {
    int equal = 0;
    bool broken = false;
    for (int t = e0 + tid; t < e1; t += kThreads) {
      const float y = to_f(x[t]);
      equal += y == m;
      broken |= isnan(y);
    }
    part = broken ? NAN : equal;
  }
  part = warp_sum(part);
  if (lane == 0) sh.sum[warp] = part;
  __syncthreads();
  if (tid == 0) {
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += sh.sum[w];
    p.sums[static_cast<long long>(row) * p.slices + slice] = make_float2(m, static_cast<float>(s));
  }
  // a sharper bound from up to 256 of the vectors set aside, as before: whole warps of them,
  // where there is more to rank than a candidate a thread
  const int aside = min(sh.count, kList), wide = min(aside, kThreads) / 32;
  const int nth = aside * E > kThreads && wide > 0 ? (p.n + wide - 1) / wide : 33;
  if (warp < wide && nth <= 32) {
    const float y = warp_nth(V{sh.vec[tid]}.largest(), nth);
    if (lane == 0) sh.red[warp] = y;
  }
  __syncthreads();
  if (nth <= 32) {               // at least the bound before
    bound = sh.red[0];
    for (int w = 1; w < wide; ++w) bound = fminf(bound, sh.red[w]);
  }
  bool full = sh.count > kList;
  if (!full) {
    for (int f = tid; f < aside * E; f += kThreads) {
      const float y = to_f(reinterpret_cast<const T*>(sh.vec)[f]);
      if (y >= bound) {
        const int at = next_place(&sh.keys);
        if (at < kList) sh.list[at] = make_key(y, sh.at[f / E] * E + f % E);
      }
    }
    __syncthreads();
    full = sh.keys > kList;
  }
  // The sample missed where the large ones are: read the slice again with the higher bound,
  // raised from what was gathered until it fits or does not rise.
  if (full) {
    float last = -INFINITY;      // below any bound
    while (bound > last) {
      __syncthreads();
      if (tid == 0) sh.keys = 0;
      __syncthreads();
      for (int t = e0 + tid; t < e1; t += kThreads) {
        const float z = to_f(x[t]);
        if (z >= bound) {
          const int at = atomicAdd(&sh.keys, 1);
          if (at < kList) sh.list[at] = make_key(z, t);
        }
      }
      __syncthreads();
      full = sh.keys > kList;
      if (!full) break;
      const float y = key_logit(sh.list[tid]);
      sh.sample[tid] = y;
      __syncthreads();
      int rank = 0;
      for (int o = 0; o < kThreads; ++o) rank += sh.sample[o] > y || (sh.sample[o] == y && o < tid);
      if (rank == p.n - 1) sh.bound = y;
      __syncthreads();
      last = bound;
      bound = sh.bound;
    }
  }
  if (!full) {
    write_ranked(sh.list, sh.keys, p.n, out);
    return;
  }
  // Rare: many values equal to the bound (a mask of the type's lowest value, coarse logits).
  // Those above it, then the first n equal ones in order of tokens, read again from memory.
  __syncthreads();
  if (tid == 0) sh.keys = 0;
  __syncthreads();
  for (int t = e0 + tid; t < e1; t += kThreads) {
    const float y = to_f(x[t]);
    if (y > bound) {
      const int at = atomicAdd(&sh.keys, 1);
      if (at < kList) sh.list[at] = make_key(y, t);
    }
  }
  __syncthreads();
  const int above = sh.keys;
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
// One CTA per request.  The n-th best of the first candidates of live beams' slices, 4 n of them, is a
// lower bound of the result's n-th best (64 x 8 beams of 151936, 16 chosen: with 1 / 2 / 4 / 8 n
// 49.2 / 49.3 / 45.6 / 46.5 us).  What reaches it is gathered, and whoever has fewer than n better ones
// writes itself to that place, so nothing depends on the order in which threads run.  Where
// few beams are far ahead that bound is loose, and the n-th best of 256 of those gathered
// raises it first: 8 requests of 32 beams, 32 chosen, scores spread by 1: 22 us in all instead of 49.
// With more of them than the list holds (many equal scores) the ranks come from binary
// searches in the sorted lists instead.
//
// Bound: latency, of three dependent reads and the two ranks: 6 us behind the slices for 8
// requests of 32 beams, 32 chosen (with 128-bit items instead of 64-bit scores and ties apart
// 8; with one thread to an item instead of four 9).

constexpr int kMergeList = 1024, kHeld = 8;
constexpr int kTokenBits = 26;   // of the vocabulary (checked on the host)

// A candidate as two numbers that order like it: the score's bits; the lower beam, then the
// larger logit, then the lower token.
struct __align__(16) MergeItem {
  unsigned long long hi, lo;
};
__device__ __forceinline__ unsigned long long ordered(double x) {
  const unsigned long long u = __double_as_longlong(x + 0.0);   // -0 and +0 are equal
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double from_ordered(unsigned long long o) {
  return __longlong_as_double(o >> 63 ? o & 0x7fffffffffffffffull : ~o);
}
__device__ __forceinline__ MergeItem make_item(double score, int beam, unsigned long long key) {
  constexpr unsigned long long tokens = (1ull << kTokenBits) - 1;
  return MergeItem{ordered(score), static_cast<unsigned long long>(kMaxBeams - 1 - beam) << 58 |
                                       (key >> 32) << kTokenBits | (key & tokens)};
}

// ln(t) for normal t: the fraction's logarithm in fp32 (6e-8), the exponent's in 64 bits
__device__ __forceinline__ double ln_sum(double t) {
  const unsigned long long u = __double_as_longlong(t);
  const int e = static_cast<int>(u >> 52) - 1023;
  const double f = __longlong_as_double((u & 0x000fffffffffffffull) | 0x3ff0000000000000ull);
  return e * kLn2 + static_cast<double>(logf(static_cast<float>(f)));
}

// over a group of N lanes; other groups of the warp may have left the loop
template <int N, typename T> __device__ __forceinline__ T group_sum(T x) {
  const uint32_t mask = ((1u << N) - 1) << (threadIdx.x & (32 - N));
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) x += __shfl_xor_sync(mask, x, o);
  return x;
}
template <int N> __device__ __forceinline__ float group_max(float x) {
  const uint32_t mask = ((1u << N) - 1) << (threadIdx.x & (32 - N));
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(mask, x, o));
  return x;
}

__global__ void __launch_bounds__(kMergeThreads, 2) beam_merge_kernel(const __grid_constant__ BeamArgs p) {
  __shared__ double lse[kMaxBeams], cum[kMaxBeams], bound;
  __shared__ float least[kMaxBeams];       // logits below are below the bound, by beam
  __shared__ unsigned long long head[kHeadItems];
  __shared__ MergeItem item[kMergeList];
  __shared__ int count;
  __shared__ bool done[kMaxBeams];
  __shared__ int live_beam[kMaxBeams], live;   // beams with candidates of their own
  const int b = blockIdx.x, tid = threadIdx.x;
  const int per_beam = p.slices * p.n, lists = p.K * p.slices, total = lists * p.n;
  if (tid == 0) {
    count = 0;
    bound = -INFINITY;
  }
  if (tid < p.K) {
    const float c = p.scores[b * p.K + tid];
    cum[tid] = c;
    done[tid] = p.finished && p.finished[b * p.K + tid];
  }
  __syncthreads();
  if (tid < 32) {
    int before = 0;
    for (int i = tid; i - tid < p.K; i += 32) {
      const bool on = i < p.K && !done[i] && isfinite(cum[i]);
      const uint32_t all_on = __ballot_sync(0xffffffffu, on);
      if (on) live_beam[before + __popc(all_on & ((1u << tid) - 1))] = i;
      before += __popc(all_on);
    }
    if (tid == 0) live = before;
  }
  __syncthreads();
  grid_wait();
  // everything that is read comes at once: up to kHeld keys a thread, the first `depth`
  // candidates of every live beam's slices (of as many as fit), and the slices' sums, eight
  // threads to a beam
  const unsigned long long* all = p.keys + static_cast<long long>(b) * total;
  unsigned long long held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    const int f = u * kMergeThreads + tid;
    held[u] = f < total ? all[f] : 0;
  }
  const int live_lists = live * p.slices;
  const int depth = live ? min(p.n, (4 * p.n + live_lists - 1) / live_lists) : 0;
  const int items = min(live_lists * depth, kHeadItems);
  unsigned long long head_key = 0;
  int head_beam = 0;
  if (tid < items) {
    const int l = tid % live_lists, i = l / p.slices;
    head_beam = live_beam[i];
    head_key = all[(head_beam * p.slices + l - i * p.slices) * p.n + tid / live_lists];
  }
  const int i8 = tid / 8, s8 = tid % 8;
  if (i8 < p.K) {
    double l = NAN;                     // not finite: a beam without candidates of its own
    const bool on = !done[i8] && isfinite(cum[i8]);
    const float2* sums = p.sums + (static_cast<long long>(b) * p.K + i8) * p.slices;
    const float2 first = on && s8 < p.slices ? sums[s8] : make_float2(-INFINITY, 0.f);
    float m = first.x;
    if (on)
      for (int s = s8 + 8; s < p.slices; s += 8) m = fmaxf(m, sums[s].x);
    m = group_max<8>(m);
    const bool huge = fabsf(m) > kHuge;
    const float c = reference(m);
    auto term = [&](float2 ms) {
      if (!(ms.x > -INFINITY || isnan(ms.y))) return 0.0;
      const float f = huge || fabsf(ms.x) > kHuge ? (ms.x == m || isnan(ms.y) ? 1.f : 0.f)
                                                  : power_of_two(reference(ms.x) - c);
      return static_cast<double>(ms.y) * f;
    };
    double t = term(first);
    if (on)
      for (int s = s8 + 8; s < p.slices; s += 8) t += term(sums[s]);
    t = group_sum<8>(t);
    // sum 2^(x L - c) with L = log2 e as rounded is e^(m (L ln 2 - 1)) 2^-c sum e^x, near enough for x
    // that are not far below m
    if (on && isfinite(m) && t > 0.0 && t < 1e300)
      l = (huge ? static_cast<double>(m) : c * kLn2 - m * (kLog2e * kLn2 - 1.0)) + ln_sum(t);
    if (s8 == 0) lse[i8] = l;
  }
  __syncthreads();
  auto score_of = [&](int i, unsigned long long k) {
    return cum[i] + (static_cast<double>(key_logit(k)) - lse[i]);
  };
  if (tid < items) {
    // all different: the last 8 bits are the place instead of the score's, which rounds down
    head[tid] = (ordered(head_key && isfinite(lse[head_beam]) ? score_of(head_beam, head_key) : -INFINITY) & ~255ull) |
                static_cast<unsigned>(tid);
  }
  __syncthreads();
  // bound = the n-th best of head's first `items`; four threads count for one
  auto rank_head = [&](int items) {
    for (int f = tid / 4; f < items; f += kMergeThreads / 4) {
      const unsigned long long sc = head[f];
      int rank = 0;
#pragma unroll 4
      for (int o = tid % 4; o < items; o += 4) rank += head[o] > sc;
      rank = group_sum<4>(rank);
      if (rank == p.n - 1) {
        const double low = from_ordered(sc & ~255ull);
        bound = isfinite(low) ? low : -INFINITY;
      }
    }
    __syncthreads();
  };
  if (items >= p.n) rank_head(items);
  double low = bound;
  for (;;) {
    // below this logit no score reaches the bound: rounded down, far below what rounding the
    // score in 64 bits can move; NaN for a beam without candidates, -inf without a bound
    if (tid < p.K) {
      const double x = low - cum[tid] + lse[tid];
      least[tid] = !isfinite(lse[tid]) ? NAN
                   : !isfinite(x)      ? -INFINITY
                                       : static_cast<float>(x - 1e-6 * (1.0 + fabs(x)));
    }
    __syncthreads();
    auto take = [&](int f, unsigned long long k) {
      const int i = static_cast<int>(div_by(f, p.per_mul, p.per_shift));
      if (k == 0 || !(key_logit(k) >= least[i])) return;
      const double sc = score_of(i, k);
      if (!(sc >= low)) return;
      const int at = next_place(&count);
      if (at < kMergeList) item[at] = make_item(sc, i, k);
    };
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (u * kMergeThreads + tid < total) take(u * kMergeThreads + tid, held[u]);
    for (int f = kHeld * kMergeThreads + tid; f < total; f += kMergeThreads) take(f, all[f]);
    if (tid < p.K && done[tid] && isfinite(cum[tid]) && cum[tid] >= low) {
      const int at = next_place(&count);
      if (at < kMergeList) item[at] = make_item(cum[tid], tid, 0);
    }
    __syncthreads();
    // Many where a few beams are far ahead of the others: the n-th best of some of them is a
    // higher bound.
    const int got = min(count, kMergeList), sample = min(got, kHeadItems);
    if (got <= kHeadItems) break;
    if (tid < sample) head[tid] = (item[tid * got / sample].hi & ~255ull) | static_cast<unsigned>(tid);
    __syncthreads();
    rank_head(sample);
    if (!(bound > low)) break;   // equal ones, ranked below
    if (tid == 0) count = 0;
    low = bound;
  }
  // (rank, score, beam, token); with a bound there are n candidates at least
  auto place = [&](int rank, double sc, int i, int token) {
    const long long at = static_cast<long long>(b) * p.n + rank;
    p.tokens[at] = done[i] ? p.eos : token;
    p.parents[at] = i;
    p.out_scores[at] = static_cast<float>(sc);
  };
  const int alive = low > -INFINITY ? p.n : count;
  if (count <= kMergeList) {
    for (int f = tid / 4; f < count; f += kMergeThreads / 4) {
      const MergeItem me = item[f];
      int rank = 0, same = 0;
#pragma unroll 4
      for (int o = tid % 4; o < count; o += 4) {
        const unsigned long long hi = item[o].hi;
        rank += hi > me.hi;
        same += hi == me.hi;
      }
      if (group_sum<4>(same) > 1)        // equal scores: by beam, logit, token
        for (int o = tid % 4; o < count; o += 4) rank += item[o].hi == me.hi && item[o].lo > me.lo;
      rank = group_sum<4>(rank);
      if (rank < p.n && tid % 4 == 0)
        place(rank, from_ordered(me.hi), kMaxBeams - 1 - static_cast<int>(me.lo >> 58),
              static_cast<int>(0xffffffffu - (static_cast<uint32_t>(me.lo) | ~((1u << kTokenBits) - 1))));
    }
  } else {
    // better ones in every list: higher scores, and equal ones of lower beams or, within the
    // beam, larger keys
    for (int f = tid; f < total + p.K; f += kMergeThreads) {
      const int i = f < total ? f / per_beam : f - total;
      unsigned long long k = ~0ull;
      double sc = cum[i];
      if (f < total) {
        k = isfinite(lse[i]) ? all[f] : 0;
        if (k == 0) continue;
        sc = score_of(i, k);
      } else if (!done[i]) {
        continue;
      }
      if (!(sc >= low) || !isfinite(sc)) continue;
      int rank = 0;
      for (int o = 0; o < p.K && rank < p.n; ++o) {
        if (done[o]) {
          rank += isfinite(cum[o]) && (cum[o] > sc || (cum[o] == sc && o < i));
          continue;
        }
        if (!isfinite(lse[o])) continue;
        for (int l = o * p.slices; l < (o + 1) * p.slices && rank < p.n; ++l) {
          int lo = 0, hi = p.n;
          while (lo < hi) {
            const int mid = (lo + hi) / 2;
            const unsigned long long q = all[l * p.n + mid];
            const double y = q ? score_of(o, q) : -INFINITY;
            if (y > sc || (y == sc && (o < i || (o == i && q > k)))) lo = mid + 1;
            else hi = mid;
          }
          rank += lo;
        }
      }
      if (rank < p.n) place(rank, sc, i, key_token(k));
    }
  }
  for (int r = alive + tid; r < p.n; r += kMergeThreads) {
    const long long at = static_cast<long long>(b) * p.n + r;
    p.tokens[at] = -1;
    p.parents[at] = -1;
    p.out_scores[at] = -INFINITY;
  }
}

// ------------------------------------------------------------------ host

// Slices of a row of 16-byte vectors with `per` logits: more while the rows alone do not
// give every SM two CTAs and a slice keeps a vector for each thread, on to 500 CTAs (of 592
// that are resident) while a slice keeps four batches, and on to twelve an SM while it keeps 65536 logits,
// or for n > 16 four batches: a longer slice sets more aside.  1 / 2 / 3 / 4 slices, n = 16: 64 x 8 rows of
// 151936 bf16 logits 45 / 43 / 47 / 48 us, 55 x 10 of 80000 28 / 30 / 36 / 39, 18 x 10 of 151936 31 / 25
// / 24 / 24, 64 x 8 of 100352 fp32 41 / 44 / 46 / 49; n = 64: 8 x 32 of 100352 bf16 92 / 53 / 42 / 46.
int slices_of(long long rows, int V, int per, int n) {
  const int vecs = (V + per - 1) / per, batches = 4 * kThreads * kBatch;
  const int enough = n <= 16 ? 65536 / per : batches;
  int s = 1;
  while (rows * s < 2 * kSMs && vecs / (2 * s) >= kThreads) s *= 2;
  while (rows * s < 500 && vecs / (s + 1) >= batches) ++s;
  while (rows * s < 12 * kSMs && vecs / (s + 1) >= enough) ++s;
  return s;
}

template <typename T>
int launch(const BeamArgs& p, cudaStream_t st) {
  const dim3 grid(p.B * p.K, p.slices);
  if (reinterpret_cast<uintptr_t>(p.logits) % 16 != 0 ||
      (p.B > 1 && p.stride_batch * sizeof(T) % 16 != 0) ||
      (p.K > 1 && p.stride_beam * sizeof(T) % 16 != 0))
    beam_slice_kernel<T, true><<<grid, kThreads, 0, st>>>(p);
  else
    beam_slice_kernel<T, false><<<grid, kThreads, 0, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return GDN_ERR_LAUNCH;
  return launch_after(beam_merge_kernel, dim3(p.B), dim3(kMergeThreads), 0, st, p) == cudaSuccess
             ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // namespace

extern "C" {

size_t gdn_beam_select_workspace_bytes(int B, int K, int V, int n) {
  if (B < 1 || K < 1 || V < 1 || n < 1) return 0;
  const long long rows = static_cast<long long>(B) * K;
  return static_cast<size_t>(rows) * std::max(slices_of(rows, V, 4, n), slices_of(rows, V, 8, n)) * (static_cast<size_t>(n) * 8 + 8);
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
  if (V > 1 << kTokenBits) return GDN_ERR_SHAPE;     // also keeps the slices of a row below 2^16
  if (workspace_bytes < gdn_beam_select_workspace_bytes(B, K, V, n)) return GDN_ERR_SHAPE;
  BeamArgs p{};
  p.logits = logits; p.scores = scores; p.finished = finished; p.tokens = tokens;
  p.parents = parents; p.out_scores = new_scores;
  p.slices = slices_of(static_cast<long long>(B) * K, V, dtype == GDN_DTYPE_FP32 ? 4 : 8, n);
  p.keys = static_cast<unsigned long long*>(workspace);
  p.sums = reinterpret_cast<float2*>(p.keys + static_cast<size_t>(B) * K * p.slices * n);
  p.stride_batch = stride_batch; p.stride_beam = stride_beam;
  p.B = B; p.K = K; p.V = V; p.n = n; p.eos = eos_token;
  div_constants(static_cast<uint32_t>(p.slices * n), p.per_mul, p.per_shift);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == GDN_DTYPE_BF16) return launch<__nv_bfloat16>(p, st);
  if (dtype == GDN_DTYPE_FP16) return launch<__half>(p, st);
  return launch<float>(p, st);
}

}  // extern "C"
