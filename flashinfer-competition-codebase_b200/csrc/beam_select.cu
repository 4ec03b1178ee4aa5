// beam_select.cu — beam search's selection over beams and vocabulary.
//
// For each request, the candidates (beam i, token t) with
//   score(i, t) = scores[i] + (logits[i, t] - lse_i),   lse_i = ln(sum_t exp(logits[i, t]))
// and, for a finished beam, the one candidate (i, eos) with score scores[i].  The n best are
// returned in descending order; candidates of one beam are ordered by logit, equal ones by
// token, and beams' candidates are merged by score in 64 bits, equal ones by beam.  What
// has no finite score (masked tokens at -inf, dead beams at -inf, rows with a NaN) is never
// chosen; places left over get token -1, parent -1, score -inf.

#include <math.h>

#include "serving_common.cuh"

namespace {

using namespace gdn_serving;

constexpr int kMaxBeams = 64, kMaxSelected = 64;

struct BeamArgs {
  const void* logits;
  const float* scores;
  const uint8_t* finished;
  int32_t* tokens;
  int32_t* parents;
  float* out_scores;
  unsigned long long* keys;   // workspace: [rows, n] keys, descending, 0 = none
  double* lse;                // workspace: [rows]
  long long stride_batch, stride_beam;
  int B, K, V, n, eos;
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

// One CTA per (request, beam): the row's lse, then its n best one after another.
template <typename T>
__global__ void __launch_bounds__(256) beam_row_kernel(BeamArgs p) {
  const int row = blockIdx.x, b = row / p.K, i = row % p.K, tid = threadIdx.x;
  const T* x = reinterpret_cast<const T*>(p.logits) + b * p.stride_batch + i * p.stride_beam;
  __shared__ double red[256];
  __shared__ unsigned long long kred[256];
  double m = -INFINITY;
  bool nan = false;
  for (int t = tid; t < p.V; t += 256) {
    const float v = to_f(x[t]);
    nan |= isnan(v);
    m = fmax(m, static_cast<double>(v));
  }
  red[tid] = m;
  nan = __syncthreads_or(nan);
  for (int o = 128; o > 0; o >>= 1) {
    if (tid < o) red[tid] = fmax(red[tid], red[tid + o]);
    __syncthreads();
  }
  m = red[0];
  __syncthreads();
  double s = 0.0;
  for (int t = tid; t < p.V; t += 256) s += exp(static_cast<double>(to_f(x[t])) - m);
  red[tid] = s;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (tid < o) red[tid] += red[tid + o];
    __syncthreads();
  }
  const bool dead = nan || !isfinite(m);
  if (tid == 0) p.lse[row] = m + log(red[0]);
  unsigned long long below = ~0ull;
  for (int r = 0; r < p.n; ++r) {
    unsigned long long best = 0;
    if (!dead)
      for (int t = tid; t < p.V; t += 256) {
        const float v = to_f(x[t]);
        if (v == -INFINITY) continue;
        const unsigned long long k = make_key(v, t);
        if (k < below && k > best) best = k;
      }
    kred[tid] = best;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
      if (tid < o && kred[tid + o] > kred[tid]) kred[tid] = kred[tid + o];
      __syncthreads();
    }
    below = kred[0];
    __syncthreads();
    if (tid == 0) p.keys[static_cast<long long>(row) * p.n + r] = below;
  }
}

// One thread per request merges its beams' sorted lists.
__global__ void beam_merge_kernel(BeamArgs p) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= p.B) return;
  int pos[kMaxBeams];
  for (int i = 0; i < p.K; ++i) pos[i] = 0;
  for (int r = 0; r < p.n; ++r) {
    double best = -INFINITY;
    int from = -1;
    for (int i = 0; i < p.K; ++i) {
      const int row = b * p.K + i;
      const double cum = p.scores[row];
      double sc = -INFINITY;
      if (p.finished && p.finished[row]) {
        if (pos[i] == 0) sc = cum;
      } else if (pos[i] < p.n) {
        const unsigned long long k = p.keys[static_cast<long long>(row) * p.n + pos[i]];
        if (k) sc = cum + (static_cast<double>(key_logit(k)) - p.lse[row]);
      }
      if (!isfinite(sc)) sc = -INFINITY;
      if (sc > best) {
        best = sc;
        from = i;
      }
    }
    int tok = -1;
    if (from >= 0) {
      const int row = b * p.K + from;
      tok = (p.finished && p.finished[row])
                ? p.eos
                : key_token(p.keys[static_cast<long long>(row) * p.n + pos[from]]);
      ++pos[from];
    }
    const long long at = static_cast<long long>(b) * p.n + r;
    p.tokens[at] = tok;
    p.parents[at] = from;
    p.out_scores[at] = static_cast<float>(best);
  }
}

}  // namespace

extern "C" {

size_t gdn_beam_select_workspace_bytes(int B, int K, int V, int n) {
  if (B < 1 || K < 1 || V < 1 || n < 1) return 0;
  return static_cast<size_t>(B) * K * (static_cast<size_t>(n) * 8 + 8);
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
  if (workspace_bytes < gdn_beam_select_workspace_bytes(B, K, V, n)) return GDN_ERR_SHAPE;
  BeamArgs p{};
  p.logits = logits; p.scores = scores; p.finished = finished; p.tokens = tokens;
  p.parents = parents; p.out_scores = new_scores;
  p.keys = static_cast<unsigned long long*>(workspace);
  p.lse = reinterpret_cast<double*>(p.keys + static_cast<size_t>(B) * K * n);
  p.stride_batch = stride_batch; p.stride_beam = stride_beam;
  p.B = B; p.K = K; p.V = V; p.n = n; p.eos = eos_token;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == GDN_DTYPE_BF16) beam_row_kernel<__nv_bfloat16><<<B * K, 256, 0, st>>>(p);
  else if (dtype == GDN_DTYPE_FP16) beam_row_kernel<__half><<<B * K, 256, 0, st>>>(p);
  else beam_row_kernel<float><<<B * K, 256, 0, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return GDN_ERR_LAUNCH;
  beam_merge_kernel<<<(B + 31) / 32, 32, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // extern "C"
