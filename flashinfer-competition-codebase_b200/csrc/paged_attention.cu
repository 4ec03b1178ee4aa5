// paged_attention.cu — softmax attention of one new token per sequence over a paged
// key-value cache, with the new token's key and value appended to the cache.
//
// Per sequence b, query head h (key-value head g = h / (HQ / HKV)) and visible tokens i:
//   x_i = scale * q_h . k_i       m = max_i x_i      p_i = exp(x_i - m)     l = sum_i p_i
//   o   = (sum_i p_i v_i) / l     lse = m + ln(l)
// in one pass over the tokens with a running maximum: when m grows, l and the sum of
// p_i v_i are scaled by exp(m_old - m_new).
//
// Visible tokens.  With n = seq_lens[b] tokens, sinks s and window w > 0 these are the
// first s and the last w; they are numbered 0 .. n_vis-1 with n_vis = min(n, s + w), and
// number j is token j when j < s, else j + (n - n_vis).  So a windowed sequence costs what
// it sees, not what it holds.

#include <math.h>

#include "serving_common.cuh"

namespace {

using namespace gdn_serving;

struct AttnArgs {
  const void* q;             // [B, HQ, D]
  char* k;                   // cache pages, byte strides below
  char* v;
  const int32_t* tables;     // [B, width], row stride table_stride
  const int32_t* lens;       // [B]
  const void* k_new;         // [B, HKV, D] or null
  const void* v_new;
  void* out;                 // [B, HQ, D]
  float* lse;                // [B, HQ] or null
  int32_t* bad;              // or null
  long long k_page, k_tok, k_head, v_page, v_tok, v_head;   // byte strides
  long long table_stride;
  float scale_log2;          // scale * log2(e): the softmax runs in base 2
  int B, HQ, HKV, group, num_pages, page_size, width, window, sinks;
};

// One sequence's lengths: tokens held, tokens visible, whether the new token is in play.
struct Seq {
  int len, vis, shift;
  bool append;
};

__device__ __forceinline__ Seq sequence(const AttnArgs& p, int b) {
  Seq s;
  const int cap = p.width * p.page_size;   // < 2^31, checked on the host
  int n = p.lens[b];
  n = n < 0 ? 0 : n;
  s.append = p.k_new != nullptr && n > 0 && n <= cap;
  s.len = n > cap ? cap : n;
  s.vis = (p.window > 0 && s.len > p.sinks + p.window) ? p.sinks + p.window : s.len;
  s.shift = s.len - s.vis;
  return s;
}

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half(x); }

// One CTA of 4 warps per (query head, sequence); warp w takes tokens w, w+4, ...; lane j
// holds dims j, j+32, ...
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_decode_kernel(AttnArgs p) {
  constexpr int N = D / 32;
  const int h = blockIdx.x, b = blockIdx.y, g = h / p.group;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Seq s = sequence(p, b);
  const int32_t* table = p.tables + b * p.table_stride;
  const T* kn = reinterpret_cast<const T*>(p.k_new) + (static_cast<long long>(b) * p.HKV + g) * D;
  const T* vn = reinterpret_cast<const T*>(p.v_new) + (static_cast<long long>(b) * p.HKV + g) * D;
  const T* q = reinterpret_cast<const T*>(p.q) + (static_cast<long long>(b) * p.HQ + h) * D;
  float qf[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    qf[i] = to_f(q[lane + 32 * i]);
    o[i] = 0.f;
  }
  if (h == 0 && threadIdx.x == 0 && p.bad && p.lens[b] > s.len) atomicAdd(p.bad, 1);
  for (int j = warp; j < s.vis; j += 4) {
    const int tok = j < p.sinks ? j : j + s.shift;
    const int page = table[tok / p.page_size], off = tok % p.page_size;
    const bool in_new = s.append && tok == s.len - 1;
    const bool ok = page >= 0 && page < p.num_pages;
    if (h == 0 && lane == 0 && p.bad && page >= p.num_pages &&
        (off == 0 || j == 0 || (j == p.sinks && p.window > 0)))
      atomicAdd(p.bad, 1);
    char* krow = p.k + (ok ? page * p.k_page + off * p.k_tok + g * p.k_head : 0);
    char* vrow = p.v + (ok ? page * p.v_page + off * p.v_tok + g * p.v_head : 0);
    if (in_new && ok && h % p.group == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        reinterpret_cast<T*>(krow)[lane + 32 * i] = kn[lane + 32 * i];
        reinterpret_cast<T*>(vrow)[lane + 32 * i] = vn[lane + 32 * i];
      }
    }
    if (!ok && !in_new) continue;
    const T* kr = in_new ? kn : reinterpret_cast<const T*>(krow);
    const T* vr = in_new ? vn : reinterpret_cast<const T*>(vrow);
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) x += qf[i] * to_f(kr[lane + 32 * i]);
    x = warp_sum(x) * p.scale_log2;
    const float mn = fmaxf(m, x);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float c = exp2f(m - base), e = exp2f(x - base);
    l = l * c + e;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * c + e * to_f(vr[lane + 32 * i]);
    m = mn;
  }
  __shared__ float sm[4], sl[4], so[4][D];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) so[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const float base = mx == -INFINITY ? 0.f : mx;
  float lt = 0.f;
  for (int w = 0; w < 4; ++w) lt += sl[w] * exp2f(sm[w] - base);
  for (int d = threadIdx.x; d < D; d += 128) {
    float acc = 0.f;
    for (int w = 0; w < 4; ++w) acc += so[w][d] * exp2f(sm[w] - base);
    reinterpret_cast<T*>(p.out)[(static_cast<long long>(b) * p.HQ + h) * D + d] =
        from_f<T>(lt == 0.f ? 0.f : acc / lt);
  }
  if (threadIdx.x == 0 && p.lse)
    p.lse[static_cast<long long>(b) * p.HQ + h] =
        lt == 0.f ? -INFINITY : (base + log2f(lt)) * 0.6931471805599453f;
}

template <typename T>
cudaError_t launch(const AttnArgs& p, int D, cudaStream_t st) {
  const dim3 grid(p.HQ, p.B);
  if (D == 64) attn_decode_kernel<T, 64><<<grid, 128, 0, st>>>(p);
  else if (D == 128) attn_decode_kernel<T, 128><<<grid, 128, 0, st>>>(p);
  else attn_decode_kernel<T, 256><<<grid, 128, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace

extern "C" {

size_t gdn_paged_attention_workspace_bytes(int B, int HQ, int HKV, int D, int max_tokens) {
  (void)B; (void)HQ; (void)HKV; (void)D; (void)max_tokens;
  return 0;
}

int gdn_paged_attention_decode(const void* q, void* k_cache, void* v_cache,
                               const int32_t* block_tables, const int32_t* seq_lens,
                               const void* k_new, const void* v_new, double scale, int window,
                               int num_sinks, void* output, float* lse, void* workspace,
                               size_t workspace_bytes, int dtype, int B, int HQ, int HKV, int D,
                               int num_pages, int page_size, int table_width,
                               int64_t table_stride, const int64_t* k_strides,
                               const int64_t* v_strides, int32_t* bad_index_count,
                               void* stream) {
  if (D != 64 && D != 128 && D != 256) return GDN_ERR_SHAPE;
  if (B < 0 || HQ < 1 || HKV < 1 || HQ % HKV != 0) return GDN_ERR_SHAPE;
  if (num_pages < 1 || page_size < 1 || table_width < 0) return GDN_ERR_SHAPE;
  if (static_cast<long long>(table_width) * page_size > 0x7fffffffLL - 1024) return GDN_ERR_SHAPE;
  if (B > 65535 || static_cast<long long>(B) * HQ > 0x7fffffffLL / 256) return GDN_ERR_SHAPE;
  if (dtype != GDN_DTYPE_BF16 && dtype != GDN_DTYPE_FP16) return GDN_ERR_ARG;
  if (window < 0 || num_sinks < 0 || window > 0x3fffffff || num_sinks > 0x3fffffff) return GDN_ERR_ARG;
  if (!isfinite(scale)) return GDN_ERR_ARG;
  if (B == 0) return GDN_OK;
  if (!q || !k_cache || !v_cache || !seq_lens || !output || !k_strides || !v_strides)
    return GDN_ERR_NULL;
  if (table_width > 0 && !block_tables) return GDN_ERR_NULL;
  if ((k_new == nullptr) != (v_new == nullptr)) return GDN_ERR_NULL;
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(output, 16) ||
      !aligned(k_new, 16) || !aligned(v_new, 16) || !aligned(block_tables, 4) ||
      !aligned(seq_lens, 4) || !aligned(lse, 4) || !aligned(bad_index_count, 4))
    return GDN_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] < 0 || v_strides[i] < 0 || k_strides[i] % 8 || v_strides[i] % 8)
      return GDN_ERR_ALIGN;
  AttnArgs p{};
  p.q = q; p.k = static_cast<char*>(k_cache); p.v = static_cast<char*>(v_cache);
  p.tables = block_tables; p.lens = seq_lens; p.k_new = k_new; p.v_new = v_new;
  p.out = output; p.lse = lse; p.bad = bad_index_count;
  p.k_page = 2 * k_strides[0]; p.k_tok = 2 * k_strides[1]; p.k_head = 2 * k_strides[2];
  p.v_page = 2 * v_strides[0]; p.v_tok = 2 * v_strides[1]; p.v_head = 2 * v_strides[2];
  p.table_stride = table_stride;
  p.scale_log2 = static_cast<float>((scale == 0.0 ? 1.0 / sqrt(static_cast<double>(D)) : scale) *
                                    1.4426950408889634);
  p.B = B; p.HQ = HQ; p.HKV = HKV; p.group = HQ / HKV; p.num_pages = num_pages;
  p.page_size = page_size; p.width = table_width; p.window = window;
  p.sinks = window > 0 ? num_sinks : 0;
  (void)workspace; (void)workspace_bytes;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == GDN_DTYPE_BF16 ? launch<__nv_bfloat16>(p, D, st) : launch<__half>(p, D, st);
  return e == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // extern "C"
