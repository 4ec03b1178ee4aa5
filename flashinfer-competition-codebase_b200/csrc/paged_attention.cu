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

#include <type_traits>

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
  float* part_o;             // workspace [2 grid, heads of a row, D]: sums of p v
  float* part_ml;            // workspace [2 grid, heads of a row, 2]: their m and l
  int4* cut;                 // workspace [grid]: the cut row that ends in this share, or none
  long long k_page, k_tok, k_head, v_page, v_tok, v_head;   // byte strides
  long long table_stride;
  float scale_log2;          // scale * log2(e): the softmax runs in base 2
  uint32_t page_mul, page_shift;
  int B, HQ, HKV, group, tiles, grid, num_pages, page_size, width, window, sinks, twin;
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

// ------------------------------------------------------------------ split of the work
//
// A "row" is (sequence, key-value head, tile of 8 or 16 of its query heads); it has
// ceil(vis / block) blocks of tokens, at least one.  All rows' blocks in a line (sequence,
// row, block) are cut into equal shares, one per CTA, so ragged batches, one long sequence
// and many short ones all load the GPU evenly.  A CTA that has all of a row writes its
// output; a row that is cut leaves partial sums (at most two per CTA: its first and its last
// row), which attn_join_kernel adds up in a fixed order.  The cut depends on lens alone, so
// no counters or flags have to be kept in memory.

constexpr int kWarps = 4;

// Shapes by head dim: tokens a warp takes at a time, ring stages, CTAs per SM.
template <int D> struct Shape {
  static constexpr int kTile = D == 64 ? 32 : 16;
  static constexpr int kBlock = kWarps * kTile;
  static constexpr int kRow = D * 2;                          // bytes of a token's row
  static constexpr int kHalf = kTile * kRow;                  // K or V part of a stage
  static constexpr int kStages = 3;
  static constexpr int kWarpBytes = kStages * 2 * kHalf;
  static constexpr int kSmem = kWarps * kWarpBytes;
  static constexpr int kResident = D == 256 ? 1 : 2;
};

template <int kBlock> __device__ __forceinline__ int blocks_of(const AttnArgs& p, int b) {
  const int vis = sequence(p, b).vis;
  return vis > 0 ? (vis + kBlock - 1) / kBlock : 1;
}

// the share of g that block i of n lies in, and the first block of share c
__device__ __forceinline__ long long share_of(long long i, long long n, long long g) {
  return ((i + 1) * g - 1) / n;
}
__device__ __forceinline__ long long share_start(long long c, long long n, long long g) {
  return c * n / g;
}

struct Share {
  long long total, count, start, end;    // blocks of all rows, shares, this CTA's blocks
  long long before;                      // blocks of one row per sequence before sequence b
  int b;                                 // the sequence of block `start`
};

// This CTA's share, by all its threads; start == end where there is none.
template <int kBlock> __device__ Share my_share(const AttnArgs& p) {
  constexpr int N = kWarps * 32;
  __shared__ long long sum[kWarps], found_before;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, rows = p.HKV * p.tiles;
  long long base = 0, first = 0;
  int n = 0;
  auto scan = [&](int b0) {              // sequences b0 ...: n and first of b0 + tid
    n = b0 + tid < p.B ? blocks_of<kBlock>(p, b0 + tid) : 0;
    long long x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();                     // the last round's readers of sum are done
    if (lane == 31) sum[warp] = x;
    __syncthreads();
    first = base + x - n;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      first += w < warp ? sum[w] : 0;
      base += sum[w];
    }
  };
  for (int b0 = 0; b0 < p.B; b0 += N) scan(b0);
  Share s;
  s.total = base * rows;
  s.count = s.total < p.grid ? s.total : p.grid;
  s.start = s.end = 0;
  if (blockIdx.x >= s.count) return s;
  s.start = share_start(blockIdx.x, s.total, s.count);
  s.end = share_start(blockIdx.x + 1, s.total, s.count);
  const long long at = s.start / rows;
  if (p.B > N) base = 0;
  for (int b0 = 0; b0 < p.B; b0 += N) {
    if (p.B > N) scan(b0);               // else n and first are still those of sequence tid
    if (n > 0 && first <= at && at < first + n) {
      found = b0 + tid;
      found_before = first;
    }
    if (p.B > N && base > at) break;     // the same for all threads
  }
  __syncthreads();
  s.b = found;
  s.before = found_before;
  return s;
}

// ------------------------------------------------------------------ matrix instructions

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// c[16 x 8] += a[16 x 16] b[16 x 8]
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// four 8 x 8 matrices of 16-bit values; lane l gives the address of row l % 8 of matrix l / 8
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// ------------------------------------------------------------------ the kernel
//
// Both products run transposed, with the tokens (then the head dims) as the 16 rows of the
// matrix instruction and 8 query heads as its columns:
//   S^T [16 tokens x 8 heads] = K Q^T        O^T [D x 8 heads] += V^T P^T
// so a group of up to 8 query heads fills the instruction, where queries as rows would
// leave half of it empty, and the accumulators of O take D / 16 x 4 registers.  The scores'
// accumulator layout becomes the second product's operand by an 8 x 8 transpose in
// registers.  p is rounded to the tensors' type for that product (its own sum l is not):
// the rounding is that of the values it multiplies, at most half a step of each weight.
//
// Every warp streams its own 16-token tiles through its own ring of kStages buffers in
// shared memory with asynchronous copies, so the main loop has no CTA barrier.  A tile's page
// numbers are loaded one tile before its copies are issued.

// A tile's row r has its 16-byte chunk c at r kRow + ((c ^ (r & 7)) << 4): the eight rows that a
// matrix load touches lie in different banks.  Stages are aligned to rows, so stepping
// along a row is one XOR on the address.

template <typename T, int D, int NG>
__global__ void __launch_bounds__(kWarps * 32, Shape<D>::kResident)
attn_decode_kernel(const __grid_constant__ AttnArgs p) {
  using S = Shape<D>;
  constexpr int kHeads = 8 * NG, KS = D / 16, CPR = D / 8;    // chunks per row
  constexpr int MT = S::kTile / 16;                           // 16-token parts of a tile
  constexpr int kRows = 32 / CPR, kIters = S::kTile / kRows;  // rows a warp copies at a time
  constexpr uint32_t kAll = S::kTile == 32 ? 0xffffffffu : 0xffffu;
  constexpr int kPad = D + 4;                                 // floats of a head in the merge
  static_assert(kHeads * kPad * 4 <= S::kWarpBytes, "the merge reuses the ring");
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ float sm_m[kWarps][kHeads], sm_l[kWarps][kHeads];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t ring = smem_addr(smem) + warp * S::kWarpBytes;

  grid_trigger();                         // the join's CTAs may take their places and wait
  const Share share = my_share<S::kBlock>(p);
  const int rows = p.HKV * p.tiles;                           // rows of one sequence
  long long at = share.start, before = share.before;
  int b = share.b;
  if (at == share.end) {
    if (tid == 0 && p.cut) p.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }

  // fixed parts of this lane's addresses
  const int copy_r = lane / CPR, copy_c = lane % CPR;
  const uint32_t copy_at = copy_r * S::kRow + ((copy_c ^ copy_r) << 4);
  const uint32_t k_at = (lane % 16) * S::kRow + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_at = ((lane & 7) + ((lane >> 4) << 3)) * S::kRow + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);

  while (at < share.end) {
    const Seq s = sequence(p, b);
    const int nb = s.vis > 0 ? (s.vis + S::kBlock - 1) / S::kBlock : 1;
    const long long in_seq = at - before * rows;
    const int row = static_cast<int>(in_seq / nb), k0 = static_cast<int>(in_seq % nb);
    const long long left = share.end - at;
    const int k1 = left < nb - k0 ? k0 + static_cast<int>(left) : nb;
    const int g = row / p.tiles, tile = row % p.tiles;
    const int head0 = g * p.group + tile * kHeads, heads = min(kHeads, p.group - tile * kHeads);
    const int32_t* table = p.tables + b * p.table_stride;
    const long long new_row = (static_cast<long long>(b) * p.HKV + g) * D * 2;
    const char* kbase = p.k + g * p.k_head;
    const char* vbase = p.v + g * p.v_head;
    const bool counts = row == 0 && p.bad != nullptr;
    if (counts && tid == 0 && k0 == 0 && p.lens[b] > s.len) atomicAdd(p.bad, 1);
    if (at == share.start && tid == 0 && p.cut) {
      const long long first = before * rows + static_cast<long long>(row) * nb;
      const int c0 = static_cast<int>(share_of(first, share.total, share.count));
      p.cut[blockIdx.x] = make_int4(k0 > 0 && k1 == nb ? b : -1, row, c0,
                                    first > share_start(c0, share.total, share.count));
    }

    // lane i looks after token i of a tile (all 32, or twice 16): its page number, its place
    auto token_of = [&](int k) {
      const int j = (k * kWarps + warp) * S::kTile + (lane & (S::kTile - 1));
      return j < s.vis ? (j < p.sinks ? j : j + s.shift) : -1;
    };
    auto page_of = [&](int k) {
      const int tok = k < k1 ? token_of(k) : -1;
      return tok < 0 ? -1 : __ldg(table + div_by(tok, p.page_mul, p.page_shift));
    };
    // whether no visible token before tok lies in its page
    auto first_in_page = [&](int tok, int off) {
      if (off == 0) return true;
      return s.shift > 0 && tok == p.sinks + s.shift &&
             (p.sinks == 0 || (p.sinks - 1) / p.page_size != tok / p.page_size);
    };
    // issue the copies of block k's tile into ring stage st; returns the tokens seen
    auto fetch = [&](int k, int st, int page) -> uint32_t {
      const int tok = token_of(k);
      const int off = tok < 0 ? 0 : tok - static_cast<int>(div_by(tok, p.page_mul, p.page_shift)) * p.page_size;
      const bool is_new = s.append && tok == s.len - 1;
      const bool in_cache = tok >= 0 && page >= 0 && page < p.num_pages;
      if (counts && lane < S::kTile && tok >= 0 && page >= p.num_pages && first_in_page(tok, off))
        atomicAdd(p.bad, 1);
      const uint32_t mask = __ballot_sync(0xffffffffu, in_cache || is_new) & kAll;
      const bool any_new = __any_sync(0xffffffffu, is_new);
      // this lane's token's row, relative to the head's first row
      long long ko = in_cache ? page * p.k_page + off * p.k_tok : 0;
      long long vo = in_cache ? page * p.v_page + off * p.v_tok : 0;
      if (is_new) {
        ko = reinterpret_cast<const char*>(p.k_new) + new_row - kbase;
        vo = reinterpret_cast<const char*>(p.v_new) + new_row - vbase;
      }
      const uint32_t dst = ring + st * 2 * S::kHalf + copy_at;
      const char* kc = kbase + copy_c * 16;
      const char* vc = vbase + copy_c * 16;
      if (mask == kAll && p.twin && !any_new) {               // nearly always
#pragma unroll
        for (int i = 0; i < kIters; ++i) {
          const long long o = __shfl_sync(0xffffffffu, ko, copy_r + i * kRows);
          const uint32_t d = (dst ^ ((i * kRows & 7) << 4)) + i * kRows * S::kRow;
          copy16_async(d, kc + o, true);
          copy16_async(d + S::kHalf, vc + o, true);
        }
      } else {
#pragma unroll 2
        for (int i = 0; i < kIters; ++i) {
          const int r = copy_r + i * kRows;
          const long long o = __shfl_sync(0xffffffffu, ko, r), w = __shfl_sync(0xffffffffu, vo, r);
          const bool ok = (mask >> r) & 1;
          const uint32_t d = (dst ^ ((i * kRows & 7) << 4)) + i * kRows * S::kRow;
          copy16_async(d, kc + o, ok);
          copy16_async(d + S::kHalf, vc + w, ok);
        }
      }
      return mask;
    };

    uint32_t mask[S::kStages - 1];
    int page = page_of(k0);
#pragma unroll
    for (int st = 0; st < S::kStages - 1; ++st) {
      mask[st] = 0;
      const int next = page_of(k0 + st + 1);
      if (k0 + st < k1) mask[st] = fetch(k0 + st, st, page);
      page = next;
      copy_commit();
    }
    // the new token's rows go into the cache once: by the first tile's owner of the last block
    if (s.append && tile == 0 && k1 == nb) {
      const int tok = s.len - 1, pi = tok / p.page_size, pg = table[pi];
      if (pg >= 0 && pg < p.num_pages && tid < 2 * CPR) {
        const int c = tid % CPR, of = tok - pi * p.page_size;
        const char* src = reinterpret_cast<const char*>(tid < CPR ? p.k_new : p.v_new) + new_row;
        char* dst = tid < CPR ? p.k + g * p.k_head + pg * p.k_page + of * p.k_tok
                              : p.v + g * p.v_head + pg * p.v_page + of * p.v_tok;
        *reinterpret_cast<uint4*>(dst + c * 16) = *reinterpret_cast<const uint4*>(src + c * 16);
      }
    }
    // queries as the right operand: head lane / 4 (+ 8 per further group), two dims a register
    uint32_t qf[NG][KS][2];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int h = n * 8 + lane / 4;
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p.q) +
                          (static_cast<long long>(b) * p.HQ + head0 + (h < heads ? h : 0)) * (D / 2);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        qf[n][i][0] = h < heads ? __ldg(q + i * 8 + lane % 4) : 0u;
        qf[n][i][1] = h < heads ? __ldg(q + i * 8 + 4 + lane % 4) : 0u;
      }
    }

    float o[NG][KS][4], m[NG][2], l[NG][2];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][i][j] = 0.f;
    }

    int st = 0;
    for (int k = k0; k < k1; ++k) {
      copy_wait<S::kStages - 2>();
      __syncwarp();
      const uint32_t buf = ring + st * 2 * S::kHalf;
      const uint32_t seen = mask[0];
      float y[MT][NG][4];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float x[NG][2][4];                // two chains of products
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[n][0][j] = x[n][1][j] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          uint32_t a[4];
          load_matrices(a, (buf + k_at + t * 16 * S::kRow) ^ (i * 32));
#pragma unroll
          for (int n = 0; n < NG; ++n) mma<T>(x[n][i & 1], a, qf[n][i][0], qf[n][i][1]);
        }
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) y[t][n][j] = (x[n][0][j] + x[n][1][j]) * p.scale_log2;
      }
      if (seen != kAll) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            if (!((seen >> (t * 16 + lane / 4)) & 1)) y[t][n][0] = y[t][n][1] = -INFINITY;
            if (!((seen >> (t * 16 + lane / 4 + 8)) & 1)) y[t][n][2] = y[t][n][3] = -INFINITY;
          }
      }
      uint32_t pb[MT][NG][2];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          t0 = fmaxf(t0, fmaxf(y[t][n][0], y[t][n][2]));
          t1 = fmaxf(t1, fmaxf(y[t][n][1], y[t][n][3]));
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, d));
          t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, d));
        }
        const float m0 = fmaxf(m[n][0], t0), m1 = fmaxf(m[n][1], t1);
        const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
        if (__any_sync(0xffffffffu, m0 > m[n][0] || m1 > m[n][1])) {
          const float c0 = exp2_fast(m[n][0] - b0), c1 = exp2_fast(m[n][1] - b1);
          l[n][0] *= c0;
          l[n][1] *= c1;
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            o[n][i][0] *= c0;
            o[n][i][1] *= c1;
            o[n][i][2] *= c0;
            o[n][i][3] *= c1;
          }
          m[n][0] = m0;
          m[n][1] = m1;
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const float p0 = exp2_fast(y[t][n][0] - b0), p1 = exp2_fast(y[t][n][1] - b1);
          const float p2 = exp2_fast(y[t][n][2] - b0), p3 = exp2_fast(y[t][n][3] - b1);
          l[n][0] += p0 + p2;
          l[n][1] += p1 + p3;
          pb[t][n][0] = transpose8(pack2<T>(p0, p1));
          pb[t][n][1] = transpose8(pack2<T>(p2, p3));
        }
      }
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          uint32_t a[4];
          load_matrices_t(a, (buf + S::kHalf + v_at + t * 16 * S::kRow) ^ (i * 32));
#pragma unroll
          for (int n = 0; n < NG; ++n) mma<T>(o[n][i], a, pb[t][n][0], pb[t][n][1]);
        }
      __syncwarp();                       // every lane is done with this stage
#pragma unroll
      for (int i = 0; i + 1 < S::kStages - 1; ++i) mask[i] = mask[i + 1];
      mask[S::kStages - 2] = 0;
      const int kn = k + S::kStages - 1;
      const int next = page_of(kn + 1);
      if (kn < k1) mask[S::kStages - 2] = fetch(kn, st == 0 ? S::kStages - 1 : st - 1, page);
      page = next;
      copy_commit();
      st = st + 1 == S::kStages ? 0 : st + 1;
    }
    copy_wait<0>();
    __syncwarp();

    // the four warps' sums, through shared memory (each in its own ring)
    float* mine = reinterpret_cast<float*>(smem + warp * S::kWarpBytes);
#pragma unroll
    for (int n = 0; n < NG; ++n) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], d);
        l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], d);
      }
      const int h = n * 8 + 2 * (lane % 4);
      if (lane < 4) {
        sm_m[warp][h] = m[n][0];
        sm_m[warp][h + 1] = m[n][1];
        sm_l[warp][h] = l[n][0];
        sm_l[warp][h + 1] = l[n][1];
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int d = i * 16 + lane / 4;
        mine[h * kPad + d] = o[n][i][0];
        mine[(h + 1) * kPad + d] = o[n][i][1];
        mine[h * kPad + d + 8] = o[n][i][2];
        mine[(h + 1) * kPad + d + 8] = o[n][i][3];
      }
    }
    __syncthreads();
    const bool whole = k0 == 0 && k1 == nb;
    const long long slot = 2 * static_cast<long long>(blockIdx.x) + (at == share.start ? 0 : 1);
    for (int f = tid; f < heads * (D / 2); f += kWarps * 32) {
      const int h = f / (D / 2), d = (f % (D / 2)) * 2;
      float mx = sm_m[0][h];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, sm_m[w][h]);
      const float base = mx == -INFINITY ? 0.f : mx;
      float lt = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float c = exp2_fast(sm_m[w][h] - base);
        const float* other = reinterpret_cast<const float*>(smem + w * S::kWarpBytes) + h * kPad + d;
        lt += sm_l[w][h] * c;
        a0 += other[0] * c;
        a1 += other[1] * c;
      }
      if (whole) {
        const long long r = static_cast<long long>(b) * p.HQ + head0 + h;
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
        reinterpret_cast<uint32_t*>(p.out)[(r * D + d) / 2] = pack2<T>(a0 * inv, a1 * inv);
        if (d == 0 && p.lse) p.lse[r] = lt == 0.f ? -INFINITY : (base + log2f(lt)) * 0.6931471805599453f;
      } else {
        *reinterpret_cast<float2*>(p.part_o + (slot * kHeads + h) * D + d) = make_float2(a0, a1);
        if (d == 0)
          *reinterpret_cast<float2*>(p.part_ml + (slot * kHeads + h) * 2) = make_float2(mx, lt);
      }
    }
    __syncthreads();                      // the ring is free for the next row
    at += k1 - k0;
    if (row == rows - 1 && k1 == nb) {
      before += nb;
      ++b;
    }
  }
}

// Adds up the parts of the rows that were cut: o = sum_i o_i 2^(m_i - m) / sum_i l_i 2^(m_i - m).
// CTA (c, y): values 512 y ... of the row whose last part is share c's, if one is.  128
// threads take four values each, two groups of them every other part.
constexpr int kJoinThreads = 256, kJoinValues = 512, kJoinParts = 3 * kSMs;

template <typename T, int D, int NG>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const __grid_constant__ AttnArgs p) {
  constexpr int kHeads = 8 * NG, kHere = kJoinValues / D;     // heads of a row, of this CTA
  __shared__ float2 ml[kJoinParts][kHere];
  __shared__ float4 acc[kJoinValues / 4];
  __shared__ float sum[kJoinValues / 4];
  const int tid = threadIdx.x, y = blockIdx.y;
  grid_wait();
  const int4 cut = p.cut[blockIdx.x];
  if (cut.x < 0) return;
  const int g = cut.y / p.tiles, tile = cut.y % p.tiles, parts = blockIdx.x - cut.z + 1;
  if (y * kHere >= p.group - tile * kHeads) return;           // heads past the group's
  auto slot = [&](int i) { return 2 * static_cast<long long>(cut.z + i) + (i == 0 ? cut.w : 0); };
  for (int f = tid; f < parts * kHere; f += kJoinThreads)
    ml[f / kHere][f % kHere] = reinterpret_cast<const float2*>(p.part_ml)[slot(f / kHere) * kHeads + y * kHere + f % kHere];
  __syncthreads();
  const int quad = tid % (kJoinValues / 4), half = tid / (kJoinValues / 4);
  const int hc = quad * 4 / D;
  float mx = -INFINITY;
  for (int i = 0; i < parts; ++i) mx = fmaxf(mx, ml[i][hc].x);
  const float base = mx == -INFINITY ? 0.f : mx;
  const float4* from = reinterpret_cast<const float4*>(p.part_o) + y * (kJoinValues / 4) + quad;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 8
  for (int i = half; i < parts; i += 2) {
    const float4 v = from[slot(i) * (kHeads * D / 4)];
    const float w = exp2_fast(ml[i][hc].x - base);
    l += w * ml[i][hc].y;
    a.x += w * v.x;
    a.y += w * v.y;
    a.z += w * v.z;
    a.w += w * v.w;
  }
  if (half) {
    acc[quad] = a;
    sum[quad] = l;
  }
  __syncthreads();
  const int h = tile * kHeads + y * kHere + hc;
  if (half || h >= p.group) return;
  const float4 v = acc[quad];
  l += sum[quad];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const long long r = static_cast<long long>(cut.x) * p.HQ + g * p.group + h;
  reinterpret_cast<uint2*>(p.out)[(r * D + quad * 4 % D) / 4] =
      make_uint2(pack2<T>((a.x + v.x) * inv, (a.y + v.y) * inv),
                 pack2<T>((a.z + v.z) * inv, (a.w + v.w) * inv));
  if (quad * 4 % D == 0 && p.lse)
    p.lse[r] = l == 0.f ? -INFINITY : (base + log2f(l)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ host

// heads of a row: one group of 8 columns, or two for larger groups of query heads
int heads_of(int group) { return group <= 8 ? 8 : 16; }

// tokens of a block, CTAs per SM
int block_of(int D) { return D == 64 ? Shape<64>::kBlock : D == 128 ? Shape<128>::kBlock : Shape<256>::kBlock; }
int resident(int D) { return D == 64 ? Shape<64>::kResident : D == 128 ? Shape<128>::kResident : Shape<256>::kResident; }

// CTAs of a call: what the GPU holds at once, or one per block of tokens if there are fewer
long long grid_of(int B, int HQ, int HKV, int D, long long max_tokens) {
  const int heads = heads_of(HQ / HKV);
  const long long rows = static_cast<long long>(B) * HKV * ((HQ / HKV + heads - 1) / heads);
  const long long nb = max_tokens > 0 ? (max_tokens + block_of(D) - 1) / block_of(D) : 1;
  const long long most = static_cast<long long>(kSMs) * resident(D);
  return rows * nb < most ? rows * nb : most;
}

template <typename T, int D, int NG>
cudaError_t launch_shape(const AttnArgs& p, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(attn_decode_kernel<T, D, NG>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
  if (e != cudaSuccess) return e;
  attn_decode_kernel<T, D, NG><<<p.grid, kWarps * 32, Shape<D>::kSmem, st>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess || !p.cut) return e;
  return launch_after(attn_join_kernel<T, D, NG>, dim3(p.grid, 8 * NG * D / kJoinValues),
                      dim3(kJoinThreads), 0, st, p);
}

template <typename T>
cudaError_t launch(const AttnArgs& p, int D, cudaStream_t st) {
  const bool wide = p.group > 8;
  if (D == 64) return wide ? launch_shape<T, 64, 2>(p, st) : launch_shape<T, 64, 1>(p, st);
  if (D == 128) return wide ? launch_shape<T, 128, 2>(p, st) : launch_shape<T, 128, 1>(p, st);
  return wide ? launch_shape<T, 256, 2>(p, st) : launch_shape<T, 256, 1>(p, st);
}

}  // namespace

extern "C" {

size_t gdn_paged_attention_workspace_bytes(int B, int HQ, int HKV, int D, int max_tokens) {
  if (B < 1 || HQ < 1 || HKV < 1 || HQ % HKV != 0 || (D != 64 && D != 128 && D != 256)) return 0;
  if (max_tokens <= block_of(D)) return 0;    // no row is ever cut
  return static_cast<size_t>(grid_of(B, HQ, HKV, D, max_tokens)) *
         (2 * static_cast<size_t>(heads_of(HQ / HKV)) * (D + 2) * 4 + sizeof(int4));
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
  const int max_tokens = table_width * page_size;
  const size_t need = gdn_paged_attention_workspace_bytes(B, HQ, HKV, D, max_tokens);
  if (need > 0 && !workspace) return GDN_ERR_NULL;
  if (!aligned(workspace, 16)) return GDN_ERR_ALIGN;
  if (workspace_bytes < need) return GDN_ERR_SHAPE;
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
  p.tiles = (p.group + heads_of(p.group) - 1) / heads_of(p.group);
  p.grid = static_cast<int>(grid_of(B, HQ, HKV, D, max_tokens));
  if (need > 0) {
    p.cut = static_cast<int4*>(workspace);
    p.part_o = reinterpret_cast<float*>(p.cut + p.grid);
    p.part_ml = p.part_o + static_cast<size_t>(2 * p.grid) * heads_of(p.group) * D;
  }
  p.twin = p.k_page == p.v_page && p.k_tok == p.v_tok;
  div_constants(static_cast<uint32_t>(page_size), p.page_mul, p.page_shift);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == GDN_DTYPE_BF16 ? launch<__nv_bfloat16>(p, D, st) : launch<__half>(p, D, st);
  return e == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // extern "C"
