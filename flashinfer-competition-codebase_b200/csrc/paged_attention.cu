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
  int4* cut;                 // workspace: the cut rows, by row or by the share they end in
  long long k_page, k_tok, k_head, v_page, v_tok, v_head;   // byte strides
  long long table_stride;
  float scale_log2;          // scale * log2(e): the softmax runs in base 2
  uint32_t page_mul, page_shift;
  int B, HQ, HKV, group, tiles, grid, num_pages, page_size, width, window, sinks, twin, by_row;
};

// One sequence's lengths: tokens held, tokens visible, whether the new token is in play.
struct Seq {
  int len, vis, shift;
  bool append;
};

__device__ __forceinline__ Seq sequence(const AttnArgs& p, int n) {   // n: its seq_lens
  Seq s;
  const int cap = p.width * p.page_size;   // < 2^31, checked on the host
  n = n < 0 ? 0 : n;
  s.append = p.k_new != nullptr && n > 0 && n <= cap;
  s.len = n > cap ? cap : n;
  s.vis = (p.window > 0 && s.len > p.sinks + p.window) ? p.sinks + p.window : s.len;
  s.shift = s.len - s.vis;
  return s;
}

// ------------------------------------------------------------------ split of the work
//
// A "row" is (sequence, key-value head, tile of 8, 16 or 24 of its query heads); it has
// ceil(vis / block) blocks of tokens, at least one.  All rows' blocks in a line (sequence,
// row, block) are cut into equal shares, one per CTA, so ragged batches and one long sequence
// load the GPU evenly.  A CTA that has all of a row writes its output; a row that is cut leaves
// partial sums (at most two per CTA: its first and its last row), which attn_join_kernel adds
// up in a fixed order.  The cut depends on lens alone, so no counters or flags have to be kept
// in memory.  In a call whose rows cannot be long, going by its table's width and its window,
// none is cut (cut == null): a row is then one unit of the line, and plan_of says how far from
// an even share that may be.

constexpr int kWarps = 4;        // that take tiles of their own, alone or as teams

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

// Warps that share a tile, each with its own 8 of the row's heads: two where one warp's
// registers do not hold 16 heads of 256 (100 sequences of 3000 tokens, 16 heads of 256 to a
// key-value head: 60 us instead of 81).
template <int D, int NG> constexpr int kTeam = D == 256 && NG == 2 ? 2 : 1;

template <int kBlock> __device__ __forceinline__ int blocks_of(const AttnArgs& p, int b) {
  const int vis = sequence(p, p.lens[b]).vis;
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
template <int kBlock, int kCtaWarps> __device__ Share my_share(const AttnArgs& p) {
  constexpr int N = kCtaWarps * 32;
  __shared__ long long sum[kCtaWarps], found_before;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, rows = p.HKV * p.tiles;
  long long base = 0, first = 0;
  int n = 0;
  Share s;
  s.start = s.end = 0;
  if (!p.cut) {                          // whole rows: the lengths do not matter
    s.total = static_cast<long long>(p.B) * rows;
    s.count = s.total < p.grid ? s.total : p.grid;
    if (blockIdx.x >= s.count) return s;
    s.start = share_start(blockIdx.x, s.total, s.count);
    s.end = share_start(blockIdx.x + 1, s.total, s.count);
    s.before = s.b = static_cast<int>(s.start / rows);
    return s;
  }
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
    for (int w = 0; w < kCtaWarps; ++w) {
      first += w < warp ? sum[w] : 0;
      base += sum[w];
    }
  };
  for (int b0 = 0; b0 < p.B; b0 += N) scan(b0);
  s.total = base * rows;
  s.count = s.total < p.grid ? s.total : p.grid;
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

// Weights are held as 2^kUp exp(x - m), l and o with them: in fp16 exp(x - m) itself would be
// subnormal from 2^-14 of the largest on and lost below 2^-25, which 131072 tokens beside a larger one
// add up to 0.4%; 2^15 of it is lost below 2^-40.
template <typename T> constexpr float kUp = std::is_same_v<T, __half> ? 15.f : 0.f;

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
// registers.  p is rounded to the tensors' type for that product (its own sum l is not), which
// takes operands of one type: at most half a step of each weight, as much as the values
// carry themselves.
//
// Every warp streams its own tiles of 16 or 32 tokens through its own ring of kStages
// buffers in shared memory with asynchronous copies, so the main loop has no CTA barrier.
// A tile's page numbers are loaded one tile before its copies are issued, and the copies run
// on into the share's next row, so a short row does not empty the pipeline.
//
// Bound: HBM; a cached byte takes part in one operation for each head of its group, far below
// the tensor cores' rate, so the warp-level instructions, whose operands need no staging
// through tensor memory, are enough.  64 sequences of 820 to 8191 tokens, 32 heads over 8 of 128: 245 us
// (1.59 GB, 6.48 TB/s, 0.98 of a copy's rate).  One of 131072 tokens, 16 heads over 2 of 256: 51 us
// (268 MB, 5.2 TB/s): 46 and the join, whose latency nothing hides.  One of 100 tokens: 5.3 us,
// the latency of a launch and five dependent reads.
//
// A tile's row r has its 16-byte chunk c at r kRow + ((c ^ (r & 7)) << 4): the eight rows that a
// matrix load touches lie in different banks.  Stages are aligned to rows, so stepping
// along a row is one XOR on the address.

template <typename T, int D, int NG>
__global__ void __launch_bounds__(kWarps * kTeam<D, NG> * 32, Shape<D>::kResident)
attn_decode_kernel(const __grid_constant__ AttnArgs p) {
  using S = Shape<D>;
  constexpr int kHeads = 8 * NG, KS = D / 16, CPR = D / 8;    // chunks per row
  constexpr int kMates = kTeam<D, NG>, G = NG / kMates;       // groups of 8 heads of one warp
  constexpr int kThreads = kWarps * kMates * 32;
  constexpr int MT = S::kTile / 16;                           // 16-token parts of a tile
  constexpr int kRows = 32 / CPR * kMates;                    // rows a team copies at a time
  constexpr int kIters = S::kTile / kRows;
  constexpr uint32_t kAll = S::kTile == 32 ? 0xffffffffu : 0xffffu;
  static_assert(kHeads * D * 4 <= 2 * S::kHalf, "the merge reuses a stage");
  static_assert(S::kStages == 3, "two tiles ahead of the one being multiplied");
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ float sm_m[kWarps][kHeads], sm_l[kWarps][kHeads], sm_c[kHeads][kWarps];
  const int tid = threadIdx.x, warp = tid / 32 / kMates, mate = tid / 32 % kMates, lane = tid % 32;
  const uint32_t ring = smem_addr(smem) + warp * S::kWarpBytes;

  grid_trigger();                         // the join's CTAs may take their places and wait
  const Share share = my_share<S::kBlock, kWarps * kMates>(p);
  const int rows = p.HKV * p.tiles;                           // rows of one sequence
  long long at = share.start, before = share.before;
  if (at == share.end) {
    if (tid == 0 && p.cut && !p.by_row) p.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }

  auto team_sync = [&]() {
    if constexpr (kMates == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + warp), "n"(kMates * 32) : "memory");
  };

  // fixed parts of this lane's addresses
  const int copy_r = mate * (32 / CPR) + lane / CPR, copy_c = lane % CPR;
  const uint32_t copy_at = copy_r * S::kRow + ((copy_c ^ copy_r) << 4);
  const uint32_t k_at = (lane % 16) * S::kRow + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_at = ((lane & 7) + ((lane >> 4) << 3)) * S::kRow + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);

  // The copies run ahead of the products, into the share's next row as well: `f` is the row
  // being copied, `row` the one being multiplied, `next` what f will be when row gets there.
  struct Row {
    int b, row, blocks, whole;
  };
  Row row = {}, next = {};
  Seq f = {};
  int f_b = share.b, f_row = 0, f_k = 0, f_k1 = 0, page = -1;
  int len_next = 0;                       // tokens of sequence f_b + 1, loaded early
  bool ahead_row = false;                 // f is `next`, not `row`
  int ahead = 0, put = 0;                 // tiles copied ahead; the stage the next one goes to
  uint32_t mask[2] = {0u, 0u};            // tokens seen of the tiles copied ahead

  // lane i looks after token i of a tile (all 32, or twice 16): its page number, its place
  auto token_of = [&](int k) {
    const int j = (k * kWarps + warp) * S::kTile + (lane & (S::kTile - 1));
    return j < f.vis ? (j < p.sinks ? j : j + f.shift) : -1;
  };
  auto page_of = [&](int k) {
    const int tok = token_of(k);
    return tok < 0 ? -1 : __ldg(p.tables + f_b * p.table_stride + div_by(tok, p.page_mul, p.page_shift));
  };
  // Turns to the row at line position `at` (of sequence f_b, whose tokens are `len`); `early`:
  // the page of this lane's token when that does not depend on len, or -1.
  auto open = [&](Row& r, int len, int early) {
    f = sequence(p, len);
    const int nb = f.vis > 0 ? (f.vis + S::kBlock - 1) / S::kBlock : 1;
    const long long in_seq = at - before * rows, left = share.end - at;
    const int units = p.cut ? nb : 1;
    f_row = static_cast<int>(in_seq / units);
    f_k = static_cast<int>(in_seq - static_cast<long long>(f_row) * units);
    f_k1 = !p.cut || left >= nb - f_k ? nb : f_k + static_cast<int>(left);
    r.b = f_b;
    r.row = f_row;
    r.blocks = f_k1 - f_k;
    r.whole = f_k == 0 && f_k1 == nb;
    page = early >= 0 && token_of(f_k) >= 0 ? early : page_of(f_k);
    if (tid == 0) {
      if (f_row == 0 && f_k == 0 && p.bad != nullptr && len > f.len) atomicAdd(p.bad, 1);
      if (p.cut && (p.by_row ? f_k1 == nb : at == share.start)) {
        const long long first = before * rows + static_cast<long long>(f_row) * nb;
        const int c0 = static_cast<int>(share_of(first, share.total, share.count));
        const int late = first > share_start(c0, share.total, share.count);   // c0's last row
        p.cut[p.by_row ? static_cast<long long>(f_b) * rows + f_row : blockIdx.x] =
            make_int4(f_k > 0 && f_k1 == nb ? f_b : -1, f_row, c0, 2 * blockIdx.x + late);
      }
    }
    // the new token's rows go into the cache once: by the first tile's owner of the last block
    const int g = f_row / p.tiles;
    if (f.append && f_row == g * p.tiles && f_k1 == nb && tid < 2 * CPR) {
      const int tok = f.len - 1, pi = tok / p.page_size, pg = p.tables[f_b * p.table_stride + pi];
      if (pg >= 0 && pg < p.num_pages) {
        const int c = tid % CPR, of = tok - pi * p.page_size;
        const long long from = (static_cast<long long>(f_b) * p.HKV + g) * (D * 2);
        const char* src = reinterpret_cast<const char*>(tid < CPR ? p.k_new : p.v_new) + from;
        char* dst = tid < CPR ? p.k + g * p.k_head + pg * p.k_page + of * p.k_tok
                              : p.v + g * p.v_head + pg * p.v_page + of * p.v_tok;
        *reinterpret_cast<uint4*>(dst + c * 16) = *reinterpret_cast<const uint4*>(src + c * 16);
      }
    }
    // where the line goes on after this row
    at += p.cut ? f_k1 - f_k : 1;
    if (f_row == rows - 1 && f_k1 == nb) {
      before += units;
      if (f_b + 1 < p.B) len_next = p.lens[f_b + 1];
    }
  };
  // whether no visible token before tok lies in its page
  auto first_in_page = [&](int tok, int off) {
    if (off == 0) return true;
    return f.shift > 0 && tok == p.sinks + f.shift &&
           (p.sinks == 0 || (p.sinks - 1) / p.page_size != tok / p.page_size);
  };
  // issue the copies of f's next tile, if there is one, and look up the pages of the one after
  auto fetch = [&]() {
    if (f_k == f_k1) return;
    const int tok = token_of(f_k);
    const int off = tok < 0 ? 0 : tok - static_cast<int>(div_by(tok, p.page_mul, p.page_shift)) * p.page_size;
    const bool is_new = f.append && tok == f.len - 1;
    const bool in_cache = tok >= 0 && page >= 0 && page < p.num_pages;
    if (f_row == 0 && p.bad != nullptr && mate == 0 && lane < S::kTile && tok >= 0 && page >= p.num_pages &&
        first_in_page(tok, off))
      atomicAdd(p.bad, 1);
    const uint32_t seen = __ballot_sync(0xffffffffu, in_cache || is_new) & kAll;
    const bool any_new = __any_sync(0xffffffffu, is_new);
    // this lane's token's row in the caches
    const int g = f_row / p.tiles;
    long long ko = in_cache ? g * p.k_head + page * p.k_page + off * p.k_tok : 0;
    const uint32_t dst = ring + put * 2 * S::kHalf + copy_at;
    const char* kc = p.k + copy_c * 16;
    if (seen == kAll && p.twin && !any_new) {                 // nearly always
      const char* vc = p.v + copy_c * 16;
#pragma unroll
      for (int i = 0; i < kIters; ++i) {
        const long long o = __shfl_sync(0xffffffffu, ko, copy_r + i * kRows);
        const uint32_t d = (dst ^ ((i * kRows & 7) << 4)) + i * kRows * S::kRow;
        copy16_async(d, kc + o, true);
        copy16_async(d + S::kHalf, vc + o, true);
      }
    } else {
      long long vo = in_cache ? g * p.v_head + page * p.v_page + off * p.v_tok : 0;
      const char* vc = p.v + copy_c * 16;
      if (is_new) {
        const long long from = (static_cast<long long>(f_b) * p.HKV + g) * (D * 2);
        ko = reinterpret_cast<const char*>(p.k_new) + from - p.k;
        vo = reinterpret_cast<const char*>(p.v_new) + from - p.v;
      }
#pragma unroll 2
      for (int i = 0; i < kIters; ++i) {
        const int r = copy_r + i * kRows;
        const long long o = __shfl_sync(0xffffffffu, ko, r), w = __shfl_sync(0xffffffffu, vo, r);
        const bool ok = (seen >> r) & 1;
        const uint32_t d = (dst ^ ((i * kRows & 7) << 4)) + i * kRows * S::kRow;
        copy16_async(d, kc + o, ok);
        copy16_async(d + S::kHalf, vc + w, ok);
      }
    }
    copy_commit();
    if (ahead == 0) mask[0] = seen;
    else mask[1] = seen;
    ++ahead;
    put = put + 1 == S::kStages ? 0 : put + 1;
    if (++f_k < f_k1) page = page_of(f_k);
  };
  // turn to the share's next row once the present one is copied and multiplication is there
  auto advance = [&]() {
    if (f_k == f_k1 && !ahead_row && at < share.end) {
      const bool same = f_row + 1 < rows;                     // the sequence has more rows
      f_b += same ? 0 : 1;
      open(next, same ? p.lens[f_b] : len_next, -1);
      ahead_row = true;
    }
  };
  // queries as the right operand: head lane / 4 (+ 8 per further group), two dims a register
  uint32_t qf[G][KS][2];
  auto load_queries = [&]() {
    const int g = row.row / p.tiles, tile = row.row - g * p.tiles;
    const int heads = min(kHeads, p.group - tile * kHeads);
#pragma unroll
    for (int n = 0; n < G; ++n) {
      const int h = (mate * G + n) * 8 + lane / 4;
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p.q) +
                          (static_cast<long long>(row.b) * p.HQ + g * p.group + tile * kHeads +
                           (h < heads ? h : 0)) * (D / 2);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        qf[n][i][0] = h < heads ? __ldg(q + i * 8 + lane % 4) : 0u;
        qf[n][i][1] = h < heads ? __ldg(q + i * 8 + 4 + lane % 4) : 0u;
      }
    }
  };

  {
    // the first row: what does not wait for its length is loaded beside it
    const int len = p.lens[f_b];
    int early = -1;
    if (!p.cut) {
      row.b = f_b;
      row.row = static_cast<int>(at - before * rows);
      load_queries();
      const int j = warp * S::kTile + (lane & (S::kTile - 1));
      if (p.window == 0 && j < p.width * p.page_size)
        early = __ldg(p.tables + f_b * p.table_stride + div_by(j, p.page_mul, p.page_shift));
    }
    open(row, len, early);
    if (p.cut) load_queries();
  }
  fetch();
  advance();
  fetch();
  advance();

  float o[G][KS][4], m[G][2], l[G][2];
  auto clear = [&]() {
#pragma unroll
    for (int n = 0; n < G; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][i][j] = 0.f;
    }
  };
  clear();
  bool first_row = true;
  int st = 0;
  while (true) {
    if (ahead == 2) copy_wait<1>();
    else copy_wait<0>();
    team_sync();
    const uint32_t buf = ring + st * 2 * S::kHalf;
    const uint32_t seen = mask[0];
    float y[MT][G][4];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      float x[G][2][4];                  // two chains of products
#pragma unroll
      for (int n = 0; n < G; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[n][0][j] = x[n][1][j] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        uint32_t a[4];
        load_matrices(a, (buf + k_at + t * 16 * S::kRow) ^ (i * 32));
#pragma unroll
        for (int n = 0; n < G; ++n) mma<T>(x[n][i & 1], a, qf[n][i][0], qf[n][i][1]);
      }
#pragma unroll
      for (int n = 0; n < G; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) y[t][n][j] = (x[n][0][j] + x[n][1][j]) * p.scale_log2;
    }
    if (seen != kAll) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < G; ++n) {
          if (!((seen >> (t * 16 + lane / 4)) & 1)) y[t][n][0] = y[t][n][1] = -INFINITY;
          if (!((seen >> (t * 16 + lane / 4 + 8)) & 1)) y[t][n][2] = y[t][n][3] = -INFINITY;
        }
    }
    uint32_t pb[MT][G][2];
#pragma unroll
    for (int n = 0; n < G; ++n) {
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
      const float s0 = b0 - kUp<T>, s1 = b1 - kUp<T>;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const float p0 = exp2_fast(y[t][n][0] - s0), p1 = exp2_fast(y[t][n][1] - s1);
        const float p2 = exp2_fast(y[t][n][2] - s0), p3 = exp2_fast(y[t][n][3] - s1);
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
        for (int n = 0; n < G; ++n) mma<T>(o[n][i], a, pb[t][n][0], pb[t][n][1]);
      }
    team_sync();                          // every lane is done with this stage
    --ahead;
    mask[0] = mask[1];
    fetch();
    advance();
    const int used = st;
    st = st + 1 == S::kStages ? 0 : st + 1;
    if (--row.blocks > 0) continue;

    // The row is done.  The four warps' sums, through the stage that each has just used;
    // the next row's first tiles and queries are on their way meanwhile.
    const Row done = row;
    const bool more = ahead_row;
    if (more) {
      row = next;
      ahead_row = false;
      load_queries();
    }
    float* mine = reinterpret_cast<float*>(smem + warp * S::kWarpBytes + used * 2 * S::kHalf);
#pragma unroll
    for (int n = 0; n < G; ++n) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], d);
        l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], d);
      }
      const int h = (mate * G + n) * 8 + 2 * (lane % 4);
      if (lane < 4) {
        sm_m[warp][h] = m[n][0];
        sm_m[warp][h + 1] = m[n][1];
        sm_l[warp][h] = l[n][0];
        sm_l[warp][h + 1] = l[n][1];
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int d = (i * 16 + lane / 4) ^ ((lane % 4) << 3);   // other heads, other banks
        mine[h * D + d] = o[n][i][0];
        mine[(h + 1) * D + d] = o[n][i][1];
        mine[h * D + (d ^ 8)] = o[n][i][2];
        mine[(h + 1) * D + (d ^ 8)] = o[n][i][3];
      }
    }
    __syncthreads();
    const int g = done.row / p.tiles, tile = done.row - g * p.tiles;
    const int head0 = g * p.group + tile * kHeads, heads = min(kHeads, p.group - tile * kHeads);
    const long long slot = 2 * static_cast<long long>(blockIdx.x) + (first_row ? 0 : 1);
    const long long out0 = static_cast<long long>(done.b) * p.HQ + head0;
    // the warps' factors for head h; `writes`: this thread writes the head's lse or m and l
    auto factors = [&](int h, bool writes, float (&c)[kWarps]) {
      float mx = sm_m[0][h], lt = 0.f;
#pragma unroll
      for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, sm_m[w][h]);
      const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        c[w] = exp2_fast(sm_m[w][h] - base);
        lt += sm_l[w][h] * c[w];
      }
      if (done.whole) {
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) c[w] *= inv;
        if (writes && p.lse)
          p.lse[out0 + h] = lt == 0.f ? -INFINITY : (base + (log2f(lt) - kUp<T>)) * 0.6931471805599453f;
      } else if (writes) {
        *reinterpret_cast<float2*>(p.part_ml + (slot * kHeads + h) * 2) = make_float2(mx, lt);
      }
    };
    // Four values a thread, several heads at once.  Where a thread has more than two heads
    // the factors are computed once for all.
    constexpr int kAtOnce = kThreads / (D / 4), kTurns = kHeads / kAtOnce;
    constexpr int kUnroll = kTurns < 4 ? kTurns : 4;
    constexpr bool kShared = kTurns > 2;
    if constexpr (kShared) {
      if (tid < kHeads) {
        float c[kWarps];
        factors(tid, tid < heads, c);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sm_c[tid][w] = c[w];
      }
      __syncthreads();
    }
    const int d = tid % (D / 4) * 4;
#pragma unroll 1
    for (int h0 = tid / (D / 4); h0 < heads; h0 += kUnroll * kAtOnce) {
      float4 a[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int h = h0 + u * kAtOnce;
        float c[kWarps];
        if constexpr (kShared) {
#pragma unroll
          for (int w = 0; w < kWarps; ++w) c[w] = sm_c[h][w];
        } else {
          factors(h, d == 0 && h < heads, c);
        }
        a[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(smem + w * S::kWarpBytes + used * 2 * S::kHalf +
                                                            (h * D + (d ^ ((h & 6) << 2))) * 4);
          a[u].x += x.x * c[w];
          a[u].y += x.y * c[w];
          a[u].z += x.z * c[w];
          a[u].w += x.w * c[w];
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int h = h0 + u * kAtOnce;
        if (h >= heads) break;
        if (done.whole)
          reinterpret_cast<uint2*>(p.out)[((out0 + h) * D + d) / 4] =
              make_uint2(pack2<T>(a[u].x, a[u].y), pack2<T>(a[u].z, a[u].w));
        else
          *reinterpret_cast<float4*>(p.part_o + (slot * kHeads + h) * D + d) = a[u];
      }
    }
    if (!more) break;
    __syncthreads();                      // the stage and the warps' sums are free
    first_row = false;
    clear();
    advance();
    if (ahead < 2) fetch();
  }
}

// Adds up the parts of the rows that were cut: o = sum_i o_i 2^(m_i - m) / sum_i l_i 2^(m_i - m).
// CTA (x, y): kValues values from y kValues of the row of cut[x].  kValues / 4 threads take
// four values each; the CTA's groups of them take every kGroups-th part.  Few rows have many
// parts each: then a CTA takes few values and has many groups.  131072 tokens, 16 heads of 128 to
// one key-value head, 296 parts: 20.5 us in all with 32 values, 21.9 with 64, 23.5 with 128; but
// 4 x 16000 tokens, 64 heads over 4 of 256, where 32 values make 2048 CTAs: 54 us, 51 with 128.
constexpr int kJoinThreads = 256, kJoinParts = 2 * kSMs;

template <typename T, int D, int NG, int kValues>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const __grid_constant__ AttnArgs p) {
  constexpr int kHeads = 8 * NG, kHere = kValues > D ? kValues / D : 1;   // heads of a row, of this CTA
  constexpr int kQuads = kValues / 4, kGroups = kJoinThreads / kQuads;
  __shared__ float2 ml[kJoinParts][kHere];
  __shared__ float4 acc[kGroups][kQuads];
  __shared__ float sum[kGroups][kQuads], top[kJoinThreads / 32][kHere];
  const int tid = threadIdx.x, head0 = blockIdx.y * kValues / D;
  grid_wait();
  const int4 cut = p.cut[blockIdx.x];
  if (cut.x < 0) return;
  const int g = cut.y / p.tiles, tile = cut.y % p.tiles, c1 = cut.w >> 1, parts = c1 - cut.z + 1;
  if (head0 >= p.group - tile * kHeads) return;               // heads past the group's
  auto slot = [&](int i) { return 2 * static_cast<long long>(cut.z + i) + (i == 0 ? cut.w & 1 : 0); };
  float most = -INFINITY;                                     // of head tid % kHere
  for (int f = tid; f < parts * kHere; f += kJoinThreads) {
    const float2 x = reinterpret_cast<const float2*>(p.part_ml)[slot(f / kHere) * kHeads + head0 + f % kHere];
    ml[f / kHere][f % kHere] = x;
    most = fmaxf(most, x.x);
  }
#pragma unroll
  for (int o = 16; o >= kHere; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (tid % 32 < kHere) top[tid / 32][tid % 32] = most;
  __syncthreads();
  const int quad = tid % kQuads, group = tid / kQuads;
  const int hc = quad * 4 / D;                                // this thread's head of kHere
  float mx = top[0][hc];
#pragma unroll
  for (int i = 1; i < kJoinThreads / 32; ++i) mx = fmaxf(mx, top[i][hc]);
  const float base = mx == -INFINITY ? 0.f : mx;
  const float4* from = reinterpret_cast<const float4*>(p.part_o) + blockIdx.y * kQuads + quad;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 8
  for (int i = group; i < parts; i += kGroups) {
    const float4 v = from[slot(i) * (kHeads * D / 4)];
    const float w = exp2_fast(ml[i][hc].x - base);
    l += w * ml[i][hc].y;
    a.x += w * v.x;
    a.y += w * v.y;
    a.z += w * v.z;
    a.w += w * v.w;
  }
  acc[group][quad] = a;
  sum[group][quad] = l;
  __syncthreads();
  const int h = tile * kHeads + head0 + hc;
  if (group || h >= p.group) return;
#pragma unroll
  for (int i = 1; i < kGroups; ++i) {
    const float4 v = acc[i][quad];
    l += sum[i][quad];
    a.x += v.x;
    a.y += v.y;
    a.z += v.z;
    a.w += v.w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const long long r = static_cast<long long>(cut.x) * p.HQ + g * p.group + h;
  const int d = (blockIdx.y * kValues + quad * 4) % D;
  reinterpret_cast<uint2*>(p.out)[(r * D + d) / 4] =
      make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
  if (d == 0 && p.lse) p.lse[r] = l == 0.f ? -INFINITY : (base + (log2f(l) - kUp<T>)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ host

// Heads of a row: one group of 8 columns, two, or, of 64 dims, three where that makes fewer rows
// (the accumulators still fit the registers).  100 sequences of 3000 tokens, heads of 64 to a key-value
// head, three groups / two: 24 heads 22.8 / 29.7 us, 32 heads 34.0 / 30.2, 48 heads 34.9 / 39.4.
int heads_of(int group, int D) {
  if (group <= 8) return 8;
  return D == 64 && (group + 23) / 24 < (group + 15) / 16 ? 24 : 16;
}

// tokens of a block, CTAs per SM
int block_of(int D) { return D == 64 ? Shape<64>::kBlock : D == 128 ? Shape<128>::kBlock : Shape<256>::kBlock; }
int resident(int D) { return D == 64 ? Shape<64>::kResident : D == 128 ? Shape<128>::kResident : Shape<256>::kResident; }

// Rows are left whole, without partial sums and a join, where neither way of sharing unevenly costs more:
//  - rows of one length leave some CTAs without a row in the last wave; cutting them would take at most
//    4 blocks from every CTA.  Not cut / cut: 1 row of 100 tokens of 128 dims 5.3 / 7.0 us, of 512 tokens
//    10.2 / 7.1 us; 512 rows of 256 tokens 14.4 / 18.0 us, of 500 tokens 27.8 / 30.0 us; 300 rows of 330
//    tokens of 64 dims 12.3 / 14.8 us; of 256 dims 75 rows 11.5 / 15.0 us, 150 rows 20.2 / 19.0 us.
//  - the longest row the call allows beside short ones gives its CTA up to 24 blocks more than one a row.
//    Not cut / cut, 296 rows of 128 dims, rows rising from 1 token to so many, and one such row among
//    rows of 16 tokens: 576 tokens 22.5 / 34.8 and 18.4 / 20.5 us, 1024 30.7 / 51.2 and 24.6 / 20.5, 2048
//    49.2 / 71.7 and 36.9 / 22.5, 8192 154 / 143 and 125 / 24.6.

struct Plan {
  long long rows, grid;      // rows of a call; CTAs: what the GPU holds at once, or fewer
  bool split;                // whether rows may be cut
  size_t cut, bytes;         // entries of `cut`, workspace
};

Plan plan_of(int B, int HQ, int HKV, int D, long long max_tokens) {
  Plan q;
  const int heads = heads_of(HQ / HKV, D);
  q.rows = static_cast<long long>(B) * HKV * ((HQ / HKV + heads - 1) / heads);
  const long long nb = max_tokens > 0 ? (max_tokens + block_of(D) - 1) / block_of(D) : 1;
  const long long most = static_cast<long long>(kSMs) * resident(D);
  const long long waves = (q.rows + most - 1) / most;
  q.split = nb * (waves * most - q.rows) > 4 * most || waves * (nb - 1) > 24;
  const long long units = q.rows * (q.split ? nb : 1);
  q.grid = units < most ? units : most;
  q.cut = static_cast<size_t>(q.rows <= q.grid ? q.rows : q.grid);
  q.bytes = q.split ? q.cut * sizeof(int4) + static_cast<size_t>(q.grid) * 2 * heads * (D + 2) * 4 : 0;
  return q;
}

template <typename T, int D, int NG>
cudaError_t launch_shape(const AttnArgs& p, const Plan& q, cudaStream_t st) {
  cudaError_t e = allow_smem<attn_decode_kernel<T, D, NG>>(Shape<D>::kSmem);
  if (e != cudaSuccess) return e;
  attn_decode_kernel<T, D, NG><<<p.grid, kWarps * kTeam<D, NG> * 32, Shape<D>::kSmem, st>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess || !q.split) return e;
  const unsigned x = static_cast<unsigned>(q.cut);
  constexpr int kAll = 8 * NG * D;                            // values of a row
  if (q.rows * (kAll / 32) <= 4 * kSMs)
    return launch_after(attn_join_kernel<T, D, NG, 32>, dim3(x, kAll / 32), dim3(kJoinThreads), 0, st, p);
  if (q.rows * 8 <= q.grid)
    return launch_after(attn_join_kernel<T, D, NG, 128>, dim3(x, kAll / 128), dim3(kJoinThreads), 0, st, p);
  return launch_after(attn_join_kernel<T, D, NG, 512>, dim3(x, kAll / 512), dim3(kJoinThreads), 0, st, p);
}

template <typename T>
cudaError_t launch(const AttnArgs& p, int D, const Plan& q, cudaStream_t st) {
  const int groups = heads_of(p.group, D) / 8;
  if (D == 64)
    return groups == 1   ? launch_shape<T, 64, 1>(p, q, st)
           : groups == 2 ? launch_shape<T, 64, 2>(p, q, st)
                         : launch_shape<T, 64, 3>(p, q, st);
  if (D == 128) return groups == 1 ? launch_shape<T, 128, 1>(p, q, st) : launch_shape<T, 128, 2>(p, q, st);
  return groups == 1 ? launch_shape<T, 256, 1>(p, q, st) : launch_shape<T, 256, 2>(p, q, st);
}

}  // namespace

extern "C" {

size_t gdn_paged_attention_workspace_bytes(int B, int HQ, int HKV, int D, int max_tokens) {
  if (B < 1 || HQ < 1 || HKV < 1 || HQ % HKV != 0 || (D != 64 && D != 128 && D != 256)) return 0;
  return plan_of(B, HQ, HKV, D, max_tokens).bytes;
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
  if (static_cast<long long>(table_width) * page_size > 0x7fffffffLL - 1024 || table_stride < 0)
    return GDN_ERR_SHAPE;
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
  // CTAs write their rows' results while others, ahead of them or behind, still read theirs
  const size_t out_bytes = static_cast<size_t>(B) * HQ * D * 2, new_bytes = static_cast<size_t>(B) * HKV * D * 2;
  const size_t table_bytes = table_width > 0 ? 4 * static_cast<size_t>((B - 1) * table_stride + table_width) : 0;
  auto cache_bytes = [&](const int64_t* st) {
    return 2 * static_cast<size_t>((num_pages - 1) * st[0] + (page_size - 1) * st[1] + (HKV - 1) * st[2] + D);
  };
  auto meets_inputs = [&](const void* x, size_t bytes) {
    return overlaps(x, bytes, q, out_bytes) || overlaps(x, bytes, k_cache, cache_bytes(k_strides)) ||
           overlaps(x, bytes, v_cache, cache_bytes(v_strides)) ||
           (k_new && (overlaps(x, bytes, k_new, new_bytes) || overlaps(x, bytes, v_new, new_bytes))) ||
           overlaps(x, bytes, block_tables, table_bytes) || overlaps(x, bytes, seq_lens, 4 * static_cast<size_t>(B));
  };
  if (meets_inputs(output, out_bytes) || (k_new && k_cache == v_cache)) return GDN_ERR_ALIAS;
  // no row sees more than its table holds, or its window and sinks
  const int held = table_width * page_size;
  const int max_tokens = window > 0 && window + num_sinks < held ? window + num_sinks : held;
  const Plan plan = plan_of(B, HQ, HKV, D, max_tokens);
  if (plan.bytes > 0 && !workspace) return GDN_ERR_NULL;
  if (!aligned(workspace, 16)) return GDN_ERR_ALIGN;
  if (workspace_bytes < plan.bytes) return GDN_ERR_SHAPE;
  const size_t lse_bytes = static_cast<size_t>(B) * HQ * 4;
  if (lse && (meets_inputs(lse, lse_bytes) || overlaps(lse, lse_bytes, output, out_bytes))) return GDN_ERR_ALIAS;
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
  p.tiles = (p.group + heads_of(p.group, D) - 1) / heads_of(p.group, D);
  p.grid = static_cast<int>(plan.grid);
  if (plan.split) {
    p.cut = static_cast<int4*>(workspace);
    p.part_o = reinterpret_cast<float*>(p.cut + plan.cut);
    p.part_ml = p.part_o + static_cast<size_t>(2 * p.grid) * heads_of(p.group, D) * D;
    p.by_row = plan.rows <= plan.grid;
  }
  // a token's row lies at the same offset in both caches
  p.twin = p.k_page == p.v_page && p.k_tok == p.v_tok && (HKV == 1 || p.k_head == p.v_head);
  div_constants(static_cast<uint32_t>(page_size), p.page_mul, p.page_shift);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == GDN_DTYPE_BF16 ? launch<__nv_bfloat16>(p, D, plan, st) : launch<__half>(p, D, plan, st);
  return e == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // extern "C"
