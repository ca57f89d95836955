// Shared by the attention kernels (paged_attn.cu, paged_attn_tc.cu): arguments, the
// geometry of a request, and how blocks find their work.
#pragma once

#include "common.cuh"
#include "runtime.h"

namespace mdlc {

// n / d for 0 <= n < 65536 and 1 <= d <= 65536 as a product: a runtime division costs some 20 instructions
struct SmallDiv {
  uint32_t m;  // ceil(2^32 / d), 0 for d = 1
};
inline SmallDiv small_div(int d) { return {d == 1 ? 0u : 0xffffffffu / (uint32_t)d + 1u}; }
MDLC_DEV int div_small(int n, const SmallDiv& s) { return s.m ? (int)__umulhi((uint32_t)n, s.m) : n; }

struct AttnArgs {
  mdlc_attn_desc d;
  const void *q, *k, *v;
  const int32_t *table, *q_starts, *kv_lens;
  void* out;
  float* lse;
  int group;          // query heads per key head
  SmallDiv group_div;
  int split_rows;     // requests with at most this many rows go to split mode
  int splits, short_splits;  // chunk mode: blocks that may share a row tile's keys; the same where their shares are short
  float scale_log2;   // scale * log2(e)
  // workspace: partial sums [slot][rows][hdp], their maxima (base-2 exponent) and sums [slot][rows]
  float *part_o, *part_m, *part_l;
  long long part_rows;    // rows of the workspace, and the error word: for the checked build
  int* err;
  int* arrived;           // split mode: arrivals at the tile that starts in block c and others share
};

// chunk mode on the tensor cores' tcgen05 form (bf16): keys of a block, rows of a block
constexpr int kTcKeys = 128;
int attn_tc_rows(int head_dim);
bool attn_tc_fits(const mdlc_attn_desc& d);
int attn_tc_smem(int head_dim);
cudaError_t attn_tc_launch(mdlc_ctx* ctx, cudaStream_t stream, const AttnArgs& a, dim3 grid);
// tensor maps of the two caches (rows of head_dim elements) with boxes of `box` rows x 64 columns, 128-byte swizzle
cudaError_t attn_tensor_maps(const AttnArgs& a, int box, CUtensorMap* k, CUtensorMap* v);

// ------------------------------------------------------------ one request's geometry
struct Request {
  int q0, q_len, kv_len;
  int shift;  // position of row 0; q_len may be fewer rows than the request has (max_q, tokens), the positions are those of all
};
MDLC_DEV Request request_of(const AttnArgs& a, int b) {
  Request r;
  const int s0 = __ldg(a.q_starts + b), s1 = __ldg(a.q_starts + b + 1);
  r.q0 = max(0, min(s0, a.d.tokens));
  r.q_len = min(max(0, min(s1, a.d.tokens) - r.q0), a.d.max_q);
  r.kv_len = max(0, min(__ldg(a.kv_lens + b), a.d.max_kv));  // the host has cut max_kv to the table's row
  r.shift = r.kv_len - max(0, s1 - r.q0);
  return r;
}

// Blocks of bt keys that the rows of tokens [i0, i1] of a request can see: blocks
// [0, n_first) hold the first tokens kept by `sinks`, the others start at `start`.
struct Span {
  int lo, hi;     // keys below lo are hidden from every row unless below sinks; keys from hi on too
  int n_first, start, n;
};
MDLC_DEV Span span_of(const AttnArgs& a, const Request& r, int i0, int i1, int bt) {
  Span s;
  s.hi = max(0, min(r.kv_len, r.shift + i1 + 1));
  s.lo = a.d.window > 0 ? (int)max(0ll, (long long)r.shift + i0 - a.d.window + 1) : 0;
  s.n_first = (min(a.d.sinks, s.lo) + bt - 1) / bt;
  s.start = s.lo / bt * bt;
  if (s.start <= s.n_first * bt) s.n_first = s.start = 0;
  s.n = s.n_first + (max(0, s.hi - s.start) + bt - 1) / bt;
  if (s.hi == 0) s.n = 0;
  return s;
}
MDLC_DEV int key_of_block(const Span& s, int blk, int bt) {
  return blk < s.n_first ? blk * bt : s.start + (blk - s.n_first) * bt;
}

// ------------------------------------------------------------ index checks (constant true but in the checked build)
MDLC_DEV bool table_ok(const AttnArgs& a, int b, int entry) {
  return MDLC_CHECK_IDX(a.err, b, a.d.batch) && MDLC_CHECK_IDX(a.err, entry, a.d.table_stride);
}
// columns [c, c + n) of a head of a token
MDLC_DEV bool out_ok(const AttnArgs& a, long long tok, int head, int c, int n) {
  return MDLC_CHECK_IDX(a.err, tok, a.d.tokens) && MDLC_CHECK_IDX(a.err, head, a.d.heads) && MDLC_CHECK_IDX(a.err, c + n - 1, a.d.head_dim);
}
MDLC_DEV bool part_ok(const AttnArgs& a, long long row) { return MDLC_CHECK_IDX(a.err, row, a.part_rows); }

// ------------------------------------------------------------ finding work
// exclusive sum over the block's threads of v; *total: the sum of all
MDLC_DEV long long block_scan(long long v, long long* warp_sums, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long run = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += x;
  }
  if (lane == 31) warp_sums[warp] = run;
  __syncthreads();
  long long before = 0, all = 0;
  for (int w = 0; w < nw; ++w) {
    if (w < warp) before += warp_sums[w];
    all += warp_sums[w];
  }
  __syncthreads();
  *total = all;
  return before + run - v;
}

struct Place {
  int b;
  long long first;  // first unit (split) or tile (chunk) of request b
};

// Chunk mode: tile `want` counted from the last one (a request's last tiles see the most
// keys, so they start first) as (request, its row tile). False: there is no such tile.
struct Tile {
  Request rq;
  int b, r0, rows;  // first row, rows of the request
};
MDLC_DEV bool find_tile(const AttnArgs& a, long long want, int tile_rows, long long* warp_sums, Place* place, Tile* t) {
  auto tiles = [&](int b) -> long long {
    const long long rows = (long long)request_of(a, b).q_len * a.group;
    return rows <= a.split_rows ? 0 : (rows + tile_rows - 1) / tile_rows;
  };
  const int per = (a.d.batch + blockDim.x - 1) / blockDim.x;
  const int b0 = min((int)threadIdx.x * per, a.d.batch), b1 = min(b0 + per, a.d.batch);
  long long mine = 0, total;
  for (int b = b0; b < b1; ++b) mine += tiles(b);
  long long at = block_scan(mine, warp_sums, &total);
  if (want >= total) return false;
  const long long u = total - 1 - want;
  if (u >= at && u < at + mine) {
    for (int b = b0;; ++b) {
      const long long n = tiles(b);
      if (u < at + n) {
        *place = {b, at};
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  t->b = place->b;
  t->rq = request_of(a, t->b);
  t->r0 = (int)(u - place->first) * tile_rows;
  t->rows = t->rq.q_len * a.group;
  return true;
}
// blocks that share a tile of n key blocks: each gets at least `least`, twice as many where more than short_splits share
MDLC_DEV int splits_of(const AttnArgs& a, int n, int least) {
  return max(1, max(min(a.short_splits, n / least), min(a.splits, n / (2 * least))));
}

template <typename T>
MDLC_DEV void store_out(T* p, float v);
template <>
MDLC_DEV void store_out<float>(float* p, float v) { *p = v; }
template <>
MDLC_DEV void store_out<__nv_bfloat16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

}  // namespace mdlc
