// Bookkeeping of a paged key / value cache: mdlc_page_plan (block tables, slot
// maps and positions from request lengths) and mdlc_rope_append (rotary
// positions on queries and keys, keys and values written to their slots).
#include <climits>

#include "paged_attn.cuh"

namespace mdlc {
namespace {

// ------------------------------------------------------------ page plan
// Integer work on a few hundred KB at most, bounded by launch and load latency,
// so it is one launch: every block scans all requests (two running sums, pages
// asked for and new tokens) into shared memory, which costs each block one pass
// over 8 bytes per request from L2, instead of a scan kernel and an expansion
// kernel with a second launch between them. Then the blocks share the tokens
// (a binary search of the token's request in the scanned starts) and the
// requests' new table entries (a warp per request).
constexpr int kPlanThreads = 512;

struct PlanPtrs {
  const int32_t *cached, *fresh, *free_list, *free_count;
  int32_t *table, *q_starts, *kv_lens, *slots, *positions, *status;
};

struct Sums {
  long long tokens, pages;
};

MDLC_DEV Sums warp_scan(Sums v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, v.tokens, o), p = __shfl_up_sync(0xffffffffu, v.pages, o);
    if (lane >= o) {
      v.tokens += t;
      v.pages += p;
    }
  }
  return v;
}

// division by the page size: a shift where it is a power of two (64-bit divisions were most of a small plan's time)
struct PageDiv {
  uint32_t page;
  int shift;  // -1: not a power of two
};
MDLC_DEV uint32_t page_index(uint32_t tok, const PageDiv& d) { return d.shift >= 0 ? tok >> d.shift : tok / d.page; }
// pages of tok tokens (two int32 lengths' sum fits 32 bits unsigned)
MDLC_DEV uint32_t pages_of(uint32_t tok, const PageDiv& d) {
  const uint32_t n = page_index(tok, d);
  return n + (n * d.page != tok);
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const mdlc_page_desc d, const PlanPtrs p, const PageDiv pd, int* err) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ int32_t plan_smem[];
  int32_t* starts = plan_smem;              // [batch + 1] first token of each request, at most d.tokens
  int32_t* held_tok = starts + d.batch + 1; // [batch] cached tokens
  int32_t* first = held_tok + d.batch;      // [batch] index in the free list of the first page taken, -1: refused
  __shared__ Sums warp_sum[kPlanThreads / 32];
  __shared__ int taken_s, refused_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) taken_s = refused_s = 0;
  int n_free = d.free_pages;
  if (p.free_count) n_free = max(0, min(n_free, __ldg(p.free_count)));

  // thread t scans requests [t * per, (t + 1) * per)
  const int per = (d.batch + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, d.batch), b1 = min(b0 + per, d.batch);
  Sums mine = {0, 0};
  // pages that request b takes (0 where it does not fit its table row), and whether it fits
  auto ask = [&](int c, int n, bool* fits) {
    const uint32_t need = pages_of((uint32_t)c + (uint32_t)n, pd);
    *fits = need <= (uint32_t)d.table_stride;
    return *fits ? need - pages_of(c, pd) : 0u;
  };
  for (int b = b0; b < b1; ++b) {
    const int c = max(0, __ldg(p.cached + b)), n = max(0, __ldg(p.fresh + b));
    bool fits;
    mine.pages += ask(c, n, &fits);
    mine.tokens += n;
  }
  // sums of the threads in front of this one, and of all
  auto scan = [&](Sums v, Sums* all) {
    Sums run = warp_scan(v, lane);
    if (lane == 31) warp_sum[warp] = run;
    __syncthreads();
    if (warp == 0) {
      Sums w = lane < kPlanThreads / 32 ? warp_sum[lane] : Sums{0, 0};
      w = warp_scan(w, lane);
      if (lane < kPlanThreads / 32) warp_sum[lane] = w;
    }
    __syncthreads();
    *all = warp_sum[kPlanThreads / 32 - 1];
    if (warp) {
      run.tokens += warp_sum[warp - 1].tokens;
      run.pages += warp_sum[warp - 1].pages;
    }
    return Sums{run.tokens - v.tokens, run.pages - v.pages};
  };
  Sums all, run = scan(mine, &all);
  // a request brings only the tokens that have rows: what lies past the last row is not planned
  auto rows_of = [&](int b, long long start) {
    return (int)min((long long)max(0, __ldg(p.fresh + b)), max(0ll, d.tokens - start));
  };
  if (all.tokens > d.tokens) {  // pages again, of those tokens alone
    Sums cut = {0, 0};
    long long at = run.tokens;
    for (int b = b0; b < b1; ++b) {
      bool fits;
      cut.pages += ask(max(0, __ldg(p.cached + b)), rows_of(b, at), &fits);
      at += max(0, __ldg(p.fresh + b));
    }
    __syncthreads();
    run.pages = scan(cut, &all).pages;
  }
  int taken = 0, refused = 0;
  for (int b = b0; b < b1; ++b) {
    const int c = max(0, __ldg(p.cached + b)), n = rows_of(b, run.tokens);
    bool fits;
    const uint32_t take = ask(c, n, &fits);
    const bool ok = fits && (take == 0 || run.pages + take <= n_free);
    starts[b] = (int32_t)min(run.tokens, (long long)d.tokens);
    held_tok[b] = c;
    first[b] = ok ? (take ? (int32_t)run.pages : 0) : -1;
    run.tokens += max(0, __ldg(p.fresh + b));
    run.pages += take;
    if (ok && take) taken = (int)run.pages;
    refused += !ok;
    if (blockIdx.x == 0) {
      p.q_starts[b] = starts[b];
      p.kv_lens[b] = ok ? c + n : c;
    }
    if (b == d.batch - 1) {
      starts[d.batch] = (int32_t)min(run.tokens, (long long)d.tokens);
      if (blockIdx.x == 0) p.q_starts[d.batch] = starts[d.batch];
    }
  }
  if (blockIdx.x == 0) {
    if (taken) atomicMax(&taken_s, taken);
    if (refused) atomicAdd(&refused_s, refused);
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    p.status[0] = taken_s;
    p.status[1] = refused_s;
  }

  // new table entries: a warp per request
  const int nwarps = gridDim.x * (kPlanThreads / 32);
  for (int b = blockIdx.x * (kPlanThreads / 32) + warp; b < d.batch; b += nwarps) {
    if (first[b] < 0) continue;
    const int c = held_tok[b];
    const int held = (int)pages_of(c, pd), take = (int)pages_of((uint32_t)c + (uint32_t)(starts[b + 1] - starts[b]), pd) - held;
    for (int j = lane; j < take; j += 32)
      if (MDLC_CHECK_IDX(err, held + j, d.table_stride) && MDLC_CHECK_IDX(err, first[b] + j, d.free_pages)) p.table[(long long)b * d.table_stride + held + j] = __ldg(p.free_list + first[b] + j);
  }

  // slots and positions
  for (int t = blockIdx.x * kPlanThreads + tid; t < d.tokens; t += gridDim.x * kPlanThreads) {
    int lo = 0, hi = d.batch;  // the number of requests that end at or before t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid + 1] <= t) lo = mid + 1; else hi = mid;
    }
    int slot = -1, pos = 0;
    if (lo < d.batch) {
      const int c = held_tok[lo];
      pos = c + (t - starts[lo]);
      if (first[lo] >= 0) {
        const int at = (int)page_index(pos, pd), held = (int)pages_of(c, pd);
        if (!MDLC_CHECK_IDX(err, at < held ? at : first[lo] + (at - held), at < held ? d.table_stride : d.free_pages)) continue;
        // a page taken by this call comes from the free list itself: its table entry may not be written yet
        const int id = at < held ? __ldg(p.table + (long long)lo * d.table_stride + at)
                                 : __ldg(p.free_list + first[lo] + (at - held));
        // an id whose slots do not fit 32 bits would wrap onto another page's
        const long long wide = (long long)id * d.page + (pos - at * d.page);
        if (id >= 0 && wide <= INT_MAX) slot = (int)wide;
        else record_error(err, MDLC_DEVERR_BOUNDS);
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

// ------------------------------------------------------------ rotary append
// Memory-bound: every element of q, k and v is read and written once. A warp (or
// a block, when there are few tokens) takes a token; a thread owns one unit of V
// pairs, reads their cosines and sines once and turns that unit of head after
// head, kRopeBatch heads' loads in flight at a time, the first ones before the angles are known. q_out may be q (so loads of a
// batch precede its stores, and no thread reads what another writes).
constexpr int kRopeThreads = 128;
constexpr int kRopeBatch = 4;

struct RopeArgs {
  mdlc_rope_desc d;
  const void *q, *k, *v;
  const int32_t* positions;
  const float2* table;
  const int32_t* slots;
  void *q_out, *k_cache, *v_cache;
  int warps_per_token;
  SmallDiv units, rest, vals;  // units of a head that turn; vectors of its rest; vectors of a value head
  int page_shift;              // log2 of the page size, -1: not a power of two
};

// V elements of T as one load or store of 16, 8 or sizeof(T) bytes
template <int BYTES>
struct RawVec;
template <>
struct RawVec<16> { using type = uint4; };
template <>
struct RawVec<8> { using type = uint2; };
template <>
struct RawVec<4> { using type = uint32_t; };
template <>
struct RawVec<2> { using type = uint16_t; };

MDLC_DEV float to_f(float v) { return v; }
MDLC_DEV float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
MDLC_DEV T from_f(float v);
template <>
MDLC_DEV float from_f<float>(float v) { return v; }
template <>
MDLC_DEV __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int V>
union Pack {
  typename RawVec<V * (int)sizeof(T)>::type raw;
  T e[V];
  MDLC_DEV Pack() {}
};

template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads, 5) rope_append_kernel(const RopeArgs a, int* err) {
  pdl_wait();
  pdl_trigger();
  using Raw = typename RawVec<V * (int)sizeof(T)>::type;
  const mdlc_rope_desc& d = a.d;
  const int nt = a.warps_per_token * 32;  // threads of one token
  const int tl = threadIdx.x % nt;
  const long long t = (long long)blockIdx.x * (kRopeThreads / nt) + threadIdx.x / nt;
  if (t >= d.tokens) return;
  const int half = d.rot_dim / 2;
  const int slot = __ldg(a.slots + t);
  int pos[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) pos[x] = x < d.axes ? __ldg(a.positions + (long long)x * d.tokens + t) : 0;
  const T* q = static_cast<const T*>(a.q) + t * d.q_stride;
  const T* k = static_cast<const T*>(a.k) + t * d.k_stride;
  const T* v = static_cast<const T*>(a.v) + t * d.v_stride;
  T* qo = a.q_out ? static_cast<T*>(a.q_out) + t * d.out_stride : nullptr;
  const int hr = d.heads + d.kv_heads, h0 = qo ? 0 : d.heads;  // heads that turn: [h0, hr)
  auto src_of = [&](int h) { return h < d.heads ? q + (long long)h * d.head_dim : k + (long long)(h - d.heads) * d.head_dim; };

  // the first batch's loads do not wait for the slot, the positions and the angles behind them
  const int units = half / V;  // per head
  const int lanes = units ? div_small(nt, a.units) : 0;
  const int hl = units ? div_small(tl, a.units) : 0, u = tl - hl * units;
  const int o0 = INTERLEAVED ? 2 * u * V : u * V, o1 = INTERLEAVED ? o0 + V : o0 + half;
  Pack<T, V> x[kRopeBatch], y[kRopeBatch];
  auto load_batch = [&](int hb) {
#pragma unroll
    for (int j = 0; j < kRopeBatch; ++j) {
      const int h = hb + j * lanes;
      if (h < hr) {
        const T* s = src_of(h);
        x[j].raw = *reinterpret_cast<const Raw*>(s + o0);
        y[j].raw = *reinterpret_cast<const Raw*>(s + o1);
      }
    }
  };
  if (hl < lanes) load_batch(h0 + hl);

  bool known = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) known &= (unsigned)pos[i] < (unsigned)d.max_pos;
  if (!known) {
    record_error(err, MDLC_DEVERR_BOUNDS);
    return;
  }
  const bool stored = slot >= 0 && slot < d.pages * d.page;
  if (slot >= 0 && !stored) record_error(err, MDLC_DEVERR_BOUNDS);
  // element offset of (slot, head 0) in a cache, and between its heads
  const long long head_step = (long long)d.page * d.head_dim;
  const int page_id = a.page_shift >= 0 ? slot >> a.page_shift : slot / d.page;
  const long long at = stored ? (long long)page_id * d.kv_heads * head_step + (long long)(slot - page_id * d.page) * d.head_dim : 0;
  T* kc = static_cast<T*>(a.k_cache) + at;
  T* vc = static_cast<T*>(a.v_cache) + at;
  const int h1 = stored ? hr : d.heads;  // heads to write
  // (the checked build: the last element of the token's last head)
  if (stored && !MDLC_CHECK_IDX(err, at + (d.kv_heads - 1) * head_step + d.head_dim - 1, (long long)d.pages * d.kv_heads * head_step)) return;
  auto dst_of = [&](int h) { return h < d.heads ? qo + (long long)h * d.head_dim : kc + (h - d.heads) * head_step; };

  if (hl < lanes) {
    float cs[V], sn[V];
    // pair i belongs to the axis whose section holds it
    const int e0 = d.section[0], e1 = e0 + d.section[1], e2 = e1 + d.section[2];  // sections past `axes` are 0
    const float2* tab = a.table + u * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int pair = u * V + i;
      const int p = pair < e0 ? pos[0] : (pair < e1 ? pos[1] : (pair < e2 ? pos[2] : pos[3]));
      const float2 w = __ldg(tab + (long long)p * half + i);
      cs[i] = w.x;
      sn[i] = w.y;
    }
    for (int hb = h0 + hl; hb < h1; hb += lanes * kRopeBatch) {
      if (hb != h0 + hl) load_batch(hb);
#pragma unroll
      for (int j = 0; j < kRopeBatch; ++j) {
        const int h = hb + j * lanes;
        if (h < h1) {
          Pack<T, V> ox, oy;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            // pair i: (x_i, y_i) of the two halves, or elements 2i, 2i + 1 of the run (x, y)
            if constexpr (INTERLEAVED) {
              const int e0 = 2 * i, e1 = 2 * i + 1;
              const float p0 = to_f(e0 < V ? x[j].e[e0 % V] : y[j].e[e0 % V]);
              const float p1 = to_f(e1 < V ? x[j].e[e1 % V] : y[j].e[e1 % V]);
              const T r0 = from_f<T>(p0 * cs[i] - p1 * sn[i]), r1 = from_f<T>(p1 * cs[i] + p0 * sn[i]);
              if (e0 < V) ox.e[e0 % V] = r0; else oy.e[e0 % V] = r0;
              if (e1 < V) ox.e[e1 % V] = r1; else oy.e[e1 % V] = r1;
            } else {
              const float p0 = to_f(x[j].e[i]), p1 = to_f(y[j].e[i]);
              ox.e[i] = from_f<T>(p0 * cs[i] - p1 * sn[i]);
              oy.e[i] = from_f<T>(p1 * cs[i] + p0 * sn[i]);
            }
          }
          T* o = dst_of(h);
          *reinterpret_cast<Raw*>(o + o0) = ox.raw;
          *reinterpret_cast<Raw*>(o + o1) = oy.raw;
        }
      }
    }
  }
  // the part of each head that does not turn, and the values
  const int rest = (d.head_dim - d.rot_dim) / V;
  if (rest) {
    for (int i = tl; i < (h1 - h0) * rest; i += nt) {
      const int hi = div_small(i, a.rest), h = h0 + hi, o = d.rot_dim + (i - hi * rest) * V;
      *reinterpret_cast<Raw*>(dst_of(h) + o) = *reinterpret_cast<const Raw*>(src_of(h) + o);
    }
  }
  if (stored) {
    const int vu = d.head_dim / V;
#pragma unroll 2
    for (int i = tl; i < d.kv_heads * vu; i += nt) {
      const int h = div_small(i, a.vals), o = (i - h * vu) * V;
      *reinterpret_cast<Raw*>(vc + h * head_step + o) = *reinterpret_cast<const Raw*>(v + (long long)h * d.head_dim + o);
    }
  }
}

template <typename T, int V>
cudaError_t launch_rope(mdlc_ctx* ctx, const RopeArgs& a) {
  const int per_block = kRopeThreads / (a.warps_per_token * 32);
  const dim3 grid((unsigned)((a.d.tokens + per_block - 1) / per_block));
  return a.d.interleaved ? launch_pdl(rope_append_kernel<T, V, true>, grid, dim3(kRopeThreads), 0, ctx->stream, a, ctx->d_err)
                         : launch_pdl(rope_append_kernel<T, V, false>, grid, dim3(kRopeThreads), 0, ctx->stream, a, ctx->d_err);
}

}  // namespace
}  // namespace mdlc

using namespace mdlc;

extern "C" int mdlc_page_plan(mdlc_ctx* ctx, const mdlc_page_desc* d, const int32_t* cached_lens, const int32_t* new_lens,
                              const int32_t* free_list, const int32_t* free_count, int32_t* block_table,
                              int32_t* q_starts, int32_t* kv_lens, int32_t* slots, int32_t* positions, int32_t* status) {
  if (!ctx) return MDLC_ERR_INVALID;
  if (!d || !cached_lens || !new_lens || !block_table || !q_starts || !kv_lens || !slots || !positions || !status)
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "page_plan: null argument");
  if (d->batch < 1 || d->batch > MDLC_MAX_REQUESTS || d->page < 1 || d->page > 1024 || d->table_stride < 1 ||
      d->tokens < 1 || d->free_pages < 0 || (d->free_pages > 0 && !free_list))
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "page_plan: bad descriptor (batch %d, page %d, table_stride %d, tokens %d, free_pages %d)",
                          d->batch, d->page, d->table_stride, d->tokens, d->free_pages);
  if ((long long)d->table_stride * d->page > INT32_MAX)
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "page_plan: table_stride * page exceeds 2^31 - 1");
  cudaSetDevice(ctx->device);
  const size_t smem = (3 * (size_t)d->batch + 1) * sizeof(int32_t);
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (3 * MDLC_MAX_REQUESTS + 1) * (int)sizeof(int32_t));
    if (e != cudaSuccess) return mdlc_cuda_status(ctx, e, "page_plan shared memory");
  }
  // two tokens per thread; the scan is repeated in each block, so no more blocks than SMs
  const int blocks = (int)min((long long)ctx->num_sms, ((long long)d->tokens + 2 * kPlanThreads - 1) / (2 * kPlanThreads));
  const PlanPtrs p = {cached_lens, new_lens, free_list, free_count, block_table, q_starts, kv_lens, slots, positions, status};
  PageDiv pd = {(uint32_t)d->page, -1};
  for (int i = 0; i <= 10; ++i)
    if (d->page == 1 << i) pd.shift = i;
  const cudaError_t e = launch_pdl(page_plan_kernel, dim3(blocks), dim3(kPlanThreads), smem, ctx->stream, *d, p, pd, ctx->d_err);
  mdlc_note_launch(ctx);
  return mdlc_cuda_status(ctx, e, "page_plan launch");
}

extern "C" int mdlc_rope_append(mdlc_ctx* ctx, const mdlc_rope_desc* d, const void* q, const void* k, const void* v,
                                const int32_t* positions, const float* table, const int32_t* slots, void* q_out,
                                void* k_cache, void* v_cache) {
  if (!ctx) return MDLC_ERR_INVALID;
  if (!d || !q || !k || !v || !positions || !table || !slots || !k_cache || !v_cache)
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "rope_append: null argument");
  if (d->tokens < 1 || d->heads < 1 || d->kv_heads < 1 || d->head_dim < 2 || d->head_dim > 256 || d->rot_dim < 0 ||
      d->rot_dim % 2 || d->rot_dim > d->head_dim || d->axes < 1 || d->axes > 4 || d->max_pos < 1 || d->page < 1 ||
      d->pages < 1 || (d->interleaved != 0 && d->interleaved != 1) || (d->dtype != MDLC_BF16 && d->dtype != MDLC_F32))
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "rope_append: bad descriptor (head_dim %d, rot_dim %d, axes %d)", d->head_dim, d->rot_dim, d->axes);
  int pairs = 0;
  for (int i = 0; i < d->axes; ++i) {
    if (d->section[i] < 0 || d->section[i] > d->rot_dim / 2) return mdlc_set_error(ctx, MDLC_ERR_INVALID, "rope_append: bad section");
    pairs += d->section[i];
  }
  if (pairs != d->rot_dim / 2)
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "rope_append: sections sum to %d pairs, rot_dim has %d", pairs, d->rot_dim / 2);
  if ((long long)d->pages * d->page > INT32_MAX)
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "rope_append: pages * page exceeds 2^31 - 1");
  const long long hw = (long long)d->heads * d->head_dim, kw = (long long)d->kv_heads * d->head_dim;
  if ((d->heads + d->kv_heads) * (long long)d->head_dim > 65535)
    return mdlc_set_error(ctx, MDLC_ERR_UNSUPPORTED, "rope_append: a token of more than 65535 elements");
  if ( d->q_stride < hw || d->k_stride < kw || d->v_stride < kw || (q_out && d->out_stride < hw))
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "rope_append: a token stride is smaller than its heads");
  const int esz = d->dtype == MDLC_BF16 ? 2 : 4;
  const uintptr_t addr = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_cache | (uintptr_t)v_cache;
  if (addr % esz || (uintptr_t)table % 8) return mdlc_set_error(ctx, MDLC_ERR_INVALID, "rope_append: misaligned pointer");
  cudaSetDevice(ctx->device);
  // the widest vector that every pointer, stride and run of pairs allows
  const long long strides = d->q_stride | d->k_stride | d->v_stride | (q_out ? d->out_stride : 0);
  auto fits = [&](int vec) { return (d->rot_dim / 2) % vec == 0 && d->head_dim % vec == 0 && strides % vec == 0 && addr % (vec * esz) == 0; };
  const int full = 16 / esz;
  const int vec = fits(full) ? full : (fits(4) ? 4 : 1), units = d->rot_dim / 2 / vec;
  RopeArgs a = {*d, q, k, v, positions, reinterpret_cast<const float2*>(table), slots, q_out, k_cache, v_cache};
  for (int i = d->axes; i < 4; ++i) a.d.section[i] = 0;
  a.units = small_div(max(1, units));
  a.rest = small_div(max(1, (d->head_dim - d->rot_dim) / vec));
  a.vals = small_div(d->head_dim / vec);
  a.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (d->page == 1 << i) a.page_shift = i;
  // Warps of a token: enough for one batch of loads per thread to hold all of its heads; few tokens, or element by element
  // (128 units): a block
  a.warps_per_token = 1;
  while (a.warps_per_token < kRopeThreads / 32 && units && a.warps_per_token * 32 / units * kRopeBatch < d->heads + d->kv_heads) a.warps_per_token *= 2;
  if (vec == 1 || d->tokens < 4 * ctx->num_sms) a.warps_per_token = kRopeThreads / 32;
  cudaError_t e;
  if (esz == 2)
    e = vec == 8 ? launch_rope<__nv_bfloat16, 8>(ctx, a) : (vec == 4 ? launch_rope<__nv_bfloat16, 4>(ctx, a) : launch_rope<__nv_bfloat16, 1>(ctx, a));
  else
    e = vec == 4 ? launch_rope<float, 4>(ctx, a) : launch_rope<float, 1>(ctx, a);
  mdlc_note_launch(ctx);
  return mdlc_cuda_status(ctx, e, "rope_append launch");
}
