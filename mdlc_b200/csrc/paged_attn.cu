// mdlc_paged_attn: attention of each request's new tokens over its cache pages.
//
// The rows of one key head are its G query heads of every new token of a request
// (row r: token r / G, head e * G + r % G), so a key or value loaded once serves them
// all. One pass over the keys with the running maximum and sum of the softmax (both
// fp32, in the base-2 exponent); scores never leave registers.
//
// attn_kernel is the mma.sync form for both types. A warp holds 16 rows; the four warps
// of a block are WM row groups x WN = 4 / WM key groups, every key group with its
// own cp.async ring of BT-key blocks (16-byte chunks swizzled by the row, so
// that ldmatrix and the fp32 fragment reads are free of bank conflicts). bf16: m16n8k16;
// fp32: every product as three tf32 products (high and low parts, the low x low term,
// 2^-22 of the product, dropped).
//   split mode (few rows per request: decoding): bounded by the cache's bytes. The
//     keys of all (request, key head) tiles form one line of 128-key units, cut evenly
//     over the blocks whatever the requests' lengths; a tile cut between blocks leaves
//     partial sums in the workspace, which attn_join_kernel adds in block order.
//   chunk mode (many rows): a block per row tile.
#include "paged_attn.cuh"

namespace mdlc {
namespace {

constexpr int kAttnThreads = 128;
constexpr int kStages = 3;
constexpr int kUnit = 128;      // keys of one unit of split work
constexpr int kMaxBlocks = 512; // split-mode blocks at most (bounds the workspace)
constexpr int kJoinThreads = 256;
constexpr int kLeastKeys = 256; // keys of a share of a chunk tile at least
constexpr int kChunkBlocks = 148;  // shares are made until chunk mode fills this many SMs

template <typename T, int HDP>
constexpr int block_keys() { return sizeof(T) * HDP <= 256 ? 32 : 16; }

// ------------------------------------------------------------ mma fragments
MDLC_DEV void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
MDLC_DEV void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
MDLC_DEV uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
MDLC_DEV void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
MDLC_DEV void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// high part (a tf32 value) and the exact rest of an fp32 number
MDLC_DEV uint32_t tf_hi(uint32_t x) { return x & 0xffffe000u; }
MDLC_DEV uint32_t tf_lo(uint32_t x) { return __float_as_uint(__uint_as_float(x) - __uint_as_float(tf_hi(x))); }
// c += a b of fp32 operands in three tf32 products, the small ones first
MDLC_DEV void mma_3tf32(float (&c)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4], uint32_t b0, uint32_t b1) {
  mma_tf32(c, lo, tf_hi(b0), tf_hi(b1));
  mma_tf32(c, hi, tf_lo(b0), tf_lo(b1));
  mma_tf32(c, hi, tf_hi(b0), tf_hi(b1));
}

MDLC_DEV void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

MDLC_DEV float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
MDLC_DEV float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// ------------------------------------------------------------ the kernel
template <typename T, int HDP, int WM>
struct Cfg {
  static constexpr int WN = 4 / WM;
  static constexpr int ROWS = 16 * WM;
  static constexpr int BT = block_keys<T, HDP>();
  static constexpr int PITCH = HDP * (int)sizeof(T);       // bytes of a key in shared memory
  static constexpr int STAGE = 2 * BT * PITCH;             // keys and values of one block
  static constexpr int RING = WN * kStages * STAGE;
  static constexpr int MERGE = WN * ROWS * (HDP + 2) * 4;  // the key groups' sums, over the ring
  static constexpr int SMEM = (RING > MERGE ? RING : MERGE);
};

// Rows [r0, r0 + 16 WM) of (request, key head e) over the span's blocks [blk0, blk1). Whole: writes out
// and lse; else leaves the sums in workspace slot `slot`.
template <typename T, int HDP, int WM>
MDLC_DEV void attn_piece(const AttnArgs& a, unsigned char* smem, uint32_t (*valid_s)[kStages], int* err, int b,
                         const Request& rq, int e, int r0, const Span& sp, int blk0, int blk1, bool whole, long long slot) {
  using K = Cfg<T, HDP, WM>;
  constexpr int BT = K::BT, WN = K::WN, PITCH = K::PITCH;
  constexpr int CH = PITCH / 16;                 // 16-byte chunks of a key
  constexpr int EC = 16 / (int)sizeof(T);        // elements of a chunk
  constexpr int GT = WM * 32;                    // threads of a key group
  constexpr bool kBf16 = sizeof(T) == 2;
  const mdlc_attn_desc& d = a.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wm = warp % WM, wn = warp / WM, gt = threadIdx.x - wn * GT;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + wn * kStages * K::STAGE;
  const int chunks = d.head_dim / EC;
  const int rows = rq.q_len * a.group;
  const int shift = rq.kv_len - rq.q_len;
  auto sync_group = [&]() {
    if constexpr (WM == 1) __syncwarp(); else named_sync(1 + wn, GT);
  };

  // this thread's two rows: their position and query
  int pos[2];
  const T* qp[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r0 + wm * 16 + h * 8 + g;
    const bool ok = r < rows;
    const int i = ok ? r / a.group : 0;
    pos[h] = ok ? shift + i : -1;
    qp[h] = ok ? static_cast<const T*>(a.q) + (long long)(rq.q0 + i) * d.q_stride + (long long)(e * a.group + r % a.group) * d.head_dim : nullptr;
  }
  constexpr int KS = kBf16 ? HDP / 16 : HDP / 8;  // steps of the score product
  uint32_t qa[KS][4];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // bf16: columns 16 ks + 2 t + (i >> 1) * 8, two of them; fp32: column 8 ks + t + (i >> 1) * 4
      const int c = kBf16 ? 16 * ks + 2 * t + (i >> 1) * 8 : 8 * ks + t + (i >> 1) * 4;
      qa[ks][i] = (qp[i & 1] && c < d.head_dim) ? __ldg(reinterpret_cast<const uint32_t*>(qp[i & 1] + c)) : 0u;
    }

  auto base_of = [&](int blk) { return key_of_block(sp, blk, BT); };
  // cache row (key `lane` of the block) or -1: hidden from every row, or no such page
  auto row_of = [&](int blk) {
    const int j = base_of(blk) + lane;
    int row = -1;
    if (blk < blk1 && lane < BT && j < rq.kv_len && (j >= sp.lo || j < d.sinks)) {
      const int id = __ldg(a.table + (long long)b * d.table_stride + j / d.page);
      if ((unsigned)id < (unsigned)d.pages) row = (id * d.kv_heads + e) * d.page + j % d.page;
      else record_error(err, MDLC_DEVERR_BOUNDS);
    }
    return row;
  };
  auto issue = [&](int blk, int row, int stage) {
    if (blk < blk1) {
      const uint32_t ks = ring + stage * K::STAGE, vs = ks + BT * PITCH;
      const uint32_t valid = __ballot_sync(0xffffffffu, row >= 0);
      if (lane == 0 && wm == 0) valid_s[wn][stage] = valid;
#pragma unroll 8
      for (int i = gt; i < BT * CH; i += GT) {
        const int key = i / CH, c = i % CH;
        const int kr = __shfl_sync(0xffffffffu, row, key);
        const bool ok = kr >= 0 && c < chunks;
        const long long off = ok ? ((long long)kr * d.head_dim + c * EC) * (int)sizeof(T) : 0;
        const uint32_t dst = key * PITCH + ((c ^ (key & 7)) << 4);
        cp_async_16(ks + dst, static_cast<const char*>(a.k) + off, ok ? 16u : 0u);
        cp_async_16(vs + dst, static_cast<const char*>(a.v) + off, ok ? 16u : 0u);
      }
    }
    cp_async_commit();
  };

  float o[HDP / 8][4] = {};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  // key group wn takes blocks blk0 + wn, blk0 + wn + WN, ...
  int row_next = -1;
  {
    int stage = 0;
    for (; stage < kStages - 1; ++stage) {
      const int blk = blk0 + wn + stage * WN;
      issue(blk, row_of(blk), stage);
    }
    row_next = row_of(blk0 + wn + stage * WN);
  }
  int stage = 0;
  for (int blk = blk0 + wn; blk < blk1; blk += WN) {
    cp_async_wait<kStages - 2>();
    sync_group();
    {
      const int ahead = blk + (kStages - 1) * WN;
      issue(ahead, row_next, stage == 0 ? kStages - 1 : stage - 1);
      row_next = row_of(ahead + WN);
    }
    const uint32_t ks_addr = ring + stage * K::STAGE, vs_addr = ks_addr + BT * PITCH;
    const uint32_t valid = valid_s[wn][stage];
    const int base = base_of(blk);

    // scores
    float s[BT / 8][4] = {};
    {
      const int mi = lane >> 3, r = lane & 7;
      const int key = (mi >> 1) * 8 + r;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int nt = 0; nt < BT / 8; nt += 2) {
          uint32_t kb[4];
          ldsm_x4(kb, ks_addr + (nt * 8 + key) * PITCH + (((2 * ks + (mi & 1)) ^ r) << 4));
          if constexpr (kBf16) {
            mma_bf16(s[nt], qa[ks], kb[0], kb[1]);
            mma_bf16(s[nt + 1], qa[ks], kb[2], kb[3]);
          } else {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              hi[i] = tf_hi(qa[ks][i]);
              lo[i] = tf_lo(qa[ks][i]);
            }
            mma_3tf32(s[nt], hi, lo, kb[0], kb[1]);
            mma_3tf32(s[nt + 1], hi, lo, kb[2], kb[3]);
          }
        }
    }
    // mask, running maximum. A block that every row sees whole (all but the span's ends) needs no mask.
    const bool open = valid == (BT == 32 ? 0xffffffffu : (1u << BT) - 1u) && base + BT - 1 <= shift + r0 / a.group &&
                      (d.window == 0 || base > shift + (min(r0 + K::ROWS, rows) - 1) / a.group - d.window || base + BT <= d.sinks);
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < BT / 8; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = s[nt][i] * a.scale_log2;
        if (!open) {
          const int c = nt * 8 + 2 * t + (i & 1), j = base + c, p = pos[i >> 1];
          const bool seen = ((valid >> c) & 1u) && j <= p && (d.window == 0 || j > p - d.window || j < d.sinks);
          x = seen ? x : -INFINITY;
        }
        s[nt][i] = x;
        top[i >> 1] = fmaxf(top[i >> 1], x);
      }
    float safe[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float mn = fmaxf(m[h], quad_max(top[h]));
      safe[h] = mn == -INFINITY ? 0.0f : mn;
      const float shrink = exp2f(m[h] - safe[h]);
      m[h] = mn;
      l[h] *= shrink;
#pragma unroll
      for (int nd = 0; nd < HDP / 8; ++nd) {
        o[nd][2 * h] *= shrink;
        o[nd][2 * h + 1] *= shrink;
      }
    }
    // the tensor cores truncate the running sum at every addition, an error that grows with the number of
    // keys: for fp32 each block is summed from zero and added with a rounded addition (over 1700 keys
    // the error falls from 1.1e-5 to the plain form's; bf16 outputs do not show it)
#pragma unroll
    for (int nt = 0; nt < BT / 8; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[nt][i] = exp2f(s[nt][i] - safe[i >> 1]);
        l[i >> 1] += s[nt][i];
      }
    // values
    if constexpr (kBf16) {
      const int mi = lane >> 3, r = lane & 7;
      const int key = (mi & 1) * 8 + r;
#pragma unroll
      for (int kt = 0; kt < BT / 16; ++kt) {
        uint32_t pa[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pa[i] = pack_bf16x2(s[2 * kt + (i >> 1)][2 * (i & 1)], s[2 * kt + (i >> 1)][2 * (i & 1) + 1]);
#pragma unroll
        for (int nd = 0; nd < HDP / 8; nd += 2) {
          uint32_t vb[4];
          ldsm_x4_t(vb, vs_addr + (kt * 16 + key) * PITCH + (((nd + (mi >> 1)) ^ r) << 4));
          mma_bf16(o[nd], pa, vb[0], vb[1]);
          mma_bf16(o[nd + 1], pa, vb[2], vb[3]);
        }
      }
    } else {
      // the order of the eight keys of a step is free: slot t takes key 2 t, slot t + 4 key 2 t + 1,
      // which is where the scores' fragment already has them
      uint32_t hi[BT / 8][4], lo[BT / 8][4];
#pragma unroll
      for (int kt = 0; kt < BT / 8; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x = __float_as_uint(s[kt][(i >> 1) + 2 * (i & 1)]);
          hi[kt][i] = tf_hi(x);
          lo[kt][i] = tf_lo(x);
        }
      const int k0 = 2 * t, k1 = 2 * t + 1;
#pragma unroll
      for (int nd = 0; nd < HDP / 8; ++nd) {
        const int c = nd * 2 + (g >> 2);
        float add[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kt = 0; kt < BT / 8; ++kt) {
          const uint32_t b0 = lds32(vs_addr + (kt * 8 + k0) * PITCH + ((c ^ k0) << 4) + (g & 3) * 4);
          const uint32_t b1 = lds32(vs_addr + (kt * 8 + k1) * PITCH + ((c ^ k1) << 4) + (g & 3) * 4);
          mma_3tf32(add, hi[kt], lo[kt], b0, b1);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nd][i] += add[i];
      }
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  cp_async_wait_all();
  __syncthreads();  // the ring is free: the key groups' sums take its place

  float* so = reinterpret_cast<float*>(smem);
  float* sm = so + WN * K::ROWS * HDP;
  float* sl = sm + WN * K::ROWS;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = wn * K::ROWS + wm * 16 + h * 8 + g;
    const float lt = quad_sum(l[h]);
    if (t == 0) {
      sm[r] = m[h];
      sl[r] = lt;
    }
#pragma unroll
    for (int nd = 0; nd < HDP / 8; ++nd) *reinterpret_cast<float2*>(so + r * HDP + nd * 8 + 2 * t) = make_float2(o[nd][2 * h], o[nd][2 * h + 1]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < K::ROWS * (HDP / 4); i += kAttnThreads) {
    const int rl = i / (HDP / 4), c = (i % (HDP / 4)) * 4, r = r0 + rl;
    if (r >= rows || c >= d.head_dim) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WN; ++w) top = fmaxf(top, sm[w * K::ROWS + rl]);
    const float safe = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < WN; ++w) {
      const float f = exp2f(sm[w * K::ROWS + rl] - safe);
      const float4 x = *reinterpret_cast<const float4*>(so + (w * K::ROWS + rl) * HDP + c);
      sum = fmaf(f, sl[w * K::ROWS + rl], sum);
      acc.x = fmaf(f, x.x, acc.x); acc.y = fmaf(f, x.y, acc.y); acc.z = fmaf(f, x.z, acc.z); acc.w = fmaf(f, x.w, acc.w);
    }
    if (whole) {
      const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
      const int tok = rq.q0 + r / a.group, head = e * a.group + r % a.group;
      T* po = static_cast<T*>(a.out) + (long long)tok * d.out_stride + (long long)head * d.head_dim + c;
      store_out<T>(po, acc.x * inv); store_out<T>(po + 1, acc.y * inv); store_out<T>(po + 2, acc.z * inv); store_out<T>(po + 3, acc.w * inv);
      if (a.lse && c == 0) a.lse[(long long)tok * d.heads + head] = (top + log2f(sum)) * 0.69314718055994531f;
    } else {
      const long long at = slot * K::ROWS + rl;
      *reinterpret_cast<float4*>(a.part_o + at * HDP + c) = acc;
      if (c == 0) {
        a.part_m[at] = top;
        a.part_l[at] = sum;
      }
    }
  }
  __syncthreads();  // the next piece takes the ring again
}

// the block that holds unit u when `units` are cut into `blocks` runs [c units / blocks, (c + 1) units / blocks)
MDLC_DEV int block_of(long long u, long long units, int blocks) { return (int)(((u + 1) * blocks - 1) / units); }

template <typename T, int HDP, int WM>
__global__ void __launch_bounds__(kAttnThreads) attn_split_kernel(const AttnArgs a, int* err) {
  using K = Cfg<T, HDP, WM>;
  constexpr int UB = kUnit / K::BT;
  extern __shared__ __align__(128) unsigned char attn_smem[];
  __shared__ uint32_t valid_s[K::WN][kStages];
  __shared__ long long warp_sums[kAttnThreads / 32];
  __shared__ Place place_s;
  pdl_wait();
  pdl_trigger();
  const mdlc_attn_desc& d = a.d;
  // units of a request and key head
  auto units_of = [&](int b) -> long long {
    const Request r = request_of(a, b);
    const long long rows = (long long)r.q_len * a.group;
    if (rows == 0 || rows > a.split_rows) return 0;
    return max(1, (span_of(a, r, 0, r.q_len - 1, K::BT).n + UB - 1) / UB);
  };
  const int per = (d.batch + kAttnThreads - 1) / kAttnThreads;
  const int b0 = min((int)threadIdx.x * per, d.batch), b1 = min(b0 + per, d.batch);
  long long mine = 0, total;
  for (int b = b0; b < b1; ++b) mine += units_of(b) * d.kv_heads;
  const long long before = block_scan(mine, warp_sums, &total);
  if (blockIdx.x == 0) {
    long long at = before;
    for (int b = b0; b < b1; ++b) {
      a.first_unit[b] = at;
      at += units_of(b) * d.kv_heads;
      if (b == d.batch - 1) a.first_unit[d.batch] = at;
    }
  }
  const int blocks = (int)min((long long)gridDim.x, total);
  if ((int)blockIdx.x >= blocks) return;
  long long u0 = (long long)blockIdx.x * total / blocks;
  const long long u1 = (long long)(blockIdx.x + 1) * total / blocks;
  if (u0 >= before && u0 < before + mine) {
    long long at = before;
    for (int b = b0;; ++b) {
      const long long n = units_of(b) * d.kv_heads;
      if (u0 < at + n) {
        place_s = {b, at};
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  Place pl = place_s;
  while (u0 < u1) {
    const Request rq = request_of(a, pl.b);
    const long long n = units_of(pl.b);
    if (u0 >= pl.first + n * d.kv_heads) {
      pl.first += n * d.kv_heads;
      ++pl.b;
      continue;
    }
    const int e = (int)((u0 - pl.first) / n);
    const long long tile0 = pl.first + e * n, end = min(u1, tile0 + n);
    const Span sp = span_of(a, rq, 0, rq.q_len - 1, K::BT);
    const int blk0 = (int)(u0 - tile0) * UB, blk1 = min((int)(end - tile0) * UB, sp.n);
    attn_piece<T, HDP, WM>(a, attn_smem, valid_s, err, pl.b, rq, e, 0, sp, blk0, blk1, u0 == tile0 && end == tile0 + n,
                           (long long)pl.b * d.kv_heads + e + blockIdx.x);
    u0 = end;
  }
}

// a block per row tile (x), key head (y) and share of its keys (z)
template <typename T, int HDP>
__global__ void __launch_bounds__(kAttnThreads) attn_chunk_kernel(const AttnArgs a, int* err) {
  using K = Cfg<T, HDP, 4>;
  extern __shared__ __align__(128) unsigned char attn_smem[];
  __shared__ uint32_t valid_s[K::WN][kStages];
  __shared__ long long warp_sums[kAttnThreads / 32];
  __shared__ Place place_s;
  pdl_wait();
  pdl_trigger();
  Tile t;
  if (!find_tile(a, blockIdx.x, K::ROWS, warp_sums, &place_s, &t)) return;
  const Span sp = span_of(a, t.rq, t.r0 / a.group, (min(t.r0 + K::ROWS, t.rows) - 1) / a.group, K::BT);
  const int ns = splits_of(a, sp.n, kLeastKeys / K::BT), z = blockIdx.z;
  if (z >= ns) return;
  attn_piece<T, HDP, 4>(a, attn_smem, valid_s, err, t.b, t.rq, blockIdx.y, t.r0, sp, (int)((long long)z * sp.n / ns),
                        (int)((long long)(z + 1) * sp.n / ns), ns == 1,
                        ((long long)blockIdx.x * a.d.kv_heads + blockIdx.y) * a.splits + z);
}

// Adds the shares of a chunk tile, in order. A warp per row.
template <typename T, int HDP>
__global__ void __launch_bounds__(kJoinThreads) attn_chunk_join_kernel(const AttnArgs a, int tile_rows, int bt) {
  pdl_wait();
  pdl_trigger();
  constexpr int V = HDP / 32;
  __shared__ long long warp_sums[kJoinThreads / 32];
  __shared__ Place place_s;
  Tile t;
  if (!find_tile(a, blockIdx.x, tile_rows, warp_sums, &place_s, &t)) return;
  const Span sp = span_of(a, t.rq, t.r0 / a.group, (min(t.r0 + tile_rows, t.rows) - 1) / a.group, bt);
  const int ns = splits_of(a, sp.n, kLeastKeys / bt);
  if (ns == 1) return;
  const mdlc_attn_desc& d = a.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.y;
  const long long slot0 = ((long long)blockIdx.x * d.kv_heads + e) * a.splits;
  const int per = (tile_rows + gridDim.z - 1) / gridDim.z, rl0 = blockIdx.z * per;
  for (int rl = rl0 + warp; rl < min(rl0 + per, min(tile_rows, t.rows - t.r0)); rl += kJoinThreads / 32) {
    const int r = t.r0 + rl;
    float top = -INFINITY, sum = 0.0f, acc[V] = {};
    for (int s = 0; s < ns; ++s) top = fmaxf(top, a.part_m[(slot0 + s) * tile_rows + rl]);
    const float safe = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
    for (int s = 0; s < ns; ++s) {
      const long long at = (slot0 + s) * tile_rows + rl;
      const float f = exp2f(a.part_m[at] - safe);
      sum = fmaf(f, a.part_l[at], sum);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(f, a.part_o[at * HDP + i * 32 + lane], acc[i]);
    }
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
    const int tok = t.rq.q0 + r / a.group, head = e * a.group + r % a.group;
    T* po = static_cast<T*>(a.out) + (long long)tok * d.out_stride + (long long)head * d.head_dim;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i * 32 + lane < d.head_dim) store_out<T>(po + i * 32 + lane, acc[i] * inv);
    if (a.lse && lane == 0) a.lse[(long long)tok * d.heads + head] = (top + log2f(sum)) * 0.69314718055994531f;
  }
}

// Adds the partial sums of every tile that several blocks share, in block order. A block per
// (key head, request); a row is given to one or several warps, which take its pieces in turn.
template <typename T, int HDP, int WM>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const AttnArgs a, int split_blocks) {
  pdl_wait();
  pdl_trigger();
  constexpr int ROWS = 16 * WM, NW = kJoinThreads / 32, V = HDP / 32;
  __shared__ float part[NW][HDP + 2];
  const mdlc_attn_desc& d = a.d;
  const int e = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long units = a.first_unit[d.batch], u0 = a.first_unit[b];
  const long long n = (a.first_unit[b + 1] - u0) / d.kv_heads;
  if (n == 0) return;
  const int blocks = (int)min((long long)split_blocks, units);
  const int c0 = block_of(u0 + e * n, units, blocks), c1 = block_of(u0 + (e + 1) * n - 1, units, blocks);
  if (c0 == c1) return;
  const Request rq = request_of(a, b);
  const int rows = rq.q_len * a.group;
  int wpr = 1;  // warps of a row
  while (wpr * 2 * rows <= NW) wpr *= 2;
  const int rpb = NW / wpr;
  for (int rb = 0; rb < rows; rb += rpb) {
    const int r = rb + warp / wpr, w = warp % wpr;
    float top = -INFINITY, sum = 0.0f, acc[V] = {};
    if (r < rows) {
#pragma unroll 4
      for (int c = c0 + w; c <= c1; c += wpr) {
        const long long at = ((long long)b * d.kv_heads + e + c) * ROWS + r;
        const float pm = a.part_m[at], pl = a.part_l[at];
        float x[V];
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = a.part_o[at * HDP + i * 32 + lane];
        const float mn = fmaxf(top, pm), safe = mn == -INFINITY ? 0.0f : mn;
        const float f0 = exp2f(top - safe), f1 = exp2f(pm - safe);
        top = mn;
        sum = sum * f0 + pl * f1;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = acc[i] * f0 + x[i] * f1;
      }
    }
    if (wpr > 1) {
      __syncthreads();
      if (lane == 0) {
        part[warp][HDP] = top;
        part[warp][HDP + 1] = sum;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) part[warp][i * 32 + lane] = acc[i];
      __syncthreads();
      if (w == 0) {
        for (int k = 1; k < wpr; ++k) {
          const float pm = part[warp + k][HDP], mn = fmaxf(top, pm), safe = mn == -INFINITY ? 0.0f : mn;
          const float f0 = exp2f(top - safe), f1 = exp2f(pm - safe);
          top = mn;
          sum = sum * f0 + part[warp + k][HDP + 1] * f1;
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = acc[i] * f0 + part[warp + k][i * 32 + lane] * f1;
        }
      }
    }
    if (w == 0 && r < rows) {
      const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
      const int tok = rq.q0 + r / a.group, head = e * a.group + r % a.group;
      T* po = static_cast<T*>(a.out) + (long long)tok * d.out_stride + (long long)head * d.head_dim;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i * 32 + lane < d.head_dim) store_out<T>(po + i * 32 + lane, acc[i] * inv);
      if (a.lse && lane == 0) a.lse[(long long)tok * d.heads + head] = (top + log2f(sum)) * 0.69314718055994531f;
    }
  }
}

// ------------------------------------------------------------ host
int padded_dim(int head_dim) { return head_dim <= 64 ? 64 : 128; }

// row groups of split mode, 0: no request goes there (more than 64 query heads per key head)
int split_groups(const mdlc_attn_desc& d) {
  const int group = d.heads / d.kv_heads;
  const long long all = (long long)d.max_q * group;
  if (all <= 16) return 1;
  if (all <= 32) return 2;
  if (all <= 64) return 4;
  // requests of many tokens go to chunk mode; the others have one
  return group <= 16 ? 1 : (group <= 32 ? 2 : (group <= 64 ? 4 : 0));
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// chunk mode's geometry: which kernel, row tiles at most (full ones, and one more per request), shares per tile
struct Chunk {
  bool used, tc;
  int rows, tiles, splits;
};
Chunk chunk_of(const mdlc_attn_desc& d) {
  const int group = d.heads / d.kv_heads;
  Chunk c = {};
  c.used = (long long)d.max_q * group > 16 * split_groups(d);
  c.tc = attn_tc_fits(d) && (long long)d.tokens * group / kTcRows + d.batch <= 65535;  // the tiles are its grid's y
  c.rows = c.tc ? kTcRows : 64;
  c.tiles = (int)min((long long)d.tokens * group / c.rows + d.batch, (long long)INT32_MAX);
  // the mma.sync kernel runs three blocks per SM
  const long long room = kChunkBlocks * (c.tc ? 1 : 3) / ((long long)c.tiles * d.kv_heads);
  c.splits = (int)max(1ll, min(room, min(16ll, (long long)d.max_kv / kLeastKeys)));
  return c;
}

struct Layout {
  size_t part_o, part_m, part_l, first_unit, total;
};
Layout layout_of(const mdlc_attn_desc& d) {
  const size_t slots = (size_t)d.batch * d.kv_heads + kMaxBlocks;
  size_t rows = slots * 16 * split_groups(d);
  const Chunk c = chunk_of(d);
  // the two modes run one after the other and share the space
  if (c.used && c.splits > 1) rows = max(rows, (size_t)c.tiles * d.kv_heads * c.splits * c.rows);
  Layout l;
  l.part_o = 0;
  l.part_m = align256(rows * padded_dim(d.head_dim) * 4);
  l.part_l = l.part_m + align256(rows * 4);
  l.first_unit = l.part_l + align256(rows * 4);
  l.total = l.first_unit + align256(((size_t)d.batch + 1) * 8);
  return l;
}

const char* check_desc(const mdlc_attn_desc* d) {
  if (d->batch < 1 || d->batch > MDLC_MAX_REQUESTS || d->tokens < 1 || d->heads < 1 || d->kv_heads < 1 ||
      d->heads % d->kv_heads || d->kv_heads > 65535)
    return "batch, tokens or heads";
  if (d->head_dim < 8 || d->head_dim > 128 || d->head_dim % 8) return "head_dim";
  if (d->page < 1 || d->page > 1024 || d->pages < 1 || d->table_stride < 1 || d->max_q < 1 || d->max_kv < 0) return "page, pages, table_stride, max_q or max_kv";
  if (d->window < 0 || d->sinks < 0) return "window or sinks";
  if (d->dtype != MDLC_BF16 && d->dtype != MDLC_F32) return "dtype";
  if ((long long)d->pages * d->page * d->kv_heads > INT32_MAX) return "pages (pages * page * kv_heads exceeds 2^31 - 1)";
  if ((long long)d->max_q * (d->heads / d->kv_heads) > (1 << 30) || (long long)d->tokens * (d->heads / d->kv_heads) > INT32_MAX - 65536) return "max_q or tokens";
  const long long w = (long long)d->heads * d->head_dim;
  if (d->q_stride < w || d->out_stride < w || d->q_stride % 8 || d->out_stride % 8) return "q_stride or out_stride";
  return nullptr;
}

template <typename T, int HDP, int WM>
cudaError_t run_split(mdlc_ctx* ctx, const AttnArgs& a) {
  const int smem = Cfg<T, HDP, WM>::SMEM;
  auto* kern = attn_split_kernel<T, HDP, WM>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  // one or two blocks per SM, as shared memory allows
  const int blocks = min(kMaxBlocks, ctx->num_sms * (smem <= 100 * 1024 ? 2 : 1));
  mdlc_note_launch(ctx);
  e = launch_pdl(kern, dim3(blocks), dim3(kAttnThreads), smem, ctx->stream, a, ctx->d_err);
  if (e != cudaSuccess) return e;
  mdlc_note_launch(ctx);
  return launch_pdl(attn_join_kernel<T, HDP, WM>, dim3(a.d.kv_heads, a.d.batch), dim3(kJoinThreads), 0, ctx->stream, a, blocks);
}

template <typename T, int HDP>
cudaError_t run_attn(mdlc_ctx* ctx, AttnArgs& a) {
  const int wm = split_groups(a.d);
  cudaError_t e = cudaSuccess;
  if (wm == 1) e = run_split<T, HDP, 1>(ctx, a);
  else if (wm == 2) e = run_split<T, HDP, 2>(ctx, a);
  else if (wm == 4) e = run_split<T, HDP, 4>(ctx, a);
  const Chunk c = chunk_of(a.d);
  if (e != cudaSuccess || !c.used) return e;
  a.splits = c.splits;
  const dim3 grid(c.tiles, a.d.kv_heads, c.splits);
  mdlc_note_launch(ctx);
  if (c.tc) {
    e = attn_tc_launch(ctx, a, grid);
  } else {
    const int smem = Cfg<T, HDP, 4>::SMEM;
    e = cudaFuncSetAttribute(attn_chunk_kernel<T, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = launch_pdl(attn_chunk_kernel<T, HDP>, grid, dim3(kAttnThreads), smem, ctx->stream, a, ctx->d_err);
  }
  if (e != cudaSuccess || c.splits == 1) return e;
  mdlc_note_launch(ctx);
  return launch_pdl(attn_chunk_join_kernel<T, HDP>, dim3(c.tiles, a.d.kv_heads, c.rows / 64), dim3(kJoinThreads), 0, ctx->stream, a, c.rows,
                    c.tc ? kTcKeys : block_keys<T, HDP>());
}

}  // namespace
}  // namespace mdlc

using namespace mdlc;

extern "C" int mdlc_paged_attn_workspace(const mdlc_attn_desc* desc, size_t* bytes) {
  if (!desc || !bytes || check_desc(desc)) return MDLC_ERR_INVALID;
  *bytes = layout_of(*desc).total;
  return MDLC_OK;
}

extern "C" int mdlc_paged_attn(mdlc_ctx* ctx, const mdlc_attn_desc* desc, const void* q, const void* k_cache,
                               const void* v_cache, const int32_t* block_table, const int32_t* q_starts,
                               const int32_t* kv_lens, void* out, float* lse, void* workspace) {
  if (!ctx) return MDLC_ERR_INVALID;
  if (!desc || !q || !k_cache || !v_cache || !block_table || !q_starts || !kv_lens || !out || !workspace)
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "paged_attn: null argument");
  if (const char* bad = check_desc(desc)) return mdlc_set_error(ctx, MDLC_ERR_INVALID, "paged_attn: bad %s", bad);
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace) % 16 || (uintptr_t)lse % 4)
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "paged_attn: misaligned pointer");
  cudaSetDevice(ctx->device);
  AttnArgs a = {};
  a.d = *desc;
  a.d.max_kv = (int)min((long long)desc->max_kv, (long long)desc->table_stride * desc->page);
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.table = block_table;
  a.q_starts = q_starts;
  a.kv_lens = kv_lens;
  a.out = out;
  a.lse = lse;
  a.group = desc->heads / desc->kv_heads;
  a.split_rows = 16 * split_groups(*desc);
  a.scale_log2 = desc->scale * 1.4426950408889634f;
  const Layout l = layout_of(*desc);
  char* ws = static_cast<char*>(workspace);
  a.part_o = reinterpret_cast<float*>(ws + l.part_o);
  a.part_m = reinterpret_cast<float*>(ws + l.part_m);
  a.part_l = reinterpret_cast<float*>(ws + l.part_l);
  a.first_unit = reinterpret_cast<long long*>(ws + l.first_unit);
  const bool bf16 = desc->dtype == MDLC_BF16;
  cudaError_t e;
  if (padded_dim(desc->head_dim) == 64) e = bf16 ? run_attn<__nv_bfloat16, 64>(ctx, a) : run_attn<float, 64>(ctx, a);
  else e = bf16 ? run_attn<__nv_bfloat16, 128>(ctx, a) : run_attn<float, 128>(ctx, a);
  return mdlc_cuda_status(ctx, e, "paged_attn launch");
}
