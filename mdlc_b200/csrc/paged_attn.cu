// mdlc_paged_attn: attention of each request's new tokens over its cache pages.
//
// The rows of one key head are its G query heads of every new token of a request
// (row r: token r / G, head e * G + r % G), so a key or value loaded once serves them
// all. One pass over the keys with the running maximum and sum of the softmax (both
// fp32, in the base-2 exponent); scores never leave registers. In bf16 the weights go into the second product as bf16 numbers
// (2^-8 of each at most, of both signs; their sum stays fp32): an fp32 weight would take three products in place of one, for an error
// that goes from 1.8e-3 to 2.3e-3 where the output's own rounding is 1.7e-3.
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
//     partial sums in the workspace, which the last of them to arrive adds in block order.
//   chunk mode (many rows): a block per row tile, or several that share its keys.
#include <climits>

#include "func_attr.h"
#include "paged_attn.cuh"

namespace mdlc {
namespace {

constexpr int kAttnThreads = 128;
constexpr int kStages = 3;
constexpr int kHiddenPage = INT_MIN;  // stands for a page that no row sees; an id of that value counts as the next one, no page either
constexpr int kSmShared = 224 * 1024;  // shared memory of an SM that blocks may ask for
constexpr int kTwoBlocks = kSmShared / 2;  // shared memory of a block of which two fit on an SM
constexpr int kUnit = 128;      // keys of one unit of split work
// What beginning and ending a tile costs, in units: without it a block whose share is many short requests ends long after
// the others (64 requests of 64 to 8192 keys: the last SM 271k cycles, the mean 189k)
constexpr int kTileCost = 2;
constexpr int kMaxBlocks = 512; // split-mode blocks at most (bounds the workspace)
constexpr int kJoinThreads = 256;
constexpr int kLeastKeys = 256; // keys of a share of a chunk tile at least, see splits_of
constexpr int kB200Sms = 148;   // shares are made for so many SMs (the workspace's size is an answer without a context)

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
MDLC_DEV void lds128(uint32_t (&v)[4], uint32_t addr) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
MDLC_DEV void sts128(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
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
// the same with the high part rounded to the nearest, for the queries: their rests then have either sign, and so has the product of
// two rests, which is dropped (an output error of 6.5e-7 over 1700 keys, 1.03e-6 without; one more integer addition each, which
// weights take 3% longer for and 6e-8 closer)
MDLC_DEV void tf_split(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = (x + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}
// a b of fp32 operands in three tf32 products, for N accumulators at once: c takes the large one, r the two small ones (a sum
// of its own: the truncation of one does not cut the other). All N products of a kind come before the next kind, so that a
// product does not wait for the one before it (64 fp32 decodes of 4000 keys, all else as it was then: 191 us; each accumulator's three
// in a row 208).
template <int N>
MDLC_DEV void mma_3tf32(float (*c)[4], float (*r)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4], const uint32_t (&b)[N][2]) {
#pragma unroll
  for (int n = 0; n < N; ++n) mma_tf32(r[n], lo, tf_hi(b[n][0]), tf_hi(b[n][1]));
#pragma unroll
  for (int n = 0; n < N; ++n) mma_tf32(c[n], hi, tf_hi(b[n][0]), tf_hi(b[n][1]));
#pragma unroll
  for (int n = 0; n < N; ++n) mma_tf32(r[n], hi, tf_lo(b[n][0]), tf_lo(b[n][1]));
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
  // fp32 heads of more than 64 columns: the queries' high and low parts behind it, fragment by fragment, since 64 registers for them
  // are too many (64 decodes of 4000 keys: 164 us, 192 from registers; heads of up to 64 columns: 98 us, 91 from registers)
  static constexpr int QAT = (RING > MERGE ? RING : MERGE);
  static constexpr bool QSHARED = sizeof(T) == 4 && HDP == 128;
  static constexpr int SMEM = QAT + (QSHARED ? WM * (HDP / 8) * 1024 : 0);
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
  const int shift = rq.shift;
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
    pos[h] = ok ? max(-1, shift + i) : -1;
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

  // fp32: this lane's fragments of step ks, split. In shared memory each thread reads what it wrote itself.
  const uint32_t q_at = smem_u32(smem) + K::QAT + wm * (HDP / 8) * 1024 + lane * 16;
  if constexpr (K::QSHARED)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) tf_split(qa[ks][i], hi[i], lo[i]);
      sts128(q_at + ks * 1024, hi);
      sts128(q_at + ks * 1024 + 512, lo);
    }
  auto query = [&](int ks, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    if constexpr (K::QSHARED) {
      lds128(hi, q_at + ks * 1024);
      lds128(lo, q_at + ks * 1024 + 512);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) tf_split(qa[ks][i], hi[i], lo[i]);
    }
  };
  auto base_of = [&](int blk) { return key_of_block(sp, blk, BT); };
  // page id of key `lane` of the block, kHiddenPage: hidden from every row. Loads only, so that several are in flight.
  auto id_of = [&](int blk) {
    const int j = base_of(blk) + lane;
    if (blk >= blk1 || lane >= BT || j >= rq.kv_len || (j < sp.lo && j >= d.sinks)) return kHiddenPage;
    if (!table_ok(a, b, j / d.page)) return kHiddenPage;
    return max(__ldg(a.table + (long long)b * d.table_stride + j / d.page), kHiddenPage + 1);
  };
  // its cache row, or -1: hidden or missing
  auto row_of = [&](int blk, int id) {
    if (id == kHiddenPage) return -1;
    if ((unsigned)id < (unsigned)d.pages) return (id * d.kv_heads + e) * d.page + (base_of(blk) + lane) % d.page;
    record_error(err, MDLC_DEVERR_BOUNDS);
    return -1;
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
  int ids[kStages];
#pragma unroll
  for (int i = 0; i < kStages; ++i) ids[i] = id_of(blk0 + wn + i * WN);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(blk0 + wn + i * WN, row_of(blk0 + wn + i * WN, ids[i]), i);
  int id_next = ids[kStages - 1];
  int stage = 0;
  for (int blk = blk0 + wn; blk < blk1; blk += WN) {
    cp_async_wait<kStages - 2>();
    sync_group();
    {
      const int ahead = blk + (kStages - 1) * WN;
      issue(ahead, row_of(ahead, id_next), stage == 0 ? kStages - 1 : stage - 1);
      id_next = id_of(ahead + WN);
    }
    const uint32_t ks_addr = ring + stage * K::STAGE, vs_addr = ks_addr + BT * PITCH;
    const uint32_t valid = valid_s[wn][stage];
    const int base = base_of(blk);

    // scores
    float s[BT / 8][4] = {};
    constexpr int ST = kBf16 ? 1 : BT / 8;
    // fp32: odd steps' products and the small ones: shorter chains of truncated additions (6.5e-7, 8.1e-7 without; 68.4 and 67.8 us)
    float s_odd[ST][4] = {}, s_low[ST][4] = {};
    {
      const int mi = lane >> 3, r = lane & 7;
      const int key = (mi >> 1) * 8 + r;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t kb[BT / 8][2];
#pragma unroll
        for (int nt = 0; nt < BT / 8; nt += 2) {
          uint32_t x[4];
          ldsm_x4(x, ks_addr + (nt * 8 + key) * PITCH + (((2 * ks + (mi & 1)) ^ r) << 4));
          kb[nt][0] = x[0], kb[nt][1] = x[1], kb[nt + 1][0] = x[2], kb[nt + 1][1] = x[3];
        }
        if constexpr (kBf16) {
#pragma unroll
          for (int nt = 0; nt < BT / 8; ++nt) mma_bf16(s[nt], qa[ks], kb[nt][0], kb[nt][1]);
        } else {
          uint32_t hi[4], lo[4];
          query(ks, hi, lo);
          mma_3tf32(ks & 1 ? s_odd : s, s_low, hi, lo, kb);
        }
      }
      if constexpr (!kBf16) {
#pragma unroll
        for (int nt = 0; nt < BT / 8; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[nt][i] += s_odd[nt][i] + s_low[nt][i];
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
    // keys: for fp32 each block is summed from zero and added with a rounded addition (over 1700 keys,
    // 1.1e-5 before this and the other measures, 6.5e-7 with them; bf16 outputs do not show it)
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
      constexpr int ND = 4;  // tiles of 8 columns at once
#pragma unroll
      for (int nd = 0; nd < HDP / 8; nd += ND) {
        float add[ND][4] = {}, low[ND][4] = {};
#pragma unroll
        for (int kt = 0; kt < BT / 8; ++kt) {
          uint32_t vb[ND][2];
#pragma unroll
          for (int i = 0; i < ND; ++i) {
            const int c = (nd + i) * 2 + (g >> 2);
            vb[i][0] = lds32(vs_addr + (kt * 8 + k0) * PITCH + ((c ^ k0) << 4) + (g & 3) * 4);
            vb[i][1] = lds32(vs_addr + (kt * 8 + k1) * PITCH + ((c ^ k1) << 4) + (g & 3) * 4);
          }
          mma_3tf32(add, low, hi[kt], lo[kt], vb);
        }
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[nd + i][j] += add[i][j] + low[i][j];
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
      if (!out_ok(a, tok, head, c, 4)) continue;
      T* po = static_cast<T*>(a.out) + (long long)tok * d.out_stride + (long long)head * d.head_dim + c;
      store_out<T>(po, acc.x * inv); store_out<T>(po + 1, acc.y * inv); store_out<T>(po + 2, acc.z * inv); store_out<T>(po + 3, acc.w * inv);
      if (a.lse && c == 0) a.lse[(long long)tok * d.heads + head] = (top + log2f(sum)) * 0.69314718055994531f;
    } else {
      const long long at = slot * K::ROWS + rl;
      if (!part_ok(a, at)) continue;
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

// Split mode: a piece of a tile that blocks c0 .. c1 share is in the workspace. The last of them to arrive adds all
// pieces, in block order whoever it is, so the result does not depend on timing.
template <typename T, int HDP, int ROWS>
MDLC_DEV void join_pieces(const AttnArgs& a, int b, int e, const Request& rq, int c0, int c1) {
  constexpr int V = HDP / 32, NW = kAttnThreads / 32;
  __shared__ float part[NW][HDP + 2];
  __shared__ int last_s;
  const mdlc_attn_desc& d = a.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    last_s = atomicAdd(a.arrived + c0, 1) == c1 - c0;
    if (last_s) a.arrived[c0] = 0;
  }
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  const int rows = rq.q_len * a.group;
  const long long slot0 = (long long)b * d.kv_heads + e;
  int wpr = 1;  // warps of a row, each with every wpr-th piece
  while (wpr * 2 * rows <= NW) wpr *= 2;
  const int rpb = NW / wpr;
  for (int rb = 0; rb < rows; rb += rpb) {
    const int r = rb + warp / wpr, w = warp % wpr;
    float top = -INFINITY, sum = 0.0f, acc[V] = {};
    if (r < rows) {
#pragma unroll 8
      for (int c = c0 + w; c <= c1; c += wpr) {
        const long long at = (slot0 + c) * ROWS + r;
        if (!part_ok(a, at)) continue;
        const float pm = __ldcg(a.part_m + at), pl = __ldcg(a.part_l + at);
        float x[V];
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = __ldcg(a.part_o + at * HDP + i * 32 + lane);
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
        if (i * 32 + lane < d.head_dim && out_ok(a, tok, head, i * 32 + lane, 1)) store_out<T>(po + i * 32 + lane, acc[i] * inv);
      if (a.lse && lane == 0 && out_ok(a, tok, head, 0, 1)) a.lse[(long long)tok * d.heads + head] = (top + log2f(sum)) * 0.69314718055994531f;
    }
  }
  __syncthreads();
}

// Split mode's line of work: calls piece(b, request, e, span, first block, end, whole, slot) for every run of this
// block's units that lies in one tile, and join(b, request, e, c0, c1) after a piece of a shared tile.
template <int BT, typename Piece, typename Join>
MDLC_DEV void split_walk(const AttnArgs& a, Piece piece, Join join) {
  constexpr int UB = kUnit / BT;
  __shared__ long long warp_sums[kAttnThreads / 32];
  __shared__ Place place_s;
  const mdlc_attn_desc& d = a.d;
  // units of a request and key head
  auto units_of = [&](int b) -> long long {
    const Request r = request_of(a, b);
    const long long rows = (long long)r.q_len * a.group;
    if (rows == 0 || rows > a.split_rows) return 0;
    return kTileCost + max(1, (span_of(a, r, 0, r.q_len - 1, BT).n + UB - 1) / UB);
  };
  const int per = (d.batch + kAttnThreads - 1) / kAttnThreads;
  const int b0 = min((int)threadIdx.x * per, d.batch), b1 = min(b0 + per, d.batch);
  long long mine = 0, total;
  for (int b = b0; b < b1; ++b) mine += units_of(b) * d.kv_heads;
  const long long before = block_scan(mine, warp_sums, &total);
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
    if (u0 >= pl.first + n * d.kv_heads) {  // (n is 0 for a request that is not split mode's)
      pl.first += n * d.kv_heads;
      ++pl.b;
      continue;
    }
    const int e = (int)((u0 - pl.first) / n);
    // the tile's keys begin kTileCost units after its place on the line; a share that ends before them has none of them
    const long long tile0 = pl.first + e * n + kTileCost, end = min(u1, tile0 + n - kTileCost), from = max(u0, tile0);
    if (from < end) {
      const Span sp = span_of(a, rq, 0, rq.q_len - 1, BT);
      const int blk0 = (int)(from - tile0) * UB, blk1 = min((int)(end - tile0) * UB, sp.n);
      const bool whole = from == tile0 && end == tile0 + n - kTileCost;
      piece(pl.b, rq, e, sp, blk0, blk1, whole, (long long)pl.b * d.kv_heads + e + blockIdx.x);
      if (!whole) join(pl.b, rq, e, block_of(tile0, total, blocks), block_of(tile0 + n - kTileCost - 1, total, blocks));
    }
    u0 = end;
  }
}

template <typename T, int HDP, int WM>
__global__ void __launch_bounds__(kAttnThreads) attn_split_kernel(const AttnArgs a, int* err) {
  using K = Cfg<T, HDP, WM>;
  extern __shared__ __align__(128) unsigned char attn_smem[];
  __shared__ uint32_t valid_s[K::WN][kStages];
  pdl_wait();
  pdl_trigger();
  split_walk<K::BT>(
      a,
      [&](int b, const Request& rq, int e, const Span& sp, int blk0, int blk1, bool whole, long long slot) {
        attn_piece<T, HDP, WM>(a, attn_smem, valid_s, err, b, rq, e, 0, sp, blk0, blk1, whole, slot);
      },
      [&](int b, const Request& rq, int e, int c0, int c1) { join_pieces<T, HDP, K::ROWS>(a, b, e, rq, c0, c1); });
}

// ------------------------------------------------------------ few rows, bf16
// Decoding in bf16 with at most 16 rows per tile and pages of 8, 16, 32, ... keys: the same split mode with the roles of the
// operands turned. The 16 rows of a product are keys (S^T = K Q^T) or output columns (O^T = V^T P^T) and the 8 columns are
// the tile's rows, so that 8 rows cost half the products, registers and exponentials that 16 would; the weights go
// from the first product's result to the second one's operand through movmatrix, the 8 x 8 transpose.
// Every warp has its own ring of 16- or 32-key blocks, filled by TMA (a box per page and 64 columns, issued
// by as many lanes). Bounded by the cache's bytes: 64 requests of 64 to 8192 keys, 500 MB: 92 us, 5.4 TB/s (the mma.sync
// form with rows as rows and one block per SM: 147 us).
template <int HDP, int NT>
struct NarrowCfg {
  static constexpr int BT = HDP == 128 ? 16 : 32;          // two blocks per SM: one streams while the other begins or ends a tile
  static constexpr int ROWS = 16;                          // workspace slots hold 16 rows
  static constexpr int TILE = BT * HDP * 2;                // keys or values of a block
  static constexpr int STAGES = 3;
  static constexpr int RING = 4 * STAGES * 2 * TILE;
  static constexpr int OP = HDP + 4;                       // floats of a row of the merge
  static constexpr int SMEM = RING + 1024;                 // 1024: alignment
};
MDLC_DEV uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
MDLC_DEV float max_over_keys(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
MDLC_DEV float sum_over_keys(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

template <int HDP, int NT>
__global__ void __launch_bounds__(kAttnThreads, 1) attn_narrow_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap,
                                                                      const __grid_constant__ CUtensorMap vmap, int* err) {
  using C = NarrowCfg<HDP, NT>;
  constexpr int BT = C::BT, HALVES = HDP / 64, MT = HDP / 16, KT = BT / 16;
  extern __shared__ unsigned char narrow_raw[];
  __shared__ __align__(8) uint64_t full_s[4][C::STAGES];
  unsigned char* smem = narrow_raw + ((1024 - (smem_u32(narrow_raw) & 1023)) & 1023);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const mdlc_attn_desc& d = a.d;
  if (threadIdx.x < 4 * C::STAGES) mbar_init(smem_u32(&full_s[0][0] + threadIdx.x), 1);
  fence_mbar_init();
  if (lane == 0) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  pdl_wait();
  pdl_trigger();
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * 2 * C::TILE;
  unsigned char* ring_p = smem + warp * C::STAGES * 2 * C::TILE;
  const int box = min(d.page, BT), boxes = BT / box;       // keys of a TMA box, boxes of a block
  const int none = d.pages * d.kv_heads * d.page;          // a row past the maps: zeros
  const int page_log2 = 31 - __clz(d.page);                // a power of two
  // this lane's box: keys or values, 64-column half, page
  const int my_page = lane % boxes, my_half = lane / boxes % HALVES, my_kv = lane / (boxes * HALVES);
  const bool mine = my_kv < 2;
  uint32_t begun = 0, used = 0;  // blocks issued and consumed by this warp so far

  auto piece = [&](int b, const Request& rq, int e, const Span& sp, int blk0, int blk1, bool whole, long long slot) {
    const int rows = rq.q_len * a.group, shift = rq.shift;
    // queries as the column operand: row 8 n + g, columns 16 ks + 2 t and + 8
    uint32_t qb[MT][NT][2];
    int pos[NT][2];  // positions of this thread's result columns, rows 8 n + 2 t and + 1
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 8 * n + g;
      const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(a.q) + (long long)(rq.q0 + min(r, rows - 1) / a.group) * d.q_stride +
                                (long long)(e * a.group + min(r, rows - 1) % a.group) * d.head_dim;
#pragma unroll
      for (int ks = 0; ks < MT; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = 16 * ks + 2 * t + 8 * i;
          qb[ks][n][i] = (r < rows && c < d.head_dim) ? __ldg(reinterpret_cast<const uint32_t*>(qp + c)) : 0u;
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) pos[n][i] = 8 * n + 2 * t + i < rows ? max(-1, shift + (8 * n + 2 * t + i) / a.group) : -1;
    }
    // page id of this lane's box, kHiddenPage: hidden from every row. Loads only, so that several are in flight.
    auto id_of = [&](int blk) {
      const int k0 = key_of_block(sp, blk, BT) + my_page * box;
      if (blk >= blk1 || !mine || k0 >= sp.hi || (k0 + box <= sp.lo && k0 >= d.sinks)) return kHiddenPage;
      if (!table_ok(a, b, k0 >> page_log2)) return kHiddenPage;
      return max(__ldg(a.table + (long long)b * d.table_stride + (k0 >> page_log2)), kHiddenPage + 1);
    };
    // its cache row, or one past the maps: hidden or missing
    auto row_of = [&](int blk, int id) {
      if (id == kHiddenPage) return none;
      if ((unsigned)id < (unsigned)d.pages) return (id * d.kv_heads + e) * d.page + ((key_of_block(sp, blk, BT) + my_page * box) & (d.page - 1));
      record_error(err, MDLC_DEVERR_BOUNDS);
      return none;
    };
    uint32_t there[C::STAGES];  // bit p: box p of the block in that stage was loaded
    auto issue = [&](int blk, int row, int st) {
      const uint32_t have = __ballot_sync(0xffffffffu, row != none);
#pragma unroll
      for (int i = 0; i < C::STAGES; ++i)
        if (i == st) there[i] = have & ((1u << boxes) - 1u);
      if (blk >= blk1) return;
      const uint32_t bar = smem_u32(&full_s[warp][st]);
      if (lane == 0) mbar_arrive_expect_tx(bar, 2 * C::TILE);
      __syncwarp();
      if (mine)
        tma_load_2d(ring + st * 2 * C::TILE + my_kv * C::TILE + my_half * (BT * 128) + my_page * box * 128, my_kv ? &vmap : &kmap, my_half * 64, row, bar);
      ++begun;
    };
    float o[MT][NT][4] = {};
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;
    // this warp takes blocks blk0 + warp, blk0 + warp + 4, ...; the stage of a use is its number modulo STAGES
    int st = used % C::STAGES;
    auto next_stage = [&](int s, int by) { return (s + by) % C::STAGES; };
    int ids[C::STAGES];
#pragma unroll
    for (int i = 0; i < C::STAGES; ++i) ids[i] = id_of(blk0 + warp + 4 * i);
#pragma unroll
    for (int i = 0; i < C::STAGES - 1; ++i) issue(blk0 + warp + 4 * i, row_of(blk0 + warp + 4 * i, ids[i]), next_stage(st, i));
    int id_next = ids[C::STAGES - 1];
    bool ok = true;
    for (int blk = blk0 + warp; blk < blk1; blk += 4) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full_s[warp][st]), (used / C::STAGES) & 1, nullptr, err, 2 * kWaitLimitNs));
      if (!ok) break;
      ++used;
      __syncwarp();  // every lane has read the stage that is filled next (the block before this one's)
      const int ahead = blk + 4 * (C::STAGES - 1);
      issue(ahead, row_of(ahead, id_next), next_stage(st, C::STAGES - 1));
      id_next = id_of(ahead + 4);
      const uint32_t ks_addr = ring + st * 2 * C::TILE, vs_addr = ks_addr + C::TILE;
      const int base = key_of_block(sp, blk, BT);
      uint32_t have = 0;
#pragma unroll
      for (int i = 0; i < C::STAGES; ++i)
        if (i == st) have = there[i];
      if (base + BT > rq.kv_len && base < rq.kv_len) {
        // values past kv_len may be anything (0 x NaN): cleared
        const int z0 = rq.kv_len - base;
        for (int i = lane; i < (BT - z0) * 8 * HALVES; i += 32) {
          const int h = i / ((BT - z0) * 8), k = i % ((BT - z0) * 8);
          *reinterpret_cast<uint4*>(ring_p + st * 2 * C::TILE + C::TILE + h * (BT * 128) + (z0 + k / 8) * 128 + (k % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      // scores: 16-key tile mt, rows 8 n + 2 t
      float s[KT][NT][4] = {};
      {
        const int mi = lane >> 3, r = lane & 7, key = (mi & 1) * 8 + r;
#pragma unroll
        for (int ks = 0; ks < MT; ++ks)
#pragma unroll
          for (int mt = 0; mt < KT; ++mt) {
            uint32_t ka[4];
            const int ch = 2 * ks + (mi >> 1);
            ldsm_x4(ka, ks_addr + (ch >> 3) * (BT * 128) + (mt * 16 + key) * 128 + (((ch & 7) ^ r) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_bf16(s[mt][n], ka, qb[ks][n][0], qb[ks][n][1]);
          }
      }
      const bool open = have == (1u << boxes) - 1u && base + BT - 1 <= shift &&
                        (d.window == 0 || base > shift + rq.q_len - 1 - d.window || base + BT <= d.sinks);
      bool grew = false;
      float safe[NT][2], shrink[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < KT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x = s[mt][n][2 * h + i] * a.scale_log2;
              if (!open) {
                const int c = mt * 16 + h * 8 + g, j = base + c, p = pos[n][i];
                const bool seen = ((have >> (c / box)) & 1u) && j <= p && (d.window == 0 || j > p - d.window || j < d.sinks);
                x = seen ? x : -INFINITY;
              }
              s[mt][n][2 * h + i] = x;
              top = fmaxf(top, x);
            }
          const float mn = fmaxf(m[n][i], max_over_keys(top));
          safe[n][i] = mn == -INFINITY ? 0.0f : mn;
          shrink[n][i] = exp2f(m[n][i] - safe[n][i]);
          grew |= mn > m[n][i];
          m[n][i] = mn;
        }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            l[n][i] *= shrink[n][i];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              o[mt][n][i] *= shrink[n][i];
              o[mt][n][2 + i] *= shrink[n][i];
            }
          }
      }
      uint32_t pb[KT][NT][2];  // weights as the column operand of the 16-key steps
#pragma unroll
      for (int mt = 0; mt < KT; ++mt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float x = exp2f(s[mt][n][2 * h] - safe[n][0]), y = exp2f(s[mt][n][2 * h + 1] - safe[n][1]);
            l[n][0] += x;
            l[n][1] += y;
            pb[mt][n][h] = transpose8x8(pack_bf16x2(x, y));
          }
      {
        const int mi = lane >> 3, r = lane & 7, key = (mi >> 1) * 8 + r;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t va[4];
            const int ch = 2 * mt + (mi & 1);
            ldsm_x4_t(va, vs_addr + (ch >> 3) * (BT * 128) + (kt * 16 + key) * 128 + (((ch & 7) ^ r) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_bf16(o[mt][n], va, pb[kt][n][0], pb[kt][n][1]);
          }
      }
      st = next_stage(st, 1);
    }
    // given up: the copies in flight must land before the shared memory changes hands
    for (; used != begun; ++used) mbar_wait(smem_u32(&full_s[warp][used % C::STAGES]), (used / C::STAGES) & 1, nullptr, err, 2 * kWaitLimitNs);
    __syncthreads();  // the rings are free: the warps' sums take their place
    float* so = reinterpret_cast<float*>(smem);
    float* sm = so + 4 * 8 * NT * C::OP;
    float* sl = sm + 4 * 8 * NT;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rl = warp * 8 * NT + 8 * n + 2 * t + i;
        const float lt = sum_over_keys(l[n][i]);
        if (g == 0) {
          sm[rl] = m[n][i];
          sl[rl] = lt;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          so[rl * C::OP + 16 * mt + g] = o[mt][n][i];
          so[rl * C::OP + 16 * mt + 8 + g] = o[mt][n][2 + i];
        }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < min(8 * NT, rows) * (HDP / 4); i += kAttnThreads) {
      const int rl = i / (HDP / 4), c = (i % (HDP / 4)) * 4;
      if (c >= d.head_dim) continue;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, sm[w * 8 * NT + rl]);
      const float base = top == -INFINITY ? 0.0f : top;
      float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = exp2f(sm[w * 8 * NT + rl] - base);
        const float4 x = *reinterpret_cast<const float4*>(so + (w * 8 * NT + rl) * C::OP + c);
        sum = fmaf(f, sl[w * 8 * NT + rl], sum);
        acc.x = fmaf(f, x.x, acc.x); acc.y = fmaf(f, x.y, acc.y); acc.z = fmaf(f, x.z, acc.z); acc.w = fmaf(f, x.w, acc.w);
      }
      if (whole) {
        const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
        const int tok = rq.q0 + rl / a.group, head = e * a.group + rl % a.group;
        if (!out_ok(a, tok, head, c, 4)) continue;
        uint2 v;
        v.x = pack_bf16x2(acc.x * inv, acc.y * inv);
        v.y = pack_bf16x2(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (long long)tok * d.out_stride + (long long)head * d.head_dim + c) = v;
        if (a.lse && c == 0) a.lse[(long long)tok * d.heads + head] = (top + log2f(sum)) * 0.69314718055994531f;
      } else {
        const long long at = slot * C::ROWS + rl;
        if (!part_ok(a, at)) continue;
        *reinterpret_cast<float4*>(a.part_o + at * HDP + c) = acc;
        if (c == 0) {
          a.part_m[at] = top;
          a.part_l[at] = sum;
        }
      }
    }
    fence_proxy_async_smem();  // the next piece's copies overwrite what was read and written here
    __syncthreads();
  };
  split_walk<BT>(a, piece, [&](int b, const Request& rq, int e, int c0, int c1) { join_pieces<__nv_bfloat16, HDP, C::ROWS>(a, b, e, rq, c0, c1); });
}

// A block per row tile, share of its keys and key head, heads fastest: blocks start in this order and the tiles come with the
// longest first, so the last to start are short (fp32, three prompts of up to 2000 tokens: 469 us, 584 with tiles fastest).
template <typename T, int HDP>
__global__ void __launch_bounds__(kAttnThreads) attn_chunk_kernel(const AttnArgs a, int* err) {
  using K = Cfg<T, HDP, 4>;
  extern __shared__ __align__(128) unsigned char attn_smem[];
  __shared__ uint32_t valid_s[K::WN][kStages];
  __shared__ long long warp_sums[kAttnThreads / 32];
  __shared__ Place place_s;
  pdl_wait();
  pdl_trigger();
  const int e = blockIdx.x % a.d.kv_heads, tile = blockIdx.x / a.d.kv_heads / a.splits, z = blockIdx.x / a.d.kv_heads % a.splits;
  Tile t;
  if (!find_tile(a, tile, K::ROWS, warp_sums, &place_s, &t)) return;
  const Span sp = span_of(a, t.rq, t.r0 / a.group, (min(t.r0 + K::ROWS, t.rows) - 1) / a.group, K::BT);
  const int ns = splits_of(a, sp.n, kLeastKeys / K::BT);
  if (z >= ns) return;
  attn_piece<T, HDP, 4>(a, attn_smem, valid_s, err, t.b, t.rq, e, t.r0, sp, (int)((long long)z * sp.n / ns),
                        (int)((long long)(z + 1) * sp.n / ns), ns == 1, ((long long)tile * a.d.kv_heads + e) * a.splits + z);
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
    if (!part_ok(a, (slot0 + ns - 1) * tile_rows + rl)) continue;
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
      if (i * 32 + lane < d.head_dim && out_ok(a, tok, head, i * 32 + lane, 1)) store_out<T>(po + i * 32 + lane, acc[i] * inv);
    if (a.lse && lane == 0 && out_ok(a, tok, head, 0, 1)) a.lse[(long long)tok * d.heads + head] = (top + log2f(sum)) * 0.69314718055994531f;
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
  int rows, tiles, splits, short_splits;
};
Chunk chunk_of(const mdlc_attn_desc& d) {
  const int group = d.heads / d.kv_heads;
  Chunk c = {};
  c.used = (long long)d.max_q * group > 16 * split_groups(d);
  c.tc = attn_tc_fits(d) && (long long)d.tokens * group / attn_tc_rows(d.head_dim) + d.batch <= 65535;  // the tiles are its grid's y
  c.rows = c.tc ? attn_tc_rows(d.head_dim) : 64;
  c.tiles = (int)min((long long)d.tokens * group / c.rows + d.batch, (long long)INT32_MAX);
  // Blocks on an SM: two of one row tile, one of two. The mma.sync kernel, of which two run at a time, has its shares made for twelve,
  // so that the last blocks to end are short; for four where that would leave a share under 512 keys, since every share costs
  // its part of the join. (`tiles` counts a part-filled tile more per request than there may be. Twenty fp32 batches of 1 to 24 requests of
  // 30 to 700 tokens on 100 to 6000 keys: twelve within 3%; 24 requests of up to 200 tokens on 6000 keys 578 us for four,
  // 441 for twelve, 24 mixed ones of 64 heads 750 and 594, 16 mixed ones on 4000 keys 165 and 99; five mixed ones on 1700 keys 66
  // and 77, twelve of up to 130 tokens on 400 keys 62 and 66.)
  const long long blocks = (long long)c.tiles * d.kv_heads;
  auto shares = [&](int per_sm, int keys) { return (int)max(1ll, min(kB200Sms * per_sm / blocks, min(16ll, (long long)d.max_kv / keys))); };
  c.short_splits = shares(c.tc ? (c.rows == 128 ? 2 : 1) : 4, kLeastKeys);
  c.splits = c.tc ? c.short_splits : max(c.short_splits, shares(12, 2 * kLeastKeys));
  return c;
}

// partial sums, maxima and sums of split mode's slots, then chunk mode's (the two run side by side)
struct Layout {
  size_t rows[2], o[2], m[2], l[2], total;
};
Layout layout_of(const mdlc_attn_desc& d) {
  const Chunk c = chunk_of(d);
  const size_t rows[2] = {((size_t)d.batch * d.kv_heads + kMaxBlocks) * 16 * split_groups(d),
                          c.used && c.splits > 1 ? (size_t)c.tiles * d.kv_heads * c.splits * c.rows : 0};
  Layout l = {};
  for (int i = 0; i < 2; ++i) {
    l.rows[i] = rows[i];
    l.o[i] = l.total;
    l.m[i] = l.o[i] + align256(rows[i] * padded_dim(d.head_dim) * 4);
    l.l[i] = l.m[i] + align256(rows[i] * 4);
    l.total = l.l[i] + align256(rows[i] * 4);
  }
  l.total = max(l.total, (size_t)256);
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
  static SmemLimit seen;
  const cudaError_t e = allow_smem(seen, ctx->device, kern, smem);
  if (e != cudaSuccess) return e;
  // one or two blocks per SM, as shared memory allows
  const int blocks = min(kMaxBlocks, ctx->num_sms * (smem <= kTwoBlocks ? 2 : 1));
  mdlc_note_launch(ctx);
  return launch_pdl(kern, dim3(blocks), dim3(kAttnThreads), smem, ctx->stream, a, ctx->d_err);
}

template <int HDP, int NT>
cudaError_t run_narrow(mdlc_ctx* ctx, const AttnArgs& a, int beside) {  // shared memory of a chunk block that runs beside, 0: none does
  using C = NarrowCfg<HDP, NT>;
  CUtensorMap maps[2];
  cudaError_t e = attn_tensor_maps(a, min(a.d.page, C::BT), &maps[0], &maps[1]);
  if (e != cudaSuccess) return e;
  static SmemLimit seen;
  e = allow_smem(seen, ctx->device, attn_narrow_kernel<HDP, NT>, C::SMEM);
  if (e != cudaSuccess) return e;
  // Two blocks per SM; one where that leaves room for a chunk block of the same call. Chunk blocks of wide heads fit beside neither one
  // nor two (40 decodes of up to 8000 keys and 20 chunks of up to 400 tokens, 128-column heads: two 324 us, one 352).
  const bool room = beside > 0 && C::SMEM + beside <= kSmShared;
  const int blocks = min(kMaxBlocks, ctx->num_sms * (room ? 1 : 2));
  mdlc_note_launch(ctx);
  return launch_pdl(attn_narrow_kernel<HDP, NT>, dim3(blocks), dim3(kAttnThreads), C::SMEM, ctx->stream, a, maps[0], maps[1], ctx->d_err);
}

// pages of 8, 16, 32, ... keys
bool narrow_fits(const mdlc_attn_desc& d) { return d.dtype == MDLC_BF16 && d.page >= 8 && (d.page & (d.page - 1)) == 0; }

template <typename T, int HDP>
cudaError_t run_chunks(mdlc_ctx* ctx, cudaStream_t stream, AttnArgs& a, const Chunk& c) {
  a.splits = c.splits;
  a.short_splits = c.short_splits;
  mdlc_note_launch(ctx);
  cudaError_t e;
  if (c.tc) {
    e = attn_tc_launch(ctx, stream, a, dim3(c.tiles, a.d.kv_heads, c.splits));
  } else {
    const int smem = Cfg<T, HDP, 4>::SMEM;
    static SmemLimit seen;
    e = allow_smem(seen, ctx->device, attn_chunk_kernel<T, HDP>, smem);
    const long long blocks = (long long)c.tiles * a.d.kv_heads * c.splits;
    if (e == cudaSuccess && blocks > INT32_MAX) e = cudaErrorInvalidConfiguration;
    if (e == cudaSuccess) e = launch_pdl(attn_chunk_kernel<T, HDP>, dim3((unsigned)blocks), dim3(kAttnThreads), smem, stream, a, ctx->d_err);
  }
  if (e != cudaSuccess || c.splits == 1) return e;
  mdlc_note_launch(ctx);
  return launch_pdl(attn_chunk_join_kernel<T, HDP>, dim3(c.tiles, a.d.kv_heads, c.rows / 16), dim3(kJoinThreads), 0, stream, a, c.rows,
                    c.tc ? kTcKeys : block_keys<T, HDP>());
}

template <typename T, int HDP>
cudaError_t run_attn(mdlc_ctx* ctx, AttnArgs& sa, AttnArgs& a) {  // split mode's and chunk mode's arguments
  const int wm = split_groups(a.d);
  const Chunk c = chunk_of(a.d);
  if (wm == 0) return run_chunks<T, HDP>(ctx, ctx->stream, a, c);
  // Both modes in one call touch different rows and parts of the workspace: chunk mode goes to the side stream, which waits for
  // the work before the call, and the compute stream for it (24 mixed requests of 64-column heads: 55.6 us, 62.1 one after the other).
  cudaError_t e = c.used ? mdlc_fork(ctx) : cudaSuccess;
  if (e != cudaSuccess) return e;
  if (wm == 1 && narrow_fits(a.d)) {
    // requests of up to 8 rows in one column tile; with more than 8 heads per key head, or several tokens, two
    const bool one = a.group <= 8 && ((long long)a.d.max_q * a.group <= 8 || (long long)a.d.max_q * a.group > 16);
    if (one) sa.split_rows = a.split_rows = 8;
    const int beside = c.used && c.tc ? attn_tc_smem(a.d.head_dim) : 0;
    e = one ? run_narrow<HDP, 1>(ctx, sa, beside) : run_narrow<HDP, 2>(ctx, sa, beside);
  } else if (wm == 1) {
    e = run_split<T, HDP, 1>(ctx, sa);
  } else if (wm == 2) {
    e = run_split<T, HDP, 2>(ctx, sa);
  } else if (wm == 4) {
    e = run_split<T, HDP, 4>(ctx, sa);
  }
  if (!c.used) return e;
  if (e == cudaSuccess) e = run_chunks<T, HDP>(ctx, ctx->side_stream, a, c);
  const cudaError_t joined = mdlc_join(ctx);
  return e != cudaSuccess ? e : joined;
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
  a.group_div = small_div(a.group);
  a.split_rows = 16 * split_groups(*desc);
  a.err = ctx->d_err;
  a.scale_log2 = desc->scale * 1.4426950408889634f;
  const Layout l = layout_of(*desc);
  char* ws = static_cast<char*>(workspace);
  auto place = [&](int mode) {
    a.part_o = reinterpret_cast<float*>(ws + l.o[mode]);
    a.part_m = reinterpret_cast<float*>(ws + l.m[mode]);
    a.part_l = reinterpret_cast<float*>(ws + l.l[mode]);
    a.part_rows = (long long)l.rows[mode];
  };
  place(0);
  AttnArgs split = a;
  place(1);
  a.arrived = ctx->d_attn_cnt;
  const bool bf16 = desc->dtype == MDLC_BF16;
  cudaError_t e;
  split.arrived = a.arrived;
  if (padded_dim(desc->head_dim) == 64) e = bf16 ? run_attn<__nv_bfloat16, 64>(ctx, split, a) : run_attn<float, 64>(ctx, split, a);
  else e = bf16 ? run_attn<__nv_bfloat16, 128>(ctx, split, a) : run_attn<float, 128>(ctx, split, a);
  return mdlc_cuda_status(ctx, e, "paged_attn launch");
}
