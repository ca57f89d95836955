// Attention of chunks on tcgen05 (bf16): the products S = Q K^T and O = P V.
//
// A block takes 256 rows (two tiles of 128, one per softmax warpgroup) of one key head, so that
// the 64 KB of keys and values of a 128-key block that it reads from L2 serve
// 256 rows: 4 x 256 x 128 x d operations per 512 d bytes. (Heads of up to 64 columns: one tile, two blocks per SM.) Roles, for two tiles:
//   warps 0-3, 4-7  softmax of row tile 0 / 1: a thread owns a row, reads its scores from
//                   tensor memory, keeps the running maximum and sum, writes the weights back
//                   to tensor memory as bf16 (the A operand of the second product)
//   warps 8, 10     issue the MMAs (one thread each) of row tile 0 / 1; warp 8 owns the tensor memory
//   warp 9          loads keys and values by TMA, a box per page, 32 lanes at once
//   (warps 8-11 give registers to the softmax warpgroups)
// Tensor memory (512 columns): scores of the two tiles [0, 256), 64 columns per half of a key block, the weights over the
// first 32 of their own half's; outputs [256, 256 + 2 HDP). Per half n of a key block the MMAs are O += P(n) V(n), then the scores of
// half n + 2 into the place that P(n) leaves (issue order makes them overwrite it only after it was read): a tile always has the next half's
// scores waiting, so its softmax does not wait for its own products.
// Outputs stay in tensor memory; they are rescaled only when a row's maximum grows by more than 2^8
// over the one in use (weights are then at most 2^8; bf16 rounding is relative, so nothing is lost),
// which after the first blocks hardly happens.
// Keys past kv_len and pages that no row sees arrive as zeros: boxes out of the map's range, and the
// last page's tail of the values is cleared in shared memory (its cache slots may hold NaN, and 0 x NaN
// would reach every row).
#include "conv.h"
#include "func_attr.h"
#include "paged_attn.cuh"

namespace mdlc {
namespace {

constexpr int kKeys = kTcKeys;
constexpr int kRing = 4;             // key / value tiles in shared memory: K(j), V(j), K(j+1), V(j+1)
constexpr float kGrow = 8.0f;        // growth of a row's maximum (base-2 exponent) that rescales the output
constexpr unsigned long long kWaitCycles = 2 * kWaitLimitNs;

template <int HDP>
struct TcCfg {
  // Row tiles of a block. Heads of up to 64 columns: one, since two such blocks fit on an SM and one's prologue and end overlap the
  // other's work; wider ones: two, for which a key block is read from L2 once.
  static constexpr int TILES = HDP == 64 ? 1 : 2;
  static constexpr int ROWS = 128 * TILES, SOFT = 4 * TILES;  // rows; softmax warps, in front of the four others
  static constexpr int THREADS = 128 * TILES + 128;
  // registers of a softmax and of another thread; their sum is what the block is launched with: 128 x (168 + 88) = 256 x 128,
  // 2 x 128 x 208 + 128 x 88 = 384 x 168
  static constexpr int SOFT_REGS = TILES == 1 ? 168 : 208, OTHER_REGS = 88;
  // Of 16 pairs of weights, how many take 2^x on the fp32 pipe beside the special-function unit (16 a clock), which the two tiles'
  // softmax share: 0.5 TFLOP of chunks in short runs on a cool chip 464 us with 3, 474 with 4, 490 with 2; with one tile, none is
  // as fast
  static constexpr int POLY = TILES == 2 ? 3 : 0;
  static constexpr int HALVES = HDP / 64;               // 128-byte wide column blocks
  static constexpr int TILE = 128 * HDP * 2;            // one Q tile, one key or value tile
  static constexpr int Q = 0;
  static constexpr int RING = TILES * TILE;
  static constexpr int BARS = RING + kRing * TILE;
  static constexpr int SMEM = BARS + 256 + 1024;        // 1024: alignment of the base
  static constexpr int O_COL = 128 * TILES, TMEM = 256 * TILES;  // outputs' first column; columns in all
};
// barriers; scores, weights and outputs have one per row tile and half of the key block (kS + 2 tile + half, ...)
enum { kFull = 0, kEmpty = kRing, kRaw = 2 * kRing, kQ, kS, kP = kS + 4, kO = kP + 4, kDrain = kO + 4, kBars = kDrain + 2 };

// instruction descriptor: bf16 x bf16 -> fp32; B stored along its N axis (values)
constexpr uint32_t idesc_bf16_nmajor(int M, int N) { return idesc_bf16(M, N) | (1u << 16); }

// B operand stored along N: 64-column (128-byte) rows, one per k; 8-row groups 1024 bytes apart (SBO), the
// next 64 columns lbo_bytes further
MDLC_DEV uint64_t umma_desc_sw128_n(uint32_t saddr, uint32_t lbo_bytes) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo_bytes >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// MMAs and commits issued by the lane that `leader` marks while the whole warp walks the loop: with operands that are
// uniform over the warp the descriptors stay in uniform registers (issued from a branch of one lane, an MMA took
// 112 cycles whatever its size, and the tensor pipe idled half of the time)
MDLC_DEV uint32_t elect_leader() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is;
}
MDLC_DEV void umma_lead(uint32_t leader, uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// A operand in tensor memory
MDLC_DEV void umma_lead_ta(uint32_t leader, uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
MDLC_DEV void commit_lead(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(leader)
      : "memory");
}
#define MDLC_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
MDLC_DEV void tmem_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : MDLC_R8(v, 0), MDLC_R8(v, 8), MDLC_R8(v, 16), MDLC_R8(v, 24)
      : "r"(taddr)
      : "memory");
}
#define MDLC_I8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
MDLC_DEV void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      MDLC_I8(v, 0), MDLC_I8(v, 8), MDLC_I8(v, 16), MDLC_I8(v, 24)
      : "memory");
}
MDLC_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
MDLC_DEV float2 add2(const float2 a, const float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_from(r);
}
template <int N>
MDLC_DEV void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
MDLC_DEV void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
MDLC_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

MDLC_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
MDLC_DEV float2 mul2(const float2 a, const float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_from(r);
}

// 2^x of two values on the fp32 pipe: x = n + f with n the nearest integer (added and taken off again at 1.5 x 2^23, where
// fp32 numbers are the integers), 2^f on [-1/2, 1/2] by a polynomial of degree 4, times 2^n made from n's bits. The
// coefficients are a fit of smallest maximal relative error on that interval (2.6e-6, far below the bf16 rounding of the
// weights). Numbers from -127 down are taken as -127, whose 2^n has the bits of 0: a hidden key (-inf) weighs exactly 0, and what is
// below 2^-126.5 counts as 0 too. NaN stays NaN: the maximum passes it on, and the last step is a product.
MDLC_DEV float2 ex2_poly(float2 x) {
  x = make_float2(max_nan(x.x, -127.0f), max_nan(x.y, -127.0f));
  const float2 t = add2(x, splat2(12582912.0f));
  const float2 f = fma2(add2(t, splat2(-12582912.0f)), splat2(-1.0f), x);
  float2 p = fma2(f, splat2(0.009570104070f), splat2(0.05591790378f));
  p = fma2(f, p, splat2(0.2402474582f));
  p = fma2(f, p, splat2(0.6931217909f));
  p = fma2(f, p, splat2(0.9999992847f));
  return mul2(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}

template <int HDP>
__global__ void __launch_bounds__(TcCfg<HDP>::THREADS, 3 - TcCfg<HDP>::TILES) attn_tc_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap,
                                                              const __grid_constant__ CUtensorMap vmap, int* err) {
  using C = TcCfg<HDP>;
  extern __shared__ unsigned char tc_smem_raw[];
  __shared__ long long warp_sums[C::THREADS / 32];
  __shared__ Place place_s;
  __shared__ uint32_t tmem_s;
  __shared__ int abort_s, missing_s;
  unsigned char* smem = tc_smem_raw + ((1024 - (smem_u32(tc_smem_raw) & 1023)) & 1023);
  const uint32_t sbase = smem_u32(smem);
  auto bar = [&](int i) { return sbase + C::BARS + 8 * i; };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const mdlc_attn_desc& d = a.d;
  volatile int* abort_flag = &abort_s;

  // what touches no global memory comes before the wait for the kernel in front
  if (warp == C::SOFT + 1 && lane == 0) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(bar(kFull + i), 1);
    }
    mbar_init(bar(kRaw), 1);
    mbar_init(bar(kQ), C::ROWS);
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(kS + i), 1);
      mbar_init(bar(kP + i), 128);
      mbar_init(bar(kO + i), 1);
    }
    for (int i = 0; i < C::TILES; ++i) mbar_init(bar(kDrain + i), 1);
    abort_s = missing_s = 0;
    fence_mbar_init();
  }
  pdl_wait();
  pdl_trigger();
  Tile t;
  if (!find_tile(a, blockIdx.y, C::ROWS, warp_sums, &place_s, &t)) return;
  const int e = blockIdx.x;
  const Span sp = span_of(a, t.rq, t.r0 / a.group, (min(t.r0 + C::ROWS, t.rows) - 1) / a.group, kKeys);
  const int ns = splits_of(a, sp.n, 2);
  if ((int)blockIdx.z >= ns) return;
  const int blk0 = (int)((long long)blockIdx.z * sp.n / ns), blk1 = (int)((long long)(blockIdx.z + 1) * sp.n / ns), nb = blk1 - blk0;
  const int shift = t.rq.shift;
  const int n_tiles = C::TILES == 2 && t.rows - t.r0 > 128 ? 2 : 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) mbar_init(bar(kEmpty + i), n_tiles);  // both tiles' MMAs give a key or value tile back
    fence_mbar_init();
  }
  if (warp == C::SOFT) {
    tmem_alloc(smem_u32(&tmem_s), C::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  // token and head of row t.r0 + rl: the tile's first ones, and a division of a small number
  const int tok0 = t.r0 / a.group, rem0 = t.r0 - tok0 * a.group;
  auto token_of = [&](int rl, int* head) {
    const int n = div_small(rem0 + rl, a.group_div);
    *head = e * a.group + rem0 + rl - n * a.group;
    return t.rq.q0 + tok0 + n;
  };

  if (warp < C::SOFT) {
    // ------------------------------------------------------------ softmax
    regs_up<C::SOFT_REGS>();
    // queries: rows of 128 bytes per 64 columns, 16-byte chunks swizzled by the row
    {
      const int chunks = d.head_dim / 8;
      constexpr int CH = HDP / 8;
      for (int i0 = threadIdx.x; i0 < C::ROWS * CH; i0 += 8 * C::ROWS) {  // eight loads at a time
        uint4 v[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int i = i0 + n * C::ROWS, rl = i / CH, c = i % CH;
          v[n] = make_uint4(0, 0, 0, 0);
          if (t.r0 + rl < t.rows && c < chunks) {
            int head;
            const int tok = token_of(rl, &head);
            v[n] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + tok * d.q_stride + (long long)head * d.head_dim) + c);
          }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int i = i0 + n * C::ROWS, rl = i / CH, c = i % CH;
          *reinterpret_cast<uint4*>(smem + C::Q + (rl >> 7) * C::TILE + (c >> 3) * 16384 + (rl & 127) * 128 + (((c & 7) ^ (rl & 7)) << 4)) = v[n];
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(bar(kQ));
    }
    const int page_log2 = 31 - __clz(d.page);  // a power of two
    // Ids that do not exist hide their keys: looked for once, so that the blocks need not look (a load from the table
    // in front of every block cost 570 cycles of 4200)
    auto missing = [&](int j) {
      return j < sp.hi && (j + min(d.page, kKeys) > sp.lo || j < d.sinks) && table_ok(a, t.b, j >> page_log2) &&
             (unsigned)__ldg(a.table + (long long)t.b * d.table_stride + (j >> page_log2)) >= (unsigned)d.pages;
    };
    {
      const int per = kKeys / min(d.page, kKeys);
      bool none = false;
      for (int i = threadIdx.x; i < nb * per; i += C::ROWS) none |= missing(key_of_block(sp, blk0 + i / per, kKeys) + i % per * min(d.page, kKeys));
      if (none) missing_s = 1;
      asm volatile("bar.sync 1, %0;" ::"n"(C::ROWS) : "memory");
    }
    const bool any_missing = *(volatile int*)&missing_s;
    const int tile = warp >> 2, rl = threadIdx.x, r = t.r0 + rl;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + tile * 128, o_addr = tmem + lanes + C::O_COL + tile * HDP;
    const bool live = r < t.rows;
    const int p = live ? max(-1, shift + r / a.group) : -1;
    const int first = t.r0 + tile * 128, last = min(first + 127, t.rows - 1);
    const int p_min = shift + first / a.group, p_max = shift + last / a.group;
    const float c = a.scale_log2;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    if (tile < n_tiles) {
      const int box = min(d.page, kKeys), box_log2 = 31 - __clz(box);  // keys of a TMA box, a power of two
      // blocks [open0, open1) of this share are seen whole by every row of the tile: no mask
      int open0 = 0, open1 = nb;
      if (any_missing) open1 = 0;
      while (open1 > 0 && key_of_block(sp, blk0 + open1 - 1, kKeys) + kKeys - 1 > p_min) --open1;
      if (d.window > 0)
        while (open0 < open1 && key_of_block(sp, blk0 + open0, kKeys) <= p_max - d.window) ++open0;
      for (int n = 0; n < 2 * nb; ++n) {
        const int j = n >> 1, h = n & 1;
        const uint32_t sh = s_addr + 64 * h;  // this half's scores, and their weights
        ok = __all_sync(0xffffffffu, mbar_wait(bar(kS + 2 * tile + h), j & 1, abort_flag, err, kWaitCycles));
        if (!ok) break;
        tc_fence_after();
        if (j < open0 || j >= open1) {
          // hidden keys to -inf, in place (a loop of its own, so that the common path stays small)
          const int base = key_of_block(sp, blk0 + j, kKeys) + 64 * h;
          const int hi = p - base, lo = d.window > 0 ? hi - d.window : -1, kept = d.window > 0 ? d.sinks - base : 0;
          uint32_t bad = 0;  // boxes of this block without a page
          if (any_missing) bad = __ballot_sync(0xffffffffu, lane < (kKeys >> box_log2) && missing(base - 64 * h + (lane << box_log2)));
          // bits [0, n) of a word, n of any sign or size
          auto below = [](int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); };
#pragma unroll 1
          for (int k0 = 0; k0 < 64; k0 += 32) {
            uint32_t see = below(hi + 1 - k0) & (~below(lo + 1 - k0) | below(kept - k0));
            if (bad) {
#pragma unroll 1
              for (int i = 0; i < 32; i += 8)
                if ((bad >> ((64 * h + k0 + i) >> box_log2)) & 1u) see &= ~(0xffu << i);
            }
            uint32_t s[32];
            tmem_ld32(sh + k0, s);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i] = (see >> i) & 1u ? s[i] : 0xff800000u;
            tmem_st32(sh + k0, s);
          }
          tmem_st_wait();
        }
        // One pass takes the weights against the maximum in use and the half's own maximum; when that has grown by more
        // than 2^8 for some row of the warp (or a row sees its first keys) the pass is repeated with the new one. The
        // weights wait in registers: their place is the scores' own.
        uint32_t w[32];
        for (;;) {
          const float mc = m == -INFINITY ? 0.0f : m * c;
          const float2 c2 = splat2(c), mc2 = splat2(-mc);
          float top[2] = {-INFINITY, -INFINITY};
          float2 sum[2] = {splat2(0.0f), splat2(0.0f)};
          uint32_t s[2][32];
          tmem_ld32(sh, s[0]);
          tmem_ld_wait();
          tmem_ld32(sh + 32, s[1]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (k) tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 x = make_float2(__uint_as_float(s[k][i]), __uint_as_float(s[k][i + 1]));
              top[(i >> 1) & 1] = max3(top[(i >> 1) & 1], x.x, x.y);
              float2 y = fma2(x, c2, mc2);
              if ((i / 2 + 1) * C::POLY / 16 > i / 2 * C::POLY / 16) y = ex2_poly(y);
              else y = make_float2(ex2(y.x), ex2(y.y));
              sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], y);
              w[16 * k + (i >> 1)] = pack_bf16x2(y.x, y.y);
            }
          }
          const float mn = fmaxf(top[0], top[1]);
          const bool fresh = m == -INFINITY && mn > -INFINITY, grow = m != -INFINITY && (mn - m) * c > kGrow;
          if (!__any_sync(0xffffffffu, fresh || grow)) {
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            break;
          }
          // a row that has summed nothing yet takes the maximum as it is
          const float f = fresh ? 0.0f : (grow ? ex2((m - mn) * c) : 1.0f);
          if (fresh || grow) m = mn;
          l *= f;
          if (__any_sync(0xffffffffu, grow)) {
            ok = mbar_wait(bar(kO + 2 * tile + (h ^ 1)), ((n - 1) >> 1) & 1, abort_flag, err, kWaitCycles);  // the half before this one
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < HDP; i += 32) {
              uint32_t o[32];
              tmem_ld32(o_addr + i, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st32(o_addr + i, o);
            }
          }
        }
        if (!ok) break;
        tmem_st32(sh, w);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar(kP + 2 * tile + h));
      }
      if (ok && nb > 0) ok = mbar_wait(bar(kO + 2 * tile + 1), (nb - 1) & 1, abort_flag, err, kWaitCycles);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      if (ok) {
        const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
        const long long slot = (((long long)blockIdx.y * d.kv_heads + e) * a.splits + blockIdx.z) * C::ROWS + rl;
        const float mlog = m == -INFINITY ? -INFINITY : m * c;
        uint32_t o[HDP];
#pragma unroll
        for (int i = 0; i < HDP; ++i) o[i] = 0;
        if (nb > 0) {
#pragma unroll
          for (int i = 0; i < HDP; i += 32) tmem_ld32(o_addr + i, o + i);
          tmem_ld_wait();
        }
        if (ns == 1) {
          // through the place of this warp's queries (their products are done), so that rows are written whole
          constexpr int CH = HDP / 8;
          unsigned char* rows = smem + C::Q + tile * C::TILE + (warp & 3) * 32 * HDP * 2;
#pragma unroll
          for (int k = 0; k < CH; ++k) {
            uint4 v;
            v.x = pack_bf16x2(__uint_as_float(o[8 * k]) * inv, __uint_as_float(o[8 * k + 1]) * inv);
            v.y = pack_bf16x2(__uint_as_float(o[8 * k + 2]) * inv, __uint_as_float(o[8 * k + 3]) * inv);
            v.z = pack_bf16x2(__uint_as_float(o[8 * k + 4]) * inv, __uint_as_float(o[8 * k + 5]) * inv);
            v.w = pack_bf16x2(__uint_as_float(o[8 * k + 6]) * inv, __uint_as_float(o[8 * k + 7]) * inv);
            *reinterpret_cast<uint4*>(rows + lane * HDP * 2 + ((k ^ (lane & 7)) << 4)) = v;
          }
          __syncwarp();
#pragma unroll 4
          for (int i = lane; i < 32 * CH; i += 32) {
            const int row = i / CH, k = i % CH, rw = warp * 32 + row;
            if (t.r0 + rw < t.rows && 8 * k < d.head_dim) {
              int head;
              const int tok = token_of(rw, &head);
              if (!out_ok(a, tok, head, 8 * k, 8)) continue;
              *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + tok * d.out_stride + (long long)head * d.head_dim + 8 * k) =
                  *reinterpret_cast<const uint4*>(rows + row * HDP * 2 + ((k ^ (row & 7)) << 4));
            }
          }
        } else if (live && part_ok(a, slot)) {
#pragma unroll
          for (int k = 0; k < HDP; k += 4)
            *reinterpret_cast<uint4*>(a.part_o + slot * HDP + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        }
        if (live) {
          if (ns > 1 && part_ok(a, slot)) {
            a.part_m[slot] = mlog;
            a.part_l[slot] = l;
          } else if (ns == 1 && a.lse) {
            int head;
            const long long tok = token_of(rl, &head);
            if (out_ok(a, tok, head, 0, 1)) a.lse[tok * d.heads + head] = (mlog + log2f(l)) * 0.69314718055994531f;
          }
        }
      }
    }
  } else {
    regs_down<C::OTHER_REGS>();  // the last four warps alike, before their ways part
    if (warp == C::SOFT || (C::TILES == 2 && warp == C::SOFT + 2)) {
    // ------------------------------------------------------------ MMA: a warp per row tile
    const uint32_t leader = elect_leader();
    const int i = warp == C::SOFT ? 0 : 1;
    const int u_nb = __shfl_sync(0xffffffffu, i < n_tiles ? nb : 0, 0);
    const uint32_t u_s = __shfl_sync(0xffffffffu, tmem + i * 128, 0), u_o = __shfl_sync(0xffffffffu, tmem + C::O_COL + i * HDP, 0);
    if (u_nb > 0) {
      constexpr uint32_t kIdS = idesc_bf16(128, 64), kIdO = idesc_bf16_nmajor(128, HDP);
      bool ok = __all_sync(0xffffffffu, mbar_wait(bar(kQ), 0, abort_flag, err, kWaitCycles));
      auto wait_tile = [&](int u) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar(kFull + u % kRing), (u / kRing) & 1, abort_flag, err, kWaitCycles)); };
      auto scores = [&](int j, int h) {  // half h of S = Q K(j)^T
        const uint32_t q = sbase + C::Q + i * C::TILE, k = sbase + C::RING + ((2 * j) % kRing) * C::TILE + h * 8192;
#pragma unroll
        for (int ks = 0; ks < HDP / 16; ++ks) {
          const uint32_t off = (ks / 4) * 16384 + (ks % 4) * 32;
          umma_lead(leader, u_s + h * 64, umma_desc_sw128(q + off), umma_desc_sw128(k + off), kIdS, ks > 0);
        }
        commit_lead(leader, bar(kS + 2 * i + h));
      };
      ok = ok && wait_tile(0);
      tc_fence_after();
      if (ok) {
        scores(0, 0);
        scores(0, 1);
        commit_lead(leader, bar(kEmpty + 0));
      }
      for (int j = 0; ok && j < u_nb; ++j) {
        ok = wait_tile(2 * j + 1);
        const uint32_t v = sbase + C::RING + ((2 * j + 1) % kRing) * C::TILE;
        for (int h = 0; ok && h < 2; ++h) {
          ok = __all_sync(0xffffffffu, mbar_wait(bar(kP + 2 * i + h), j & 1, abort_flag, err, kWaitCycles));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_lead_ta(leader, u_o, u_s + h * 64 + ks * 8, umma_desc_sw128_n(v + (4 * h + ks) * 2048, 16384), kIdO, j > 0 || h > 0 || ks > 0);
          commit_lead(leader, bar(kO + 2 * i + h));
          if (h) commit_lead(leader, bar(kEmpty + (2 * j + 1) % kRing));
          if (j + 1 < u_nb) {
            if (!h) {
              ok = wait_tile(2 * j + 2);
              if (!ok) break;
              tc_fence_after();
            }
            scores(j + 1, h);
            if (h) commit_lead(leader, bar(kEmpty + (2 * j + 2) % kRing));
          }
        }
      }
      // everything issued is done before the tensor memory goes back
      commit_lead(leader, bar(kDrain + i));
      mbar_wait(bar(kDrain + i), 0, nullptr, err, kWaitCycles);
    }
    __syncwarp();
    } else if (warp == C::SOFT + 1) {
    // ------------------------------------------------------------ keys and values
    const int box = min(d.page, kKeys), boxes = kKeys / box;
    const int page_i = lane % boxes, half = lane / boxes;   // this lane's box: boxes x HALVES <= 32 of them
    const bool mine = half < C::HALVES;
    const int none = d.pages * d.kv_heads * d.page;         // a row past the map: zeros
    bool ok = true;
    int u = 0, raw = 0;
    for (int j = 0; ok && j < nb; ++j) {
      const int base = key_of_block(sp, blk0 + j, kKeys);
      const int k0 = base + page_i * box;
      int row = none;
      if (mine && k0 < sp.hi && (k0 + box > sp.lo || k0 < d.sinks)) {
        const int id = table_ok(a, t.b, k0 / d.page) ? __ldg(a.table + (long long)t.b * d.table_stride + k0 / d.page) : -1;
        if ((unsigned)id < (unsigned)d.pages) row = (id * d.kv_heads + e) * d.page + k0 % d.page;
        else record_error(err, MDLC_DEVERR_BOUNDS);
      }
      for (int kv = 0; kv < 2; ++kv, ++u) {
        const int st = u % kRing;
        // values whose last page ends inside this block: cleared from kv_len on before the MMA may read them
        const bool tail = kv == 1 && base < t.rq.kv_len && t.rq.kv_len < base + kKeys && t.rq.kv_len % d.page != 0;
        if (u >= kRing) ok = mbar_wait(bar(kEmpty + st), ((u / kRing) & 1) ^ 1, abort_flag, err, kWaitCycles);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t full = tail ? bar(kRaw) : bar(kFull + st);
        if (lane == 0) mbar_arrive_expect_tx(full, C::TILE);
        __syncwarp();
        const uint32_t dst = sbase + C::RING + st * C::TILE;
        if (mine) tma_load_2d(dst + half * 16384 + page_i * box * 128, kv ? &vmap : &kmap, half * 64, row, full);
        if (tail) {
          ok = __all_sync(0xffffffffu, mbar_wait(bar(kRaw), raw & 1, nullptr, err, kWaitCycles));
          ++raw;
          if (!ok) break;
          const int z0 = t.rq.kv_len - base, z1 = min(kKeys, (z0 / box + 1) * box);
          for (int i = lane; i < (z1 - z0) * 8 * C::HALVES; i += 32) {
            const int h = i / ((z1 - z0) * 8), k = i % ((z1 - z0) * 8);
            *reinterpret_cast<uint4*>(smem + C::RING + st * C::TILE + h * 16384 + (z0 + k / 8) * 128 + (k % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(kFull + st));
        }
      }
    }
    if (!ok) {
      // given up: this block's copies must land before its shared memory goes back
      for (int i = max(0, u - kRing); i < u; ++i) mbar_wait(bar(kFull + i % kRing), (i / kRing) & 1, nullptr, err, kWaitCycles);
    }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == C::SOFT) tmem_dealloc(tmem, C::TMEM);
}

template <int HDP>
cudaError_t launch(mdlc_ctx* ctx, cudaStream_t stream, const AttnArgs& a, dim3 grid) {
  CUtensorMap maps[2];
  cudaError_t e = attn_tensor_maps(a, min(a.d.page, kKeys), &maps[0], &maps[1]);
  if (e != cudaSuccess) return e;
  static SmemLimit seen;
  e = allow_smem(seen, ctx->device, attn_tc_kernel<HDP>, TcCfg<HDP>::SMEM);
  if (e != cudaSuccess) return e;
  // key heads fastest: the tiles that see the most keys start first in all of them
  return launch_pdl(attn_tc_kernel<HDP>, dim3(grid.y, grid.x, grid.z), dim3(TcCfg<HDP>::THREADS), TcCfg<HDP>::SMEM, stream, a, maps[0], maps[1], ctx->d_err);
}

}  // namespace

cudaError_t attn_tensor_maps(const AttnArgs& a, int box, CUtensorMap* k, CUtensorMap* v) {
  const auto encode = tensor_map_encoder();
  if (!encode) return cudaErrorNotSupported;
  const mdlc_attn_desc& d = a.d;
  const cuuint64_t dims[2] = {(cuuint64_t)d.head_dim, (cuuint64_t)d.pages * d.kv_heads * d.page}, strides[1] = {(cuuint64_t)d.head_dim * 2};
  const cuuint32_t size[2] = {64, (cuuint32_t)box}, steps[2] = {1, 1};
  for (int i = 0; i < 2; ++i)
    if (encode(i ? v : k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(i ? a.v : a.k), dims, strides, size, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  return cudaSuccess;
}

// bf16, pages that tile a 128-key block, a positive scale (the running maximum is that of the raw scores)
bool attn_tc_fits(const mdlc_attn_desc& d) {
  const bool page = d.page >= 8 && (d.page & (d.page - 1)) == 0;
  return d.dtype == MDLC_BF16 && page && d.scale > 0.0f && d.heads / d.kv_heads <= 4096;  // (small divisions by the group)
}

int attn_tc_rows(int head_dim) { return head_dim <= 64 ? TcCfg<64>::ROWS : TcCfg<128>::ROWS; }

int attn_tc_smem(int head_dim) { return head_dim <= 64 ? TcCfg<64>::SMEM : TcCfg<128>::SMEM; }

cudaError_t attn_tc_launch(mdlc_ctx* ctx, cudaStream_t stream, const AttnArgs& a, dim3 grid) {
  return a.d.head_dim <= 64 ? launch<64>(ctx, stream, a, grid) : launch<128>(ctx, stream, a, grid);
}

}  // namespace mdlc
