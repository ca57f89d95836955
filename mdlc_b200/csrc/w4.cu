// mdlc_gemv_w4: products of a few rows with 4-bit weights and group scales.
//
// Memory-bound: half a byte of weight per 2 m operations. At the copy bandwidth an SM receives 48
// weights a clock, so what decides, besides bytes in flight, is how many instructions a weight
// costs. The products run on the bf16 tensor pipe (mma.sync m16n8k16, fp32 sums), every one of them exact:
//   * the weights are the 16-row operand. A code c or-ed into the low mantissa bits of 2^-5 is 2^-5 + c 2^-12, and less
//     2^-5 + z 2^-12 (z the zero point) it is (c - z) 2^-12 exactly: eleven operations for eight codes. The factor, which the
//     end takes off again, keeps a group's sums below the largest |x| of it.
//   * x is the 8-column operand: a bf16 row is one column as it is, an fp32 row three, whose sum it is exactly (8 bits each, cut
//     off in turn; below 2^-110 the last bits go). No scale is shared between columns of x, so a large one that meets weights of
//     zero takes nothing from its neighbours. (Fixed-point digits with a shared scale on the int8 pipe cost three operations for
//     eight codes - one row of 65536 x 8192 55-59 us, here 68-73 us, 3.8-4.1 TB/s - but an error that followed the largest |x| of 128
//     columns, and three columns for a bf16 row too: 16 rows of 14336 x 4096 51 us, here 34 us.)
//   * a group is summed from zero in the tensor core, scaled and added to the row's fp32 sum.
// The order of the columns inside a product is free as long as both operands agree, so a thread keeps
// the 32 consecutive codes of its 16-byte load. For groups under 128 columns the four threads of a row hold different
// groups; a 4 x 4 exchange of words inside the quad then puts 32 consecutive columns into each product.
//
// Blocks are persistent: 16 R output columns at a time, the 8 warps taking 128-column steps of k in turn
// (adjacent warps read adjacent bytes of a row); the weights of the next steps, across tiles too, are on their way
// through cp.async, and the warps' sums are added in warp order, so results do not depend on timing.
#include "common.cuh"
#include "func_attr.h"
#include "runtime.h"

namespace mdlc {
namespace {

constexpr int kW4Warps = 8;
constexpr int kW4Depth = 4;        // 128-column steps of weights on their way per warp
// A single row up to this long is split by every block itself (fp32, 8192 columns, 28672 outputs: 50.8 us, 56.2 with a kernel in front;
// bf16, 28672 columns, 8192 outputs: 42.7 and 39.5)
constexpr int kW4OwnColumns = 12288;
constexpr uint32_t kCode0 = 0x3d003d00u;  // two bf16 numbers 2^-5; one more in the last place is 2^-12
constexpr float kCodeUnit = 4096.0f;      // 2^12

struct W4Args {
  mdlc_w4_desc d;
  const void* x;
  const uint8_t* codes;
  const uint16_t* scales;  // bf16 bits
  const uint8_t* zeros;
  const float* bias;
  void* y;
  int rows_per_chunk;   // x rows of one grid.y chunk
  int parts;            // columns of an x row: 1 (bf16) or 3 (fp32)
  int pitch;            // columns kept per 8 of k
  int step_bytes;       // x of one step: 16 units of 8 columns x pitch x 16 bytes
  int span, buffers;    // steps in shared memory at a time, and their buffers
  const uint8_t* ready; // x in parts, [chunk][step], or null: the block makes them itself
  bool ready_wanted;
  int* err;
};

// 16-byte copy to shared memory, always whole
MDLC_DEV void cp_async_16_all(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

MDLC_DEV void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the codes in bits 0-3 and 16-19 as two bf16 numbers (code - z) 2^-12; zero: kCode0 with z in both halves
MDLC_DEV uint32_t code_pair(uint32_t w, uint32_t zero) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(0x000f000fu), "r"(kCode0));  // (a & b) | c
  asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(zero));
  return v;
}

// word i of the four threads of a quad <-> thread i's words: w[i] becomes thread i's word t
MDLC_DEV void quad_transpose(uint32_t (&w)[4], int t) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint32_t got = __shfl_xor_sync(0xffffffffu, (t & 1) ? w[i] : w[i + 1], 1);
    if (t & 1) w[i] = got; else w[i + 1] = got;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t got = __shfl_xor_sync(0xffffffffu, (t & 2) ? w[i] : w[i + 2], 2);
    if (t & 2) w[i] = got; else w[i + 2] = got;
  }
}

// x in parts, one 128-column step of k after the other, each: 16 units of 8 columns x pitch columns x 16 bytes (bf16, columns
// 0 4 1 5 2 6 3 7 of the unit, as the codes of a word come). Units and columns are permuted so that the four units a warp reads
// at once, 4 apart or adjacent, lie in different banks for each pair of columns.
MDLC_DEV int x_place(int unit, int col, int pitch) {
  const int turn = (unit ^ (unit >> 2)) & 3;
  if (pitch == 1) return (unit & ~3) | turn;
  if (pitch == 4) return ((unit & ~3) | turn) * 4 + (col ^ (turn & 2));
  return unit * pitch + (col ^ (2 * turn));
}

// Unit u of an x row in its parts, written to the step that holds it (past k: zeros). col0: the row's first column
template <bool BF16>
MDLC_DEV void x_unit(const W4Args& a, const uint4 (&raw)[2], int u, int col0, uint8_t* dst) {
  uint4* units = reinterpret_cast<uint4*>(dst);
  if (BF16) {
    const uint4 p = raw[0];
    units[x_place(u & 15, col0, a.pitch)] = make_uint4(__byte_perm(p.x, p.z, 0x5410), __byte_perm(p.x, p.z, 0x7632), __byte_perm(p.y, p.w, 0x5410),
                                                       __byte_perm(p.y, p.w, 0x7632));
    return;
  }
  const uint32_t f[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
  uint32_t part[3][8];  // bf16 in the upper half
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t top = f[e] & 0x7fffffffu;
    part[0][e] = top > 0x7f800000u ? 0x7fc00000u : f[e] & 0xffff0000u;  // (a NaN's upper bits alone may be an infinity's)
    const float rest = top < 0x7f800000u ? __uint_as_float(f[e]) - __uint_as_float(part[0][e]) : 0.0f;
    part[1][e] = __float_as_uint(rest) & 0xffff0000u;
    part[2][e] = __float_as_uint(rest - __uint_as_float(part[1][e]));
  }
#pragma unroll
  for (int p = 0; p < 3; ++p)
    units[x_place(u & 15, col0 + p, a.pitch)] = make_uint4(__byte_perm(part[p][0], part[p][4], 0x7632), __byte_perm(part[p][1], part[p][5], 0x7632),
                                                           __byte_perm(part[p][2], part[p][6], 0x7632), __byte_perm(part[p][3], part[p][7], 0x7632));
}
template <bool BF16>
MDLC_DEV void x_load(const W4Args& a, int row, int u, bool ok, uint4 (&raw)[2]) {
  raw[0] = raw[1] = make_uint4(0, 0, 0, 0);
  if (!ok || !MDLC_CHECK_IDX(a.err, row, a.d.m) || !MDLC_CHECK_IDX(a.err, u * 8 + 7, a.d.k)) return;
  const long long at = (long long)row * a.d.x_stride + u * 8;
  if (BF16) {
    raw[0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.x) + at));
  } else {
    raw[0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(a.x) + at));
    raw[1] = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(a.x) + at) + 1);
  }
}

// x in parts in global memory, for the blocks of gemv_w4_kernel to copy: a thread per row and unit
template <bool BF16>
__global__ void __launch_bounds__(128) w4_parts_kernel(const W4Args a, uint8_t* ready) {
  pdl_wait();
  pdl_trigger();
  const int steps = (a.d.k + 127) / 128, u = blockIdx.x * 128 + threadIdx.x, row = blockIdx.y;
  if (u >= 16 * steps) return;
  uint4 raw[2];
  x_load<BF16>(a, row, u, u < a.d.k / 8, raw);
  const int chunk = row / a.rows_per_chunk;
  if (!MDLC_CHECK_IDX(a.err, ((long long)chunk * steps + u / 16 + 1) * a.step_bytes - 1, kSplitWsBytes)) return;
  x_unit<BF16>(a, raw, u, a.parts * (row - chunk * a.rows_per_chunk), ready + ((long long)chunk * steps + u / 16) * a.step_bytes);
}

// all of one row into shared memory, by the whole block
template <bool BF16>
MDLC_DEV void x_own(const W4Args& a, int row, int steps, uint8_t* xs) {
  const int units = a.d.k / 8;
  constexpr int N = kW4Warps * 32;
  for (int u0 = threadIdx.x; u0 < 16 * steps; u0 += 2 * N) {  // two loads at a time
    const int u1 = u0 + N;
    uint4 r0[2], r1[2];
    x_load<BF16>(a, row, u0, u0 < units, r0);
    x_load<BF16>(a, row, u1, u1 < units, r1);
    x_unit<BF16>(a, r0, u0, 0, xs + u0 / 16 * a.step_bytes);
    if (u1 < 16 * steps) x_unit<BF16>(a, r1, u1, 0, xs + u1 / 16 * a.step_bytes);
  }
}

// a run of bytes (16-byte aligned, a multiple of 16) into shared memory, completing on an mbarrier
MDLC_DEV void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// NT: 8-column tiles; R: 16-row tiles; GROUP: columns of a group; ZEROS: zero points given
template <int NT, int R>
constexpr int w4_min_blocks() { return NT * R <= 3 ? 2 : 1; }

template <int NT, int R, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kW4Warps * 32, w4_min_blocks<NT, R>()) gemv_w4_kernel(const W4Args a) {
  pdl_wait();
  pdl_trigger();
  constexpr int kRing = kW4Warps * 32 * kW4Depth * R * 2 * 16;
  extern __shared__ __align__(128) unsigned char w4_smem[];  // at 16 mod 128 the whole kernel is 15% slower
  // weights on their way: a thread reads back only what it copied itself, so no barrier is needed
  const uint32_t ring = smem_u32(w4_smem) + threadIdx.x * 16;
  const mdlc_w4_desc& d = a.d;
  const int pitch = a.pitch, x_bytes = a.span * a.step_bytes;
  uint8_t* xs = w4_smem + kRing;
  float* red = reinterpret_cast<float*>(xs + a.buffers * x_bytes);
  __shared__ __align__(8) uint64_t x_bar[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.y * a.rows_per_chunk, mc = min(a.rows_per_chunk, d.m - m0);
  constexpr bool G128 = GROUP == 128;
  const int groups = d.k / GROUP, half = d.k / 2;
  const int steps = (d.k + 127) / 128, tiles = (d.n + 16 * R - 1) / (16 * R);

  // This block's tiles are blockIdx.x, + gridDim.x, ...; the warp's steps of all of them form one line, along which
  // weights (kW4Depth - 1 steps) and scales (one step) are fetched ahead, past the end of a tile too.
  // rows past n repeat the last one and are not stored
  auto row_of = [&](int tile, int r, int h) { return (long long)min(tile * 16 * R + r * 16 + h * 8 + g, d.n - 1); };
  int w_tile = blockIdx.x, w_step = warp;
  const uint8_t* wp[R][2];
  auto enter = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long row = row_of(w_tile, r, h);
        wp[r][h] = a.codes + row * half + 16 * t;
        // the row's first scales, which are fetched one step ahead only
        if (w_tile < tiles) asm volatile("prefetch.global.L1 [%0];" ::"l"(a.scales + row * groups));
      }
  };
  auto load = [&](uint32_t dst) {
    if (w_tile < tiles && (G128 ? w_step < steps : w_step * 128 + 32 * t < d.k)) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (MDLC_CHECK_IDX(a.err, wp[r][h] + (uint32_t)w_step * 64 + 15 - a.codes, (long long)d.n * half)) cp_async_16_all(dst + (r * 2 + h) * (kW4Warps * 32 * 16), wp[r][h] + (uint32_t)w_step * 64);
    }
    cp_async_commit();
    w_step += kW4Warps;
    if (w_step >= steps) {
      w_tile += gridDim.x;
      w_step = warp;
      enter();
    }
  };
  // scales and zero points of a step's groups (past k: 0, for columns whose x is 0)
  constexpr int SETS = 128 / GROUP;
  uint32_t sc[SETS][R][2] = {}, sc_next[SETS][R][2] = {}, zr[SETS][R][2] = {}, zr_next[SETS][R][2] = {};
  int s_tile = blockIdx.x, s_step = warp;
  const uint16_t* sp[R][2];
  const uint8_t* zp[R][2];
  auto enter_scales = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long at = row_of(s_tile, r, h) * groups;
        sp[r][h] = a.scales + at;
        if (ZEROS) zp[r][h] = a.zeros + at;
      }
  };
  auto load_scales = [&]() {
    if (s_tile < tiles && s_step < steps) {
#pragma unroll
      for (int i = 0; i < SETS; ++i) {
        const int grp = s_step * SETS + i;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!MDLC_CHECK_IDX(a.err, sp[r][h] - a.scales + min(grp, groups - 1), (long long)d.n * groups)) continue;
            sc_next[i][r][h] = G128 || grp < groups ? __ldg(sp[r][h] + grp) : 0;
            if (ZEROS) zr_next[i][r][h] = G128 || grp < groups ? __ldg(zp[r][h] + grp) : 0;
          }
      }
    }
    s_step += kW4Warps;
    if (s_step >= steps) {
      s_tile += gridDim.x;
      s_step = warp;
      enter_scales();
    }
  };
  constexpr uint32_t kSlot = R * 2 * kW4Warps * 32 * 16;  // bytes of a step in the ring
  enter();
#pragma unroll
  for (int i = 0; i < kW4Depth - 1; ++i) load(ring + i * kSlot);
  enter_scales();
  load_scales();
  // where this thread's four units of a step lie (column tile j: 128 bytes on)
  uint32_t x_off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x_off[i] = 16 * x_place(G128 ? 4 * t + i : 4 * i + t, pitch == 4 ? g & 3 : g, pitch);
  const uint32_t xs_addr = smem_u32(xs);

  // x: one buffer for all of it, or two that the spans of every tile take in turn, the next one on its way
  const int spans = (steps + a.span - 1) / a.span;
  int q = 0;  // spans begun
  auto fetch_x = [&](int which) {
    const int sp = which % spans, n = min(a.span, steps - sp * a.span);
    const uint32_t bar = smem_u32(&x_bar[which & 1]), bytes = (uint32_t)n * a.step_bytes;
    mbar_arrive_expect_tx(bar, bytes);
    bulk_load(xs_addr + (which & 1) * x_bytes, a.ready + ((long long)blockIdx.y * steps + sp * a.span) * a.step_bytes, bytes, bar);
  };
  if (a.ready) {
    if (threadIdx.x == 0) {
      mbar_init(smem_u32(&x_bar[0]), 1);
      mbar_init(smem_u32(&x_bar[1]), 1);
      fence_mbar_init();
      fetch_x(0);
    }
  } else if (d.x_type == MDLC_BF16) {
    x_own<true>(a, m0, steps, xs);
  } else {
    x_own<false>(a, m0, steps, xs);
  }
  __syncthreads();

  uint32_t slot = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    float2 out[R][NT][2] = {};
    for (int s0 = 0; s0 < steps; s0 += a.span) {
      if (a.ready && (spans > 1 || q == 0)) {
        const bool ok = mbar_wait(smem_u32(&x_bar[q & 1]), (q >> 1) & 1, nullptr, a.err, 2 * kWaitLimitNs);
        if (!__syncthreads_and(ok)) {  // every warp is done with the other buffer
          cp_async_wait_all();
          return;
        }
        if (spans > 1 && threadIdx.x == 0 && (s0 + a.span < steps || tile + (int)gridDim.x < tiles)) fetch_x(q + 1);
        ++q;
      }
      const uint8_t* buf = xs + (spans > 1 ? (q - 1) & 1 : 0) * x_bytes;
      const int s1 = min(steps, s0 + a.span);
      for (int s = s0 + ((warp - s0) & (kW4Warps - 1)); s < s1; s += kW4Warps) {  // step s is warp s % 8's
#pragma unroll
        for (int i = 0; i < SETS; ++i)
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              sc[i][r][h] = sc_next[i][r][h];
              zr[i][r][h] = zr_next[i][r][h];
            }
        load(ring + ((slot + kW4Depth - 1) % kW4Depth) * kSlot);
        load_scales();
        cp_async_wait<kW4Depth - 1>();
        uint32_t w[R][2][4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 v = *reinterpret_cast<const uint4*>(w4_smem + threadIdx.x * 16 + slot * kSlot + (r * 2 + h) * (kW4Warps * 32 * 16));
            w[r][h][0] = v.x; w[r][h][1] = v.y; w[r][h][2] = v.z; w[r][h][3] = v.w;
            if constexpr (!G128) quad_transpose(w[r][h], t);
          }
        slot = (slot + 1) % kW4Depth;
        const uint8_t* x_at = buf + (s - s0) * a.step_bytes;
        float acc[R][NT][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // word i holds columns 32 t + 8 i of this step (G128) or, after the exchange, 32 i + 8 t
          const bool first = G128 ? i == 0 : 32 * i % GROUP == 0, last = G128 ? i == 3 : 32 * (i + 1) % GROUP == 0;
          const int set = G128 ? 0 : 32 * i / GROUP;
          if (first) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][j][e] = 0.0f;
          }
          // columns without an x row read what lies there (a single row's are read several times): their sums are not used
          uint4 b[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j) b[j] = *reinterpret_cast<const uint4*>(x_at + x_off[i] + 128 * j);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            uint32_t c[4][2];  // columns n and n + 4 of the word, rows g and g + 8
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t zero = ZEROS ? kCode0 + (zr[set][r][h] & 15u) * 0x00010001u : kCode0 + 0x00080008u;
#pragma unroll
              for (int n = 0; n < 4; ++n) c[n][h] = code_pair(w[r][h][i] >> (4 * n), zero);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_bf16(acc[r][j], c[0][0], c[0][1], c[1][0], c[1][1], b[j].x, b[j].y);
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_bf16(acc[r][j], c[2][0], c[2][1], c[3][0], c[3][1], b[j].z, b[j].w);
          }
          if (last) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float2 scale = splat2(__uint_as_float(sc[set][r][h] << 16));
#pragma unroll
                for (int j = 0; j < NT; ++j) out[r][j][h] = fma2(scale, make_float2(acc[r][j][2 * h], acc[r][j][2 * h + 1]), out[r][j][h]);
              }
          }
        }
      }
    }

    // sums of the parts and of the warps: eight neighbouring threads per output, a warp's sums each, added in a fixed tree
    constexpr int RP = 8 * NT + 2, ROWS = 16 * R;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) *reinterpret_cast<float2*>(red + (warp * ROWS + r * 16 + h * 8 + g) * RP + 8 * j + 2 * t) = out[r][j][h];
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * mc * kW4Warps; i += kW4Warps * 32) {
      const int w = i % kW4Warps, o = i / kW4Warps % ROWS, xr = i / (kW4Warps * ROWS), n = tile * ROWS + o;
      const float* p = red + (w * ROWS + o) * RP + xr * a.parts;
      // the small parts first; they do not change an infinity (an infinite scale may have made them 0 x inf)
      float v = a.parts == 1 || isinf(p[0]) ? p[0] : (p[2] + p[1]) + p[0];
#pragma unroll
      for (int x = 1; x < kW4Warps; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
      if (w == 0 && n < d.n) {
        v *= kCodeUnit;
        if (a.bias) v += __ldg(a.bias + n);
        const long long at = (long long)(m0 + xr) * d.y_stride + n;
        if (!MDLC_CHECK_IDX(a.err, m0 + xr, d.m)) continue;
        if (d.y_type == MDLC_BF16) static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
        else static_cast<float*>(a.y)[at] = v;
      }
    }
    __syncthreads();
  }
  cp_async_wait_all();
}

// shared memory, blocks and rounds of one configuration
struct W4Plan {
  int span, buffers, smem, blocks, tiles;  // span 0: does not fit
  int rounds() const { return (tiles + blocks - 1) / blocks; }
};
template <int NT, int R>
W4Plan w4_plan(const W4Args& a, int num_sms) {
  W4Plan p = {};
  const int steps = (a.d.k + 127) / 128, rest = kW4Warps * 32 * kW4Depth * R * 2 * 16 + kW4Warps * 16 * R * (8 * NT + 2) * 4;
  p.tiles = (a.d.n + 16 * R - 1) / (16 * R);
  // per_sm blocks on an SM: all of x where it fits beside the rest, else two buffers of a whole number of the warps' rounds
  auto fit = [&](int per_sm) {
    W4Plan q = p;
    const int room = 226 * 1024 / per_sm - 1024 - rest;
    if ((long long)steps * a.step_bytes <= room) {
      q.span = steps;
      q.buffers = 1;
    } else {
      q.span = a.ready_wanted ? max(0, room) / 2 / a.step_bytes : 0;
      if (q.span > kW4Warps) q.span -= q.span % kW4Warps;  // whole rounds of the warps, where there is room for one
      q.buffers = 2;
    }
    q.smem = rest + q.buffers * q.span * a.step_bytes;
    q.blocks = num_sms * per_sm;
    return q;
  };
  const W4Plan one = fit(1);
  if (w4_min_blocks<NT, R>() < 2) return one;
  const W4Plan two = fit(2);
  // two buffers read x again for every tile: worth two blocks on an SM only where that is little beside the weights
  const bool little = two.buffers == 1 || (double)p.tiles * steps * a.step_bytes <= 0.5 * a.d.n * a.d.k;
  return two.span && (!one.span || (little && two.rounds() < one.rounds())) ? two : one;
}

template <int NT, int R>
cudaError_t launch_w4(mdlc_ctx* ctx, W4Args& a, const W4Plan& p) {
  a.span = p.span;
  a.buffers = p.buffers;
  const dim3 grid(min(p.tiles, p.blocks), (a.d.m + a.rows_per_chunk - 1) / a.rows_per_chunk);
  static SmemLimit seen[6];
  auto go = [&](int which, auto* kern) {
    const cudaError_t e = allow_smem(seen[which], ctx->device, kern, p.smem);
    return e != cudaSuccess ? e : launch_pdl(kern, grid, dim3(kW4Warps * 32), p.smem, ctx->stream, a);
  };
  if (a.d.group == 128) return a.zeros ? go(0, gemv_w4_kernel<NT, R, 128, true>) : go(1, gemv_w4_kernel<NT, R, 128, false>);
  if (a.d.group == 64) return a.zeros ? go(2, gemv_w4_kernel<NT, R, 64, true>) : go(3, gemv_w4_kernel<NT, R, 64, false>);
  if constexpr (R == 1) return a.zeros ? go(4, gemv_w4_kernel<NT, R, 32, true>) : go(5, gemv_w4_kernel<NT, R, 32, false>);
  return cudaErrorInvalidValue;  // groups of 32 take one row tile
}

template <int NT>
cudaError_t launch_w4_cols(mdlc_ctx* ctx, W4Args& a) {
  a.parts = a.d.x_type == MDLC_BF16 ? 1 : 3;
  a.rows_per_chunk = 8 * NT / a.parts;
  a.pitch = a.d.m == 1 ? (a.parts == 1 ? 1 : 4) : 8 * NT;
  a.step_bytes = 256 * a.pitch;
  const long long steps = ((long long)a.d.k + 127) / 128;
  const bool ready = a.ready_wanted = a.d.m > 1 || a.d.k > kW4OwnColumns;
  // several rows: one kernel splits them for all blocks, as many chunks of rows at a time as the context's workspace holds
  const long long fit = (long long)kSplitWsBytes / (steps * a.step_bytes);
  if (ready && fit == 0) return cudaErrorNotSupported;
  const int m = a.d.m, batch = ready ? (int)min((long long)m, fit * a.rows_per_chunk) : m;
  const W4Plan one = w4_plan<NT, 1>(a, ctx->num_sms), two = w4_plan<NT, 2>(a, ctx->num_sms);
  // Two row tiles share a read of x: a round of them takes less than two of single ones. The fewer and fuller
  // rounds win (one row of 65536 x 8192: 7 rounds of two tiles 68 us, 14 of one 80; 24 rows of 28672 x 4096: 78 and 98; 4096 outputs: one round
  // either way), but for groups of 32, whose scales take the registers of a second tile (one row of 14336 x 4096: two tiles 33 us, one 27;
  // 8 rows of 4096 x 14336: 36 and 33).
  const bool pair = a.d.group > 32 && two.span && (!one.span || 3 * two.rounds() < 2 * one.rounds());
  for (int m0 = 0; m0 < m; m0 += batch) {
    W4Args b = a;
    b.d.m = min(batch, m - m0);
    b.x = static_cast<const char*>(a.x) + (long long)m0 * a.d.x_stride * (a.d.x_type == MDLC_BF16 ? 2 : 4);
    b.y = static_cast<char*>(a.y) + (long long)m0 * a.d.y_stride * (a.d.y_type == MDLC_BF16 ? 2 : 4);
    if (ready) {
      uint8_t* parts = reinterpret_cast<uint8_t*>(ctx->d_split_ws);
      mdlc_note_launch(ctx);
      const dim3 grid((unsigned)((steps * 16 + 127) / 128), b.d.m);
      const cudaError_t e = a.parts == 1 ? launch_pdl(w4_parts_kernel<true>, grid, dim3(128), 0, ctx->stream, b, parts)
                                         : launch_pdl(w4_parts_kernel<false>, grid, dim3(128), 0, ctx->stream, b, parts);
      if (e != cudaSuccess) return e;
      b.ready = parts;
    }
    mdlc_note_launch(ctx);
    const cudaError_t e = pair ? launch_w4<NT, 2>(ctx, b, two) : launch_w4<NT, 1>(ctx, b, one);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t launch_w4_rows(mdlc_ctx* ctx, W4Args& a) {
  // Up to six column tiles at once: 48 bf16 rows, 16 fp32 rows. Fewer where the parts of one chunk would not fit the workspace.
  const long long steps = ((long long)a.d.k + 127) / 128;
  const int parts = a.d.x_type == MDLC_BF16 ? 1 : 3;
  int nt = (int)min(6ll, ((long long)parts * a.d.m + 7) / 8);
  nt = (int)min((long long)nt, max(1ll, (long long)kSplitWsBytes / (steps * 256 * 8)));
  if (nt == 5) nt = 6 * steps * 256 * 8 <= (long long)kSplitWsBytes ? 6 : 4;
  switch (nt) {
    case 1: return launch_w4_cols<1>(ctx, a);
    case 2: return launch_w4_cols<2>(ctx, a);
    case 3: return launch_w4_cols<3>(ctx, a);
    case 4: return launch_w4_cols<4>(ctx, a);
    default: return launch_w4_cols<6>(ctx, a);
  }
}

}  // namespace
}  // namespace mdlc

using namespace mdlc;

extern "C" int mdlc_gemv_w4(mdlc_ctx* ctx, const mdlc_w4_desc* d, const void* x, const uint8_t* codes, const void* scales,
                            const uint8_t* zeros, const float* bias, void* y) {
  if (!ctx) return MDLC_ERR_INVALID;
  if (!d || !x || !codes || !scales || !y) return mdlc_set_error(ctx, MDLC_ERR_INVALID, "gemv_w4: null argument");
  if (d->m < 1 || d->n < 1 || d->k < 1 || (d->group != 32 && d->group != 64 && d->group != 128) || d->k % d->group)
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "gemv_w4: bad sizes (m %d, n %d, k %d, group %d)", d->m, d->n, d->k, d->group);
  if ((d->x_type != MDLC_BF16 && d->x_type != MDLC_F32) || (d->y_type != MDLC_BF16 && d->y_type != MDLC_F32))
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "gemv_w4: types must be bf16 or fp32");
  if (d->x_stride < d->k || d->y_stride < d->n || d->x_stride % 8)
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "gemv_w4: bad strides (x %lld, y %lld)", (long long)d->x_stride, (long long)d->y_stride);
  if ((uintptr_t)x % 16 || (uintptr_t)codes % 16 || (uintptr_t)scales % 2 || (uintptr_t)bias % 4 ||
      (uintptr_t)y % (d->y_type == MDLC_BF16 ? 2 : 4))
    return mdlc_set_error(ctx, MDLC_ERR_INVALID, "gemv_w4: misaligned pointer");
  if (d->m > 65535) return mdlc_set_error(ctx, MDLC_ERR_UNSUPPORTED, "gemv_w4: %d rows (at most 65535)", d->m);
  cudaSetDevice(ctx->device);
  W4Args a = {*d, x, codes, static_cast<const uint16_t*>(scales), zeros, bias, y, 0, 0, 0, 0, 0, 0, nullptr, false, ctx->d_err};
  const cudaError_t e = launch_w4_rows(ctx, a);
  if (e == cudaErrorNotSupported) return mdlc_set_error(ctx, MDLC_ERR_UNSUPPORTED, "gemv_w4: k = %d does not fit the workspace", d->k);
  return mdlc_cuda_status(ctx, e, "gemv_w4 launch");
}
