// mdlc_gemv_w4: products of a few rows with 4-bit weights and group scales.
//
// Memory-bound: half a byte of weight per 2 m operations. At the copy bandwidth an SM receives 48
// weights a clock, so what decides, besides bytes in flight, is how many instructions a weight
// costs. The products therefore run on the int8 tensor pipe (mma.sync m16n8k32, exact int32 sums), where
// eight codes need three integer operations and one product:
//   * the weights are the 16-row operand. Code - 8 of the high nibbles of a word is
//     (w & 0xf0f0f0f0) ^ 0x80808080, read as four signed bytes 16 (code - 8); the low nibbles likewise
//     after one shift. (As bf16 operands they took 11 operations, two of them per pair of
//     codes, and the kernel was bound by the integer pipe: 79 us at one row of 65536 x 8192 where this
//     one takes 56 us, 4.9 TB/s.)
//   * x is written once as fixed-point numbers of 23 bits, a power of two per row and 128 columns
//     (the largest magnitude just below 2^22), cut into three balanced signed base-256 digits, each a
//     column of the 8-column operand. The error is at most 2^-23 of the largest |x| of those columns: what an fp32 product
//     with that element would round.
//   * a group's int32 sums (below 2^21) start from the bits of 1.5 x 2^23, so they are fp32 numbers as they
//     stand; they are scaled and added to the row's fp32 sum once per group. A zero point z other
//     than 8 adds (8 - z) times the digits' sum.
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
constexpr int kW4OwnX = 41 * 1024;  // x that a block turns into digits itself (one row) at most
constexpr uint32_t kMagic = 0x4b400000u;  // 1.5 x 2^23: adding an integer below 2^22 to the bits adds it to the number

struct W4Args {
  mdlc_w4_desc d;
  const void* x;
  const uint8_t* codes;
  const uint16_t* scales;  // bf16 bits
  const uint8_t* zeros;
  const float* bias;
  void* y;
  int rows_per_chunk;   // x rows of one grid.y chunk
  int pitch;            // columns kept per 8 of k
  int step_bytes;       // x of one step, see w4_step_bytes
  int span, buffers;    // steps in shared memory at a time, and their buffers
  const uint8_t* ready; // x as digits, [chunk][step], or null: the block makes them itself
  bool ready_wanted;
  int* err;
};

// 16-byte copy to shared memory, always whole
MDLC_DEV void cp_async_16_all(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

MDLC_DEV void mma_s8(uint32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the high nibble of each byte as a signed byte 16 (code - 8)
MDLC_DEV uint32_t high_codes(uint32_t w) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(v) : "r"(w), "r"(0xf0f0f0f0u), "r"(0x80808080u));  // (a & b) ^ c
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

// x as digits, one 128-column step of k after the other, each: 16 units of 8 columns x pitch columns x 8 bytes (the digits of
// columns 0, 2, 4, 6 and 1, 3, 5, 7; units and columns permuted so that the four units a warp reads at once,
// 4 apart or adjacent, lie in different banks); the columns' weights / 256 (fp32); per group of the weights the digits' sums (fp32)
MDLC_DEV int x_place(int unit, int col, int pitch) {
  const int v = unit ^ ((unit >> 2) & 3);
  return v * pitch + (pitch == 4 ? col : col ^ ((v & 2) << 1));
}
__host__ __device__ inline int w4_step_bytes(int pitch, int group) { return pitch * (128 + 4 + 128 / group * 4); }

// Eight columns of an x row as digits, by one lane; the 16 lanes of a step (neighbours) share an exponent. u: unit; dst: the
// step that holds it. Every lane of the warp calls this; `ok`: the unit is one of a step's (past k: zeros).
MDLC_DEV void x_digits(const float (&f)[8], int u, int col0, int group, int pitch, uint8_t* dst, bool ok) {
  const int per = group / 8;
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  // |x| < 2^(ex - 126); below 2^-96 the digits get shorter
  const bool finite = top < 0x7f800000u;
  const int ex = max((int)(top >> 23), 30);
  const float up = __uint_as_float((uint32_t)(275 - ex) << 23);  // 2^(148 - ex)
  uint32_t y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    y[e] = (__float_as_uint(fminf(fmaxf(f[e] * up, -4194303.0f), 4194303.0f) + __uint_as_float(kMagic)) - kMagic + 0x808080u) ^ 0x808080u;
  // 1/16 for the weights' factor, and 1/16 that the end restores: no digit's sum overflows where their sum does not
  float down = __uint_as_float((uint32_t)(ex - 29) << 23);  // 2^(ex - 156)
  if (!finite) {
    // infinities become the digit +-1 (the finite columns beside them 0) of an infinite weight, NaN a NaN weight
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (__float_as_uint(f[e]) & 0x7fffffffu) == 0x7f800000u ? (f[e] > 0.0f ? 1u : 0xffu) : 0u;
    down = __uint_as_float(top);
  }
  uint2* units = reinterpret_cast<uint2*>(dst);
  float* xf = reinterpret_cast<float*>(dst + 128 * pitch);
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    const uint32_t two = p | ((4 + p) << 4);
    uint2 b;
    b.x = __byte_perm(__byte_perm(y[0], y[2], two), __byte_perm(y[4], y[6], two), 0x5410);
    b.y = __byte_perm(__byte_perm(y[1], y[3], two), __byte_perm(y[5], y[7], two), 0x5410);
    if (ok) units[x_place(u & 15, col0 + p, pitch)] = b;
    int sum = __dp4a((int)b.x, 0x01010101, __dp4a((int)b.y, 0x01010101, 0));
    for (int o = 1; o < per; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (ok && (u & 15) == 0) xf[col0 + p] = p == 0 ? down : (finite ? down * (p == 1 ? 256.0f : 65536.0f) : 0.0f);
    if (ok && (u & (per - 1)) == 0) xf[(1 + (u & 15) / per) * pitch + col0 + p] = (float)sum;
  }
}
MDLC_DEV void x_load(const W4Args& a, int row, int u, bool ok, float (&f)[8]) {
  uint4 p = make_uint4(0, 0, 0, 0), v = p;
  if (ok) {
    const long long at = (long long)row * a.d.x_stride + u * 8;
    if (a.d.x_type == MDLC_BF16) {
      p = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.x) + at));
    } else {
      p = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(a.x) + at));
      v = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(a.x) + at) + 1);
    }
  }
  if (a.d.x_type == MDLC_BF16) {
    f[0] = bf16_lo(p.x); f[1] = bf16_hi(p.x); f[2] = bf16_lo(p.y); f[3] = bf16_hi(p.y);
    f[4] = bf16_lo(p.z); f[5] = bf16_hi(p.z); f[6] = bf16_lo(p.w); f[7] = bf16_hi(p.w);
  } else {
    f[0] = __uint_as_float(p.x); f[1] = __uint_as_float(p.y); f[2] = __uint_as_float(p.z); f[3] = __uint_as_float(p.w);
    f[4] = __uint_as_float(v.x); f[5] = __uint_as_float(v.y); f[6] = __uint_as_float(v.z); f[7] = __uint_as_float(v.w);
  }
}

// x as digits in global memory, for the blocks of gemv_w4_kernel to copy: a warp per row and 256 columns
__global__ void __launch_bounds__(128) w4_digits_kernel(const W4Args a, uint8_t* ready) {
  pdl_wait();
  pdl_trigger();
  const int units = a.d.k / 8, lane = threadIdx.x & 31, steps = (a.d.k + 127) / 128;
  const int u = (blockIdx.x * 4 + (threadIdx.x >> 5)) * 32 + lane, row = blockIdx.y;
  float f[8];
  x_load(a, row, u, u < units, f);
  const int chunk = row / a.rows_per_chunk;
  uint8_t* dst = ready + ((long long)chunk * steps + min(u / 16, steps - 1)) * a.step_bytes;
  x_digits(f, u, 3 * (row - chunk * a.rows_per_chunk), a.d.group, a.pitch, dst, u < 16 * steps);
}

// a run of bytes (16-byte aligned, a multiple of 16) into shared memory, completing on an mbarrier
MDLC_DEV void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

MDLC_DEV float2 add2(const float2 a, const float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_from(r);
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
        for (int h = 0; h < 2; ++h) cp_async_16_all(dst + (r * 2 + h) * (kW4Warps * 32 * 16), wp[r][h] + (uint32_t)w_step * 64);
    }
    cp_async_commit();
    w_step += kW4Warps;
    if (w_step >= steps) {
      w_tile += gridDim.x;
      w_step = warp;
      enter();
    }
  };
  // scales and zero points of a step's groups (past k: the last group's, for columns whose digits are 0)
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
        const uint32_t grp = G128 ? s_step : min(s_step * SETS + i, groups - 1);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            sc_next[i][r][h] = __ldg(sp[r][h] + grp);
            if (ZEROS) zr_next[i][r][h] = __ldg(zp[r][h] + grp);
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
  // where this thread's four units of a step lie (column tile j: 64 bytes on)
  uint32_t x_off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x_off[i] = 8 * x_place(G128 ? 4 * t + i : 4 * i + t, pitch == 4 ? g & 3 : g, pitch);
  const uint32_t xs_addr = smem_u32(xs), f_off = 128 * pitch + 4 * (pitch == 4 ? (2 * t) & 3 : 2 * t);

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
  } else {
    const int units = d.k / 8;
    for (int u0 = warp * 32; u0 < 16 * steps; u0 += 2 * kW4Warps * 32) {  // two loads at a time
      const int u1 = u0 + kW4Warps * 32 + lane, ua = u0 + lane;
      float fa[8], fb[8];
      x_load(a, m0, ua, ua < units, fa);
      x_load(a, m0, u1, u1 < units, fb);
      x_digits(fa, ua, 0, GROUP, pitch, xs + min(ua / 16, steps - 1) * a.step_bytes, ua < 16 * steps);
      x_digits(fb, u1, 0, GROUP, pitch, xs + min(u1 / 16, steps - 1) * a.step_bytes, u1 < 16 * steps);
    }
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
      for (int s = s0 + warp; s < s1; s += kW4Warps) {
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
        uint32_t acc[R][NT][4];
        float2 part[R][NT][2] = {};  // the step's sums of scaled groups
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // word i holds columns 32 t + 8 i of this step (G128) or, after the exchange, 32 i + 8 t
          const bool first = G128 ? i == 0 : 32 * i % GROUP == 0;
          if (first) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][j][e] = kMagic;
          }
          // columns without an x row read what lies there (a single row's are read twice): their sums are not used
          uint2 b[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j) b[j] = *reinterpret_cast<const uint2*>(x_at + x_off[i] + 64 * j);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const uint32_t a0 = high_codes(w[r][0][i] << 4), a1 = high_codes(w[r][1][i] << 4);
            const uint32_t a2 = high_codes(w[r][0][i]), a3 = high_codes(w[r][1][i]);
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_s8(acc[r][j], a0, a1, a2, a3, b[j].x, b[j].y);
          }
          const bool last = G128 ? i == 3 : 32 * (i + 1) % GROUP == 0;
          if (last) {
            const int set = G128 ? 0 : 32 * i / GROUP;
            const uint8_t* dp = x_at + f_off + (1 + set) * pitch * 4;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              float2 dx = splat2(0.0f);
              if (ZEROS) dx = *reinterpret_cast<const float2*>(dp + 32 * j);
#pragma unroll
              for (int r = 0; r < R; ++r)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  float2 f = splat2(-12582912.0f);
                  if (ZEROS) f = fma2(splat2(__uint_as_float(kMagic + 128u - 16u * (zr[set][r][h] & 15u)) - 12582912.0f), dx, f);
                  f = add2(make_float2(__uint_as_float(acc[r][j][2 * h]), __uint_as_float(acc[r][j][2 * h + 1])), f);
                  part[r][j][h] = fma2(splat2(__uint_as_float(sc[set][r][h] << 16)), f, part[r][j][h]);
                }
            }
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float2 fx = *reinterpret_cast<const float2*>(x_at + f_off + 32 * j);
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) out[r][j][h] = fma2(fx, part[r][j][h], out[r][j][h]);
        }
      }
    }

    // sums of the digits and of the warps: eight neighbouring threads per output, a warp's sums each, added in a fixed tree
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
      const float* p = red + (w * ROWS + o) * RP + xr * 3;
      float v = (p[0] + p[1]) + p[2];  // the small digits first
#pragma unroll
      for (int x = 1; x < kW4Warps; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
      if (w == 0 && n < d.n) {
        v *= 16.0f;
        if (a.bias) v += __ldg(a.bias + n);
        const long long at = (long long)(m0 + xr) * d.y_stride + n;
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
      q.span = a.ready_wanted ? max(0, room) / 2 / a.step_bytes / kW4Warps * kW4Warps : 0;
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
  return a.zeros ? go(4, gemv_w4_kernel<NT, R, 32, true>) : go(5, gemv_w4_kernel<NT, R, 32, false>);
}

template <int NT>
cudaError_t launch_w4_cols(mdlc_ctx* ctx, W4Args& a) {
  a.rows_per_chunk = 8 * NT / 3;
  a.pitch = a.d.m == 1 ? 4 : 8 * NT;
  a.step_bytes = w4_step_bytes(a.pitch, a.d.group);
  const long long steps = ((long long)a.d.k + 127) / 128;
  const bool ready = a.ready_wanted = a.d.m > 1 || steps * a.step_bytes > kW4OwnX;
  // several rows: one kernel makes the digits for all blocks, as many chunks of rows at a time as the context's workspace holds
  const long long fit = (long long)kSplitWsBytes / (steps * a.step_bytes);
  if (ready && fit == 0) return cudaErrorNotSupported;
  const int m = a.d.m, batch = ready ? (int)min((long long)m, fit * a.rows_per_chunk) : m;
  const W4Plan one = w4_plan<NT, 1>(a, ctx->num_sms), two = w4_plan<NT, 2>(a, ctx->num_sms);
  // Two row tiles share a read of x: a round of them takes less than two of single ones. The fewer and fuller
  // rounds win (65536 rows: 7 rounds of two tiles 56 us, 14 of one 66 us; 4096 rows: one round either way).
  const bool pair = two.span && (!one.span || 3 * two.rounds() < 2 * one.rounds());
  for (int m0 = 0; m0 < m; m0 += batch) {
    W4Args b = a;
    b.d.m = min(batch, m - m0);
    b.x = static_cast<const char*>(a.x) + (long long)m0 * a.d.x_stride * (a.d.x_type == MDLC_BF16 ? 2 : 4);
    b.y = static_cast<char*>(a.y) + (long long)m0 * a.d.y_stride * (a.d.y_type == MDLC_BF16 ? 2 : 4);
    if (ready) {
      uint8_t* digits = reinterpret_cast<uint8_t*>(ctx->d_split_ws);
      mdlc_note_launch(ctx);
      const cudaError_t e = launch_pdl(w4_digits_kernel, dim3((unsigned)((steps * 16 + 127) / 128), b.d.m), dim3(128), 0, ctx->stream, b, digits);
      if (e != cudaSuccess) return e;
      b.ready = digits;
    }
    mdlc_note_launch(ctx);
    const cudaError_t e = pair ? launch_w4<NT, 2>(ctx, b, two) : launch_w4<NT, 1>(ctx, b, one);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t launch_w4_rows(mdlc_ctx* ctx, W4Args& a) {
  // Three columns per row, up to 16 rows in six column tiles at once. (Fewer tiles at once would let all of x stay in shared memory, but
  // read the weights again: 16 rows of 14336 x 4096 in six tiles 40 us, in three, twice, 53 us.)
  const int need = (int)min(6ll, (3ll * a.d.m + 7) / 8), nt = need == 5 ? 6 : need;
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
  W4Args a = {*d, x, codes, static_cast<const uint16_t*>(scales), zeros, bias, y, 0, 0, 0, 0, 0, nullptr, false, ctx->d_err};
  const cudaError_t e = launch_w4_rows(ctx, a);
  if (e == cudaErrorNotSupported) return mdlc_set_error(ctx, MDLC_ERR_UNSUPPORTED, "gemv_w4: k = %d does not fit the workspace", d->k);
  return mdlc_cuda_status(ctx, e, "gemv_w4 launch");
}
