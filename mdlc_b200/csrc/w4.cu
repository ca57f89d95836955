// mdlc_gemv_w4: products of a few rows with 4-bit weights and group scales.
//
// Memory-bound: half a byte of weight per 2 m operations, so the kernel has to (1) keep
// enough weight bytes in flight and (2) spend few instructions per weight. At the
// copy bandwidth an SM receives about 48 weights a clock; one multiply-add and
// one conversion per weight on the fp32 lanes would already fill them. So the
// products run on the tensor pipe, m16n8k16 bf16 with fp32 sums: the weights are the
// 16-row operand, the x rows the 8 columns, and a code costs one and-or and
// one paired subtract per two weights:
//   * a code q becomes bf16 128 + q by or-ing it into the mantissa of 128
//     (0x4300 | q: steps of one at 128), two at a time: nibbles s and s + 4 of a
//     word land in the two halves of (w >> 4s) & 0x000f000f;
//   * minus (128 + zero) is exact, so the products are those of the integers;
//   * the scale multiplies the fp32 sum of a group once.
// The order of the columns inside a product is free as long as both operands agree,
// so a thread simply keeps the 32 consecutive codes of its 16-byte load and
// takes its x values in the same order. For groups under 128 columns the four threads
// of a row hold different groups; a 4 x 4 exchange of words inside the quad then
// puts 32 consecutive columns, one group, into each pair of products.
// An fp32 x is cut into three bf16 parts of 8 bits each (exact), one column each.
//
// A block owns 16 R output columns; its 8 warps take 128-column steps of k in turn
// (adjacent warps read adjacent bytes of a row) and add their sums in warp order
// through shared memory, so results do not depend on timing.
#include "common.cuh"
#include "runtime.h"

namespace mdlc {
namespace {

constexpr int kW4Warps = 8;

struct W4Args {
  mdlc_w4_desc d;
  const void* x;
  const uint8_t* codes;
  const __nv_bfloat16* scales;
  const uint8_t* zeros;
  const float* bias;
  void* y;
  int rows_per_chunk;  // x rows of one grid.y chunk
};

MDLC_DEV uint4 ldg_stream(const void* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

MDLC_DEV void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// nibbles s and s + 4 of w as bf16 (code - zero); zp: bf16 pair of 128 + zero
MDLC_DEV uint32_t dequant(uint32_t w, int s, uint32_t zp) {
  uint32_t v, r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w >> (4 * s)), "r"(0x000f000fu), "r"(0x43004300u));  // (a & b) | c
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(zp));
  return r;
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

// eight consecutive x values of one column as four bf16 pairs (s, s + 4)
MDLC_DEV void x_pairs(const __nv_bfloat16* x, int, bool ok, uint32_t (&p)[4]) {
  const uint4 v = ok ? __ldg(reinterpret_cast<const uint4*>(x)) : make_uint4(0, 0, 0, 0);
  p[0] = __byte_perm(v.x, v.z, 0x5410);
  p[1] = __byte_perm(v.x, v.z, 0x7632);
  p[2] = __byte_perm(v.y, v.w, 0x5410);
  p[3] = __byte_perm(v.y, v.w, 0x7632);
}
// the fp32 form: `part` 0, 1, 2 of x's 24 bits, eight each; truncation, so that no part
// overflows; an infinity has no further parts
MDLC_DEV float rest_of(float v) {
  const float head = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
  return head == v ? 0.0f : v - head;
}
MDLC_DEV void x_pairs(const float* x, int part, bool ok, uint32_t (&p)[4]) {
  float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (ok) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(x)), b = __ldg(reinterpret_cast<const float4*>(x) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float r1 = rest_of(f[i]), r2 = rest_of(r1);
    f[i] = part == 0 ? f[i] : (part == 1 ? r1 : r2);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) p[s] = __byte_perm(__float_as_uint(f[s]), __float_as_uint(f[s + 4]), 0x7632);
}

// XT: x's type; NT: 8-column tiles; R: 16-row tiles; G128: groups of 128 columns
template <typename XT, int NT, int R, bool G128>
__global__ void __launch_bounds__(kW4Warps * 32) gemv_w4_kernel(const W4Args a) {
  pdl_wait();
  pdl_trigger();
  constexpr int kParts = sizeof(XT) == 4 ? 3 : 1;
  constexpr int kCols = 8 * NT;
  __shared__ float red[kW4Warps][16 * R][kCols + 1];
  const mdlc_w4_desc& d = a.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16 * R;
  const int m0 = blockIdx.y * a.rows_per_chunk, mc = min(a.rows_per_chunk, d.m - m0);
  const int groups = d.k / d.group, half = d.k / 2;
  const int steps = (d.k + 127) / 128;

  // rows past n repeat the last one and are not stored
  const uint8_t* wp[R][2];
  int row[R][2];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      row[r][h] = min(n0 + r * 16 + h * 8 + g, d.n - 1);
      wp[r][h] = a.codes + (long long)row[r][h] * half + 16 * t;
    }
  const XT* xp[NT];
  int part[NT];
  bool xok[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int c = 8 * j + g, i = c / kParts;
    part[j] = c % kParts;
    xok[j] = i < mc;
    xp[j] = static_cast<const XT*>(a.x) + (long long)(m0 + (xok[j] ? i : 0)) * d.x_stride;
  }

  float out[R][NT][4] = {};
  uint4 cur[R][2], nxt[R][2];
  auto load = [&](int s, uint4 (&w)[R][2]) {
    const bool ok = s < steps && s * 128 + 32 * t < d.k;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) w[r][h] = ok ? ldg_stream(wp[r][h] + s * 64) : make_uint4(0, 0, 0, 0);
  };
  load(warp, cur);
  for (int s = warp; s < steps; s += kW4Warps) {
    load(s + kW4Warps, nxt);
    uint32_t w[R][2][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        w[r][h][0] = cur[r][h].x; w[r][h][1] = cur[r][h].y; w[r][h][2] = cur[r][h].z; w[r][h][3] = cur[r][h].w;
        if constexpr (!G128) quad_transpose(w[r][h], t);
      }
    float acc[R][NT][4] = {};
    float sc[R][2];
    uint32_t zp[R][2];
    auto scales_of = [&](int grp) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const long long at = (long long)row[r][h] * groups + grp;
          sc[r][h] = __bfloat162float(a.scales[at]);
          zp[r][h] = (0x4300u | (a.zeros ? (uint32_t)__ldg(a.zeros + at) & 15u : 8u)) * 0x10001u;
        }
    };
    auto flush = [&]() {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            out[r][j][e] = fmaf(sc[r][e >> 1], acc[r][j][e], out[r][j][e]);
            acc[r][j][e] = 0.0f;
          }
    };
    if constexpr (G128) scales_of(s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // columns of word i: G128: 32 t + 8 i of this step; else, after the exchange, 32 i + 8 t
      const int col = s * 128 + (G128 ? 32 * t + 8 * i : 32 * i + 8 * t);
      if constexpr (!G128) {
        if (s * 128 + 32 * i >= d.k) break;
        scales_of((s * 128 + 32 * i) / d.group);
      }
      uint32_t b[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) x_pairs(xp[j] + col, part[j], xok[j], b[j]);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          const uint32_t a0 = dequant(w[r][0][i], q, zp[r][0]), a1 = dequant(w[r][1][i], q, zp[r][1]);
          const uint32_t a2 = dequant(w[r][0][i], q + 1, zp[r][0]), a3 = dequant(w[r][1][i], q + 1, zp[r][1]);
#pragma unroll
          for (int j = 0; j < NT; ++j) mma_bf16(acc[r][j], a0, a1, a2, a3, b[j][q], b[j][q + 1]);
        }
      if constexpr (!G128) flush();
    }
    if constexpr (G128) flush();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      cur[r][0] = nxt[r][0];
      cur[r][1] = nxt[r][1];
    }
  }

  // sums of the warps, in warp order
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[warp][r * 16 + (e >> 1) * 8 + g][8 * j + 2 * t + (e & 1)] = out[r][j][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * R * mc; i += kW4Warps * 32) {
    const int o = i % (16 * R), xr = i / (16 * R);
    if (n0 + o >= d.n) continue;
    float v = 0.0f;
#pragma unroll
    for (int p = kParts - 1; p >= 0; --p)  // the small parts first
#pragma unroll
      for (int w = 0; w < kW4Warps; ++w) v += red[w][o][xr * kParts + p];
    if (a.bias) v += __ldg(a.bias + n0 + o);
    const long long at = (long long)(m0 + xr) * d.y_stride + n0 + o;
    if (d.y_type == MDLC_BF16) static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
    else static_cast<float*>(a.y)[at] = v;
  }
}

template <typename XT, int NT, int R>
cudaError_t launch_w4(mdlc_ctx* ctx, const W4Args& a) {
  const dim3 grid((a.d.n + 16 * R - 1) / (16 * R), (a.d.m + a.rows_per_chunk - 1) / a.rows_per_chunk);
  return a.d.group == 128 ? launch_pdl(gemv_w4_kernel<XT, NT, R, true>, grid, dim3(kW4Warps * 32), 0, ctx->stream, a)
                          : launch_pdl(gemv_w4_kernel<XT, NT, R, false>, grid, dim3(kW4Warps * 32), 0, ctx->stream, a);
}

template <typename XT>
cudaError_t launch_w4_rows(mdlc_ctx* ctx, W4Args& a) {
  constexpr int kParts = sizeof(XT) == 4 ? 3 : 1;
  const int cols = min(32, a.d.m * kParts);
  const int nt = cols <= 8 ? 1 : (cols <= 16 ? 2 : 4);
  a.rows_per_chunk = 8 * nt / kParts;
  // two row tiles share x's loads where that still leaves two blocks per SM
  const bool two = a.d.n >= 32 * 2 * ctx->num_sms;
  if (nt == 1) return two ? launch_w4<XT, 1, 2>(ctx, a) : launch_w4<XT, 1, 1>(ctx, a);
  if (nt == 2) return two ? launch_w4<XT, 2, 2>(ctx, a) : launch_w4<XT, 2, 1>(ctx, a);
  return two ? launch_w4<XT, 4, 2>(ctx, a) : launch_w4<XT, 4, 1>(ctx, a);
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
  W4Args a = {*d, x, codes, static_cast<const __nv_bfloat16*>(scales), zeros, bias, y, 0};
  const cudaError_t e = d->x_type == MDLC_BF16 ? launch_w4_rows<__nv_bfloat16>(ctx, a) : launch_w4_rows<float>(ctx, a);
  mdlc_note_launch(ctx);
  return mdlc_cuda_status(ctx, e, "gemv_w4 launch");
}
