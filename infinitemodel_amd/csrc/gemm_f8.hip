// imq_linear_f8: y = x W^T of block-scaled e4m3 operands (f8_tile.h), x quantized first if it is not handed over
// quantized.
#include "f8_gemv.h"
#include "f8_tile.h"

namespace imq {
int quant_rows_f8(const void* x, int64_t sx, int dt, int64_t M, int64_t K, uint8_t* q, int64_t sq, float* sc, int64_t ssm,
                  int64_t ssk, hipStream_t st);
}

namespace {

// Sum of the K ranges' fp32 partials in range order, rounded once to bf16: 4 columns a thread where the rows are whole
// quads.
__global__ __launch_bounds__(256) void f8_sum_kernel(const float* __restrict__ part, int splits, int64_t M, int64_t N,
                                                     FastDiv quads, uint16_t* __restrict__ y, int64_t sy, bool vec) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= M * quads.d) return;
  const int64_t m = div_fast((uint32_t)id, quads), n = (id - m * quads.d) * 4;
  float v[4] = {};
  for (int s = 0; s < splits; ++s) {
    const float* p = part + (s * M + m) * N + n;
    if (vec) {
      const f32x4_t d = *(const f32x4_t*)p;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += d[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += n + i < N ? p[i] : 0.f;
    }
  }
  uint16_t* o = y + m * sy + n;
  if (vec) {
    *(u32x2_t*)o = u32x2_t{cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < N) o[i] = (uint16_t)f32_to_bf16_bits(v[i]);
  }
}

// The tiles a call may run in, and what they take: with one tile on a CU a step of 128 columns costs `one` us, with two
// at once both together `two` (0: one workgroup fills the CU); `base` is the time before the first and after the last
// step. Measured on M 24 .. 4096, N 1024 .. 28672, K 2048 .. 14336 with weights in the caches; the model below orders
// the tiles as the measurements do in 13 of 15 shapes and is never over 8% off the best of them. Large tiles move the
// fewest bytes a product (4096^3 from memory: 256 x 256 71, 128 x 128 81, 64 x 64 129 us), small ones fill the CUs (512 x
// 4096 -> 4096: 256 x 256 55, 128 x 128 30, 64 x 64 18 us).
struct TileCost {
  int bn, bm;
  float one, two, base;
};
constexpr TileCost kTiles[] = {
    {256, 256, 1.65f, 0.f, 9.f}, {128, 128, 0.7f, 0.96f, 6.f}, {128, 64, 0.43f, 0.58f, 5.f}, {64, 64, 0.27f, 0.38f, 4.5f}, {64, 32, 0.22f, 0.3f, 4.f}};

// How a call runs, by its sizes alone. waves > 0: the few-row kernel, x quantized inside it (inside), copied quantized to
// LDS by workgroups of several tiles (copy) or read quantized by those of one; else tile kTiles[tile], the K in `splits` ranges.
struct Plan {
  int waves = 0;
  bool inside = false, copy = false;
  int tile = 0, splits = 1;
};

Plan plan_of(int64_t M, int64_t N, int64_t nb, bool given, const DevInfo& d) {
  Plan p;
  if (M <= 16) {
    p.waves = nb >= 48 ? 16 : nb >= 12 ? 8 : 4;
    p.inside = !given && M * nb <= 128 && f8_gemv_lds(p.waves, 0, false, M, nb) <= d.max_lds;
    p.copy = !p.inside && N > 32 * d.cus && f8_gemv_lds(16, 0, false, M, nb) <= d.max_lds;
    if (p.copy) p.waves = 16;
    return p;
  }
  const int64_t quads = M * imq_cdiv(N, 4);              // threads of the launch that sums K ranges
  double best = 0;
  for (int i = 0; i < (int)(sizeof(kTiles) / sizeof(kTiles[0])); ++i) {
    const TileCost& c = kTiles[i];
    const int64_t tiles = imq_cdiv(M, c.bm) * imq_cdiv(N, c.bn);
    for (int s = 1; s <= 8 && (s == 1 || (nb >= 4 * s && quads <= 0x7fffffff)); ++s) {
      const int64_t on = imq_cdiv(tiles * s, d.cus);      // tiles on the fullest CU
      double us = c.base + (double)imq_cdiv(nb, s) * (c.two > 0.f ? (double)(on / 2) * c.two + (on & 1) * c.one : on * c.one);
      // the fp32 partials, written and read at 4.5 TB/s, and the launch that sums them
      if (s > 1) us += 2.5 + (double)s * M * N * 8 / 4.5e6;
      if (best == 0 || us < best) {
        best = us;
        p.tile = i;
        p.splits = s;
      }
    }
  }
  return p;
}

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

template <int BN, int BM, int WN, int WM, int S>
int go(const F8Tile& a, int cus, hipStream_t st) {
  constexpr int lds = f8_tile_lds(BN, BM, WN * WM, S, 0);
  constexpr auto kern = f8_tile_kernel<BN, BM, WN, WM, S, 0>;
  if (const hipError_t e = f8_allow_lds<kern>(lds); e != hipSuccess) return (int)e;
  kern<<<dim3((unsigned)f8_tile_grid((int64_t)a.mt * a.nt * a.splits, WN * WM, S, lds, cus)), dim3(64 * WN * WM), lds, st>>>(a);
  IMQ_LAUNCH_CHECK();
  return IMQ_OK;
}

template <int W, bool XG>
int go_gemv(const F8Gemv& a, int64_t grid, hipStream_t st) {
  const int64_t lds = f8_gemv_lds(W, 0, XG, a.M, a.nb);
  constexpr auto kern = f8_gemv_kernel<W, 0, XG>;
  if (const hipError_t e = f8_allow_lds<kern>(lds); e != hipSuccess) return (int)e;
  kern<<<dim3((unsigned)grid), dim3(64 * W), (size_t)lds, st>>>(a);
  IMQ_LAUNCH_CHECK();
  return IMQ_OK;
}

bool float_type(int dt) { return dt == IMQ_DT_BF16 || dt == IMQ_DT_FP16 || dt == IMQ_DT_FP32; }

}  // namespace

namespace imq {

// imq_launch_plan's answer for imq_linear_f8.
void linear_f8_plan_query(int64_t M, int64_t N, int64_t K_pad, bool given, int cus, int max_lds, int64_t* out) {
  const int64_t nb = K_pad / F8_BLOCK;
  const Plan p = plan_of(M, N, nb, given, DevInfo{cus, max_lds});
  const TileCost& t = kTiles[p.tile];
  constexpr int lds[] = {f8_tile_lds(256, 256, 8, 2, 0), f8_tile_lds(128, 128, 4, 2, 0), f8_tile_lds(128, 64, 4, 3, 0),
                         f8_tile_lds(64, 64, 4, 4, 0), f8_tile_lds(64, 32, 2, 5, 0)};
  out[0] = 1;
  out[1] = p.waves > 0 ? 0 : t.bn;
  out[2] = p.waves > 0 ? p.waves : t.bm;
  out[3] = p.waves > 0 ? (p.inside ? 1 : p.copy ? 2 : 0) : p.splits;
  out[4] = p.waves > 0 ? f8_gemv_lds(p.waves, 0, !p.inside && !p.copy, M, nb) : lds[p.tile];
}

}  // namespace imq

extern "C" int64_t imq_linear_f8_workspace_bytes(int64_t M, int64_t N, int64_t K_pad, int x_dtype) {
  if (M < 0 || N < 0 || K_pad < 0 || K_pad % F8_BLOCK || !(float_type(x_dtype) || x_dtype == IMQ_DT_F8)) return -1;
  if (M == 0 || N == 0 || K_pad == 0) return 0;
  if (M > 0x7fffffff || N > 0x7fffffff || K_pad > 0x7fffffff) return -1;
  const Plan p = plan_of(M, N, K_pad / F8_BLOCK, x_dtype == IMQ_DT_F8, device_info());
  int64_t b = p.splits > 1 ? up256((int64_t)p.splits * M * N * 4) : 0;
  if (x_dtype != IMQ_DT_F8 && !p.inside) b += up256(M * K_pad) + up256(M * (K_pad / F8_BLOCK) * 4);
  return b;
}

extern "C" int imq_linear_f8(const void* x, int64_t x_row_stride, int x_dtype, int64_t M, int64_t K, const float* x_scale,
                             int64_t xs_stride_m, int64_t xs_stride_b, const void* qweight, int64_t q_row_stride,
                             const float* scale, int64_t s_stride_r, int64_t s_stride_b, int64_t N, int64_t K_pad, void* y,
                             int64_t y_row_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  const bool given = x_dtype == IMQ_DT_F8;
  if (M < 0 || N < 0 || K < 1 || K > K_pad || K_pad % F8_BLOCK || K_pad - K >= F8_BLOCK || !(given || float_type(x_dtype)))
    return IMQ_ERR_INVALID;
  if (M == 0 || N == 0) return IMQ_OK;
  if (!x || !qweight || !scale || !y || (given && !x_scale) || workspace_bytes < 0) return IMQ_ERR_INVALID;
  if (x_row_stride < (M > 1 ? (given ? K_pad : K) : 0) || q_row_stride < (N > 1 ? K_pad : 0) || y_row_stride < (M > 1 ? N : 0) ||
      (given && K != K_pad))
    return IMQ_ERR_INVALID;
  if (((uintptr_t)qweight & 15) || (q_row_stride & 15) || ((uintptr_t)y & 1) || ((uintptr_t)scale & 3) ||
      (given && (((uintptr_t)x & 15) || (x_row_stride & 15) || ((uintptr_t)x_scale & 3))) || ((uintptr_t)workspace & 15))
    return IMQ_ERR_ALIGN;
  const int64_t lim = 0x7fffffff, nb = K_pad / F8_BLOCK;
  if (M > lim || N > lim || M > lim / 4 / nb || q_row_stride > lim / 257 || K_pad > lim / 257 || (given && x_row_stride > lim / 257))
    return IMQ_ERR_UNSUPPORTED;
  const DevInfo dev = device_info();
  const Plan p = plan_of(M, N, nb, given, dev);
  // the tile kernel takes a row's scales at 32-bit offsets
  if (given && (xs_stride_m < 0 || xs_stride_b < 0 || xs_stride_m > lim / M || xs_stride_b > lim / nb ||
                xs_stride_m * M + xs_stride_b * nb > lim / 4))
    return IMQ_ERR_UNSUPPORTED;
  const TileCost& tc = kTiles[p.tile];
  if (imq_cdiv(M, tc.bm) * imq_cdiv(N, tc.bn) * p.splits > lim) return IMQ_ERR_UNSUPPORTED;
  if (workspace_bytes < imq_linear_f8_workspace_bytes(M, N, K_pad, x_dtype) || (!workspace && ((!given && !p.inside) || p.splits > 1)))
    return IMQ_ERR_SCRATCH;
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  F8Tile a{};
  if (given) {
    a.x = (const uint8_t*)x;
    a.sx = x_row_stride;
    a.xs = x_scale;
    a.xsm = xs_stride_m;
    a.xsb = xs_stride_b;
  } else if (!p.inside) {
    uint8_t* xq = (uint8_t*)ws;
    float* xs = (float*)(ws + up256(M * K_pad));
    ws += up256(M * K_pad) + up256(M * nb * 4);
    const int rc = imq::quant_rows_f8(x, x_row_stride, x_dtype, M, K, xq, K_pad, xs, 1, M, st);
    if (rc != IMQ_OK) return rc;
    a.x = xq;
    a.sx = K_pad;
    a.xs = xs;
    a.xsm = 1;
    a.xsb = M;
  }
  if (p.waves > 0) {
    F8Gemv v{};
    v.x = p.inside ? x : a.x;
    v.sx = p.inside ? x_row_stride : a.sx;
    v.xdt = x_dtype;
    v.xs = a.xs;
    v.xsm = a.xsm;
    v.xsb = a.xsb;
    v.M = (int)M;
    v.K = (int)K;
    v.w = (const uint8_t*)qweight;
    v.sw = q_row_stride;
    v.ws = scale;
    v.wsr = s_stride_r;
    v.wsb = s_stride_b;
    v.N = (int)N;
    v.nb = (int)nb;
    v.tiles = (int)imq_cdiv(N, 16);
    v.y = y;
    v.sy = y_row_stride;
    v.nbd = fast_div((uint32_t)nb);
    const int64_t grid = f8_gemv_grid(v.tiles, (int64_t)dev.cus * (16 / p.waves));
    if (p.inside || p.copy)
      return p.waves == 16 ? go_gemv<16, false>(v, grid, st) : p.waves == 8 ? go_gemv<8, false>(v, grid, st) : go_gemv<4, false>(v, grid, st);
    return p.waves == 16 ? go_gemv<16, true>(v, grid, st) : p.waves == 8 ? go_gemv<8, true>(v, grid, st) : go_gemv<4, true>(v, grid, st);
  }
  a.w = (const uint8_t*)qweight;
  a.sw = q_row_stride;
  a.ws = scale;
  a.wsr = s_stride_r;
  a.wsb = s_stride_b;
  a.M = (int)M;
  a.N = (int)N;
  a.nb = (int)nb;
  a.y = (uint16_t*)y;
  a.sy = y_row_stride;
  a.part = (float*)ws;
  a.splits = p.splits;
  a.mt = (int)imq_cdiv(M, tc.bm);
  a.nt = (int)imq_cdiv(N, tc.bn);
  int rc;
  switch (p.tile) {
    case 0: rc = go<256, 256, 2, 4, 2>(a, dev.cus, st); break;
    case 1: rc = go<128, 128, 2, 2, 2>(a, dev.cus, st); break;
    case 2: rc = go<128, 64, 4, 1, 3>(a, dev.cus, st); break;
    case 3: rc = go<64, 64, 2, 2, 4>(a, dev.cus, st); break;
    default: rc = go<64, 32, 2, 1, 5>(a, dev.cus, st); break;
  }
  if (rc != IMQ_OK || p.splits == 1) return rc;
  const int64_t quads = imq_cdiv(N, 4);
  const bool vec = N % 4 == 0 && y_row_stride % 4 == 0 && ((uintptr_t)y & 7) == 0;
  f8_sum_kernel<<<dim3((unsigned)imq_cdiv(M * quads, 256)), dim3(256), 0, st>>>(a.part, p.splits, M, N, fast_div((uint32_t)quads),
                                                                              (uint16_t*)y, y_row_stride, vec);
  IMQ_LAUNCH_CHECK();
  return IMQ_OK;
}
