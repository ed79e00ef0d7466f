// imq_moe_experts_f8: one MoE layer's routed experts on block-scaled e4m3 weights.
//   [g | u] = x W_gu^T, h = silu(g) u, y = h W_dn^T, out[t] = sum_j w[t, j] y[t, j],
// x and h quantized by rows in blocks of 128 columns (h from its fp32 values). The routed rows are sorted by expert,
// so that an expert's weights are read once a row tile (f8_tile.h), and combined in routed order: no result
// depends on the order in which workgroups run.
#include <cmath>

#include "f8_gemv.h"
#include "f8_tile.h"

namespace {

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

constexpr int kChunk = 2048;             // routed rows a workgroup counts and places

// A chunk's experts: thread tid holds those of rows b0 + 256 i + tid (-1 past the end); all reads go out before the first is
// waited for.
struct Chunk {
  int b0, at[kChunk / 256];
};
IMQ_DEV Chunk f8_chunk(const void* ids, int is64, int B, int E, int chunk) {
  Chunk c;
  c.b0 = chunk * kChunk;
#pragma unroll
  for (int i = 0; i < kChunk / 256; ++i) {
    const int b = c.b0 + i * 256 + (int)threadIdx.x;
    c.at[i] = b < B ? f8_expert(ids, is64, E, b) : -1;
  }
  return c;
}

// Places a chunk's rows, sorted by expert. lds: [E] rows of the expert over all chunks, [E] those of the chunks before this
// one (then the next place). The first workgroup to call it writes the row tiles of bm rows. The order of an expert's rows
// among themselves is free, as every row's result is its own.
IMQ_DEV void f8_place(const Chunk& c, int E, int bm, int32_t* lds, bool first, int32_t* __restrict__ perm,
                      int32_t* __restrict__ tiles) {
  int32_t *all = lds, *next = lds + E;
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid < 64) {
    const int per = (E + 63) / 64, e0 = tid * per, e1 = e0 + per < E ? e0 + per : E;
    int rows = 0, blks = 0;
    for (int e = e0; e < e1; ++e) {
      rows += all[e];
      blks += (all[e] + bm - 1) / bm;
    }
    int rs = rows, bs = blks;
    for (int d = 1; d < 64; d <<= 1) {
      const int r = __shfl_up(rs, d, 64), q = __shfl_up(bs, d, 64);
      if (tid >= d) {
        rs += r;
        bs += q;
      }
    }
    int run = rs - rows, tile = bs - blks;
    for (int e = e0; e < e1; ++e) {
      const int n = all[e];
      if (first)
        for (int r0 = 0; r0 < n; r0 += bm, ++tile) {
          tiles[1 + 3 * tile] = e;
          tiles[2 + 3 * tile] = run + r0;
          tiles[3 + 3 * tile] = run + (r0 + bm < n ? r0 + bm : n);
        }
      next[e] += run;
      run += n;
    }
    if (tid == 63 && first) tiles[0] = bs;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kChunk / 256; ++i)
    if (c.at[i] >= 0) perm[atomicAdd(&next[c.at[i]], 1)] = c.b0 + i * 256 + tid;
}

// Workgroups [0, chunks) count their rows' experts, the others quantize the hidden rows (16 blocks each, as
// quant_rows_kernel). A single chunk is placed at once; more take f8_place_kernel.
template <int DT>
__global__ __launch_bounds__(256) void f8_count_kernel(const void* __restrict__ ids, int is64, int B, int E, int chunks, int bm,
                                                       int32_t* __restrict__ counts, int32_t* __restrict__ perm,
                                                       int32_t* __restrict__ tiles, const void* __restrict__ x, int64_t sx,
                                                       int64_t blocks, int64_t K, FastDiv nbd,
                                                       uint8_t* __restrict__ q, float* __restrict__ sc, int64_t ssb) {
  extern __shared__ int32_t cnt[];       // [E] counts, [E] zeros of a single chunk
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < chunks) {
    const Chunk c = f8_chunk(ids, is64, B, E, blockIdx.x);
    for (int e = tid; e < E * (chunks == 1 ? 2 : 1); e += 256) cnt[e] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kChunk / 256; ++i)
      if (c.at[i] >= 0) atomicAdd(&cnt[c.at[i]], 1);
    if (chunks == 1) {
      f8_place(c, E, bm, cnt, true, perm, tiles);
      return;
    }
    __syncthreads();
    for (int e = tid; e < E; e += 256) counts[(int64_t)blockIdx.x * E + e] = cnt[e];
    return;
  }
  const int64_t id = (int64_t)(blockIdx.x - chunks) * 16 + (tid >> 4);
  if (id >= blocks) return;
  const int64_t m = div_fast((uint32_t)id, nbd), b = id - m * nbd.d;
  const int64_t k = b * F8_BLOCK + (tid & 15) * 8;
  const F8Raw<DT> raw = f8_load8<DT>(x, m * sx, k, K);
  const float s = f8_scale(f8_amax_f32<DT>(row_max16(f8_amax<DT>(raw))));
  const float r = 1.f / s;
  float v[8];
  f8_values<DT>(raw, v);
  u32x2_t w;
  w[0] = f8_codes4(v, s, r);
  w[1] = f8_codes4(v + 4, s, r);
  *(u32x2_t*)(q + m * nbd.d * F8_BLOCK + k) = w;
  if ((tid & 15) == 0) sc[b * ssb + m] = s;
}

// Several chunks: every workgroup sums the counts and places its own.
__global__ __launch_bounds__(256) void f8_place_kernel(const void* __restrict__ ids, int is64, int B, int E, int chunks, int bm,
                                                       const int32_t* __restrict__ counts, int32_t* __restrict__ perm,
                                                       int32_t* __restrict__ tiles) {
  extern __shared__ int32_t lds[];
  const Chunk c = f8_chunk(ids, is64, B, E, blockIdx.x);
  for (int e = threadIdx.x; e < E; e += 256) {
    int sum = 0, before = 0;
#pragma unroll 8
    for (int q = 0; q < chunks; ++q) {
      if (q == (int)blockIdx.x) before = sum;
      sum += counts[(int64_t)q * E + e];
    }
    lds[e] = sum;
    lds[E + e] = before;
  }
  f8_place(c, E, bm, lds, blockIdx.x == 0, perm, tiles);
}

// out[t] = sum over j, in order, of w[t, j] y[t k + j] in fp32: 8 columns a thread. y: fp32, rows padded to whole eights.
__global__ __launch_bounds__(256) void f8_combine_kernel(const float* __restrict__ y, int64_t sy, const void* __restrict__ w, int wdt,
                                                         int k, int64_t H, FastDiv per, int64_t total, uint16_t* __restrict__ out,
                                                         int64_t so) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int64_t t = div_fast((uint32_t)id, per), n = (id - t * per.d) * 8;
  float v[8] = {};
#pragma unroll 4
  for (int j = 0; j < k; ++j) {
    const int64_t b = t * k + j;
    const float c = f8_weight_at(w, wdt, b);
    const f32x4_t d0 = *(const f32x4_t*)(y + b * sy + n), d1 = *(const f32x4_t*)(y + b * sy + n + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = fmaf(c, d0[i], v[i]);
      v[4 + i] = fmaf(c, d1[i], v[4 + i]);
    }
  }
  uint16_t* o = out + t * so + n;
  if (n + 8 <= H && ((uintptr_t)o & 15) == 0) {
    *(u32x4_t*)o = u32x4_t{cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3]), cvt_pk_bf16(v[4], v[5]), cvt_pk_bf16(v[6], v[7])};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < H) o[i] = (uint16_t)f32_to_bf16_bits(v[i]);
  }
}

// How a call runs, by its sizes alone: direct (each routed row on its own, two launches), or sorted by expert in
// tiles of bm rows (four launches, five of more than 2048 routed rows).
struct Plan {
  bool direct;
  int wg, wd;            // direct: waves of the gate_up and of the down kernel
  int bm;
};

Plan plan_of(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I, const DevInfo& d) {
  const int64_t B = T * k, hb = imq_cdiv(H, F8_BLOCK), ib = imq_cdiv(I, F8_BLOCK), per = B / E;
  Plan p;
  p.wg = hb >= 12 ? 8 : 4;
  p.wd = k * ib >= 32 ? 16 : k * ib >= 12 ? 8 : 4;
  // What the weights take at 5.6 (direct, once per routed row) or 5.2 TB/s (sorted, once per expert that some row goes to, as
  // if all were alike), and the launches: measured on 1 .. 12 tokens of 8 and 64 experts.
  const double w = 3.0 * H * I / 1e6, hit = (double)E * (1.0 - pow(1.0 - (double)(k < E ? k : E) / E, (double)T));
  p.direct = B <= 64 && B * w / 5.6 + 6.0 <= hit * w / 5.2 + 14.0 && f8_gemv_lds(p.wg, 1, false, 1, hb) <= d.max_lds && f8_gemv_lds(p.wd, 2, false, k, ib) <= d.max_lds &&
             (k * ib + 1) * 128 < 0x7fffffff;
  // Rows a tile by the mean rows an expert: short experts leave a tall tile empty, tall tiles read the weights less often. us in
  // tiles of 192 and of 128 rows: 200 rows an expert, 64 experts of 2048 x 1408 362 and 336; 250 rows, 64 of 2048 x 1024 301 and
  // 288, but 8 of 4096 x 1792 134 and 158; 256 rows, 64 of 2048 x 768 243 and 240, 16 of 2048 x 1024 93 and 115; 512 rows, 64
  // of 2048 x 1024 525 and 539. Between 200 and 256 the border follows the larger differences.
  p.bm = per > 224 ? 192 : per > 64 ? 128 : per > 24 ? 64 : 32;
  return p;
}

struct Ws {
  int64_t xq, xs, hq, hs, y, counts, perm, tiles, total, sy;
};

Ws ws_of(const Plan& p, int64_t T, int64_t k, int64_t E, int64_t H, int64_t I) {
  const int64_t B = T * k, hb = imq_cdiv(H, F8_BLOCK), ib = imq_cdiv(I, F8_BLOCK);
  Ws w{};
  if (p.direct) {                        // h in fp32, rows of I padded to 4
    w.total = up256(B * ((I + 3) / 4 * 4) * 4);
    return w;
  }
  w.sy = (H + 7) / 8 * 8;
  w.xq = 0;
  w.xs = w.xq + up256(T * hb * F8_BLOCK);
  w.hq = w.xs + up256(T * hb * 4);
  w.hs = w.hq + up256(B * ib * F8_BLOCK);
  w.y = w.hs + up256(B * ib * 4);
  w.counts = w.y + up256(B * w.sy * 4);
  w.perm = w.counts + up256(imq_cdiv(B, kChunk) * E * 4);
  w.tiles = w.perm + up256(B * 4);
  w.total = w.tiles + up256((1 + 3 * (B / p.bm + (B < E ? B : E))) * 4);
  return w;
}

template <int BN, int BM, int WN, int WM, int S, int MODE>
int go(const F8Tile& a, int64_t tiles, int cus, hipStream_t st) {
  constexpr int lds = f8_tile_lds(BN, BM, WN * WM, S, MODE);
  constexpr auto kern = f8_tile_kernel<BN, BM, WN, WM, S, MODE>;
  if (const hipError_t e = f8_allow_lds<kern>(lds); e != hipSuccess) return (int)e;
  kern<<<dim3((unsigned)f8_tile_grid(tiles * a.nt, WN * WM, S, lds, cus)), dim3(64 * WN * WM), lds, st>>>(a);
  IMQ_LAUNCH_CHECK();
  return IMQ_OK;
}

template <int W, int MODE>
int go_gemv(const F8Gemv& a, int64_t grid, int64_t gy, int64_t rows, hipStream_t st) {
  const int64_t lds = f8_gemv_lds(W, MODE, false, rows, a.nb);
  constexpr auto kern = f8_gemv_kernel<W, MODE, false>;
  if (const hipError_t e = f8_allow_lds<kern>(lds); e != hipSuccess) return (int)e;
  kern<<<dim3((unsigned)grid, (unsigned)gy), dim3(64 * W), (size_t)lds, st>>>(a);
  IMQ_LAUNCH_CHECK();
  return IMQ_OK;
}

bool float_type(int dt) { return dt == IMQ_DT_BF16 || dt == IMQ_DT_FP16 || dt == IMQ_DT_FP32; }
constexpr int64_t kMaxExperts = 4096;

// Sizes whose offsets the kernels can hold in 32 bits; each limit by division, so that no product of sizes overflows.
bool sizes_fit(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I, const DevInfo& dev) {
  const int64_t lim = 0x7fffffff;
  if (E > kMaxExperts || k > lim || T > lim / k || H > lim || I > lim / 2) return false;
  const int64_t hp = imq_cdiv(H, F8_BLOCK) * F8_BLOCK, ip = imq_cdiv(I, F8_BLOCK) * F8_BLOCK, B = T * k;
  if (T > lim / hp || B > lim / ip || 2 * I > lim / hp || H > lim / ip) return false;
  const Plan p = plan_of(T, k, E, H, I, dev);
  const int64_t tiles = B / p.bm + (B < E ? B : E);
  return p.direct || (tiles <= lim / imq_cdiv(H, F8_BLOCK) / 8 && tiles <= lim / imq_cdiv(I, F8_BLOCK) / 8);
}

}  // namespace

namespace imq {

// imq_launch_plan's answer for imq_moe_experts_f8 (LDS: gate_up's).
void moe_f8_plan_query(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I, int cus, int max_lds, int64_t* out) {
  const DevInfo dev{cus, max_lds};
  if (!sizes_fit(T, k, E, H, I, dev)) return;
  const Plan p = plan_of(T, k, E, H, I, dev);
  out[0] = 1;
  out[1] = p.direct ? 0 : p.bm;
  out[2] = p.direct ? p.wg : 0;
  out[3] = p.direct ? p.wd : 0;
  out[4] = p.direct ? f8_gemv_lds(p.wg, 1, false, 1, imq_cdiv(H, F8_BLOCK))
           : p.bm == 192 ? f8_tile_lds(256, 192, 8, 2, 1) : p.bm == 128 ? f8_tile_lds(256, 128, 8, 2, 1)
           : p.bm == 64 ? f8_tile_lds(256, 64, 4, 3, 1) : f8_tile_lds(256, 32, 4, 4, 1);
}

}  // namespace imq

extern "C" int64_t imq_moe_f8_workspace_bytes(int64_t T, int64_t top_k, int64_t E, int64_t H, int64_t I) {
  if (T < 0 || top_k < 1 || E < 1 || H < 1 || I < 1) return -1;
  if (T == 0) return 0;
  const DevInfo dev = device_info();
  return sizes_fit(T, top_k, E, H, I, dev) ? ws_of(plan_of(T, top_k, E, H, I, dev), T, top_k, E, H, I).total : -1;
}

extern "C" int imq_moe_experts_f8(const void* hidden, int64_t h_row_stride, int h_dtype, int64_t T, int64_t H, int64_t top_k,
                                  const void* topk_idx, int idx_dtype, const void* topk_w, int w_dtype, int64_t E,
                                  const void* gu_q, int64_t gu_q_stride_e, int64_t gu_q_row_stride, const float* gu_s,
                                  int64_t gu_s_stride_e, int64_t gu_s_stride_r, int64_t I, const void* dn_q,
                                  int64_t dn_q_stride_e, int64_t dn_q_row_stride, const float* dn_s, int64_t dn_s_stride_e,
                                  int64_t dn_s_stride_r, void* out, int64_t out_row_stride, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (T < 0 || H < 1 || I < 1 || top_k < 1 || E < 1 || !float_type(h_dtype) || !float_type(w_dtype) ||
      (idx_dtype != IMQ_DT_I32 && idx_dtype != IMQ_DT_I64))
    return IMQ_ERR_INVALID;
  if (T == 0) return IMQ_OK;
  if (H > (int64_t)1 << 40 || I > (int64_t)1 << 40) return IMQ_ERR_UNSUPPORTED;
  const int64_t hp = imq_cdiv(H, F8_BLOCK) * F8_BLOCK, ip = imq_cdiv(I, F8_BLOCK) * F8_BLOCK;
  if (!hidden || !topk_idx || !topk_w || !gu_q || !gu_s || !dn_q || !dn_s || !out || h_row_stride < (T > 1 ? H : 0) ||
      out_row_stride < (T > 1 ? H : 0) || gu_q_row_stride < hp || dn_q_row_stride < (H > 1 ? ip : 0))
    return IMQ_ERR_INVALID;
  if (((uintptr_t)gu_q & 15) || (gu_q_row_stride & 15) || (gu_q_stride_e & 15) || ((uintptr_t)dn_q & 15) || (dn_q_row_stride & 15) ||
      (dn_q_stride_e & 15) || ((uintptr_t)gu_s & 3) || ((uintptr_t)dn_s & 3) || ((uintptr_t)out & 1) || ((uintptr_t)workspace & 15))
    return IMQ_ERR_ALIGN;
  const int64_t lim = 0x7fffffff;
  const DevInfo dev = device_info();
  if (!sizes_fit(T, top_k, E, H, I, dev) || 2 * I > lim / gu_q_row_stride ||
      (dn_q_row_stride > 0 && H > lim / dn_q_row_stride))      // one row of down needs no stride
    return IMQ_ERR_UNSUPPORTED;
  const int64_t B = T * top_k;
  const Plan p = plan_of(T, top_k, E, H, I, dev);
  const Ws L = ws_of(p, T, top_k, E, H, I);
  if (!workspace || workspace_bytes < L.total) return IMQ_ERR_SCRATCH;
  char* ws = (char*)workspace;
  hipStream_t st = (hipStream_t)stream;
  const int is64 = idx_dtype == IMQ_DT_I64;
  const int64_t hb = hp / F8_BLOCK, ib = ip / F8_BLOCK;
  int rc;
  if (p.direct) {
    F8Gemv g{};
    g.x = hidden;
    g.sx = h_row_stride;
    g.xdt = h_dtype;
    g.M = 1;
    g.K = (int)H;
    g.w = (const uint8_t*)gu_q;
    g.sw = gu_q_row_stride;
    g.swe = gu_q_stride_e;
    g.ws = gu_s;
    g.wse = gu_s_stride_e;
    g.wsr = gu_s_stride_r;
    g.wsb = 1;
    g.N = (int)I;
    g.nb = (int)hb;
    g.tiles = (int)imq_cdiv(I, 16);
    g.y = ws;
    g.sy = (I + 3) / 4 * 4;
    g.ids = topk_idx;
    g.is64 = is64;
    g.E = (int)E;
    g.k = (int)top_k;
    g.nbd = fast_div((uint32_t)hb);
    const int64_t gg = f8_gemv_grid(g.tiles, imq_cdiv((int64_t)dev.cus * (32 / p.wg), B));
    rc = p.wg == 8 ? go_gemv<8, 1>(g, gg, B, 1, st) : go_gemv<4, 1>(g, gg, B, 1, st);
    if (rc != IMQ_OK) return rc;
    F8Gemv d = g;
    d.x = ws;
    d.sx = g.sy;
    d.xdt = IMQ_DT_FP32;
    d.K = (int)I;
    d.w = (const uint8_t*)dn_q;
    d.sw = dn_q_row_stride;
    d.swe = dn_q_stride_e;
    d.ws = dn_s;
    d.wse = dn_s_stride_e;
    d.wsr = dn_s_stride_r;
    d.N = (int)H;
    d.nb = (int)ib;
    d.tiles = (int)imq_cdiv(H, 16);
    d.y = out;
    d.sy = out_row_stride;
    d.rw = topk_w;
    d.rwdt = w_dtype;
    d.nbd = fast_div((uint32_t)ib);
    const int64_t dg = f8_gemv_grid(d.tiles, imq_cdiv((int64_t)dev.cus * (32 / p.wd), T));
    return p.wd == 16 ? go_gemv<16, 2>(d, dg, T, top_k, st) : p.wd == 8 ? go_gemv<8, 2>(d, dg, T, top_k, st)
                                                                         : go_gemv<4, 2>(d, dg, T, top_k, st);
  }
  const int bm = p.bm;
  const int64_t tiles = B / bm + (B < E ? B : E), blocks = T * hb, chunks = imq_cdiv(B, kChunk);
  uint8_t *xq = (uint8_t*)(ws + L.xq), *hq = (uint8_t*)(ws + L.hq);
  float *xs = (float*)(ws + L.xs), *hs = (float*)(ws + L.hs);
  int32_t *counts = (int32_t*)(ws + L.counts), *perm = (int32_t*)(ws + L.perm), *tl = (int32_t*)(ws + L.tiles);
  const dim3 grid((unsigned)(chunks + imq_cdiv(blocks, 16)));
#define IMQ_GO(DT)                                                                                                     \
  f8_count_kernel<DT><<<grid, dim3(256), (size_t)E * 8, st>>>(topk_idx, is64, (int)B, (int)E, (int)chunks, bm, counts, perm, tl, \
                                                              hidden, h_row_stride, blocks, H, fast_div((uint32_t)hb), xq, xs, T)
  if (h_dtype == IMQ_DT_BF16) IMQ_GO(IMQ_DT_BF16);
  else if (h_dtype == IMQ_DT_FP16) IMQ_GO(IMQ_DT_FP16);
  else IMQ_GO(IMQ_DT_FP32);
#undef IMQ_GO
  IMQ_LAUNCH_CHECK();
  if (chunks > 1) {
    f8_place_kernel<<<dim3((unsigned)chunks), dim3(256), (size_t)E * 8, st>>>(topk_idx, is64, (int)B, (int)E, (int)chunks, bm, counts,
                                                                            perm, tl);
    IMQ_LAUNCH_CHECK();
  }
  F8Tile g{};
  g.x = xq;
  g.sx = hp;
  g.xs = xs;
  g.xsm = 1;
  g.xsb = T;
  g.w = (const uint8_t*)gu_q;
  g.sw = gu_q_row_stride;
  g.swe = gu_q_stride_e;
  g.ws = gu_s;
  g.wse = gu_s_stride_e;
  g.wsr = gu_s_stride_r;
  g.wsb = 1;
  g.N = (int)I;
  g.nb = (int)(hp / F8_BLOCK);
  g.splits = 1;
  g.tiles = tl;
  g.perm = perm;
  g.kd = fast_div((uint32_t)top_k);
  g.I = (int)I;
  g.h = hq;
  g.sh = ip;
  g.hs = hs;
  g.hsb = B;
  g.nt = (int)ib;
  rc = bm == 192 ? go<256, 192, 2, 4, 2, 1>(g, tiles, dev.cus, st) : bm == 128 ? go<256, 128, 2, 4, 2, 1>(g, tiles, dev.cus, st)
       : bm == 64 ? go<256, 64, 4, 1, 3, 1>(g, tiles, dev.cus, st) : go<256, 32, 4, 1, 4, 1>(g, tiles, dev.cus, st);
  if (rc != IMQ_OK) return rc;
  F8Tile d{};
  d.x = hq;
  d.sx = ip;
  d.xs = hs;
  d.xsm = 1;
  d.xsb = B;
  d.w = (const uint8_t*)dn_q;
  d.sw = dn_q_row_stride;
  d.swe = dn_q_stride_e;
  d.ws = dn_s;
  d.wse = dn_s_stride_e;
  d.wsr = dn_s_stride_r;
  d.wsb = 1;
  d.N = (int)H;
  d.nb = (int)(ip / F8_BLOCK);
  d.splits = 1;
  d.tiles = tl;
  d.perm = perm;
  d.rows = (float*)(ws + L.y);
  d.sy = L.sy;
  d.nt = (int)imq_cdiv(H, bm == 192 ? 256 : 128);
  rc = bm == 192 ? go<256, 192, 2, 4, 2, 2>(d, tiles, dev.cus, st) : bm == 128 ? go<128, 128, 2, 2, 2, 2>(d, tiles, dev.cus, st)
       : bm == 64 ? go<128, 64, 4, 1, 3, 2>(d, tiles, dev.cus, st) : go<128, 32, 4, 1, 3, 2>(d, tiles, dev.cus, st);
  if (rc != IMQ_OK) return rc;
  const int64_t cols = imq_cdiv(H, 8), total = T * cols;
  f8_combine_kernel<<<dim3((unsigned)imq_cdiv(total, 256)), dim3(256), 0, st>>>(
      d.rows, d.sy, topk_w, w_dtype, (int)top_k, H, fast_div((uint32_t)cols), total, (uint16_t*)out, out_row_stride);
  IMQ_LAUNCH_CHECK();
  return IMQ_OK;
}
