// Quantizers to block-scaled e4m3: rows in blocks of 128 columns (activations) and weights in blocks of
// 128 x 128. A block's scale is s = max(amax |x| / 448, 2^-100) in fp32 (IEEE division), its codes are
// e4m3(x / s), the exact quotient rounded once to nearest even. Columns past K up to K_pad, the next
// multiple of 128, get code 0. A block that holds a NaN or an infinity gets scale NaN and codes 0.
#include "f8_common.h"

namespace {

// 16 lanes of 8 columns hold a block; a workgroup takes 16 U consecutive blocks in row-major order, all of its loads
// out before the first is used. HBM-bound: two thirds of the bytes are read, one third written (8192 x 8192 bf16: 43.8 us,
// 4.6 TB/s; a device copy of torch's 5.5). The codes are stored as usual: the product reads them next.
template <int DT, int U>
__global__ __launch_bounds__(256) void quant_rows_kernel(const void* __restrict__ x, int64_t sx, uint32_t blocks,
                                                         int64_t K, FastDiv nbd, uint8_t* __restrict__ q, int64_t sq,
                                                         float* __restrict__ sc, int64_t ssm, int64_t ssb) {
  const int part = threadIdx.x & 15;
  F8Raw<DT> raw[U];
  int64_t m[U], b[U];
  bool in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t id = (blockIdx.x * U + u) * 16 + (threadIdx.x >> 4);
    in[u] = id < blocks;
    m[u] = div_fast(in[u] ? id : blocks - 1, nbd);
    b[u] = (in[u] ? id : blocks - 1) - m[u] * nbd.d;
    raw[u] = f8_load8<DT>(x, m[u] * sx, b[u] * F8_BLOCK + part * 8, K);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float s = f8_scale(f8_amax_f32<DT>(row_max16(f8_amax<DT>(raw[u]))));
    const float r = 1.f / s;
    float v[8];
    f8_values<DT>(raw[u], v);
    u32x2_t w;
    w[0] = f8_codes4(v, s, r);
    w[1] = f8_codes4(v + 4, s, r);
    if (!in[u]) continue;
    *(u32x2_t*)(q + m[u] * sq + b[u] * F8_BLOCK + part * 8) = w;
    if (part == 0) sc[m[u] * ssm + b[u] * ssb] = s;
  }
}

// A workgroup per 128 x 128 block: 16 lanes of 8 columns per row, 16 rows at a time, the block's 64 values a
// thread held in registers between the maximum and the division. HBM-bound, with the quotients' arithmetic (about 12
// operations a value) at two thirds of that time: 28672 x 4096 bf16 65.6 us, 5.4 TB/s. The codes of a load-time
// conversion are not read soon, so they are stored past the caches (69.7 us without).
template <int DT>
__global__ __launch_bounds__(256) void pack_f8_kernel(const void* __restrict__ W, int64_t swe, int64_t sw, int64_t N,
                                                      int64_t K, int64_t mb, int64_t nb, uint8_t* __restrict__ q,
                                                      float* __restrict__ sc) {
  __shared__ uint32_t most[4];
  const int64_t id = blockIdx.x, en = id / nb, b = id - en * nb, e = en / mb, nblk = en - e * mb;
  const int part = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int64_t k = b * F8_BLOCK + part * 8;
  F8Raw<DT> raw[8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = nblk * F8_BLOCK + i * 16 + r0;
    raw[i] = f8_load8<DT>(W, e * swe + (n < N ? n : N - 1) * sw, k, n < N ? K : 0);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = f8_amax<DT>(raw[i]);
    m = a > m ? a : m;
  }
  m = row_max16(m);
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    const uint32_t a = (uint32_t)__shfl_xor((int)m, o, 64);
    m = a > m ? a : m;
  }
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(most[0], most[1]), max(most[2], most[3]));
  const float s = f8_scale(f8_amax_f32<DT>(m));
  const float r = 1.f / s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = nblk * F8_BLOCK + i * 16 + r0;
    float v[8];
    f8_values<DT>(raw[i], v);
    u32x2_t w;
    w[0] = f8_codes4(v, s, r);
    w[1] = f8_codes4(v + 4, s, r);
    if (n < N) __builtin_nontemporal_store(w, (u32x2_t*)(q + ((e * N + n) * nb + b) * F8_BLOCK + part * 8));
  }
  if (threadIdx.x == 0) sc[id] = s;
}

bool float_type(int dt) { return dt == IMQ_DT_BF16 || dt == IMQ_DT_FP16 || dt == IMQ_DT_FP32; }

}  // namespace

namespace imq {

int quant_rows_f8(const void* x, int64_t sx, int dt, int64_t M, int64_t K, uint8_t* q, int64_t sq, float* sc, int64_t ssm,
                  int64_t ssk, hipStream_t st) {
  const int64_t nb = imq_cdiv(K, F8_BLOCK);
  if (M > 0x7fffffff / nb) return IMQ_ERR_UNSUPPORTED;
  const int64_t blocks = M * nb;
  // two blocks a lane group where that still leaves eight workgroups a CU (8192 x 8192: 43.8 us, one
  // 45.3, four 44.7; 2048 x 14336: 19.5, 19.5, 20.8)
  const int U = blocks >= 32 * 8 * (int64_t)device_info().cus ? 2 : 1;
  const dim3 grid((unsigned)imq_cdiv(blocks, 16 * U));
  const FastDiv nbd = fast_div((uint32_t)nb);
#define IMQ_GO(DT)                                                                                                       \
  do {                                                                                                                   \
    if (U == 2) quant_rows_kernel<DT, 2><<<grid, dim3(256), 0, st>>>(x, sx, (uint32_t)blocks, K, nbd, q, sq, sc, ssm, ssk); \
    else quant_rows_kernel<DT, 1><<<grid, dim3(256), 0, st>>>(x, sx, (uint32_t)blocks, K, nbd, q, sq, sc, ssm, ssk);        \
  } while (0)
  if (dt == IMQ_DT_BF16) IMQ_GO(IMQ_DT_BF16);
  else if (dt == IMQ_DT_FP16) IMQ_GO(IMQ_DT_FP16);
  else IMQ_GO(IMQ_DT_FP32);
#undef IMQ_GO
  IMQ_LAUNCH_CHECK();
  return IMQ_OK;
}

}  // namespace imq

extern "C" int imq_quant_f8(const void* x, int64_t x_row_stride, int x_dtype, int64_t M, int64_t K, void* q,
                            int64_t q_row_stride, void* scale, int64_t s_stride_m, int64_t s_stride_b, void* stream) {
  if (M < 0 || K < 1 || !float_type(x_dtype)) return IMQ_ERR_INVALID;
  if (M == 0) return IMQ_OK;
  const int64_t kp = imq_cdiv(K, F8_BLOCK) * F8_BLOCK;
  if (!x || !q || !scale || x_row_stride < (M > 1 ? K : 0) || q_row_stride < kp) return IMQ_ERR_INVALID;
  if (((uintptr_t)q & 7) || (q_row_stride & 7) || ((uintptr_t)scale & 3)) return IMQ_ERR_ALIGN;
  return imq::quant_rows_f8(x, x_row_stride, x_dtype, M, K, (uint8_t*)q, q_row_stride, (float*)scale, s_stride_m,
                            s_stride_b, (hipStream_t)stream);
}

extern "C" int imq_pack_f8(const void* W, int64_t w_stride_e, int64_t w_row_stride, int w_dtype, int64_t E, int64_t N,
                           int64_t K, void* qweight, void* scale, void* stream) {
  if (E < 0 || N < 0 || K < 1 || !float_type(w_dtype)) return IMQ_ERR_INVALID;
  if (E == 0 || N == 0) return IMQ_OK;
  if (!W || !qweight || !scale || w_row_stride < (N > 1 ? K : 0) || w_stride_e < 0) return IMQ_ERR_INVALID;
  if (((uintptr_t)qweight & 7) || ((uintptr_t)scale & 3)) return IMQ_ERR_ALIGN;
  const int64_t nb = imq_cdiv(K, F8_BLOCK), mb = imq_cdiv(N, F8_BLOCK);
  const int64_t lim = 0x7fffffff;
  if (mb > lim || nb > lim / mb || E > lim / (mb * nb)) return IMQ_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)(E * mb * nb));
  hipStream_t st = (hipStream_t)stream;
#define IMQ_GO(DT) \
  pack_f8_kernel<DT><<<grid, dim3(256), 0, st>>>(W, w_stride_e, w_row_stride, N, K, mb, nb, (uint8_t*)qweight, (float*)scale)
  if (w_dtype == IMQ_DT_BF16) IMQ_GO(IMQ_DT_BF16);
  else if (w_dtype == IMQ_DT_FP16) IMQ_GO(IMQ_DT_FP16);
  else IMQ_GO(IMQ_DT_FP32);
#undef IMQ_GO
  IMQ_LAUNCH_CHECK();
  return IMQ_OK;
}
