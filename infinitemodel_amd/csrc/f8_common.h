// Device helpers of the block-scaled fp8 kernels: e4m3 (1-4-3, finite, largest value 448) codes with one
// fp32 scale per 128 columns of an activation row and per 128 x 128 block of a weight.
#pragma once

#include "imq_common.h"

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int F8_BLOCK = 128;
constexpr float F8_TOP = 448.f;
// The least scale: blocks of zeros (and of values below 448 2^-100) divide by it, and neither the quotient
// nor its remainder leaves the normal range above it.
constexpr float F8_LEAST = 0x1p-100f;

// The scale of a block from the bits of its largest magnitude (NaN > infinity > finite as integers): NaN for
// a block that is not finite, so that every product taken from it is NaN.
IMQ_DEV float f8_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return fmaxf(__uint_as_float(amax_bits) / F8_TOP, F8_LEAST);
}

// v / s, s > 0, r = 1 / s correctly rounded, as an fp32 value that rounds to e4m3 as the exact quotient does:
// one Newton step on |v| gives a faithful quotient q, whose exact remainder says on which side of q the quotient
// lies. Where it is not q itself, q is moved to the next value toward zero if it is too large, and its last bit is set
// (rounding to odd): no e4m3 midpoint (20 zero bits at the end) is met by accident, so the conversion's own
// rounding to nearest even is the only one. Four fma and six integer operations a value, against about ten
// for an IEEE division that would still round twice.
IMQ_DEV float f8_quotient(float v, float s, float r) {
  const float a = fabsf(v);
  float q = a * r;
  q = fmaf(fmaf(-q, s, a), r, q);
  const float rem = fmaf(-q, s, a);
  const uint32_t u = (__float_as_uint(q) + (uint32_t)((int32_t)__float_as_uint(rem) >> 31)) | (rem != 0.f ? 1u : 0u);
  return copysignf(__uint_as_float(u), v);
}

// Four values (fp32) of a block -> four e4m3 codes. s NaN gives codes 0.
IMQ_DEV uint32_t f8_codes4(const float* v, float s, float r) {
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = f8_quotient(v[i], s, r);
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
  return s != s ? 0u : (uint32_t)w;
}

// silu(g) u = g u / (1 + e^-g) to a few steps of fp32, from e = e^-|g|, which cannot overflow: g / (1 + e) where g is positive, g e /
// (1 + e) where it is negative. e by the hardware's exponential of t = -|g| / ln 2, whose rounding (and that of 1 / ln 2)
// is carried on in `lo`; the reciprocal is off by one step. Half the operations of expf and a division, which
// were half of the gate_up tile's epilogue. |g| is cut at 87, so e is a normal number; silu of less than -87, below 2^-119
// in magnitude, is taken as 0. NaN and -inf (infinity times 0) give NaN.
IMQ_DEV float f8_silu_mul(float g, float u) {
  const float a = fabsf(g), m = fminf(a, 87.f), t = m * -1.44269504f;
  const float lo = fmaf(m, -1.92596302e-8f, fmaf(m, -1.44269504f, -t));
  float e = __builtin_amdgcn_exp2f(t);
  e = fmaf(e, lo * 0.693147181f, e);
  const float f = g >= 0.f ? 1.f : a > 87.f ? 0.f : e;
  return g * f * __builtin_amdgcn_rcpf(1.f + e) * u;
}

// 16x16x128: A lane l = row l % 16, B lane l = column l % 16, 32 of the 128 bytes in lanes l / 16; D lane l holds
// column l % 16, rows 4 (l / 16) .. + 3.
IMQ_DEV f32x4_t mfma_f8_16x16x128(i32x8_t a, i32x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

// The same product by the bf16 matrix instructions (every e4m3 value is a bf16 value). The e4m3 instruction cuts the
// products of 8 neighbouring columns off at 2^-13 of the largest among them before it adds them in fp32 (measured: 1.5e-5
// of a 128-column sum of normal values, and the same for every e4m3 shape of the instruction); the bf16 one keeps them
// (1e-8). Half the rate and a conversion of two values per instruction: taken where the result is quantized again. There a sum's
// error decides which code a value near a border gets, a few in ten thousand, and each is off by a whole step: with the e4m3
// instruction in gate and up the experts' result was 2.5e-3 off where its rounding to bf16 is 1.7e-3 (4096 tokens; up to 4.4e-3
// for 40), with this one 1.7e-3.
struct F8Wide {
  bf16x8_t p[4];
};
IMQ_DEV F8Wide f8_widen(i32x8_t a) {
  F8Wide w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u32x4_t r;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int v = a[2 * i + q];
      r[2 * q] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.f, false));
      r[2 * q + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.f, true));
    }
    w.p[i] = __builtin_bit_cast(bf16x8_t, r);
  }
  return w;
}
IMQ_DEV f32x4_t mfma_f8_wide(const F8Wide& a, const F8Wide& b, f32x4_t c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = mfma16x16x32(a.p[i], b.p[i], c);
  return c;
}

IMQ_DEV i32x8_t f8_join(u32x4_t lo, u32x4_t hi) {
  i32x8_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = lo[i], b = hi[i];
    r[i] = (int)a;
    r[4 + i] = (int)b;
  }
  return r;
}

// The largest of 16 lanes' (a DPP row's) integers, in every lane.
IMQ_DEV uint32_t row_max16(uint32_t v) {
  uint32_t o;
  o = dpp_row_ror<8>(v); v = v > o ? v : o;
  o = dpp_row_ror<4>(v); v = v > o ? v : o;
  o = dpp_row_ror<2>(v); v = v > o ? v : o;
  o = dpp_row_ror<1>(v); v = v > o ? v : o;
  return v;
}

// 8 consecutive elements of a row, zero past `end`. Rows may start at any element: the loads ask for no more alignment than
// the elements have.
template <int DT>
struct F8Raw {
  uint32_t d[DT == IMQ_DT_FP32 ? 8 : 4];
};
template <int DT>
IMQ_DEV F8Raw<DT> f8_load8(const void* x, int64_t row, int64_t k, int64_t end) {
  F8Raw<DT> r;
  if (k + 8 <= end) {
    if constexpr (DT == IMQ_DT_FP32) {
      typedef uint32_t v4_t __attribute__((ext_vector_type(4), aligned(4)));
      const v4_t a = *(const v4_t*)((const float*)x + row + k), b = *(const v4_t*)((const float*)x + row + k + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r.d[i] = a[i];
        r.d[4 + i] = b[i];
      }
    } else {
      typedef uint32_t v4_t __attribute__((ext_vector_type(4), aligned(2)));
      const v4_t a = *(const v4_t*)((const uint16_t*)x + row + k);
#pragma unroll
      for (int i = 0; i < 4; ++i) r.d[i] = a[i];
    }
    return r;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t e = k + i < end ? load_raw_bits<DT>(x, row + k + i) : 0;
    if constexpr (DT == IMQ_DT_FP32) r.d[i] = e;
    else r.d[i >> 1] = i & 1 ? r.d[i >> 1] | e << 16 : e;
  }
  return r;
}
template <int DT>
IMQ_DEV void f8_values(const F8Raw<DT>& r, float* v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (DT == IMQ_DT_FP32) v[i] = __uint_as_float(r.d[i]);
    else if constexpr (DT == IMQ_DT_BF16) v[i] = __uint_as_float(i & 1 ? r.d[i >> 1] & 0xffff0000u : r.d[i >> 1] << 16);
    else v[i] = f16_bits_to_f32(i & 1 ? r.d[i >> 1] >> 16 : r.d[i >> 1] & 0xffffu);
  }
}

// The largest magnitude's bits, as integers of the type's own width (two at a time of the 16-bit types); f8_amax_f32 of the
// whole block's gives them as an fp32 value's.
template <int DT>
IMQ_DEV uint32_t f8_amax(const F8Raw<DT>& r) {
  if constexpr (DT == IMQ_DT_FP32) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = r.d[i] & 0x7fffffffu;
      m = a > m ? a : m;
    }
    return m;
  } else {
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    u16x2_t m = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, r.d[i] & 0x7fff7fffu));
    return m[0] > m[1] ? m[0] : m[1];
  }
}
template <int DT>
IMQ_DEV uint32_t f8_amax_f32(uint32_t m) {
  return DT == IMQ_DT_FP32 ? m : DT == IMQ_DT_BF16 ? m << 16 : __float_as_uint(f16_bits_to_f32(m));
}

// A kernel of more than 64 KB of LDS asks for it, once per device.
template <auto KERN>
inline hipError_t f8_allow_lds(int64_t lds) {
  if (lds <= 65536) return hipSuccess;
  static uint64_t done;                  // one bit a device
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit) return hipSuccess;
  const hipError_t e = hipFuncSetAttribute((const void*)KERN, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  if (e == hipSuccess && bit) __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
  return e;
}
