// Device helpers that the 8-bit cache's kernels share (k_kv8.cu,
// k_kv8_prompt.cu).
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "kv8.h"

namespace grx {

namespace {

constexpr uint32_t FULL = 0xffffffffu;
constexpr int kSMs = 148;
constexpr int kRangeError = -5;  // GRX_ERANGE, what the status word gets

enum { ROPE_NONE = 0, ROPE_PAIRS = 1, ROPE_HALVES = 2 };

__device__ __forceinline__ void report(const Kv8Args& a) {
  if (a.status) *a.status = kRangeError;
}

__device__ __forceinline__ float wide(float x) { return x; }
__device__ __forceinline__ float wide(__half h) { return __half2float(h); }
__device__ __forceinline__ float wide(__nv_bfloat16 h) { return __bfloat162float(h); }
// A lane's values 64j + 16·tg + e of a row of float32 (type 0), float16 (1)
// or bfloat16 (2), zeros where there is no row; `vec` where the address of
// four is a multiple of their size together. All loads go out before the
// first value is used: with a choice of the type around each four they came
// one after the other, 2.5 µs for a row of 128.
template <int D>
__device__ __forceinline__ void load_row(const void* p, int64_t off, int type, bool vec, bool there, float (&x)[D / 64][16]) {
  constexpr int H2 = D / 64;
  if (!there) {
#pragma unroll
    for (int j = 0; j < H2; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) x[j][e] = 0.f;
  } else if (type == 0) {
    const float* f = static_cast<const float*>(p) + off;
    if (vec) {
#pragma unroll
      for (int j = 0; j < H2; j++)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 v = *reinterpret_cast<const float4*>(f + 64 * j + e);
          x[j][e] = v.x, x[j][e + 1] = v.y, x[j][e + 2] = v.z, x[j][e + 3] = v.w;
        }
    } else {
#pragma unroll
      for (int j = 0; j < H2; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) x[j][e] = f[64 * j + e];
    }
  } else {
    const uint16_t* h = static_cast<const uint16_t*>(p) + off;
    uint32_t w[H2][8];
    if (vec) {
#pragma unroll
      for (int j = 0; j < H2; j++)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(h + 64 * j + 2 * e);
          w[j][e] = v.x, w[j][e + 1] = v.y;
        }
    } else {
#pragma unroll
      for (int j = 0; j < H2; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) w[j][e] = h[64 * j + 2 * e] | uint32_t(h[64 * j + 2 * e + 1]) << 16;
    }
#pragma unroll
    for (int j = 0; j < H2; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const uint32_t v = w[j][e / 2];
        x[j][e] = type == 1 ? __half2float(__ushort_as_half(uint16_t(e & 1 ? v >> 16 : v)))
                            : __uint_as_float(e & 1 ? v & 0xffff0000u : v << 16);
      }
  }
}

__device__ __forceinline__ float ninf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float qnan() { return __int_as_float(0x7fc00000); }
// A page's scales of keys and values, both NaN where one is not finite or the
// values' is below 0: then a query that sees the page has a sum, and with it
// an output and a log-sum-exp, that are no numbers.
__device__ __forceinline__ float2 sound_scales(float2 s) {
  const bool sound = isfinite(s.x) && isfinite(s.y) && s.y >= 0.f;
  return sound ? s : make_float2(qnan(), qnan());
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Weights are counted in units of a power of two W = 2^(e − 127), kept as its
// exponent field e: of the number `most` (not below 0), within the range in
// which W, 1/W and 2^11/W are normal numbers.
__device__ __forceinline__ int unit_of(float most) { return min(max(int(__float_as_uint(most) >> 23), 12), 253); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(uint32_t(e) << 23); }  // 2^(e − 127)
// 1/x of a unit of weights: powers of two for two float16s a weight, exact; for
// one any number (the largest weight itself is then exact), off by 2^-23.
template <int NP>
__device__ __forceinline__ float inverse(float x) {
  if (NP == 2) return __uint_as_float((254u << 23) - __float_as_uint(x));
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^11/W for weights as NP float16s, W being about `most`, the largest weight:
// that itself for one (which is then exact, as it is where it comes again), the
// power of two below it for two (whose sums then move exactly). *slack: log2 of
// 2^4·W, where W moves again.
template <int NP>
__device__ __forceinline__ float weight_scale(float most, float* slack) {
  const float W = fminf(fmaxf(most, 0x1p-115f), 0x1p126f);
  *slack = __fadd_rn(lg2(W), 4.f);
  return NP == 1 ? __fmul_rn(2048.f, inverse<1>(W)) : pow2(265 - unit_of(W));
}
// Two floats as float16s, lo in the low half.
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
// Values 16·tg .. 16·tg + 15 of each 64 of a query at the position `pos`,
// rotated, by four lanes together.
template <int D>
__device__ __forceinline__ void rotate16(float (&x)[D / 64][16], const Kv8Args& a, int pos, int tg) {
  constexpr int H2 = D / 64;
  if (a.rope_mode == ROPE_NONE) return;
  // a slot that holds nothing has no position; its scores are not used
  const float2* cs = reinterpret_cast<const float2*>(a.rope) + int64_t(max(pos, 0)) * (D / 2);
  if (a.rope_mode == ROPE_PAIRS) {
#pragma unroll
    for (int j = 0; j < H2; j++)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float2 f = cs[(64 * j + 16 * tg + e) / 2];
        const float p = x[j][e], q = x[j][e + 1];
        x[j][e] = __fmaf_rn(p, f.x, -__fmul_rn(q, f.y));
        x[j][e + 1] = __fmaf_rn(p, f.y, __fmul_rn(q, f.x));
      }
  } else if (D == 64) {
    // the partner is 32 values on: two lanes away
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const float o = __shfl_xor_sync(FULL, x[0][e], 2);
      const float2 f = cs[(16 * tg + e) & 31];
      x[0][e] = __fmaf_rn(x[0][e], f.x, tg < 2 ? -__fmul_rn(o, f.y) : __fmul_rn(o, f.y));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const float2 f = cs[16 * tg + e];
      const float p = x[0][e], q = x[H2 - 1][e];
      x[0][e] = __fmaf_rn(p, f.x, -__fmul_rn(q, f.y));
      x[H2 - 1][e] = __fmaf_rn(p, f.y, __fmul_rn(q, f.x));
    }
  }
}

constexpr float kQueryUnits = 4194304.f;  // a query's largest value

// The largest magnitude of the values that four lanes hold, NaN where one is
// not finite. `lanes`: those that take part.
template <int D>
__device__ __forceinline__ float group_amax(const float (&x)[D / 64][16], uint32_t lanes) {
  float m = 0.f, nan = 0.f;
#pragma unroll
  for (int j = 0; j < D / 64; j++)
#pragma unroll
    for (int e = 0; e < 16; e++) {
      m = fmaxf(m, fabsf(x[j][e]));
      nan = __fmaf_rn(0.f, x[j][e], nan);  // 0·inf and 0·NaN
    }
  m = __fadd_rn(m, nan);
  const float a = __shfl_xor_sync(lanes, m, 1);
  m = m > a || isnan(m) ? m : a;
  const float b = __shfl_xor_sync(lanes, m, 2);
  return m > b || isnan(m) ? m : b;
}
// The factor that makes the largest value kQueryUnits (0 for rows of zeros
// or of no numbers); tiny rows are lifted first, so that it stays in range.
template <int D>
__device__ __forceinline__ float lift_row(float (&x)[D / 64][16], float amax) {
  if (amax < 1e-30f) {
    amax = __fmul_rn(amax, 1e30f);
#pragma unroll
    for (int j = 0; j < D / 64; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) x[j][e] = __fmul_rn(x[j][e], 1e30f);
  }
  return amax > 0.f ? __fdiv_rn(kQueryUnits, amax) : 0.f;
}
// n + 1.5·2^23 → n's three signed digits in base 256, a byte each: with 128
// added to every digit they are the bytes of n + 0x808080.
__device__ __forceinline__ uint32_t digits_of(float y) {
  return (__float_as_uint(y) - MAGIC_BITS + 0x808080u) ^ 0x808080u;
}
// Byte `at` of four words.
__device__ __forceinline__ uint32_t take_bytes(const uint32_t* n, int at) {
  const uint32_t pick = at | (at + 4) << 4;
  return __byte_perm(__byte_perm(n[0], n[1], pick), __byte_perm(n[2], n[3], pick), 0x5410);
}

__device__ __forceinline__ void put(const Kv8Attend& t, int type, int64_t at, float y) {
  void* op = const_cast<void*>(t.out.p);
  if (type == 0)
    static_cast<float*>(op)[at] = y;
  else if (type == 1)
    static_cast<__half*>(op)[at] = __float2half_rn(y);
  else
    static_cast<__nv_bfloat16*>(op)[at] = __float2bfloat16_rn(y);
}
__device__ __forceinline__ float lse_of(float top, float sum) {
  return sum == 0.f ? ninf() : __fmaf_rn(top, 0.693147181f, logf(sum));
}


// Whether groups of `count` elements of rows that begin at p with these
// strides lie at multiples of their size.
template <class T>
bool aligned(const Kv8Rows& r, int count) {
  const uintptr_t b = sizeof(T) * count;
  return reinterpret_cast<uintptr_t>(r.p) % b == 0 && (r.row * sizeof(T)) % b == 0 && (r.head * sizeof(T)) % b == 0;
}

}  // namespace

}  // namespace grx
