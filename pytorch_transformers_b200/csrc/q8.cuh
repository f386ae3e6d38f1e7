// The cache in 8 bits: e4m3 codes and one exponent for each block of 64 tokens (a page) and K/V head; a value is code * 2^exponent.
//
// The scale is a power of two. e4m3 is a floating format, so a scale that brings the largest entry exactly to 448 would win half a
// bit there and nothing elsewhere; a power makes a value exact in bfloat16 and rounding a page's codes again, when its
// exponent rises, exact but for codes that turn subnormal (they lose half of 2^-9 * 2^exponent, 2^-18 of what the page can hold).
#pragma once
#include "common.cuh"

constexpr int Q8_EXP_MIN = -126, Q8_EXP_MAX = 119;   // 2^-e and 448 * 2^e are normal, finite float32 (and the latter bfloat16) numbers

// 2^e, e in [-126, 127]
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// The smallest e in range with amax <= 448 * 2^e: amax = m 2^k with m in [1/2, 1), and 448 = 7/8 * 2^9.
__device__ __forceinline__ int q8_exponent(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 126 - 9 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return min(max(e, Q8_EXP_MIN), Q8_EXP_MAX);        // zero and subnormal amax: the lowest
}

// Four codes of four scaled numbers, rounded to nearest even. What is infinite, no number or past the largest code's upper half step
// (only entries above 448 * 2^119 are) becomes the code of no number: the conversion alone would make it 448 without a word.
__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d) {
  const float nan = __int_as_float(0x7fffffff);
  a = fabsf(a) <= 464.f ? a : nan;
  b = fabsf(b) <= 464.f ? b : nan;
  c = fabsf(c) <= 464.f ? c : nan;
  d = fabsf(d) <= 464.f ? d : nan;
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(hi) : "f"(d), "f"(c));
  return uint32_t(lo) | (uint32_t(hi) << 16);
}
// four codes as two pairs of float16 numbers, exactly (the first in the lower half)
__device__ __forceinline__ void q8_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}\n" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ void q8_unpack4(uint32_t w, float (&f)[4]) {
  uint32_t lo, hi;
  q8_halves(w, lo, hi);
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}\n" : "=f"(f[0]), "=f"(f[1]) : "r"(lo));
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}\n" : "=f"(f[2]), "=f"(f[3]) : "r"(hi));
}

// Eight entries from the eighth `c` of a bfloat16 row, rotated: `P` pairs (i, i + P), or (2 i, 2 i + 1), by the angles whose cosines and
// sines are given. The rotation's products and sums are those of rotate_pair; nothing is rounded to bfloat16 after it.
__device__ __forceinline__ void load_rotated8(const __nv_bfloat16* row, int c, const float* rc, const float* rs, int P, int interleaved,
                                              float (&x)[8]) {
  const int d0 = 8 * c;
  unpack_bf16x8(*reinterpret_cast<const uint4*>(row + d0), x);
  if (d0 >= 2 * P) return;
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const int e = (d0 + i) >> 1;
      if (e < P) rotate_pair(x[i], x[i + 1], rc[e], rs[e], x[i], x[i + 1]);
    }
  } else if ((P & 7) == 0) {
    const bool upper = d0 >= P;
    const int e0 = upper ? d0 - P : d0;
    float y[8];
    unpack_bf16x8(*reinterpret_cast<const uint4*>(row + (upper ? e0 : e0 + P)), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float ra, rb;
      rotate_pair(upper ? y[i] : x[i], upper ? x[i] : y[i], rc[e0 + i], rs[e0 + i], ra, rb);
      x[i] = upper ? rb : ra;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = d0 + i;
      if (d >= 2 * P) continue;
      const bool upper = d >= P;
      const int e = upper ? d - P : d;
      const float y = __bfloat162float(row[upper ? e : e + P]);
      float ra, rb;
      rotate_pair(upper ? y : x[i], upper ? x[i] : y, rc[e], rs[e], ra, rb);
      x[i] = upper ? rb : ra;
    }
  }
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

// Job `at` of a list that names, sequence after sequence, count(seq) jobs each: its sequence, and in `at` its place among that sequence's.
// -1 behind the last. A whole warp calls it with the same `at`.
template <typename Count>
__device__ __forceinline__ int find_job(int n_seqs, int& at, Count count) {
  const int lane = threadIdx.x & 31;
  for (int s0 = 0; s0 < n_seqs; s0 += 32) {
    const int mine = s0 + lane < n_seqs ? count(s0 + lane) : 0;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const int total = __shfl_sync(0xffffffffu, sum, 31);
    if (at < total) {
      const int l = __ffs(__ballot_sync(0xffffffffu, sum > at)) - 1;
      at -= __shfl_sync(0xffffffffu, sum - mine, l);
      return s0 + l;
    }
    at -= total;
  }
  return -1;
}
