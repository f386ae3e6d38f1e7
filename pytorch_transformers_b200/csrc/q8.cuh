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

__device__ __forceinline__ void load_angles(const float* rc, const float* rs, int e0, float (&c)[8], float (&s)[8]) {
  if (((reinterpret_cast<uintptr_t>(rc + e0) | reinterpret_cast<uintptr_t>(rs + e0)) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(rc + e0 + i);
      *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(rs + e0 + i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = rc[e0 + i], s[i] = rs[e0 + i];
  }
}

// Eighths of rows of the projection on their way (a row's own and the one that holds its pairs' other halves), and the angles of an
// eighth, which are the same for all rows: what a lane rotates in registers once all of its loads are out.
struct Angles {
  float c[8], s[8];
  int mode;      // 0: not rotated; 1: pairs within the eighth; 2: the pairs' other halves in the eighth `other`; 3: entry by entry
  int other;
  bool upper;
};
__device__ __forceinline__ Angles angles_of(int c, const float* rc, const float* rs, int P, int interleaved) {
  Angles a;
  const int d0 = 8 * c;
  a.other = c;
  a.upper = d0 >= P;
  a.mode = d0 >= 2 * P ? 0 : interleaved ? 1 : (P & 7) == 0 ? 2 : 3;
  if (a.mode == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d0 / 2 + i < P) a.c[i] = rc[d0 / 2 + i], a.s[i] = rs[d0 / 2 + i];
      else a.c[i] = 1.f, a.s[i] = 0.f;
  } else if (a.mode == 2) {
    const int e0 = a.upper ? d0 - P : d0;
    a.other = (a.upper ? e0 : e0 + P) / 8;
    load_angles(rc, rs, e0, a.c, a.s);
  }
  return a;
}
__device__ __forceinline__ void rotate8(const Angles& a, const uint4& own, const uint4& other, float (&x)[8]) {
  unpack_bf16x8(own, x);
  if (a.mode == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (a.c[i] != 1.f || a.s[i] != 0.f) rotate_pair(x[2 * i], x[2 * i + 1], a.c[i], a.s[i], x[2 * i], x[2 * i + 1]);
  } else if (a.mode == 2) {
    float y[8];
    unpack_bf16x8(other, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float ra, rb;
      rotate_pair(a.upper ? y[i] : x[i], a.upper ? x[i] : y[i], a.c[i], a.s[i], ra, rb);
      x[i] = a.upper ? rb : ra;
    }
  }
}
// both halves of pairs (i, i + P): `low` of the first P entries, `high` of the next P
__device__ __forceinline__ void rotate_halves(const float (&c)[8], const float (&s)[8], const uint4& low, const uint4& high, float (&x)[8], float (&y)[8]) {
  unpack_bf16x8(low, x);
  unpack_bf16x8(high, y);
#pragma unroll
  for (int i = 0; i < 8; ++i) rotate_pair(x[i], y[i], c[i], s[i], x[i], y[i]);
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

// One token's key (or value) into its page, by one warp: the rule of store_q8_kernel for a page that gets one row. The row's codes go to
// `copy` as well (or null), and the page's exponent is returned; `rose`: it is larger than before, and the earlier codes have been
// rounded again, seen by all who read them after the block's next barrier.
__device__ __forceinline__ int append_row(const __nv_bfloat16* row, const float* rc, const float* rs, int P, int interleaved, uint8_t* codes, int8_t* exps,
                          int at, int dim, unsigned char* copy, bool& rose) {
  const int lane = threadIdx.x & 31;
  const int old = at > 0 ? int(__ldcg(reinterpret_cast<const signed char*>(exps))) : Q8_EXP_MIN;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, most = 0.f;
  if (lane * 8 < dim) {
    load_rotated8(row, lane, rc, rs, P, interleaved, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, finite_abs(x[e]));
  }
  const int e = max(q8_exponent(warp_max(most)), old);
  rose = at > 0 && e > old;
  if (rose) {
    const float down = power_of_two(max(old - e, -126));
    for (int i = lane; i < at * dim / 16; i += 32) {
      uint4 w = __ldcg(reinterpret_cast<const uint4*>(codes) + i);
      uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[4];
        q8_unpack4(u[k], f);
        u[k] = q8_pack4(f[0] * down, f[1] * down, f[2] * down, f[3] * down);
      }
      reinterpret_cast<uint4*>(codes)[i] = w;
    }
  }
  const float by = power_of_two(-e);
  if (lane * 8 < dim) {
    const uint2 w = make_uint2(q8_pack4(x[0] * by, x[1] * by, x[2] * by, x[3] * by), q8_pack4(x[4] * by, x[5] * by, x[6] * by, x[7] * by));
    *reinterpret_cast<uint2*>(codes + size_t(at) * dim + lane * 8) = w;
    if (copy) *reinterpret_cast<uint2*>(copy + lane * 8) = w;
  }
  if (lane == 0) *exps = int8_t(e);
  if (rose) {      // the accelerator reads them next
    __threadfence();
    asm volatile("fence.proxy.async;\n" ::: "memory");
  }
  return e;
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
