// The 8-bit context cache: layout, argument records and the fragment helpers its kernels share.
//
// Keys and values are kept in blocks of 64 rows.  A (group, head, block) has one record of 128 * Dh code bytes (the
// keys row by row, then the values transposed), two scales, and the smallest / largest key code per channel.
// A code c stands for (c - 128) * scale.  Codes are unsigned because a byte then becomes a half-precision number in
// one permute and one subtraction (0x6400 | byte is 1024 + byte), exactly; whole numbers up to 127 are exact in
// half precision, so products with them cost no accuracy beyond the other operand's.
//
// Order inside a record, chosen so that every thread of a warp reads its mma.m16n8k16 fragments as one contiguous
// piece (g = lane / 4, t = lane % 4):
//   keys     [64][Dh]; the four k indices of thread t in k step s are channels t * Dh/4 + 4 s + {0,1,2,3}, so the
//            thread reads Dh/4 bytes of a row at once
//   values   [Dh][64]; place 16 t + 4 s + 2 h + e of a channel holds row 16 s + 8 h + 2 t + e, so the thread reads the 16
//            bytes of its four k steps at once
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace artab {

constexpr int kCacheBlock = 64;
constexpr int kMostListed = 1 << 30;   // blocks of a list: the kernels step through it, and past its end, in 32 bits

// Rows of a [.., .., rows, Dh] tensor by strides (in elements) of its three leading axes.
struct RowView {
  const void* p;
  long s0, s1, s2;
};

// strides as the entry points take them: null for a contiguous tensor
inline RowView row_view(const void* p, const int64_t* strides, int n1, int n2, int dh) {
  if (!strides) return {p, (long)n1 * n2 * dh, (long)n2 * dh, (long)dh};
  return {p, (long)strides[0], (long)strides[1], (long)strides[2]};
}

// ---- whole numbers nearest to a quotient ------------------------------------------------------------------
// The nearest whole number to x / scale in exact arithmetic, ties to even.  A first value c comes from one fused product
// with the reciprocal, rounded by adding 1.5 * 2^23 (the low byte of the sum is then the code).  Next to a tie it may be
// off by one, and ties are not rare (rows of eight-bit numbers such as bf16 meet one in some 200): the rest x - c * scale,
// one fused operation that is exact next to a tie, is compared with half the scale.  Steps below 2^-125, and kept rows next to a tie (whose x is a product itself), go through 64 bits.
constexpr float kRound = 12582912.0f + 128.0f;   // 1.5 * 2^23, and the 128 that is added to a code
constexpr float kLeastStep = 2.350988701644575e-38f;   // 2^-125: half of it is a normal number, so halves of steps are exact

__device__ __forceinline__ uint32_t low_bytes(const uint32_t (&w)[4]) {
  return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}
// bytes of a word as numbers less 128
__device__ __forceinline__ void code_values(uint32_t w, float (&x)[4]) {
  const uint32_t u[4] = {__byte_perm(w, 0x4b000000u, 0x7440), __byte_perm(w, 0x4b000000u, 0x7441),
                         __byte_perm(w, 0x4b000000u, 0x7442), __byte_perm(w, 0x4b000000u, 0x7443)};
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(u[j]) - 8388736.0f;
}
static __device__ __noinline__ uint32_t exact_codes(float x0, float x1, float x2, float x3, float was, float scale) {
  const float x[4] = {x0, x1, x2, x3};
  uint32_t w = 0;
  for (int j = 0; j < 4; ++j) {
    const double c = rint((double)x[j] * (double)was / (double)scale);
    w |= (uint32_t)(128 + (int)fmin(fmax(c, -127.0), 127.0)) << (8 * j);
  }
  return w;
}
// Four codes of x at a step of `scale` (> 0)
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float scale, float inv) {
  uint32_t w[4];
  float rest[4];
  const float half = 0.5f * scale;
  bool sure = scale >= kLeastStep;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float r = fmaf(x[j], inv, kRound);
    rest[j] = fmaf(kRound - r, scale, x[j]);
    sure = sure && fabsf(rest[j]) < half;             // false for what is not finite, too
    w[j] = __float_as_uint(r);
  }
  if (!sure) {
    if (scale < kLeastStep) return exact_codes(x[0], x[1], x[2], x[3], 1.0f, scale);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool off = fabsf(rest[j]) > half || (fabsf(rest[j]) == half && (w[j] & 1u));
      w[j] += off ? (rest[j] > 0.0f ? 1u : 0xffffffffu) : 0u;
    }
  }
  return low_bytes(w);
}
// Four codes of bf16 numbers x whose largest magnitude gave the step.  x = a 2^i and that magnitude b 2^j have a, b < 256, so
// 127 x / (b 2^j) is either a tie or more than 2^-16 of itself away from one; the step is off from b 2^j / 127 by at most 2^-24.  A
// reciprocal that is 2^-19 too small (`over`: step * 127 above the magnitude) or too large decides every tie as the exact
// quotient by the step does, and nothing else.  `over` 0: ties of the step itself, which this cannot decide.
constexpr float kTieShift = 1.9073486328125e-6f;
__device__ __forceinline__ float shifted(float inv, float over) { return inv * (over > 0.0f ? 1.0f - kTieShift : 1.0f + kTieShift); }
__device__ __forceinline__ uint32_t codes_of_bf16(const float (&x)[4], float inv_shifted) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(fmaf(x[j], inv_shifted, kRound));
  return low_bytes(w);
}
// Four codes of x * was (whole numbers x at an older step `was`) at a step of `scale`.  The first quotient is off by less
// than 3e-5: closer than 5e-5 to a tie it is formed again.
__device__ __forceinline__ uint32_t kept_codes(const float (&x)[4], float was, float scale, float inv) {
  uint32_t w[4];
  bool sure = scale >= kLeastStep;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float y = x[j] * was, r = fmaf(y, inv, kRound);
    sure = sure && fabsf(fmaf(y, inv, kRound - r)) <= 0.49995f;
    w[j] = __float_as_uint(r);
  }
  return sure ? low_bytes(w) : exact_codes(x[0], x[1], x[2], x[3], was, scale);
}

// ---- fragments -------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// two neighbouring code bytes -> two halves (byte - 128); `high`: bytes 2, 3 of the word instead of 0, 1
__device__ __forceinline__ uint32_t codes_to_halves(uint32_t w, bool high) {
  const uint32_t x = __byte_perm(w, 0x64646464u, high ? 0x4342u : 0x4140u);  // 1024 + byte
  const uint32_t off = 0x64806480u;                                         // 1152
  return h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&off)));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {  // 8 x 8 halves over the warp, two per thread
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void cache_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cache_cp8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Power of two that brings a row with largest magnitude `top` into [1, 2), and its inverse.  Queries go to the
// tensor cores as one or two half-precision parts (11 bits each) of the scaled row: what falls below the range of
// halves is then less than 2^-24 of the row's largest element.  Both are normal numbers for every finite row.
__device__ __forceinline__ void row_scale(float top, float& to, float& back) {
  int e = (int)((__float_as_uint(top) >> 23) & 255u);
  e = e < 1 ? 1 : e > 253 ? 253 : e;
  to = __uint_as_float((uint32_t)(254 - e) << 23);
  back = __uint_as_float((uint32_t)e << 23);
}

// NN consecutive elements of a query row as floats; `vec`: the row is aligned to the 16 (8, 4) bytes read at a time
template <typename T, int NN>
__device__ __forceinline__ void load_elements(const T* p, bool vec, float (&x)[NN]) {
  constexpr int kBytes = NN * (int)sizeof(T);
  if (vec) {
    constexpr int kUnit = kBytes >= 16 ? 16 : 8;
    constexpr int kPer = kUnit / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < NN / kPer; ++i) {
      uint32_t w[4];
      if constexpr (kUnit == 16) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      } else {
        const uint2 v = reinterpret_cast<const uint2*>(p)[i];
        w[0] = v.x, w[1] = v.y;
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if constexpr (sizeof(T) == 4)
          x[i * kPer + j] = __uint_as_float(w[j]);
        else
          x[i * kPer + j] = __uint_as_float((j & 1) ? (w[j >> 1] & 0xffff0000u) : (w[j >> 1] << 16));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NN; ++i) x[i] = to_f32<T>(p[i]);
  }
}

// A cache and query tensor that fit each other: checked by every entry point that takes queries.
int check_cache(const artab_cache* c, const char* what);
int check_queries(int dtype, const void* q, int n_streams, int n_q, const artab_cache* c, const char* what);
// every strided row starts on a 16-byte (fp32, bf16 with at least eight elements per thread) boundary
inline bool rows_aligned(const RowView& v, int elem) {
  return ((reinterpret_cast<uintptr_t>(v.p) | (uintptr_t)(v.s0 * elem) | (uintptr_t)(v.s1 * elem) | (uintptr_t)(v.s2 * elem)) & 15) == 0;
}

}  // namespace artab
