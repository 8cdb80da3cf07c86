// A warp's tile of a few query rows against blocks of the 8-bit context cache (see cache_attn.cu).
#pragma once
#include "cache_attn.cuh"

namespace artab {

// numerators are 2^14 times exp(s - max): halves keep 11 bits of them down to 2^-28 of the largest
constexpr float kLift = 14.0f;
// outputs are kept without that factor: of the size of the sums that they stand for, which fit where those do
constexpr float kUnlift = 6.103515625e-5f;

template <int DH, int PARTS>
struct Tile {
  static constexpr int KS = DH / 16;      // k steps of a score, 16-channel tiles of the output
  static constexpr int R = 3 - PARTS;     // query rows of a thread
  static constexpr int ROWS = 8 / PARTS;
  uint32_t q[KS][2];
  float f[R];                             // score units to log2
  float m[R], l[R], o[KS][2][R];          // o: channels 16 md + g, 16 md + 8 + g of the thread's rows

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = -CUDART_INF_F, l[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) o[i][j][r] = 0.0f;
  }

  // `row`: this thread's row of the query fragment (row g / PARTS of the tile), or null
  template <typename T>
  __device__ __forceinline__ void load_queries(const T* row, bool vec, float scale_log2) {
    constexpr int NE = DH / 4;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float x[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) x[i] = 0.0f;
    if (row) load_elements<T, NE>(row + t * NE, vec, x);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i) top = fmaxf(top, fabsf(x[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float to, back;
    row_scale(top, to, back);
    back *= scale_log2;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      __half2 p[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float a = x[4 * s + 2 * j] * to, b = x[4 * s + 2 * j + 1] * to;
        p[j] = __floats2half2_rn(a, b);
        if (PARTS == 2 && (g & 1)) p[j] = __floats2half2_rn(a - __low2float(p[j]), b - __high2float(p[j]));
      }
      q[s][0] = h2_bits(p[0]);
      q[s][1] = h2_bits(p[1]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) f[r] = __shfl_sync(0xffffffffu, back, PARTS == 2 ? 8 * t : 8 * t + 4 * r);
  }

  // one block: record in shared memory, its scales, its rows in use (1 .. 64)
  __device__ __forceinline__ void block(const uint8_t* rec, float ks, float vs, int live) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float x[4][2][R];                     // scores of rows 16 mt + g, 16 mt + 8 + g
    float mx[R];
#pragma unroll
    for (int r = 0; r < R; ++r) mx[r] = m[r];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      uint32_t wa[KS], wb[KS];
      load_codes(rec + (16 * mt + g) * DH + t * (DH / 4), wa);
      load_codes(rec + (16 * mt + 8 + g) * DH + t * (DH / 4), wb);
#pragma unroll
      for (int s = 0; s < KS; ++s)
        mma_f16(c, codes_to_halves(wa[s], false), codes_to_halves(wb[s], false), codes_to_halves(wa[s], true),
                codes_to_halves(wb[s], true), q[s][0], q[s][1]);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float s = (PARTS == 2 ? c[2 * j] + c[2 * j + 1] : c[2 * j + r]) * (f[r] * ks);
          if (live < kCacheBlock && 16 * mt + 8 * j + g >= live) s = -CUDART_INF_F;
          x[mt][j][r] = s;
          mx[r] = fmaxf(mx[r], s);
        }
    }
    float alpha[R], ref[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], o));
      const float base = mx[r] == -CUDART_INF_F ? 0.0f : mx[r];
      alpha[r] = ex2(m[r] - base);
      m[r] = mx[r];
      ref[r] = base - kLift;
      l[r] *= alpha[r];
    }
    uint32_t p[4][2];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float e[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          e[r] = ex2(x[mt][j][r] - ref[r]);
          l[r] += e[r];
        }
        __half2 u;
        if constexpr (PARTS == 2) {
          const __half hi = __float2half_rn(e[0]);
          u = __halves2half2(hi, __float2half_rn(e[0] - __half2float(hi)));
        } else {
          u = __floats2half2_rn(e[0], e[R - 1]);
        }
        p[mt][j] = transpose_8x8(h2_bits(u));
      }
    const uint8_t* vals = rec + kCacheBlock * DH;
#pragma unroll
    for (int md = 0; md < KS; ++md) {
      const uint4 a = *reinterpret_cast<const uint4*>(vals + (16 * md + g) * kCacheBlock + 16 * t);
      const uint4 b = *reinterpret_cast<const uint4*>(vals + (16 * md + 8 + g) * kCacheBlock + 16 * t);
      const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
      float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < 4; ++s)
        mma_f16(c, codes_to_halves(wa[s], false), codes_to_halves(wb[s], false), codes_to_halves(wa[s], true),
                codes_to_halves(wb[s], true), p[s][0], p[s][1]);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r)
          o[md][j][r] = fmaf(o[md][j][r], alpha[r], vs * (kUnlift * (PARTS == 2 ? c[2 * j] + c[2 * j + 1] : c[2 * j + r])));
    }
  }

 private:
  static __device__ __forceinline__ void load_codes(const uint8_t* p, uint32_t (&w)[KS]) {
    if constexpr (KS == 1) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (KS == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
  }
};

}  // namespace artab
