// Writing rows into the 8-bit context cache, and reading them back.
//
// write: one CTA per (group, head, touched block), half of its threads on the keys, half on the values, 16 elements a
// thread.  The scale of a block is its largest magnitude / 127; rows that come behind others of a block may raise
// it, and the older rows are then rounded again to the new step.
// Keys go out as they came in; of the values a thread holds the four rows that are neighbours in a channel's order, so
// that it turns 4 x 4 bytes with permutes, and shared memory brings the words into the order of the record.
// 64 contexts x 2048 rows x 6 heads of size 32 (B200): fp32 48 us for 251 MB (5.2 TB/s, HBM), bf16 38 us for 151 MB: some 310
// instructions a warp and block (80 % of issue slots).  Reading the same back
// as fp32: 40 us for 252 MB (6.3 TB/s), as bf16 32 us for 151 MB.  100 rows behind 2000 of 64 contexts: 8 heads of size 64 16 us (fp32;
// bf16 15.5), 6 of size 32 7.5: two or three blocks a (group, head), a CTA each, a chain of lengths, rows, barrier, codes and stores.
#include "cache8.cuh"

namespace artab {
namespace {

constexpr int kMostRows = 1 << 30;   // of a cache, or to write or read at once

struct WriteArgs {
  artab_cache c;
  RowView k, v;
  const int32_t* start;    // [G], or null: 0
  const int32_t* counts;   // [G], or null: n_rows
  int n_rows;
  int fresh;               // the whole cache is laid out: every block of it is given scales and bounds
  int set_lens;            // lens[g] = end of the rows written here
  int by_group;            // a CTA (of cache_append_row_kernel) has all heads of a group: it may move the lens[g] that it reads
  int vec_k, vec_v;
  int per_cta;             // blocks of a CTA
};

// the group's first row to write, and the row behind its last one
__device__ __forceinline__ void write_range(const WriteArgs& a, int g, int& start, int& end) {
  const int cap = a.c.n_blocks * kCacheBlock;
  int s = a.start ? a.start[g] : 0;
  int n = a.counts ? a.counts[g] : a.n_rows;
  s = s < 0 ? 0 : s > cap ? cap : s;
  n = n < 0 ? 0 : n > a.n_rows ? a.n_rows : n;
  start = s;
  end = n > cap - s ? cap : s + n;
}

// 4 x 4 bytes: word r of the result holds byte r of every word
__device__ __forceinline__ void turn(uint32_t (&w)[4]) {
  const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
  const uint32_t c = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);
  w[0] = __byte_perm(a, b, 0x5410), w[1] = __byte_perm(a, b, 0x7632);
  w[2] = __byte_perm(c, d, 0x5410), w[3] = __byte_perm(c, d, 0x7632);
}
// first of the four rows {r, r + 1, r + 8, r + 9} that are neighbours in word `word` (0 .. 15) of a value channel
__device__ __forceinline__ int first_row(int word) { return 16 * (word & 3) + 2 * (word >> 2); }

__device__ __forceinline__ float step_of(uint32_t top_bits) {
  const float x = __uint_as_float(top_bits);
  if (x < 1e-30f) return __fdiv_rn(x, 127.0f);
  // the quotient by 127, correctly rounded: a first value, its exact rest, one correction (Markstein, "Computation of elementary
  // functions on the IBM RISC System/6000 processor", 1990)
  const float c = 1.0f / 127.0f, q = x * c;
  return top_bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : fmaf(fmaf(-127.0f, q, x), c, q);
}
// 1 / x to one step in the last place, for what is checked or moved by more than that afterwards
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// a block with a value that is not finite has NaN for its scale, for good
__device__ __forceinline__ float larger_step(float a, float b) { return a != a ? a : b != b ? b : fmaxf(a, b); }

template <int DH>
struct Half {                      // threads of a CTA that work on the keys; as many again on the values
  static constexpr int C4 = DH / 4, N = 16 * C4, WARPS = N / 32, VP = 17;   // VP: words of a padded value channel
};

__device__ __forceinline__ float larger_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// four neighbouring elements as they are stored
template <typename T>
struct Four;
template <>
struct Four<float> {
  using Raw = uint4;
  __device__ static __forceinline__ void values(const Raw& r, float (&x)[4]) {
    x[0] = __uint_as_float(r.x), x[1] = __uint_as_float(r.y), x[2] = __uint_as_float(r.z), x[3] = __uint_as_float(r.w);
  }
  __device__ static __forceinline__ Raw zero() { return make_uint4(0u, 0u, 0u, 0u); }
  __device__ static __forceinline__ float largest(const Raw (&r)[4]) {   // magnitude, NaN if there is one
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[4];
      values(r[i], x);
#pragma unroll
      for (int j = 0; j < 4; ++j) top = larger_or_nan(top, fabsf(x[j]));
    }
    return top;
  }
};
template <>
struct Four<__nv_bfloat16> {
  using Raw = uint2;
  __device__ static __forceinline__ void values(const Raw& r, float (&x)[4]) {
    x[0] = __uint_as_float(r.x << 16), x[1] = __uint_as_float(r.x & 0xffff0000u);
    x[2] = __uint_as_float(r.y << 16), x[3] = __uint_as_float(r.y & 0xffff0000u);
  }
  __device__ static __forceinline__ Raw zero() { return make_uint2(0u, 0u); }
  __device__ static __forceinline__ float largest(const Raw (&r)[4]) {
    uint32_t top = 0u;                               // magnitudes; the signs are of no use
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(r[i].x));
      asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(r[i].y));
    }
    return larger_or_nan(__uint_as_float(top << 16 & 0x7fffffffu), __uint_as_float(top & 0x7fff0000u));
  }
};
template <typename T>
__device__ __noinline__ typename Four<T>::Raw load_unaligned(const T* p) {
  typename Four<T>::Raw r;
  T* to = reinterpret_cast<T*>(&r);
  for (int j = 0; j < 4; ++j) to[j] = p[j];
  return r;
}
// FRESH: the whole cache is laid out, several neighbouring blocks a CTA, the rows of the next on their way while one is
// worked on; else one block a CTA and as many CTAs of an SM as there can be, for latencies that follow one another.
template <typename T, int DH, bool FRESH>
__global__ void __launch_bounds__(2 * Half<DH>::N, (FRESH ? 1024 : 1280) / (2 * Half<DH>::N)) cache_write_kernel(const WriteArgs a) {
  using F = Half<DH>;
  using Raw = typename Four<T>::Raw;
  constexpr int C4 = F::C4;
  __shared__ uint32_t s_v[DH * F::VP];
  __shared__ uint32_t s_top[2 * F::WARPS];
  __shared__ uint2 s_lo[F::WARPS][C4], s_hi[F::WARPS][C4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool vals = threadIdx.x >= F::N;
  const int tid = vals ? threadIdx.x - F::N : threadIdx.x, c4 = tid % C4, word = tid / C4;
  const int h = blockIdx.y, g = blockIdx.z;
  int start, end;
  write_range(a, g, start, end);
  if (a.set_lens && blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.c.lens[g] = end;
  // the blocks of this CTA: `per_cta` neighbours
  const int per_cta = FRESH ? a.per_cta : 1;
  int blk = (FRESH ? 0 : start / kCacheBlock) + (int)blockIdx.x * per_cta;
  const int last = blk + per_cta < a.c.n_blocks ? blk + per_cta : a.c.n_blocks;
  const size_t rec0 = ((size_t)g * a.c.n_heads + h) * a.c.n_blocks;
  const RowView& src = vals ? a.v : a.k;
  // the rows of a thread's four pieces: of keys 16 apart, of values those of a word
  const int row0 = vals ? first_row(word) : word, d1 = vals ? 1 : 16, d2 = vals ? 8 : 32;
  const long p1 = d1 * src.s2, p2 = d2 * src.s2;
  const T* from = reinterpret_cast<const T*>(src.p) + g * src.s0 + h * src.s1 + ((long)blk * kCacheBlock + row0 - start) * src.s2 + c4 * 4;
  const int vec = vals ? a.vec_v : a.vec_k;
  const auto load = [&](int b, const T* p, Raw (&raw)[4]) {      // new rows of block b, zeros for the others
    const int lo = start - b * kCacheBlock, hi = end - b * kCacheBlock;
    if (FRESH && vec && hi >= kCacheBlock) {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = *reinterpret_cast<const Raw*>(p + (i & 1) * p1 + (i >> 1) * p2);
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + (i & 1) * d1 + (i >> 1) * d2;
      const T* at = p + (i & 1) * p1 + (i >> 1) * p2;
      raw[i] = Four<T>::zero();
      if (row >= lo && row < hi) raw[i] = vec ? *reinterpret_cast<const Raw*>(at) : load_unaligned(at);
    }
  };
  Raw next[4];
  if (blk < last) load(blk, from, next);
  for (; blk < last; ++blk) {
    const int base = blk * kCacheBlock;
    float* scales = a.c.scales + (rec0 + blk) * 2;
    __half* bounds = reinterpret_cast<__half*>(a.c.bounds) + (rec0 + blk) * 2 * DH;
    if (end <= base) {                               // no row of this block
      if (!FRESH) return;
      if (threadIdx.x < 2) scales[threadIdx.x] = 0.0f;
      if (threadIdx.x < 2 * DH) bounds[threadIdx.x] = __float2half(0.0f);
      continue;
    }
    uint32_t* codes = reinterpret_cast<uint32_t*>(a.c.codes + (rec0 + blk) * (size_t)(2 * kCacheBlock * DH)) + (vals ? kCacheBlock * C4 : 0);
    const int n_old = !FRESH && start > base ? start - base : 0;     // rows that are there already
    const int n_live = end - base < kCacheBlock ? end - base : kCacheBlock;
    Raw raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = next[i];
    from += kCacheBlock * src.s2;
    if (FRESH && blk + 1 < last) load(blk + 1, from, next);
    const float was = n_old ? scales[vals] : 0.0f;
    const float top = Four<T>::largest(raw);
    const uint32_t warp_top = __reduce_max_sync(0xffffffffu, __float_as_uint(top));   // NaN above all
    if (lane == 0) s_top[warp] = warp_top;
    // Codes that are there: of keys all (for the bounds), of values at first only words that new rows go into.
    const bool mine = row0 < n_live && row0 + d1 + d2 >= n_old;     // may have a new row among its four
    uint32_t old[4] = {0u, 0u, 0u, 0u};
    const auto load_old = [&]() {
#pragma unroll
      for (int i = 0; i < 4; ++i) old[i] = vals ? codes[(c4 * 4 + i) * 16 + word] : codes[(word + 16 * i) * C4 + c4];
      if (vals) turn(old);
    };
    if (n_old && (!vals || mine)) load_old();
    __syncthreads();   // also: every thread has read the old codes and scales
    uint32_t block_top = 0;
#pragma unroll
    for (int w = 0; w < F::WARPS; ++w) block_top = max(block_top, s_top[(vals ? F::WARPS : 0) + w]);
    // a step of zero (or NaN) has zero codes
    const float step = larger_step(was, step_of(block_top)), inv = reciprocal(step);
    const float over = fmaf(step, 127.0f, -__uint_as_float(block_top)), inv_shifted = shifted(inv, over);
    const bool shift = FRESH && sizeof(T) == 2 && step >= kLeastStep && over != 0.0f;
    // rows that stay, at a scale that stays, are not written again
    const bool stays = !FRESH && n_old > 0 && !(step > was);
    if (n_old && vals && !mine && !stays) load_old();
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + (i & 1) * d1 + (i >> 1) * d2;
      w[i] = 0x80808080u;
      if (FRESH || (row >= n_old && row < n_live)) {   // of a whole cache, rows that are not in use are zeros
        float x[4];
        Four<T>::values(raw[i], x);
        if (shift)
          w[i] = codes_of_bf16(x, inv_shifted);
        else if (step > 0.0f)
          w[i] = codes_of(x, step, inv);
      } else if (row < n_old) {
        w[i] = old[i];
        if (step > was) {
          float y[4];
          code_values(old[i], y);
          w[i] = kept_codes(y, was, step, inv);
        }
      }
    }
    if (vals && stays) {
      if (mine) {
        turn(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) codes[(c4 * 4 + i) * 16 + word] = w[i];
      }
    } else if (vals) {
      turn(w);
#pragma unroll
      for (int i = 0; i < 4; ++i) s_v[(c4 * 4 + i) * F::VP + word] = w[i];
    } else {
      // smallest and largest code of the channels, as halves 1024 + byte
      __half2 lo[2], hi[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) lo[j] = __float2half2_rn(2048.0f), hi[j] = __float2half2_rn(0.0f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!stays || row0 + 16 * i >= n_old) codes[(word + 16 * i) * C4 + c4] = w[i];
        if (row0 + 16 * i >= n_live) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t u = __byte_perm(w[i], 0x64646464u, j ? 0x4342u : 0x4140u);
          lo[j] = __hmin2(lo[j], *reinterpret_cast<const __half2*>(&u));
          hi[j] = __hmax2(hi[j], *reinterpret_cast<const __half2*>(&u));
        }
      }
#pragma unroll
      for (int o = C4; o < 32; o <<= 1)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          lo[j] = __hmin2(lo[j], __shfl_xor_sync(0xffffffffu, lo[j], o));
          hi[j] = __hmax2(hi[j], __shfl_xor_sync(0xffffffffu, hi[j], o));
        }
      if (lane < C4) {
        s_lo[warp][lane] = make_uint2(h2_bits(lo[0]), h2_bits(lo[1]));
        s_hi[warp][lane] = make_uint2(h2_bits(hi[0]), h2_bits(hi[1]));
      }
    }
    __syncthreads();
    if (vals) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (stays) break;
        const int at = tid + i * F::N;
        codes[at] = s_v[(at / 16) * F::VP + at % 16];
      }
    } else if (tid < 2 * C4) {                       // a thread per four channels of either bound
      const bool upper = tid >= C4;
      uint2 best = upper ? s_hi[0][tid - C4] : s_lo[0][tid];
      const __half2 off = __float2half2_rn(1152.0f);
#pragma unroll
      for (int r = 1; r < F::WARPS; ++r) {
        const uint2 u = upper ? s_hi[r][tid - C4] : s_lo[r][tid];
        const __half2 x = *reinterpret_cast<const __half2*>(&u.x), y = *reinterpret_cast<const __half2*>(&u.y);
        __half2 &bx = *reinterpret_cast<__half2*>(&best.x), &by = *reinterpret_cast<__half2*>(&best.y);
        bx = upper ? __hmax2(bx, x) : __hmin2(bx, x);
        by = upper ? __hmax2(by, y) : __hmin2(by, y);
      }
      best.x = h2_bits(__hsub2(*reinterpret_cast<__half2*>(&best.x), off));
      best.y = h2_bits(__hsub2(*reinterpret_cast<__half2*>(&best.y), off));
      reinterpret_cast<uint2*>(bounds)[tid] = best;
    }
    if (tid == 0) scales[vals] = step;
  }
}

// One new row a context: the step of a decode.  A warp does a (group, head): the new row's codes by a lane or two a channel,
// the bounds from the block's older keys, which 16 bytes a lane hold while they are looked through; older codes are
// written only where a scale rises.  512 contexts x 6 heads of size 32: 15.4 us with cache_write_kernel, which goes through
// whole blocks with a CTA each, 4.8 here (17 heads, in two launches, 10).  Up to kGroupHeads heads a CTA takes a group, and the length moves in the same launch;
// beyond, four warps of any groups, and cache_advance_kernel.
constexpr int kGroupHeads = 16;
__device__ __forceinline__ int value_place(int row) { return 16 * ((row >> 1) & 3) + 4 * (row >> 4) + 2 * ((row >> 3) & 1) + (row & 1); }

template <typename T, int DH>
__global__ void __launch_bounds__(32 * kGroupHeads) cache_append_row_kernel(const WriteArgs a) {
  constexpr int NV = DH / 16;          // new numbers of a lane: number v = lane + 32 i is channel v % DH of keys (v < DH) or values
  constexpr int NQ = DH / 8;           // 16-byte pieces of a lane: piece lane + 32 i, 16 channels of a key
  constexpr int PARTS = DH / 16;       // pieces of a row
  const int lane = threadIdx.x & 31, H = a.c.n_heads;
  const long unit = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (unit >= (long)a.c.n_groups * H) return;
  const int g = (int)(unit / H), h = (int)(unit % H);
  int start, end;
  write_range(a, g, start, end);
  if (a.by_group) __syncthreads();                                 // every warp has read lens
  if ((a.by_group || a.set_lens) && h == 0 && lane == 0) a.c.lens[g] = end;
  const int blk = start / kCacheBlock, at = start % kCacheBlock;   // `at` rows of the block are kept
  const bool fresh_row = end > start;
  if (blk >= a.c.n_blocks || at + fresh_row == 0) return;
  const size_t rec = (size_t)unit * a.c.n_blocks + blk;
  uint8_t* codes = a.c.codes + rec * (size_t)(2 * kCacheBlock * DH);
  float2* scales = reinterpret_cast<float2*>(a.c.scales) + rec;
  uint4 q[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    q[i] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
    if ((lane + 32 * i) / PARTS < at) q[i] = reinterpret_cast<const uint4*>(codes)[lane + 32 * i];
  }
  const float2 was = at ? *scales : make_float2(0.0f, 0.0f);
  float x[NV];
  uint32_t top_k = 0, top_v = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = lane + 32 * i, d = v % DH;
    x[i] = 0.0f;
    if (fresh_row)
      x[i] = v < DH ? to_f32<T>(reinterpret_cast<const T*>(a.k.p)[g * a.k.s0 + h * a.k.s1 + d])
                    : to_f32<T>(reinterpret_cast<const T*>(a.v.p)[g * a.v.s0 + h * a.v.s1 + d]);
    const uint32_t bits = __float_as_uint(x[i]) & 0x7fffffffu;
    top_k = max(top_k, v < DH ? bits : 0u), top_v = max(top_v, v < DH ? 0u : bits);
  }
  const float2 step = make_float2(larger_step(was.x, step_of(__reduce_max_sync(0xffffffffu, top_k))),
                                  larger_step(was.y, step_of(__reduce_max_sync(0xffffffffu, top_v))));
  if (at && step.x > was.x) {
    const float inv = 1.0f / step.x;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&q[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float y[4];
        code_values(w[e], y);
        w[e] = kept_codes(y, was.x, step.x, inv);
      }
      if ((lane + 32 * i) / PARTS < at) reinterpret_cast<uint4*>(codes)[lane + 32 * i] = q[i];
    }
  }
  if (at && step.y > was.y) {          // every place of the values: those of rows that are not in use do not matter
    const float inv = 1.0f / step.y;
    uint32_t* v = reinterpret_cast<uint32_t*>(codes + kCacheBlock * DH);
#pragma unroll 1
    for (int i = lane; i < kCacheBlock * DH / 4; i += 32) {
      float y[4];
      code_values(v[i], y);
      v[i] = kept_codes(y, was.y, step.y, inv);
    }
  }
  if (!at) {                           // a block begins: no row of it is in use yet
#pragma unroll
    for (int i = 0; i < 2 * NQ; ++i)
      reinterpret_cast<uint4*>(codes)[lane + 32 * i] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
  }
  __syncwarp();
  uint32_t mine[NV];                   // codes of the new numbers
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = lane + 32 * i, d = v % DH;
    const float s = v < DH ? step.x : step.y, y[4] = {x[i], 0.0f, 0.0f, 0.0f};
    mine[i] = s > 0.0f ? codes_of(y, s, 1.0f / s) & 255u : 128u;
    if (fresh_row) codes[v < DH ? at * DH + d : kCacheBlock * DH + d * kCacheBlock + value_place(at)] = (uint8_t)mine[i];
  }
  // bounds: halves 1024 + code of this lane's 16 channels over its rows, then over the lanes of the same channels
  __half2 lo[8], hi[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) lo[j] = __float2half2_rn(2048.0f), hi[j] = __float2half2_rn(0.0f);
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    if ((lane + 32 * i) / PARTS >= at) continue;
    const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t u = __byte_perm(w[j >> 1], 0x64646464u, j & 1 ? 0x4342u : 0x4140u);
      lo[j] = __hmin2(lo[j], *reinterpret_cast<const __half2*>(&u));
      hi[j] = __hmax2(hi[j], *reinterpret_cast<const __half2*>(&u));
    }
  }
#pragma unroll
  for (int o = PARTS; o < 32; o <<= 1)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = __hmin2(lo[j], __shfl_xor_sync(0xffffffffu, lo[j], o));
      hi[j] = __hmax2(hi[j], __shfl_xor_sync(0xffffffffu, hi[j], o));
    }
  // the new key's codes of channels 16 part .. + 15: number v is with lane v % 32, there of register v / 32
  const int part = lane % PARTS;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t c[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int v = 16 * part + 2 * j + e;
      uint32_t got = __shfl_sync(0xffffffffu, mine[0], v % 32);
      if (DH == 64) {
        const uint32_t upper = __shfl_sync(0xffffffffu, mine[NV > 1 ? 1 : 0], v % 32);
        got = v >= 32 ? upper : got;
      }
      c[e] = got;
    }
    const uint32_t u = 0x64006400u | c[0] | c[1] << 16;
    if (fresh_row) {
      lo[j] = __hmin2(lo[j], *reinterpret_cast<const __half2*>(&u));
      hi[j] = __hmax2(hi[j], *reinterpret_cast<const __half2*>(&u));
    }
  }
  if (lane < PARTS) {
    const __half2 off = __float2half2_rn(1152.0f);
    __half2* to = reinterpret_cast<__half2*>(reinterpret_cast<__half*>(a.c.bounds) + rec * 2 * DH);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      to[8 * part + j] = __hsub2(lo[j], off);
      to[DH / 2 + 8 * part + j] = __hsub2(hi[j], off);
    }
  }
  if (lane == 0) *scales = step;
}

// lens[g] moves behind the rows that cache_write_kernel has put there from lens[g] on
__global__ void cache_advance_kernel(const WriteArgs a) {
  const int g = blockIdx.x * blockDim.x + threadIdx.x;
  if (g >= a.c.n_groups) return;
  int start, end;
  write_range(a, g, start, end);
  a.c.lens[g] = end;
}

struct ReadArgs {
  artab_cache c;
  const int32_t* start;
  int n_rows;
  void *k, *v;
};

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    __nv_bfloat162 y[2] = {__floats2bfloat162_rn(x[0], x[1]), __floats2bfloat162_rn(x[2], x[3])};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(y);
  }
}

template <typename T, int DH>
__global__ void __launch_bounds__(2 * Half<DH>::N) cache_read_kernel(const ReadArgs a) {
  using F = Half<DH>;
  constexpr int C4 = F::C4;
  __shared__ uint32_t s_v[DH * F::VP];
  const bool vals = threadIdx.x >= F::N;
  const int tid = vals ? threadIdx.x - F::N : threadIdx.x, c4 = tid % C4, word = tid / C4;
  const int h = blockIdx.y, g = blockIdx.z;
  const int cap = a.c.n_blocks * kCacheBlock;
  int len = a.c.lens[g], start = a.start ? a.start[g] : 0;
  len = len < 0 ? 0 : len > cap ? cap : len;
  start = start < 0 ? 0 : start;
  const long base = ((long)(start / kCacheBlock) + blockIdx.x) * kCacheBlock;
  if (base >= (long)start + a.n_rows) return;
  const bool any = base < len;
  const size_t rec = ((size_t)g * a.c.n_heads + h) * a.c.n_blocks + (any ? base / kCacheBlock : 0);
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(a.c.codes + rec * (size_t)(2 * kCacheBlock * DH)) + (vals ? kCacheBlock * C4 : 0);
  uint32_t w[4] = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
  const float step = any ? a.c.scales[rec * 2 + vals] : 0.0f;
  if (any) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = codes[tid + i * F::N];
  }
  if (vals) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = tid + i * F::N;
      s_v[(at / 16) * F::VP + at % 16] = w[i];
    }
  }
  __syncthreads();
  if (vals) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = s_v[(c4 * 4 + i) * F::VP + word];
    turn(w);
  }
  T* out = reinterpret_cast<T*>(vals ? a.v : a.k) + ((size_t)g * a.c.n_heads + h) * a.n_rows * DH + c4 * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = vals ? first_row(word) + (i & 1) + 8 * (i >> 1) : word + 16 * i;
    const long at = base + row - start;
    if (at < 0 || at >= a.n_rows) continue;
    float x[4];
    code_values(w[i], x);
    const bool live = base + row < len;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = live ? x[j] * step : 0.0f;
    store4<T>(out + at * DH, x);
  }
}

template <template <typename, int> class Launch, typename A>
int by_type_and_size(int dtype, int head_dim, const A& a, dim3 grid, cudaStream_t s) {
  if (dtype == ARTAB_F32) {
    if (head_dim == 16) return Launch<float, 16>::go(a, grid, s);
    if (head_dim == 32) return Launch<float, 32>::go(a, grid, s);
    return Launch<float, 64>::go(a, grid, s);
  }
  if (head_dim == 16) return Launch<__nv_bfloat16, 16>::go(a, grid, s);
  if (head_dim == 32) return Launch<__nv_bfloat16, 32>::go(a, grid, s);
  return Launch<__nv_bfloat16, 64>::go(a, grid, s);
}
template <typename T, int DH>
struct LaunchWrite {
  static int go(const WriteArgs& a, dim3 grid, cudaStream_t s) {
    count_launch();
    if (a.fresh)
      cache_write_kernel<T, DH, true><<<grid, 2 * Half<DH>::N, 0, s>>>(a);
    else
      cache_write_kernel<T, DH, false><<<grid, 2 * Half<DH>::N, 0, s>>>(a);
    return check_launch("cache_write");
  }
};
template <typename T, int DH>
struct LaunchAppendRow {
  static int go(const WriteArgs& a, dim3 grid, cudaStream_t s) {
    count_launch();
    cache_append_row_kernel<T, DH><<<grid, a.by_group ? 32 * a.c.n_heads : 128, 0, s>>>(a);
    return check_launch("cache_append_row");
  }
};
template <typename T, int DH>
struct LaunchRead {
  static int go(const ReadArgs& a, dim3 grid, cudaStream_t s) {
    count_launch();
    cache_read_kernel<T, DH><<<grid, 2 * Half<DH>::N, 0, s>>>(a);
    return check_launch("cache_read");
  }
};

}  // namespace

int check_cache(const artab_cache* c, const char* what) {
  ARTAB_REQUIRE(c && c->codes && c->scales && c->bounds && c->lens, ARTAB_EINVAL, "%s: null pointer", what);
  ARTAB_REQUIRE(c->head_dim == 16 || c->head_dim == 32 || c->head_dim == 64, ARTAB_EINVAL,
                "%s: head_dim %d not supported (16, 32, 64)", what, c->head_dim);
  ARTAB_REQUIRE(c->n_groups >= 1 && c->n_groups <= 65535 && c->n_heads >= 1 && c->n_heads <= 65535 && c->n_blocks >= 1 &&
                    c->n_blocks <= kMostRows / kCacheBlock,
                ARTAB_EINVAL, "%s: bad cache sizes", what);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(c->codes) | reinterpret_cast<uintptr_t>(c->bounds);
  ARTAB_REQUIRE(bits % 16 == 0 && reinterpret_cast<uintptr_t>(c->scales) % 8 == 0, ARTAB_EINVAL,
                "%s: cache tensors must be 16-byte aligned", what);
  return ARTAB_OK;
}

}  // namespace artab

using namespace artab;

extern "C" {

int artab_cache_write(int dtype, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                      int n_rows, const int32_t* start, const int32_t* counts, int fresh, artab_cache* c,
                      void* stream) {
  int rc = check_cache(c, "cache_write");
  if (rc) return rc;
  ARTAB_REQUIRE(dtype == ARTAB_F32 || dtype == ARTAB_BF16, ARTAB_EINVAL, "cache_write: bad dtype %d", dtype);
  ARTAB_REQUIRE(k && v && n_rows >= 1 && n_rows <= kMostRows, ARTAB_EINVAL, "cache_write: bad number of rows");
  ARTAB_REQUIRE(!(fresh && start), ARTAB_EINVAL, "cache_write: a fresh cache starts at row 0");
  ARTAB_REQUIRE(!fresh || (n_rows + kCacheBlock - 1) / kCacheBlock <= c->n_blocks, ARTAB_ECAPACITY,
                "cache_write: %d rows in a cache of %d", n_rows, c->n_blocks * kCacheBlock);
  cudaStream_t s = (cudaStream_t)stream;
  WriteArgs a;
  a.c = *c;
  a.k = row_view(k, k_strides, c->n_heads, n_rows, c->head_dim);
  a.v = row_view(v, v_strides, c->n_heads, n_rows, c->head_dim);
  a.start = fresh ? nullptr : start ? start : c->lens;
  a.counts = counts;
  a.n_rows = n_rows;
  a.fresh = fresh != 0;
  // rows counted from lens itself: every CTA still reads it, a second launch moves it
  const auto reads_lens = [c](const int32_t* p) { return p && p < c->lens + c->n_groups && p + c->n_groups > c->lens; };
  a.set_lens = !reads_lens(a.start) && !reads_lens(counts);
  ARTAB_REQUIRE(a.set_lens || ((!reads_lens(a.start) || a.start == c->lens) && (!reads_lens(counts) || counts == c->lens)),
                ARTAB_EINVAL, "cache_write: start / counts overlap the lengths of the cache");
  const int elem = dtype == ARTAB_F32 ? 4 : 2;
  a.vec_k = rows_aligned(a.k, elem);
  a.vec_v = rows_aligned(a.v, elem);
  long nb = fresh ? c->n_blocks : (n_rows + 2L * kCacheBlock - 2) / kCacheBlock;   // n rows from anywhere in a block
  if (nb > c->n_blocks) nb = c->n_blocks;
  // several blocks a CTA once there are many: the rows of the next are on their way while one is worked on
  const long all = nb * c->n_heads * c->n_groups;
  a.per_cta = !fresh || all / (148L * 16) < 1 ? 1 : all / (148L * 16) > 8 ? 8 : (int)(all / (148L * 16));
  a.by_group = !fresh && n_rows == 1 && !a.set_lens && c->n_heads <= kGroupHeads;
  if (!fresh && n_rows == 1)
    rc = by_type_and_size<LaunchAppendRow>(dtype, c->head_dim, a,
                                           dim3(a.by_group ? c->n_groups : (unsigned)(((long)c->n_groups * c->n_heads + 3) / 4)), s);
  else
    rc = by_type_and_size<LaunchWrite>(dtype, c->head_dim, a,
                                       dim3((unsigned)((nb + a.per_cta - 1) / a.per_cta), c->n_heads, c->n_groups), s);
  if (rc || a.set_lens || a.by_group) return rc;
  count_launch();
  cache_advance_kernel<<<(c->n_groups + 255) / 256, 256, 0, s>>>(a);
  return check_launch("cache_advance");
}

int artab_cache_read(int dtype, const artab_cache* c, const int32_t* start, int n_rows, void* k, void* v, void* stream) {
  int rc = check_cache(c, "cache_read");
  if (rc) return rc;
  ARTAB_REQUIRE(dtype == ARTAB_F32 || dtype == ARTAB_BF16, ARTAB_EINVAL, "cache_read: bad dtype %d", dtype);
  ARTAB_REQUIRE(k && v && n_rows >= 1 && n_rows <= kMostRows, ARTAB_EINVAL, "cache_read: bad number of rows");
  ARTAB_REQUIRE((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0, ARTAB_EINVAL,
                "cache_read: outputs must be 16-byte aligned");
  ReadArgs a;
  a.c = *c;
  a.start = start;
  a.n_rows = n_rows;
  a.k = k;
  a.v = v;
  const long nb = (n_rows + kCacheBlock - 1L) / kCacheBlock + (start ? 1 : 0);
  return by_type_and_size<LaunchRead>(dtype, c->head_dim, a, dim3((unsigned)nb, c->n_heads, c->n_groups),
                                      (cudaStream_t)stream);
}

}  // extern "C"
