// Writing rows into the 8-bit context cache, and reading them back.
//
// write: one CTA per (group, head, touched block).  The scale of a block is its largest magnitude / 127; rows that
// come behind others of a block may raise it, and the older rows are then rounded again to the new step.  Code
// of x: the whole number nearest to x / scale in exact arithmetic, ties to even.  It is taken from a product with
// the reciprocal in fp32; that is off by less than 3e-5, so where it lies closer than 5e-5 to a tie the quotient is
// formed in 64 bits (once in 10 000 elements).
// Both kernels move each byte once and are bounded by HBM for whole contexts, by one launch for a few rows.
#include "cache8.cuh"

namespace artab {
namespace {

constexpr int kWriteThreads = 256;

struct WriteArgs {
  artab_cache c;
  RowView k, v;
  const int32_t* start;    // [G], or null: 0
  const int32_t* counts;   // [G], or null: n_rows
  int n_rows;
  int fresh;               // the whole cache is laid out: every block of it is given scales and bounds
  int set_lens;            // lens[g] = end of the rows written here
  int vec_k, vec_v;
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

__device__ __forceinline__ int nearest_code(float x, float scale, float inv) {
  const float f = x * inv;
  float c = rintf(f);
  if (!(fabsf(f - c) < 0.49995f)) c = (float)rint((double)x / (double)scale);
  return (int)fminf(fmaxf(c, -127.0f), 127.0f);
}
__device__ __forceinline__ int moved_code(int code, float was, float scale, float inv) {
  const float f = (float)code * was * inv;
  float c = rintf(f);
  if (!(fabsf(f - c) < 0.49995f)) c = (float)rint((double)code * (double)was / (double)scale);
  return (int)fminf(fmaxf(c, -127.0f), 127.0f);
}
__device__ __forceinline__ float step_of(uint32_t top_bits) {
  return top_bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __fdiv_rn(__uint_as_float(top_bits), 127.0f);
}
// a block with a value that is not finite has NaN for its scale, for good
__device__ __forceinline__ float larger_step(float a, float b) { return a != a ? a : b != b ? b : fmaxf(a, b); }

template <typename T, int DH>
__global__ void __launch_bounds__(kWriteThreads) cache_write_kernel(const WriteArgs a) {
  constexpr int C4 = DH / 4;                       // four-channel pieces of a row
  constexpr int NC = kCacheBlock * C4 / kWriteThreads;
  constexpr int VP = kCacheBlock + 4;              // padded value channel: byte stores of a warp spread over the banks
  __shared__ __align__(16) uint8_t s_k[kCacheBlock * DH];
  __shared__ __align__(16) uint8_t s_v[DH * VP];
  __shared__ uint32_t s_top[2][8];
  __shared__ uint32_t s_lo[8][C4], s_hi[8][C4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.y, g = blockIdx.z;
  int start, end;
  write_range(a, g, start, end);
  if (a.set_lens && blockIdx.x == 0 && h == 0 && tid == 0) a.c.lens[g] = end;
  const int blk = a.fresh ? (int)blockIdx.x : start / kCacheBlock + (int)blockIdx.x;
  if (blk >= a.c.n_blocks) return;
  const int base = blk * kCacheBlock;
  const size_t rec = ((size_t)g * a.c.n_heads + h) * a.c.n_blocks + blk;
  float* scales = a.c.scales + rec * 2;
  __half* bounds = reinterpret_cast<__half*>(a.c.bounds) + rec * 2 * DH;
  if (end <= base) {                               // no row of this block
    if (a.fresh) {
      if (tid < 2) scales[tid] = 0.0f;
      if (tid < 2 * DH) bounds[tid] = __float2half(0.0f);
    }
    return;
  }
  uint8_t* codes = a.c.codes + rec * (size_t)(2 * kCacheBlock * DH);
  const int n_old = start > base ? start - base : 0;     // rows that are there already
  const int n_live = end - base < kCacheBlock ? end - base : kCacheBlock;
  const T* k0 = reinterpret_cast<const T*>(a.k.p) + g * a.k.s0 + h * a.k.s1;
  const T* v0 = reinterpret_cast<const T*>(a.v.p) + g * a.v.s0 + h * a.v.s1;
  const int c4 = tid % C4;
  float x[2][NC][4];
  uint32_t top_k = 0, top_v = 0;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int row = (tid + i * kWriteThreads) / C4;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[0][i][j] = x[1][i][j] = 0.0f;
    if (row >= n_old && row < n_live) {
      const long src = base + row - start;
      load_elements<T, 4>(k0 + src * a.k.s2 + c4 * 4, a.vec_k, x[0][i]);
      load_elements<T, 4>(v0 + src * a.v.s2 + c4 * 4, a.vec_v, x[1][i]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {                  // magnitudes order like their bit patterns, NaN above all
      top_k = max(top_k, __float_as_uint(x[0][i][j]) & 0x7fffffffu);
      top_v = max(top_v, __float_as_uint(x[1][i][j]) & 0x7fffffffu);
    }
  }
  top_k = __reduce_max_sync(0xffffffffu, top_k);
  top_v = __reduce_max_sync(0xffffffffu, top_v);
  if (lane == 0) s_top[0][warp] = top_k, s_top[1][warp] = top_v;
  const float was_k = n_old ? scales[0] : 0.0f, was_v = n_old ? scales[1] : 0.0f;
  __syncthreads();
  top_k = top_v = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) top_k = max(top_k, s_top[0][w]), top_v = max(top_v, s_top[1][w]);
  const float ks = larger_step(was_k, step_of(top_k)), vs = larger_step(was_v, step_of(top_v));
  // a step of zero (or NaN) has zero codes: the reciprocal is then zero and no quotient is formed
  const float ki = ks > 0.0f ? 1.0f / ks : 0.0f, vi = vs > 0.0f ? 1.0f / vs : 0.0f;
  uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int row = (tid + i * kWriteThreads) / C4;
    uint32_t wk = 0x80808080u, wv = 0x80808080u;
    if (row < n_old) {
      wk = *reinterpret_cast<const uint32_t*>(codes + row * DH + c4 * 4);
      wv = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        wv |= (uint32_t)codes[kCacheBlock * DH + (c4 * 4 + j) * kCacheBlock + cache_value_place(row)] << (8 * j);
      if (ks > was_k) {
        uint32_t y = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          y |= (uint32_t)(moved_code((int)((wk >> (8 * j)) & 255u) - 128, was_k, ks, ki) + 128) << (8 * j);
        wk = y;
      }
      if (vs > was_v) {
        uint32_t y = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          y |= (uint32_t)(moved_code((int)((wv >> (8 * j)) & 255u) - 128, was_v, vs, vi) + 128) << (8 * j);
        wv = y;
      }
    } else if (row < n_live) {
      wk = wv = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        wk |= (uint32_t)((ks > 0.0f ? nearest_code(x[0][i][j], ks, ki) : 0) + 128) << (8 * j);
        wv |= (uint32_t)((vs > 0.0f ? nearest_code(x[1][i][j], vs, vi) : 0) + 128) << (8 * j);
      }
    }
    if (row < n_live) lo = __vminu4(lo, wk), hi = __vmaxu4(hi, wk);
    *reinterpret_cast<uint32_t*>(s_k + row * DH + c4 * 4) = wk;
#pragma unroll
    for (int j = 0; j < 4; ++j) s_v[(c4 * 4 + j) * VP + cache_value_place(row)] = (uint8_t)(wv >> (8 * j));
  }
#pragma unroll
  for (int o = C4; o < 32; o <<= 1) {
    lo = __vminu4(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = __vmaxu4(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (lane < C4) s_lo[warp][lane] = lo, s_hi[warp][lane] = hi;
  __syncthreads();   // also: every thread has read the old codes and scales
#pragma unroll
  for (int i = tid; i < kCacheBlock * DH / 16; i += kWriteThreads)
    reinterpret_cast<uint4*>(codes)[i] = reinterpret_cast<const uint4*>(s_k)[i];
#pragma unroll
  for (int i = tid; i < kCacheBlock * DH / 4; i += kWriteThreads)
    reinterpret_cast<uint32_t*>(codes + kCacheBlock * DH)[i] =
        *reinterpret_cast<const uint32_t*>(s_v + (i / 16) * VP + (i % 16) * 4);
  if (tid < C4) {
#pragma unroll
    for (int w = 0; w < 8; ++w) lo = __vminu4(w ? lo : s_lo[0][tid], s_lo[w][tid]), hi = __vmaxu4(w ? hi : s_hi[0][tid], s_hi[w][tid]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bounds[tid * 4 + j] = __int2half_rn((int)((lo >> (8 * j)) & 255u) - 128);
      bounds[DH + tid * 4 + j] = __int2half_rn((int)((hi >> (8 * j)) & 255u) - 128);
    }
  }
  if (tid == 0) scales[0] = ks, scales[1] = vs;
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

template <typename T, int DH>
__global__ void __launch_bounds__(kWriteThreads) cache_read_kernel(const ReadArgs a) {
  constexpr int C4 = DH / 4, NC = kCacheBlock * C4 / kWriteThreads, VP = kCacheBlock + 4;
  __shared__ __align__(16) uint8_t s_v[DH * VP];
  const int tid = threadIdx.x, h = blockIdx.y, g = blockIdx.z;
  const int cap = a.c.n_blocks * kCacheBlock;
  int len = a.c.lens[g], start = a.start ? a.start[g] : 0;
  len = len < 0 ? 0 : len > cap ? cap : len;
  start = start < 0 ? 0 : start;
  const long base = ((long)(start / kCacheBlock) + blockIdx.x) * kCacheBlock;
  if (base >= (long)start + a.n_rows) return;
  const size_t out0 = ((size_t)g * a.c.n_heads + h) * a.n_rows;
  const bool any = base < len;
  const size_t rec = ((size_t)g * a.c.n_heads + h) * a.c.n_blocks + (any ? base / kCacheBlock : 0);
  const uint8_t* codes = a.c.codes + rec * (size_t)(2 * kCacheBlock * DH);
  float ks = 0.0f, vs = 0.0f;
  uint32_t wk[NC];
  if (any) {
    ks = a.c.scales[rec * 2], vs = a.c.scales[rec * 2 + 1];
#pragma unroll
    for (int i = 0; i < NC; ++i) wk[i] = reinterpret_cast<const uint32_t*>(codes)[tid + i * kWriteThreads];
#pragma unroll
    for (int i = tid; i < kCacheBlock * DH / 4; i += kWriteThreads)
      *reinterpret_cast<uint32_t*>(s_v + (i / 16) * VP + (i % 16) * 4) =
          reinterpret_cast<const uint32_t*>(codes + kCacheBlock * DH)[i];
  }
  __syncthreads();
  const int c4 = tid % C4;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int row = (tid + i * kWriteThreads) / C4;
    const long at = base + row - start;
    if (at < 0 || at >= a.n_rows) continue;
    float k[4] = {0.0f, 0.0f, 0.0f, 0.0f}, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (base + row < len) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        k[j] = (float)((int)((wk[i] >> (8 * j)) & 255u) - 128) * ks;
        v[j] = (float)((int)s_v[(c4 * 4 + j) * VP + cache_value_place(row)] - 128) * vs;
      }
    }
    const size_t o = (out0 + (size_t)at) * DH + c4 * 4;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.k) + o) = make_float4(k[0], k[1], k[2], k[3]);
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.v) + o) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      __nv_bfloat162 p[2] = {__floats2bfloat162_rn(k[0], k[1]), __floats2bfloat162_rn(k[2], k[3])};
      __nv_bfloat162 r[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
      *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.k) + o) = *reinterpret_cast<uint2*>(p);
      *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.v) + o) = *reinterpret_cast<uint2*>(r);
    }
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
    cache_write_kernel<T, DH><<<grid, kWriteThreads, 0, s>>>(a);
    return check_launch("cache_write");
  }
};
template <typename T, int DH>
struct LaunchRead {
  static int go(const ReadArgs& a, dim3 grid, cudaStream_t s) {
    count_launch();
    cache_read_kernel<T, DH><<<grid, kWriteThreads, 0, s>>>(a);
    return check_launch("cache_read");
  }
};

}  // namespace

int check_cache(const artab_cache* c, const char* what) {
  ARTAB_REQUIRE(c && c->codes && c->scales && c->bounds && c->lens, ARTAB_EINVAL, "%s: null pointer", what);
  ARTAB_REQUIRE(c->head_dim == 16 || c->head_dim == 32 || c->head_dim == 64, ARTAB_EINVAL,
                "%s: head_dim %d not supported (16, 32, 64)", what, c->head_dim);
  ARTAB_REQUIRE(c->n_groups >= 1 && c->n_groups <= 65535 && c->n_heads >= 1 && c->n_heads <= 65535 && c->n_blocks >= 1 &&
                    c->n_blocks <= (1 << 24),
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
  ARTAB_REQUIRE(k && v && k_strides && v_strides && n_rows >= 1, ARTAB_EINVAL, "cache_write: no rows");
  ARTAB_REQUIRE(!(fresh && start), ARTAB_EINVAL, "cache_write: a fresh cache starts at row 0");
  ARTAB_REQUIRE(!fresh || (n_rows + kCacheBlock - 1) / kCacheBlock <= c->n_blocks, ARTAB_ECAPACITY,
                "cache_write: %d rows in a cache of %d", n_rows, c->n_blocks * kCacheBlock);
  cudaStream_t s = (cudaStream_t)stream;
  WriteArgs a;
  a.c = *c;
  a.k = {k, (long)k_strides[0], (long)k_strides[1], (long)k_strides[2]};
  a.v = {v, (long)v_strides[0], (long)v_strides[1], (long)v_strides[2]};
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
  rc = by_type_and_size<LaunchWrite>(dtype, c->head_dim, a, dim3((unsigned)nb, c->n_heads, c->n_groups), s);
  if (rc || a.set_lens) return rc;
  count_launch();
  cache_advance_kernel<<<(c->n_groups + 255) / 256, 256, 0, s>>>(a);
  return check_launch("cache_advance");
}

int artab_cache_read(int dtype, const artab_cache* c, const int32_t* start, int n_rows, void* k, void* v, void* stream) {
  int rc = check_cache(c, "cache_read");
  if (rc) return rc;
  ARTAB_REQUIRE(dtype == ARTAB_F32 || dtype == ARTAB_BF16, ARTAB_EINVAL, "cache_read: bad dtype %d", dtype);
  ARTAB_REQUIRE(k && v && n_rows >= 1, ARTAB_EINVAL, "cache_read: no rows");
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
