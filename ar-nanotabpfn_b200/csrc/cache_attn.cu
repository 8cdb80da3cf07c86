// Attention of queries over the 8-bit context cache, all of its rows or a list of blocks per query.
//
//   out = sum_n exp(s_n) v_n / sum_n exp(s_n),  s_n = scale * ks * (q . (k code)),  v_n = vs * (v code),  lse = log sum_n exp(s_n)
//
// The scales of a block are factors of whole products, so codes go to the tensor cores as the whole numbers they are
// (exact in half precision) and nothing is rounded on the way but the other operand: queries and softmax numerators
// are taken in two half-precision parts (22 bits, both types of input; PARTS = 2) or one (bf16 inputs; PARTS = 1: a bf16
// query is exact in it, numerators keep 11 bits where bf16 would keep 8).  Sums, maxima and outputs are fp32.
//
// cache_attn_kernel: the codes are the 16-row operand, the queries the 8 columns.  PARTS = 2: four queries, column
// 2 r + p is part p of query r, and a thread holds both parts of a score of its own query t.  PARTS = 1: eight
// queries.  Numerators become the second product's columns by one 8 x 8 transposition per 8 rows.  Each warp
// walks blocks of its own with a running maximum; its ring of records is filled by 16-byte asynchronous copies
// and no warp waits for another until the end, where the warps of a CTA and the CTAs of a cluster (up to eight
// share the rows of a context) merge maximum, sum and output through shared memory.
#include <math_constants.h>

#include "cache8.cuh"
#include "cluster.cuh"

namespace artab {
namespace {

constexpr int kWarps = 8;

struct AttnArgs {
  artab_cache c;
  RowView q;
  int n_streams, n_q;
  int rows;               // query rows of a group
  int tiles;              // tiles of a group's rows
  long units;             // (group, head, tile) or (stream, head, query)
  int splits;             // CTAs of a cluster
  const int32_t* list;    // [B][H][Lq][n_list], or null: every block
  int n_list;
  float scale_log2;       // scale * log2 e
  int vec_q;
  void* out;              // [B][H][Lq][Dh]
  float* lse;             // [B][H][Lq]
};

// numerators are 2^14 times exp(s - max): halves keep 11 bits of them down to 2^-28 of the largest
constexpr float kLift = 14.0f;

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
          o[md][j][r] = fmaf(o[md][j][r], alpha[r], vs * (PARTS == 2 ? c[2 * j] + c[2 * j + 1] : c[2 * j + r]));
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

template <int DH>
struct Ring {
  static constexpr int kRecord = 2 * kCacheBlock * DH;
  static constexpr int kStages = DH == 64 ? 2 : 3;
  static constexpr int kBytes = kStages * (kRecord + 16);
};

// Partial results of a CTA's warps and of the cluster's CTAs: [row][DH + 2] (output not yet divided, maximum, sum)
template <int DH, int PARTS>
constexpr int partial_floats() {
  return Tile<DH, PARTS>::ROWS * (DH + 2);
}

template <typename T, int DH, int PARTS, bool LIST>
__global__ void __launch_bounds__(kWarps * 32) cache_attn_kernel(const AttnArgs a) {
  using R = Ring<DH>;
  using Tl = Tile<DH, PARTS>;
  constexpr int ROWS = LIST ? 1 : Tl::ROWS, P = DH + 2;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int rank = (int)(blockIdx.x % a.splits);
  const long unit = blockIdx.x / a.splits;
  const int H = a.c.n_heads;
  int group, h, row0, n_rows;
  if (LIST) {
    h = (int)(unit / a.n_q % H);
    const int b = (int)(unit / a.n_q / H);
    group = a.c.n_groups == 1 ? 0 : b;
    row0 = (a.c.n_groups == 1 ? b * a.n_q : 0) + (int)(unit % a.n_q);
    n_rows = row0 + 1;
  } else {
    row0 = (int)(unit % a.tiles) * ROWS;
    h = (int)(unit / a.tiles % H);
    group = (int)(unit / a.tiles / H);
    n_rows = a.rows;
  }
  const bool one = a.c.n_groups == 1;
  const auto stream_of = [&](int row) { return one ? row / a.n_q : group; };
  const auto query_of = [&](int row) { return one ? row % a.n_q : row; };

  int len = a.c.lens[group];
  const int cap = a.c.n_blocks * kCacheBlock;
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int held = (len + kCacheBlock - 1) / kCacheBlock;
  const int n = LIST ? a.n_list : held;                      // blocks of the unit
  const int32_t* list = LIST ? a.list + unit * a.n_list : nullptr;
  const size_t gh = (size_t)group * H + h;
  const uint8_t* codes = a.c.codes + gh * a.c.n_blocks * (size_t)R::kRecord;
  const float* scales = a.c.scales + gh * a.c.n_blocks * 2;

  uint8_t* ring = smem + warp * R::kBytes;
  const uint32_t ring_addr = smem_u32(ring);
  const int first = rank * kWarps + warp, step = a.splits * kWarps;
  const auto block_of = [&](int i) {                          // -1: nothing there
    if (i >= n) return -1;
    if (!LIST) return i;
    const int b = list[i];
    return b < 0 || b >= held ? -1 : b;
  };
  const auto fetch = [&](int blk, int stage) {
    if (blk >= 0) {
      const uint8_t* src = codes + (size_t)blk * R::kRecord;
      const uint32_t dst = ring_addr + stage * R::kRecord;
#pragma unroll
      for (int i = 0; i < R::kRecord / 512; ++i) cache_cp16(dst + (i * 32 + lane) * 16, src + (i * 32 + lane) * 16);
      if (lane == 0) cache_cp8(ring_addr + R::kStages * R::kRecord + stage * 16, scales + (size_t)blk * 2);
    }
    cp_commit();
  };
  int ahead[R::kStages - 1];
#pragma unroll
  for (int i = 0; i < R::kStages - 1; ++i) {
    ahead[i] = block_of(first + i * step);
    fetch(ahead[i], i);
  }
  Tl tile;
  tile.reset();
  {
    const int row = row0 + g / PARTS;
    const bool there = LIST ? g / PARTS == 0 : row < n_rows;
    const T* q = reinterpret_cast<const T*>(a.q.p) + stream_of(row) * a.q.s0 + h * a.q.s1 + query_of(row) * a.q.s2;
    tile.template load_queries<T>(there ? q : nullptr, a.vec_q, a.scale_log2);
  }
  int stage = 0;
  for (int i = first; i < n; i += step) {
    const int next = block_of(i + (R::kStages - 1) * step);
    fetch(next, stage == 0 ? R::kStages - 1 : stage - 1);
    cp_wait<R::kStages - 1>();
    __syncwarp();
    const int blk = ahead[0];
    if (blk >= 0) {
      const float2 sc = *reinterpret_cast<const float2*>(ring + R::kStages * R::kRecord + stage * 16);
      const int live = len - blk * kCacheBlock;
      tile.block(ring + stage * R::kRecord, sc.x, sc.y, live < kCacheBlock ? live : kCacheBlock);
    }
    __syncwarp();   // the stage is free for the next copy
#pragma unroll
    for (int j = 0; j + 1 < R::kStages - 1; ++j) ahead[j] = ahead[j + 1];
    ahead[R::kStages - 2] = next;
    stage = stage + 1 == R::kStages ? 0 : stage + 1;
  }
  cp_wait<0>();
  __syncthreads();

  // the warps' results, then the CTA's
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int r = 0; r < Tl::R; ++r) {
    float l = tile.l[r];
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const int row = PARTS == 2 ? t : 2 * t + r;
    if (row < ROWS) {
      float* to = part + (warp * ROWS + row) * P;
#pragma unroll
      for (int md = 0; md < Tl::KS; ++md)
#pragma unroll
        for (int j = 0; j < 2; ++j) to[16 * md + 8 * j + g] = tile.o[md][j][r];
      if (g == 0) to[DH] = tile.m[r], to[DH + 1] = l;
    }
  }
  __syncthreads();
  float* mine = part + kWarps * ROWS * P;
  const auto merge = [&](auto at, int count, int e, float& m, float& l, float& o) {
    const int row = e / DH, d = e % DH;
    m = -CUDART_INF_F;
    for (int w = 0; w < count; ++w) m = fmaxf(m, at(w, row * P + DH));
    const float base = m == -CUDART_INF_F ? 0.0f : m;
    l = 0.0f, o = 0.0f;
    for (int w = 0; w < count; ++w) {
      const float x = ex2(at(w, row * P + DH) - base);
      l = fmaf(at(w, row * P + DH + 1), x, l);
      o = fmaf(at(w, row * P + d), x, o);
    }
  };
  const auto store = [&](int e, float m, float l, float o) {
    const int row = row0 + e / DH, d = e % DH;
    if (row >= n_rows) return;
    const size_t at = ((size_t)stream_of(row) * H + h) * a.n_q + query_of(row);
    reinterpret_cast<T*>(a.out)[at * DH + d] = from_f32<T>(l == 0.0f ? 0.0f : o / l);
    if (d == 0) a.lse[at] = l == 0.0f ? -CUDART_INF_F : (m - kLift) * kLn2 + logf(l);
  };
  for (int e = tid; e < ROWS * DH; e += kWarps * 32) {
    float m, l, o;
    merge([&](int w, int i) { return part[w * ROWS * P + i]; }, kWarps, e, m, l, o);
    if (a.splits == 1) {
      store(e, m, l, o);
    } else {
      mine[e / DH * P + e % DH] = o;
      if (e % DH == 0) mine[e / DH * P + DH] = m, mine[e / DH * P + DH + 1] = l;
    }
  }
  if (a.splits == 1) return;
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const uint32_t base = smem_u32(mine);
  for (int e = rank * kWarps * 32 + tid; e < ROWS * DH; e += a.splits * kWarps * 32) {
    float m, l, o;
    merge([&](int w, int i) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_rank(base + i * 4, w)) : "memory");
      return v;
    }, a.splits, e, m, l, o);
    store(e, m, l, o);
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, int DH, int PARTS, bool LIST>
int launch(const AttnArgs& a, cudaStream_t s) {
  static SmemConfig config;
  const auto kernel = cache_attn_kernel<T, DH, PARTS, LIST>;
  const size_t part = (size_t)(kWarps + 1) * partial_floats<DH, PARTS>() * sizeof(float);
  const size_t ring = (size_t)kWarps * Ring<DH>::kBytes;
  const size_t smem = part > ring ? part : ring;
  cudaError_t e = config.ensure(kernel, smem, true);
  ARTAB_REQUIRE(e == cudaSuccess, ARTAB_ELAUNCH, "cache_attention: %s", cudaGetErrorString(e));
  ARTAB_REQUIRE(a.units * a.splits <= 0x7fffffffL, ARTAB_EINVAL, "cache_attention: too many query rows");
  PlainLaunchScope plain;
  count_launch();
  e = launch_dependent_cluster(kernel, dim3((unsigned)(a.units * a.splits)), dim3(kWarps * 32), smem, s,
                               (unsigned)a.splits, a);
  ARTAB_REQUIRE(e == cudaSuccess, ARTAB_ELAUNCH, "cache_attention: %s", cudaGetErrorString(e));
  return ARTAB_OK;
}

template <typename T, int DH>
int by_form(AttnArgs& a, cudaStream_t s) {
  if (a.list) return launch<T, DH, 2, true>(a, s);
  if (sizeof(T) == 2 && a.rows > 4) {
    a.tiles = (a.rows + 7) / 8;
    a.units *= a.tiles;
    return launch<T, DH, 1, false>(a, s);
  }
  a.tiles = (a.rows + 3) / 4;
  a.units *= a.tiles;
  return launch<T, DH, 2, false>(a, s);
}

// CTAs that share the blocks of a unit: as many as fill the GPU twice, none without a block for every warp
int plan_splits(long units, long blocks) {
  int s = 1;
  while (s < 8 && units * s * 2 <= 2 * 148 && blocks >= 2L * s * kWarps) s *= 2;
  return s;
}

int attention(int dtype, const void* q, const int64_t* strides, int n_streams, int n_q, const artab_cache* c,
              int max_len, const int32_t* list, int n_list, float scale, void* out, float* lse, cudaStream_t s,
              const char* what) {
  int rc = check_cache(c, what);
  if (rc) return rc;
  rc = check_queries(dtype, q, strides, n_streams, n_q, c, what);
  if (rc) return rc;
  ARTAB_REQUIRE(out && lse, ARTAB_EINVAL, "%s: null pointer", what);
  AttnArgs a;
  a.c = *c;
  a.q = {q, (long)strides[0], (long)strides[1], (long)strides[2]};
  a.n_streams = n_streams;
  a.n_q = n_q;
  a.rows = c->n_groups == 1 ? n_streams * n_q : n_q;
  a.tiles = 1;
  a.list = list;
  a.n_list = n_list;
  a.scale_log2 = scale * kLog2e;
  a.vec_q = rows_aligned(a.q, dtype == ARTAB_F32 ? 4 : 2);
  a.out = out;
  a.lse = lse;
  a.units = list ? (long)n_streams * c->n_heads * n_q : (long)c->n_groups * c->n_heads;
  const long blocks = list ? n_list : (max_len + kCacheBlock - 1L) / kCacheBlock;
  const int per = list ? 1 : dtype == ARTAB_BF16 && a.rows > 4 ? 8 : 4;
  a.splits = plan_splits(list ? a.units : a.units * ((a.rows + per - 1) / per), blocks);
  if (dtype == ARTAB_F32) {
    if (c->head_dim == 16) return by_form<float, 16>(a, s);
    if (c->head_dim == 32) return by_form<float, 32>(a, s);
    return by_form<float, 64>(a, s);
  }
  if (c->head_dim == 16) return by_form<__nv_bfloat16, 16>(a, s);
  if (c->head_dim == 32) return by_form<__nv_bfloat16, 32>(a, s);
  return by_form<__nv_bfloat16, 64>(a, s);
}

}  // namespace

int check_queries(int dtype, const void* q, const int64_t* strides, int n_streams, int n_q, const artab_cache* c,
                  const char* what) {
  ARTAB_REQUIRE(dtype == ARTAB_F32 || dtype == ARTAB_BF16, ARTAB_EINVAL, "%s: bad dtype %d", what, dtype);
  ARTAB_REQUIRE(q && strides, ARTAB_EINVAL, "%s: null pointer", what);
  ARTAB_REQUIRE(n_streams >= 1 && n_q >= 1 && (long)n_streams * n_q <= (1L << 28), ARTAB_EINVAL, "%s: bad query sizes",
                what);
  ARTAB_REQUIRE(c->n_groups == 1 || c->n_groups == n_streams, ARTAB_EINVAL,
                "%s: %d contexts for %d streams (one, or one each)", what, c->n_groups, n_streams);
  return ARTAB_OK;
}

}  // namespace artab

using namespace artab;

extern "C" {

int artab_cache_attention(int dtype, const void* q, const int64_t* q_strides, int n_streams, int n_q,
                          const artab_cache* c, int max_len, float scale, void* out, float* lse, void* stream) {
  return attention(dtype, q, q_strides, n_streams, n_q, c, max_len, nullptr, 0, scale, out, lse, (cudaStream_t)stream,
                   "cache_attention");
}

int artab_cache_block_attention(int dtype, const void* q, const int64_t* q_strides, int n_streams, int n_q,
                                const artab_cache* c, const int32_t* blocks, int n_list, float scale, void* out,
                                float* lse, void* stream) {
  ARTAB_REQUIRE(blocks && n_list >= 1, ARTAB_EINVAL, "cache_block_attention: no blocks");
  return attention(dtype, q, q_strides, n_streams, n_q, c, 0, blocks, n_list, scale, out, lse, (cudaStream_t)stream,
                   "cache_block_attention");
}

}  // extern "C"
