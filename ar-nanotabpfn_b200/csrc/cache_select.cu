// For every query the blocks of the 8-bit context cache with the largest upper bound of a score.
//
// With the query rounded to whole numbers (largest magnitude -> 127) the bound over a block's rows is
//   ks * sum_d max(qi_d * lo_d, qi_d * hi_d) = ks * (max(qi, 0) . hi + min(qi, 0) . lo),
// lo / hi the smallest and largest key code of channel d.  The sum is a whole number below 2^21, formed exactly by
// half-precision products with fp32 sums whatever their order, and one fp32 product follows: the choice does not
// depend on tiling, and ties (broken by the lowest index) are real ties.
//
// One CTA = 16 queries of a (group, head): scores of all blocks into shared memory as ordered keys (products of
// 16 queries x 8 blocks a warp), then a warp takes two queries at a time, finds their n-th largest keys by bisection
// and writes the chosen indices in ascending order.  1024 queries x 6 heads x 256 blocks (B200): 12.4 us; one CTA alone takes 8.
// 384 CTAs fill the GPU once, with 53 % of the issue slots busy: each of some 15 steps of bisection counts every key of a row (eight
// compares and sums a lane, a reduction), behind a chain of loads and barriers.
#include "cache8.cuh"

namespace artab {
namespace {

constexpr int kThreads = 256, kRows = 16, kMaxBlocks = 3456;   // 16 rows of keys in 227 KB

struct SelectArgs {
  artab_cache c;
  RowView q;
  int n_q, rows, tiles, n_pick;
  int pitch;               // keys of a row
  int vec_q;
  int32_t* index;          // [B][H][Lq][n_pick]
};

constexpr int kHeld = 8;   // keys of a lane that are kept in registers: contexts of up to 16384 rows

// Finds the n-th largest of `held` keys (n < held; lanes i, i + 32, ... hold key i) by bisection between two values, `lo` with
// at least n keys from it on and `hi` with fewer, and writes the n indices chosen.  It ends when exactly n keys lie from lo
// on, or when lo is a key that is there several times.  A first lower value comes from the largest keys of the 32 lanes alone, at
// a vote a step: from their n-th on there are n keys, and few more.
struct Pick {
  uint32_t key[kHeld];
  const uint32_t* row;
  uint32_t lo, hi;
  int at_least;            // keys from lo on

  template <typename F>
  __device__ __forceinline__ int count(int held, F f) const {
    int n = 0;
    if (held <= 32 * kHeld) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) n += f(key[i]);
    } else {
      for (int i = threadIdx.x & 31; i < held; i += 32) n += f(row[i]);
    }
    return __reduce_add_sync(0xffffffffu, n);
  }
  __device__ __forceinline__ void start(const uint32_t* r, int held, int n) {
    const int lane = threadIdx.x & 31;
    row = r;
    uint32_t top = 0, least = 0xffffffffu;
    if (held <= 32 * kHeld) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        key[i] = i * 32 + lane < held ? r[i * 32 + lane] : 0u;       // 0: below every key
        top = max(top, key[i]);
      }
      least = lane < held ? top : 0xffffffffu;
    } else {
      for (int i = lane; i < held; i += 32) top = max(top, r[i]), least = min(least, r[i]);
      if (n <= 32) least = top;
    }
    hi = __reduce_max_sync(0xffffffffu, top) + 1u;
    lo = __reduce_min_sync(0xffffffffu, least);
    if (n > 32) {                                    // the lanes' own maxima tell nothing
      if (held <= 32 * kHeld) lo = 1u;
    } else {
      uint32_t above = hi;
      int lanes = min(held, 32);
      while (lanes > n && above - lo > 1u) {
        const uint32_t mid = lo + (above - lo) / 2;
        const int c = __popc(__ballot_sync(0xffffffffu, top >= mid));
        if (c >= n)
          lo = mid, lanes = c;
        else
          above = mid;
      }
    }
    const uint32_t from = lo;
    at_least = count(held, [from](uint32_t k) { return k >= from ? 1 : 0; });
  }
  __device__ __forceinline__ bool done(int n) const { return at_least == n || hi - lo == 1u; }
  __device__ __forceinline__ void narrow(int held, int n) {
    const uint32_t mid = lo + (hi - lo) / 2;
    const int c = count(held, [mid](uint32_t k) { return k >= mid ? 1 : 0; });
    if (c >= n)
      lo = mid, at_least = c;
    else
      hi = mid;
  }
  __device__ __forceinline__ void write(int held, int n, int32_t* out) const {
    const int lane = threadIdx.x & 31;
    const uint32_t below = (1u << lane) - 1u, last = lo;
    int done = 0;
    if (at_least == n) {                             // every key from lo on
      for (int i0 = 0; i0 < held && done < n; i0 += 32) {
        const bool take = i0 + lane < held && row[i0 + lane] >= last;
        const uint32_t taken = __ballot_sync(0xffffffffu, take);
        if (take) out[done + __popc(taken & below)] = i0 + lane;
        done += __popc(taken);
      }
      return;
    }
    // every key above lo, and the first of those equal to it
    int ties = n - count(held, [last](uint32_t k) { return k > last ? 1 : 0; });
    for (int i0 = 0; i0 < held && done < n; i0 += 32) {
      const bool there = i0 + lane < held;
      const uint32_t k = there ? row[i0 + lane] : 0u;
      const uint32_t tied = __ballot_sync(0xffffffffu, there && k == last);
      const bool take = there && (k > last || (k == last && __popc(tied & below) < ties));
      const uint32_t taken = __ballot_sync(0xffffffffu, take);
      if (take) out[done + __popc(taken & below)] = i0 + lane;
      ties -= min(ties, __popc(tied));
      done += __popc(taken);
    }
  }
};

template <typename T, int DH>
__global__ void __launch_bounds__(kThreads) cache_select_kernel(const SelectArgs a) {
  constexpr int KS = DH / 8;       // k steps over the 2 * DH products
  constexpr int NE = DH / 2;       // channels of a thread
  extern __shared__ __align__(16) uint32_t s_key[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int H = a.c.n_heads;
  const int tile = (int)(blockIdx.x % a.tiles), h = (int)(blockIdx.x / a.tiles % H);
  const int group = (int)(blockIdx.x / a.tiles / H), row0 = tile * kRows;
  const bool one = a.c.n_groups == 1;
  int len = a.c.lens[group];
  const int cap = a.c.n_blocks * kCacheBlock;
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int held = (len + kCacheBlock - 1) / kCacheBlock;
  const size_t gh = (size_t)group * H + h;

  // bounds and scales of a warp's eight blocks, asked for while those before them (at first: the queries) are worked on
  constexpr int kStep = kThreads / 32 * 8;
  const uint4* bounds = reinterpret_cast<const uint4*>(reinterpret_cast<const __half*>(a.c.bounds) + gh * a.c.n_blocks * 2 * DH + t * NE);
  const float* scales = a.c.scales + gh * a.c.n_blocks * 2;
  uint4 next[NE / 8];
  float next_ks[2];
  const auto load = [&](int j) {
    if (j >= held) return;
    const uint4* src = bounds + (size_t)min(j + g, held - 1) * (2 * DH / 8);
#pragma unroll
    for (int i = 0; i < NE / 8; ++i) next[i] = src[i];
#pragma unroll
    for (int e = 0; e < 2; ++e) next_ks[e] = scales[(size_t)min(j + 2 * t + e, held - 1) * 2];
  };
  load(warp * 8);
  // the queries as whole numbers, four channels a thread
  constexpr int C4 = DH / 4;
  __shared__ __align__(16) __half s_q[kRows][DH];
  for (int i = tid; i < kRows * C4; i += kThreads) {     // 64 - 256 pieces: whole warps
    const int row = row0 + i / C4, c4 = i % C4;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (row < a.rows) {
      const int b = one ? row / a.n_q : group, l = one ? row % a.n_q : row;
      load_elements<T, 4>(reinterpret_cast<const T*>(a.q.p) + b * a.q.s0 + h * a.q.s1 + l * a.q.s2 + c4 * 4, a.vec_q, x);
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < C4; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float step = top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top), 127.0f) : 0.0f;  // not finite: all zero
    const uint32_t w = step > 0.0f ? codes_of(x, step, 1.0f / step) : 0x80808080u;
    *reinterpret_cast<uint2*>(&s_q[i / C4][c4 * 4]) = make_uint2(codes_to_halves(w, false), codes_to_halves(w, true));
  }
  __syncthreads();
  // thread t < 2: negative parts of channels t * NE .., for the lower bounds; t >= 2: positive parts, upper bounds
  uint32_t qa[KS][4];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint2 v = *reinterpret_cast<const uint2*>(&s_q[g + 8 * half][(t & 1) * NE + 4 * s]);
      const __half2 zero = __float2half2_rn(0.0f);
      const __half2 x = *reinterpret_cast<const __half2*>(&v.x), y = *reinterpret_cast<const __half2*>(&v.y);
      qa[s][half] = h2_bits(t < 2 ? __hmin2(x, zero) : __hmax2(x, zero));
      qa[s][2 + half] = h2_bits(t < 2 ? __hmin2(y, zero) : __hmax2(y, zero));
    }
  for (int j = warp * 8; j < held; j += kStep) {
    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f}, ks[2] = {next_ks[0], next_ks[1]};
    uint32_t w[KS][2];
#pragma unroll
    for (int i = 0; i < NE / 8; ++i)
      w[2 * i][0] = next[i].x, w[2 * i][1] = next[i].y, w[2 * i + 1][0] = next[i].z, w[2 * i + 1][1] = next[i].w;
    load(j + kStep);
#pragma unroll
    for (int s = 0; s < KS; ++s) mma_f16(c, qa[s][0], qa[s][1], qa[s][2], qa[s][3], w[s][0], w[s][1]);
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = j + 2 * t + e;
      if (col >= held) continue;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // a block whose scale is not a number ranks first: what is wrong with it shows in the output
        const float v = ks[e] == ks[e] ? c[2 * half + e] * ks[e] : __uint_as_float(0x7f800000u);
        const uint32_t bits = __float_as_uint(v + 0.0f);   // -0 -> 0: equal scores have equal keys
        s_key[(g + 8 * half) * a.pitch + col] = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
      }
    }
  }
  __syncthreads();
  // two queries a warp, side by side: the steps of one hide in the latencies of the other
  Pick pick[2];
  int32_t* out[2];
  const int n = a.n_pick;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = row0 + 2 * warp + i;
    const int b = one ? row / a.n_q : group, l = one ? row % a.n_q : row;
    out[i] = row < a.rows ? a.index + (((size_t)b * H + h) * a.n_q + l) * n : nullptr;
  }
  if (!out[0]) return;
  if (held > n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) pick[i].start(s_key + (2 * warp + i) * a.pitch, held, n);   // of a row of zeros, if need be
    while (!pick[0].done(n) || !pick[1].done(n)) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (!pick[i].done(n)) pick[i].narrow(held, n);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (!out[i]) continue;
    if (held > n) {
      pick[i].write(held, n, out[i]);
    } else {
      for (int j = lane; j < n; j += 32) out[i][j] = j < held ? j : -1;
    }
  }
}

template <typename T, int DH>
int launch(const SelectArgs& a, cudaStream_t s) {
  static SmemConfig config;
  const auto kernel = cache_select_kernel<T, DH>;
  const size_t smem = (size_t)kRows * a.pitch * sizeof(uint32_t);
  cudaError_t e = config.ensure(kernel, smem);
  ARTAB_REQUIRE(e == cudaSuccess, ARTAB_ELAUNCH, "cache_select: %s", cudaGetErrorString(e));
  const long ctas = (long)a.tiles * a.c.n_heads * a.c.n_groups;
  ARTAB_REQUIRE(ctas <= 0x7fffffffL, ARTAB_EINVAL, "cache_select: too many query rows");
  count_launch();
  kernel<<<(unsigned)ctas, kThreads, smem, s>>>(a);
  return check_launch("cache_select");
}

}  // namespace
}  // namespace artab

using namespace artab;

extern "C" int artab_cache_select(int dtype, const void* q, const int64_t* q_strides, int n_streams, int n_q,
                                  const artab_cache* c, int max_len, int n_pick, int32_t* index, void* stream) {
  int rc = check_cache(c, "cache_select");
  if (rc) return rc;
  rc = check_queries(dtype, q, n_streams, n_q, c, "cache_select");
  if (rc) return rc;
  ARTAB_REQUIRE(index && n_pick >= 1, ARTAB_EINVAL, "cache_select: no blocks asked for");
  ARTAB_REQUIRE(n_pick <= kMostListed, ARTAB_EINVAL, "cache_select: %d blocks a query", n_pick);
  ARTAB_REQUIRE(c->n_blocks <= kMaxBlocks, ARTAB_EINVAL, "cache_select: a cache of more than %d rows is not supported",
                kMaxBlocks * kCacheBlock);
  (void)max_len;   // room for keys goes by the capacity: lens may have grown past the bound in a replayed graph
  SelectArgs a;
  a.c = *c;
  a.q = row_view(q, q_strides, c->n_heads, n_q, c->head_dim);
  a.n_q = n_q;
  a.rows = c->n_groups == 1 ? n_streams * n_q : n_q;
  a.tiles = (a.rows + kRows - 1) / kRows;
  a.n_pick = n_pick;
  a.pitch = c->n_blocks | 1;
  a.vec_q = rows_aligned(a.q, dtype == ARTAB_F32 ? 4 : 2);
  a.index = index;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == ARTAB_F32) {
    if (c->head_dim == 16) return launch<float, 16>(a, s);
    if (c->head_dim == 32) return launch<float, 32>(a, s);
    return launch<float, 64>(a, s);
  }
  if (c->head_dim == 16) return launch<__nv_bfloat16, 16>(a, s);
  if (c->head_dim == 32) return launch<__nv_bfloat16, 32>(a, s);
  return launch<__nv_bfloat16, 64>(a, s);
}
