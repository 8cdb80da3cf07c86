// For every query the blocks of the 8-bit context cache with the largest upper bound of a score.
//
// With the query rounded to whole numbers (largest magnitude -> 127) the bound over a block's rows is
//   ks * sum_d max(qi_d * lo_d, qi_d * hi_d) = ks * (max(qi, 0) . hi + min(qi, 0) . lo),
// lo / hi the smallest and largest key code of channel d.  The sum is a whole number below 2^21, formed exactly by
// half-precision products with fp32 sums whatever their order, and one fp32 product follows: the choice does not
// depend on tiling, and ties (broken by the lowest index) are real ties.
//
// One CTA = 16 queries of a (group, head): scores of all blocks into shared memory as ordered keys (products of
// 16 queries x 8 blocks a warp), then one warp per query finds the n-th largest key bit by bit and writes the chosen
// indices in ascending order.
#include "cache8.cuh"

namespace artab {
namespace {

constexpr int kThreads = 256, kRows = 16, kMaxBlocks = 3456;   // 16 rows of keys in 227 KB

struct SelectArgs {
  artab_cache c;
  RowView q;
  int n_streams, n_q, rows, tiles, n_pick;
  int pitch;               // keys of a row
  int vec_q;
  int32_t* index;          // [B][H][Lq][n_pick]
};

__device__ __forceinline__ float nearest_whole(float x, float step, float inv) {
  const float f = x * inv;
  float c = rintf(f);
  if (!(fabsf(f - c) < 0.49995f)) c = (float)rint((double)x / (double)step);
  return fminf(fmaxf(c, -127.0f), 127.0f);
}

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

  // thread t < 2: negative parts of channels t * NE .., for the lower bounds; t >= 2: positive parts, upper bounds
  uint32_t qa[KS][4];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = row0 + g + 8 * half;
    float x[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) x[i] = 0.0f;
    if (row < a.rows) {
      const int b = one ? row / a.n_q : group, l = one ? row % a.n_q : row;
      load_elements<T, NE>(reinterpret_cast<const T*>(a.q.p) + b * a.q.s0 + h * a.q.s1 + l * a.q.s2 + (t & 1) * NE, a.vec_q, x);
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NE; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const float step = top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top), 127.0f) : 0.0f;  // not finite: all zero
    const float inv = step > 0.0f ? 1.0f / step : 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      x[i] = step > 0.0f ? nearest_whole(x[i], step, inv) : 0.0f;
      x[i] = t < 2 ? fminf(x[i], 0.0f) : fmaxf(x[i], 0.0f);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qa[s][half] = h2_bits(__floats2half2_rn(x[4 * s], x[4 * s + 1]));
      qa[s][2 + half] = h2_bits(__floats2half2_rn(x[4 * s + 2], x[4 * s + 3]));
    }
  }
  const __half* bounds = reinterpret_cast<const __half*>(a.c.bounds) + gh * a.c.n_blocks * 2 * DH;
  const float* scales = a.c.scales + gh * a.c.n_blocks * 2;
  for (int j = warp * 8; j < held; j += kThreads / 32 * 8) {
    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int blk = j + g < held ? j + g : held - 1;
    const uint4* src = reinterpret_cast<const uint4*>(bounds + (size_t)blk * 2 * DH + t * NE);
    uint32_t w[KS][2];
#pragma unroll
    for (int i = 0; i < NE / 8; ++i) {
      const uint4 v = src[i];
      w[2 * i][0] = v.x, w[2 * i][1] = v.y, w[2 * i + 1][0] = v.z, w[2 * i + 1][1] = v.w;
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) mma_f16(c, qa[s][0], qa[s][1], qa[s][2], qa[s][3], w[s][0], w[s][1]);
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = j + 2 * t + e;
      if (col >= held) continue;
      const float ks = scales[(size_t)col * 2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // a block whose scale is not a number ranks first: what is wrong with it shows in the output
        const float v = ks == ks ? c[2 * half + e] * ks : __uint_as_float(0x7f800000u);
        const uint32_t bits = __float_as_uint(v + 0.0f);   // -0 -> 0: equal scores have equal keys
        s_key[(g + 8 * half) * a.pitch + col] = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
      }
    }
  }
  __syncthreads();
  for (int r = warp; r < kRows; r += kThreads / 32) {
    const int row = row0 + r;
    if (row >= a.rows) break;
    const uint32_t* key = s_key + r * a.pitch;
    const int b = one ? row / a.n_q : group, l = one ? row % a.n_q : row;
    int32_t* out = a.index + (((size_t)b * H + h) * a.n_q + l) * a.n_pick;
    int done = 0;
    if (held <= a.n_pick) {
      for (int i = lane; i < held; i += 32) out[i] = i;
      done = held;
    } else {
      uint32_t nth = 0;                                    // the n-th largest key
      int at_least = held;                                 // keys >= nth
      for (uint32_t bit = 0x80000000u; bit && at_least > a.n_pick; bit >>= 1) {
        const uint32_t trial = nth | bit;
        int count = 0;
        for (int i = lane; i < held; i += 32) count += key[i] >= trial;
        count = __reduce_add_sync(0xffffffffu, count);
        if (count >= a.n_pick) nth = trial, at_least = count;
      }
      // every key above nth, and the first of those equal to it
      int above = 0;
      if (at_least > a.n_pick) {
        for (int i = lane; i < held; i += 32) above += key[i] > nth;
        above = __reduce_add_sync(0xffffffffu, above);
      }
      int ties = at_least > a.n_pick ? a.n_pick - above : a.n_pick;
      for (int i0 = 0; i0 < held && done < a.n_pick; i0 += 32) {
        const uint32_t k = i0 + lane < held ? key[i0 + lane] : 0u;
        const bool in = i0 + lane < held && k > nth, tie = i0 + lane < held && k == nth;
        const uint32_t tied = __ballot_sync(0xffffffffu, tie);
        const bool take = in || (tie && __popc(tied & ((1u << lane) - 1u)) < ties);
        const uint32_t taken = __ballot_sync(0xffffffffu, take);
        if (take) out[done + __popc(taken & ((1u << lane) - 1u))] = i0 + lane;
        ties -= min(ties, __popc(tied));
        done += __popc(taken);
      }
    }
    for (int i = done + lane; i < a.n_pick; i += 32) out[i] = -1;
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
  rc = check_queries(dtype, q, q_strides, n_streams, n_q, c, "cache_select");
  if (rc) return rc;
  ARTAB_REQUIRE(index && n_pick >= 1, ARTAB_EINVAL, "cache_select: no blocks asked for");
  ARTAB_REQUIRE(c->n_blocks <= kMaxBlocks, ARTAB_EINVAL, "cache_select: a cache of more than %d rows is not supported",
                kMaxBlocks * kCacheBlock);
  (void)max_len;
  SelectArgs a;
  a.c = *c;
  a.q = {q, (long)q_strides[0], (long)q_strides[1], (long)q_strides[2]};
  a.n_streams = n_streams;
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
