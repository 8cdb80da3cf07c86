// Attention over listed blocks when many queries share a context: by block instead of by query.
//
// A query that takes its blocks one by one reads and turns 64 rows for itself alone, one of eight columns of a product in
// use.  Where lists of many queries hold the same blocks, cache_by_block_kernel goes through the blocks: a CTA per
// (group, head, block) looks its block up in all lists of the head (four bytes an entry), gathers the queries
// that hold it, eight (bf16) or four (fp32) a warp, and writes for each entry the partial result of its block: output not
// yet divided, maximum, sum.  cache_join_kernel merges the entries of a query in the order of its list.  The
// order in which a CTA finds entries varies, what it computes for an entry does not.
// 1024 queries x 6 heads x 16 of 256 blocks (B200), bf16 / fp32, beside one by one: size 32 35 / 43.5 us (63; 402 MB out of L2), 16
// 31 / 37 (44), 64 51 / 61 (99); of the 35 us 28 + 7.  With 5 CTAs an SM that look at 4096 entries at a time 40 us, with 6 and 8192
// 34.5.  Of some 1500 instructions a warp two fifths are the products and a fifth the look-up; issue slots are 60 % busy, waits for
// queries and entries (long scoreboard) the largest stall.  Six CTAs an SM take 40 registers a thread, at the cost of spills (size 32, bf16:
// 28 bytes stored and 24 read a thread); at size 64 shared memory lets five onto an SM, and the bound spills
// 200 bytes there (bf16).
#include <type_traits>

#include "cache_tile.cuh"

namespace artab {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps, kChunk = 32 * kThreads;   // entries looked at between two rounds of work

struct JoinArgs {
  AttnArgs a;
  float* o;       // [B][H][Lq][n_list][Dh]
  float2* ml;     // [B][H][Lq][n_list]
};

template <typename T, int DH, int PARTS>
__global__ void __launch_bounds__(kThreads, 6) cache_by_block_kernel(const JoinArgs j) {
  using Tl = Tile<DH, PARTS>;
  const AttnArgs& a = j.a;
  constexpr int kRecord = 2 * kCacheBlock * DH;
  __shared__ __align__(16) uint8_t rec[kRecord];
  __shared__ int found[kWarps * Tl::ROWS + kChunk];
  __shared__ int n_found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int blk = blockIdx.x, h = blockIdx.y, group = blockIdx.z, H = a.c.n_heads;
  const bool one = a.c.n_groups == 1;
  int len = a.c.lens[group];
  const int cap = a.c.n_blocks * kCacheBlock;
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int live = len - blk * kCacheBlock;
  if (live <= 0) return;
  const size_t at = ((size_t)group * H + h) * a.c.n_blocks + blk;
  for (int i = tid; i < kRecord / 16; i += kThreads)
    reinterpret_cast<uint4*>(rec)[i] = reinterpret_cast<const uint4*>(a.c.codes + at * kRecord)[i];
  const float2 sc = reinterpret_cast<const float2*>(a.c.scales)[at];
  if (tid == 0) n_found = 0;
  __syncthreads();

  const int per = a.n_q * a.n_list;                               // entries of a stream and head, contiguous
  const int entries = one ? a.n_streams * per : per, first = one ? 0 : group;
  const bool by4 = per % 4 == 0 && reinterpret_cast<uintptr_t>(a.list) % 16 == 0;
  const auto offer = [&](int index, int p) {
    if (index == blk) found[atomicAdd(&n_found, 1)] = p;
  };
  // a thread's entries lie `stride` apart: stream and place of the next one follow from those of this one
  const int wide = by4 ? 4 : 1, stride = kThreads * wide, step_b = stride / per, step_i = stride % per;
  int b_at = tid * wide / per, i_at = tid * wide % per;
  for (int e0 = 0;; e0 += kChunk) {
    const bool last = e0 + kChunk >= entries;
    const auto look = [&](auto wide_) {
      constexpr int W = decltype(wide_)::value;
#pragma unroll 4
      for (int e = e0 + tid * W; e < min(e0 + kChunk, entries); e += kThreads * W) {
        const int p = ((first + b_at) * H + h) * per + i_at;
        if constexpr (W == 4) {
          const int4 v = *reinterpret_cast<const int4*>(a.list + p);
          if (v.x == blk || v.y == blk || v.z == blk || v.w == blk)
            offer(v.x, p), offer(v.y, p + 1), offer(v.z, p + 2), offer(v.w, p + 3);
        } else {
          offer(a.list[p], p);
        }
        b_at += step_b, i_at += step_i;
        if (i_at >= per) i_at -= per, ++b_at;
      }
    };
    if (by4)
      look(std::integral_constant<int, 4>());
    else
      look(std::integral_constant<int, 1>());
    __syncthreads();
    const int n = n_found, full = last ? n : n / (kWarps * Tl::ROWS) * (kWarps * Tl::ROWS);   // whole rounds for all warps
    for (int r0 = warp * Tl::ROWS; r0 < full; r0 += kWarps * Tl::ROWS) {
      Tl tile;
      tile.reset();
      const int mine = r0 + g / PARTS;
      const T* q = nullptr;
      if (mine < full) {
        const int row = found[mine] / a.n_list, b = row / a.n_q / H;
        q = reinterpret_cast<const T*>(a.q.p) + b * a.q.s0 + h * a.q.s1 + row % a.n_q * a.q.s2;
      }
      tile.template load_queries<T>(q, a.vec_q, a.scale_log2);
      tile.block(rec, sc.x, sc.y, live < kCacheBlock ? live : kCacheBlock);
#pragma unroll
      for (int r = 0; r < Tl::R; ++r) {
        float l = tile.l[r];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const int i = r0 + (PARTS == 2 ? t : 2 * t + r);
        if (i >= full) continue;
        const size_t p = found[i];
#pragma unroll
        for (int md = 0; md < Tl::KS; ++md)
#pragma unroll
          for (int k = 0; k < 2; ++k) j.o[p * DH + 16 * md + 8 * k + g] = tile.o[md][k][r];
        if (g == 0) j.ml[p] = make_float2(tile.m[r], l);
      }
    }
    if (last) return;
    __syncthreads();
    const int rest = n - full;                                    // kept for the next round
    const int keep = tid < rest ? found[full + tid] : 0;
    __syncthreads();
    if (tid < rest) found[tid] = keep;
    if (tid == 0) n_found = rest;
    __syncthreads();
  }
}

template <typename T, int DH>
__global__ void __launch_bounds__(256) cache_join_kernel(const JoinArgs j) {
  const AttnArgs& a = j.a;
  const long u = ((long)blockIdx.x * 256 + threadIdx.x) / DH;     // (stream, head, query)
  const int d = threadIdx.x % DH;
  if (u >= a.units) return;
  const int group = a.c.n_groups == 1 ? 0 : (int)(u / a.n_q / a.c.n_heads);
  int len = a.c.lens[group];
  const int cap = a.c.n_blocks * kCacheBlock;
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int held = (len + kCacheBlock - 1) / kCacheBlock;
  float top = -CUDART_INF_F, sum = 0.0f, out = 0.0f;
#pragma unroll 8
  for (int s = 0; s < a.n_list; ++s) {
    const long p = u * a.n_list + s;
    const int index = a.list[p];
    float2 ml = j.ml[p];
    float o = j.o[p * DH + d];
    if (index < 0 || index >= held) ml = make_float2(-CUDART_INF_F, 0.0f), o = 0.0f;   // nothing was written for it
    const float m = fmaxf(top, ml.x), base = m == -CUDART_INF_F ? 0.0f : m;
    const float x = ex2(top - base), y = ex2(ml.x - base);
    sum = fmaf(sum, x, ml.y * y);
    out = fmaf(out, x, o * y);
    top = m;
  }
  reinterpret_cast<T*>(a.out)[u * DH + d] = from_f32<T>(sum == 0.0f ? 0.0f : out / (kUnlift * sum));
  if (d == 0) a.lse[u] = sum == 0.0f ? -CUDART_INF_F : (top - kLift) * kLn2 + logf(sum);
}

template <typename T, int DH>
int launch_by_block(const JoinArgs& j, cudaStream_t s) {
  constexpr int kParts = sizeof(T) == 2 ? 1 : 2;
  count_launch();
  cache_by_block_kernel<T, DH, kParts><<<dim3(j.a.c.n_blocks, j.a.c.n_heads, j.a.c.n_groups), kThreads, 0, s>>>(j);
  int rc = check_launch("cache_by_block");
  if (rc) return rc;
  count_launch();
  cache_join_kernel<T, DH><<<(unsigned)((j.a.units * DH + 255) / 256), 256, 0, s>>>(j);
  return check_launch("cache_join");
}

}  // namespace

// Going through the blocks pays from so many entries a block on (in the mean), as long as looking an entry up in every
// block does not cost more than the records that are read once less, and the partial results stay below a gigabyte.  By block / one
// by one (us), 6 heads, 16 of 256 blocks, 128, 192 and 256 queries (8, 12 and 16 entries a block):
//   size 16 bf16 13.4 / 9.9, 14.4 / 11.7, 15.3 / 15.6; fp32 13.5 / 9.9, 15.2 / 11.7, 16.4 / 15.6   (16 would suit it better)
//   size 32 bf16 14.3 / 12.8, 15.4 / 15.4, 16.0 / 20.1; fp32 14.7 / 12.7, 16.4 / 15.6, 18.1 / 20.3
//   size 64 bf16 19.1 / 16.7, 20.8 / 23.2, 22.4 / 30.8; fp32 19.2 / 17.0, 21.3 / 23.0, 23.8 / 30.6
// 16 of 1024 blocks, 1024 queries: size 16 64 / 44.5, 32 71 / 63, 64 102 / 99.  Blocks are those of the capacity: the rows in use are
// known on the device only, so a cache with much room (16384 rows in a capacity of 65536: 63 us, in one of 16384 35) goes one by one.
constexpr int kLeastShared = 12;
constexpr int64_t kMostWorkspace = 1LL << 30;
int64_t by_block_workspace(const artab_cache* c, int n_streams, int n_q, int n_list) {
  const int64_t rows = c->n_groups == 1 ? (int64_t)n_streams * n_q : n_q;
  const int64_t entries = (int64_t)n_streams * c->n_heads * n_q * n_list;
  const int64_t bytes = entries * (c->head_dim * 4 + 8);
  const int form = debug_cache_form();
  if (form == 1 || entries > (1 << 27) || bytes > kMostWorkspace) return 0;
  if (form == 0 && (rows * n_list < (int64_t)kLeastShared * c->n_blocks || c->n_blocks * 4 > 64 * c->head_dim || entries < 8192))
    return 0;
  return bytes;
}

int launch_cache_by_block(int dtype, const AttnArgs& a, void* workspace, cudaStream_t s) {
  JoinArgs j;
  j.a = a;
  const int64_t entries = a.units * (int64_t)a.n_list;
  j.o = reinterpret_cast<float*>(workspace);
  j.ml = reinterpret_cast<float2*>(j.o + entries * a.c.head_dim);
  const int dh = a.c.head_dim;
  if (dtype == ARTAB_F32) return dh == 16 ? launch_by_block<float, 16>(j, s) : dh == 32 ? launch_by_block<float, 32>(j, s) : launch_by_block<float, 64>(j, s);
  return dh == 16 ? launch_by_block<__nv_bfloat16, 16>(j, s) : dh == 32 ? launch_by_block<__nv_bfloat16, 32>(j, s) : launch_by_block<__nv_bfloat16, 64>(j, s);
}

}  // namespace artab
