// What the attention kernels of the 8-bit context cache share: arguments, constants, the merge of partial results.
#pragma once
#include <math_constants.h>

#include "cache8.cuh"
#include "cluster.cuh"

namespace artab {

struct AttnArgs {
  artab_cache c;
  RowView q;
  int n_streams, n_q;
  int rows;               // query rows of a group
  int tiles;              // tiles of a group's rows
  long units;             // (group, head, tile) or (stream, head, query)
  int splits;             // CTAs of a cluster, which share the blocks of a unit
  const int32_t* list;    // [B][H][Lq][n_list], or null: every block
  int n_list;
  float scale_log2;       // scale * log2 e
  int vec_q;
  void* out;              // [B][H][Lq][Dh]
  float* lse;             // [B][H][Lq]
};

constexpr int kSms = 148;
// Where value scales are factors of the numerators (the kernels of many rows), they are so relative to the largest of the context, and
// a row's maximum is that of score + log2(ratio): a numerator is as large as what its row adds to the output, so a block of small
// values keeps all its bits wherever the output is made of it.  Ratios below 2^-80, blocks of zeros among them, count as 2^-80
// (sums of numerators over their ratios stay within fp32: 2^41 numerators, times 2^80).
constexpr float kLeastRatio = 8.271806125530277e-25f;

template <typename T>
int launch_cache_attn_tc(const AttnArgs& a, cudaStream_t s);
int64_t by_block_workspace(const artab_cache* c, int n_streams, int n_q, int n_list);
int launch_cache_by_block(int dtype, const AttnArgs& a, void* workspace, cudaStream_t s);

__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_rank(addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(map_to_rank(addr, rank))
               : "memory");
  return v;
}

// A partial result of a query row: output not yet divided, maximum in log2 units, sum of numerators (2^lift times
// exp(s - maximum)); padded so that four channels are read at once.
template <int DH>
constexpr int kPartial = DH + 4;

// Merges the partial results of `rows` query rows and writes output and log-sum-exp: `per_cta` of them lie in every CTA of
// the cluster, [per_cta][rows][kPartial] from shared-memory address `base` on.  The calling thread takes every `step`-th
// group of four channels from `first` on.  `factor`: of quotients of outputs and sums; a factor of sums would not fit fp32 where
// values are large.
template <typename T, int DH>
__device__ __forceinline__ void merge_rows(const AttnArgs& a, uint32_t base, int per_cta, int first, int step, int rows,
                                           int row0, int h, int group, float lift, float factor) {
  constexpr int P = kPartial<DH>;
  const int count = per_cta * a.splits;
  for (int e = first; e < rows * (DH / 4); e += step) {
    const int r = e / (DH / 4), d = e % (DH / 4) * 4, row = row0 + r;
    if (row >= a.rows) return;
    const auto at = [&](int w) { return base + (uint32_t)((w % per_cta * rows + r) * P * 4); };
    float top = -CUDART_INF_F, sum = 0.0f;
    float4 out = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int w = 0; w < count; ++w) top = fmaxf(top, ld_cluster(at(w) + DH * 4, w / per_cta));
    const float from = top == -CUDART_INF_F ? 0.0f : top;
#pragma unroll 4
    for (int w = 0; w < count; ++w) {
      const float x = ex2(ld_cluster(at(w) + DH * 4, w / per_cta) - from);
      sum = fmaf(ld_cluster(at(w) + DH * 4 + 4, w / per_cta), x, sum);
      const float4 o = ld_cluster4(at(w) + d * 4, w / per_cta);
      out.x = fmaf(o.x, x, out.x), out.y = fmaf(o.y, x, out.y), out.z = fmaf(o.z, x, out.z), out.w = fmaf(o.w, x, out.w);
    }
    const bool one = a.c.n_groups == 1;
    const int b = one ? row / a.n_q : group, l = one ? row % a.n_q : row;
    const size_t to = ((size_t)b * a.c.n_heads + h) * a.n_q + l;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    out.x = out.x * inv * factor, out.y = out.y * inv * factor, out.z = out.z * inv * factor, out.w = out.w * inv * factor;
    T* dst = reinterpret_cast<T*>(a.out) + to * DH + d;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(dst) = make_float4(out.x, out.y, out.z, out.w);
    } else {
      __nv_bfloat162 y[2] = {__floats2bfloat162_rn(out.x, out.y), __floats2bfloat162_rn(out.z, out.w)};
      *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(y);
    }
    if (d == 0) a.lse[to] = sum == 0.0f ? -CUDART_INF_F : (top - lift) * kLn2 + logf(sum);
  }
}

// One launch: `units` clusters of `splits` CTAs.
template <typename K, typename... E>
int launch_attn(K kernel, SmemConfig& config, size_t smem, int threads, const AttnArgs& a, cudaStream_t s, E... extra) {
  cudaError_t e = config.ensure(kernel, smem, true);
  ARTAB_REQUIRE(e == cudaSuccess, ARTAB_ELAUNCH, "cache_attention: %s", cudaGetErrorString(e));
  const long ctas = a.units * a.splits;
  ARTAB_REQUIRE(ctas <= 0x7fffffffL, ARTAB_EINVAL, "cache_attention: too many query rows");
  PlainLaunchScope plain;   // the caller's earlier launches are unknown: see common.cuh
  count_launch();
  e = launch_dependent_cluster(kernel, dim3((unsigned)ctas), dim3(threads), smem, s, (unsigned)a.splits, a, extra...);
  ARTAB_REQUIRE(e == cudaSuccess, ARTAB_ELAUNCH, "cache_attention: %s", cudaGetErrorString(e));
  return ARTAB_OK;
}

}  // namespace artab
