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
  int per_cta;            // units of a CTA (lists; else 1)
  const int32_t* list;    // [B][H][Lq][n_list], or null: every block
  int n_list;
  float scale_log2;       // scale * log2 e
  int vec_q;
  void* out;              // [B][H][Lq][Dh]
  float* lse;             // [B][H][Lq]
};

constexpr int kSms = 148;
// Smallest value scale, relative to the largest of the context, that is told apart where value scales are factors of the
// numerators: below it codes count as much as they would at it, an error of 2^-20 of the largest value.
constexpr float kLeastRatio = 9.5367431640625e-7f;

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

// Merges `count` partial results of `rows` query rows (at(w, i): element i of partial result w, [row][DH + 2] = output not
// yet divided, maximum in log2 units, sum of numerators, which are 2^lift times exp(s - max)) and writes output and
// log-sum-exp.  The calling thread takes every `step`-th element from `first` on.
template <typename T, int DH, typename F>
__device__ __forceinline__ void merge_rows(const AttnArgs& a, F at, int count, int first, int step, int rows, int row0, int h,
                                           int group, float lift) {
  constexpr int P = DH + 2;
  for (int e = first; e < rows * DH; e += step) {
    const int r = e / DH, d = e % DH, row = row0 + r;
    if (row >= a.rows) return;
    float top = -CUDART_INF_F, sum = 0.0f, out = 0.0f;
    for (int w = 0; w < count; ++w) top = fmaxf(top, at(w, r * P + DH));
    const float from = top == -CUDART_INF_F ? 0.0f : top;
    for (int w = 0; w < count; ++w) {
      const float x = ex2(at(w, r * P + DH) - from);
      sum = fmaf(at(w, r * P + DH + 1), x, sum);
      out = fmaf(at(w, r * P + d), x, out);
    }
    const bool one = a.c.n_groups == 1;
    const int b = one ? row / a.n_q : group, l = one ? row % a.n_q : row;
    const size_t to = ((size_t)b * a.c.n_heads + h) * a.n_q + l;
    reinterpret_cast<T*>(a.out)[to * DH + d] = from_f32<T>(sum == 0.0f ? 0.0f : out / sum);
    if (d == 0) a.lse[to] = sum == 0.0f ? -CUDART_INF_F : (top - lift) * kLn2 + logf(sum);
  }
}

// One launch: ceil(units / per_cta) clusters of `splits` CTAs.
template <typename K, typename... E>
int launch_attn(K kernel, SmemConfig& config, size_t smem, int threads, const AttnArgs& a, cudaStream_t s, E... extra) {
  cudaError_t e = config.ensure(kernel, smem, true);
  ARTAB_REQUIRE(e == cudaSuccess, ARTAB_ELAUNCH, "cache_attention: %s", cudaGetErrorString(e));
  const long ctas = (a.units + a.per_cta - 1) / a.per_cta * a.splits;
  ARTAB_REQUIRE(ctas <= 0x7fffffffL, ARTAB_EINVAL, "cache_attention: too many query rows");
  PlainLaunchScope plain;   // the caller's earlier launches are unknown: see common.cuh
  count_launch();
  e = launch_dependent_cluster(kernel, dim3((unsigned)ctas), dim3(threads), smem, s, (unsigned)a.splits, a, extra...);
  ARTAB_REQUIRE(e == cudaSuccess, ARTAB_ELAUNCH, "cache_attention: %s", cudaGetErrorString(e));
  return ARTAB_OK;
}

}  // namespace artab
