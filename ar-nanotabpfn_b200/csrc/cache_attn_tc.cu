// Attention over the 8-bit context cache for many query rows of bf16, on the 5th-generation tensor cores.
//
// The formulas are those of cache_attn.cu.  One CTA = 128 query rows of a (group, head) and a share of its blocks of 64 rows,
// 384 threads:
//   warps 0-3, 4-7   two softmax warpgroups; a thread owns one query row (TMEM lane).  Each warpgroup takes every other
//                    block, with scores, numerators and an output accumulator of its own in tensor memory, a running
//                    reference and sum in registers: the two meet only at the end, like two key splits
//   warps 8, 9       turn codes into half-precision tiles (K-major, swizzled) of a ring of four blocks
//   warps 10, 11     one issuing thread for the MMAs of each warpgroup (MMAs of one thread cost 100 cycles each whatever
//                    their width; those of several threads overlap)
// S = Q . codes^T is M 128, N 64; O += P . codes is M 128, N = Dh with P from tensor memory.  All operands are halves:
// queries of bf16 are exact in them (scaled by a power of two per row), codes are whole numbers, numerators keep
// 11 bits.  Scales of keys go into the exponent's factor, scales of values into its offset (relative to the largest of the
// context, taken out of the row sum again), so O accumulates over all blocks.
// What bounds it is the exponential: 64 per row and block, 16 a clock and SM on the special-function unit; a
// quarter of them is computed on the FMA pipe.  Two CTAs share an SM (256 TMEM columns each), so four warpgroups are in
// different phases of their blocks.  head_dim 64 has no room for P beside S: it overwrites the scores it came from, and the
// next scores wait for P . V.
// Every wait is bounded; a CTA that gives up writes NaN for its rows.
#include "cache_attn.cuh"

namespace artab {
namespace {

constexpr int BM = 128, BN = kCacheBlock, kStages = 4, kThreads = 384, kConvert = 64;
constexpr uint32_t kTmemCols = 256;
// numerators are 2^6 times exp(s - reference); the reference lags by at most 2^8 before it is raised
constexpr float kLiftTc = 6.0f, kLag = 8.0f;
// 2^f on [-0.5, 0.5]: least largest relative error, 2.6e-6
constexpr float kExp0 = 0.999999285f, kExp1 = 0.69312185f, kExp2 = 0.240247443f, kExp3 = 0.0559177138f, kExp4 = 0.00957003608f;
#ifndef ARTAB_CACHE_POLY_OF_8
#define ARTAB_CACHE_POLY_OF_8 2
#endif

struct Ctl {
  int abort_flag, pad;
  long long limit;
};
template <int DH>
struct __align__(1024) TcSmem {
  uint8_t k[kStages][BN * DH * 2];       // [64 rows][DH] halves
  uint8_t v[kStages][DH * 128];          // [DH][64 rows] halves
  uint8_t q[BM * DH * 2];
  uint64_t q_full, kv_full[kStages], kv_empty[kStages];
  uint64_t s_full[2], s_free[2], p_full[2], o_full[2];
  float vmax[kThreads / 32];
  uint32_t tmem_base;
  Ctl ctl;
  static constexpr int kFree = kStages * (BN * DH * 2 + DH * 128) + BM * DH * 2;   // bytes that the merge may use
};

__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
// false when the CTA is giving up (this wait or another one ran out)
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile Ctl* ctl) {
  const uint32_t b = smem_u32(bar);
  if (mbar_try(b, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
    if (mbar_try(b, parity)) return true;
    if (ctl->abort_flag) return false;
    if (clock64() - t0 > ctl->limit) {
      ctl->abort_flag = 1;
      return false;
    }
  }
}

// K-major tile of rows of 32, 64 or 128 bytes: swizzle of that span, groups of eight rows behind one another
template <int ROW_BYTES>
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) {   // byte offset of a 16-byte chunk
  constexpr uint32_t kMask = ROW_BYTES / 16 - 1;
  constexpr uint32_t kShift = ROW_BYTES == 128 ? 0 : ROW_BYTES == 64 ? 1 : 2;
  return row * ROW_BYTES + ((chunk ^ ((row >> kShift) & kMask)) << 4);
}
template <int ROW_BYTES>
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr) {
  constexpr uint64_t kLayout = ROW_BYTES == 128 ? 2 : ROW_BYTES == 64 ? 4 : 6;
  uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)1 << 16;                               // leading byte offset: unused for a swizzled K-major tile
  d |= (uint64_t)(8 * ROW_BYTES >> 4) << 32;            // distance of groups of eight rows
  d |= (uint64_t)1 << 46;                               // descriptor version (sm_100)
  d |= kLayout << 61;
  return d;
}
// kind::f16, fp32 accumulators, A and B halves, both K-major
constexpr uint32_t idesc(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }

__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(desc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ float2 pk_fma(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 pk_add(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// 2^x on the FMA pipe for x <= 16: the nearest integer n by adding 1.5 * 2^23, a polynomial of degree four for
// 2^f, f = x - n in [-0.5, 0.5] (relative error 2.6e-6), n into the exponent field.  Below
// 2^-125 the result is nothing; a NaN stays one.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
  const float2 y = make_float2(x.x < -125.0f ? -125.0f : x.x, x.y < -125.0f ? -125.0f : x.y);
  const float2 r = pk_add(y, make_float2(12582912.0f, 12582912.0f));
  const float2 n = pk_add(r, make_float2(-12582912.0f, -12582912.0f));
  const float2 f = pk_fma(n, make_float2(-1.0f, -1.0f), y);
  float2 p = pk_fma(make_float2(kExp4, kExp4), f, make_float2(kExp3, kExp3));
  p = pk_fma(p, f, make_float2(kExp2, kExp2));
  p = pk_fma(p, f, make_float2(kExp1, kExp1));
  p = pk_fma(p, f, make_float2(kExp0, kExp0));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23)),
                     __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23)));
}

template <int DH>
__global__ void __launch_bounds__(kThreads, 2) cache_attn_tc_kernel(const AttnArgs a, long long wait_cycles, int drop_commits) {
  constexpr bool kAlias = DH == 64;                  // P in the columns of S
  constexpr uint32_t kColP = kAlias ? 0 : BN, kColO = kAlias ? BN : BN + BN / 2, kColsWg = kTmemCols / 2;
  constexpr int KS = DH / 16, P = DH + 2, KB = DH * 2;
  extern __shared__ uint8_t smem_raw[];
  using S = TcSmem<DH>;
  S* sm = reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)(blockIdx.x % a.splits);
  const long unit = blockIdx.x / a.splits;
  const int H = a.c.n_heads, row0 = (int)(unit % a.tiles) * BM, h = (int)(unit / a.tiles % H);
  const int group = (int)(unit / a.tiles / H);
  const bool one = a.c.n_groups == 1;
  const auto stream_of = [&](int row) { return one ? row / a.n_q : group; };
  const auto query_of = [&](int row) { return one ? row % a.n_q : row; };
  int len = a.c.lens[group];
  const int cap = a.c.n_blocks * kCacheBlock;
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int held = (len + kCacheBlock - 1) / kCacheBlock;
  const int nb = held > rank ? (held - rank + a.splits - 1) / a.splits : 0;      // blocks of this CTA: rank, rank + splits, ...
  const size_t gh = (size_t)group * H + h;
  const uint8_t* codes = a.c.codes + gh * a.c.n_blocks * (size_t)(2 * kCacheBlock * DH);
  const float2* scales = reinterpret_cast<const float2*>(a.c.scales) + gh * a.c.n_blocks;
  volatile Ctl* ctl = &sm->ctl;

  if (tid == 0) {
    mbar_init(&sm->q_full, BM);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm->kv_full[s], kConvert);
      mbar_init(&sm->kv_empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sm->s_full[w], 1);
      mbar_init(&sm->s_free[w], BM);
      mbar_init(&sm->p_full[w], BM);
      mbar_init(&sm->o_full[w], 1);
    }
    sm->ctl.abort_flag = 0;
    sm->ctl.limit = wait_cycles;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 10) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm->tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  float vmax = 0.0f;                                  // largest value scale of the context
  for (int i = tid; i < held; i += kThreads) vmax = fmaxf(vmax, scales[i].y);
  vmax = warp_max(vmax);
  if (lane == 0) sm->vmax[warp] = vmax;
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sm->tmem_base;

  bool ok = true;
  float m = -CUDART_INF_F, l = 0.0f, poison = 0.0f;
  const int wg = warp >> 2, row = tid & (BM - 1);     // softmax threads
  const uint32_t t_row = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (wg & 1) * kColsWg;
  const int steps = wg < 2 ? (nb - wg + 1) / 2 : 0;   // blocks of the warpgroup

  if (warp >= 10) {
    // ------------------------------ MMA issuers ------------------------------
    const int w = warp - 10, n = (nb - w + 1) / 2;
    if (lane == 0 && n > 0) {
      const uint32_t t_wg = tmem + w * kColsWg, q_addr = smem_u32(sm->q);
      ok = mbar_wait(&sm->q_full, 0, ctl);
      const auto scores = [&](int i) {                // S = Q . K^T of step i
        const int j = 2 * i + w, st = j % kStages;
        if (!mbar_wait(&sm->kv_full[st], (j / kStages) & 1, ctl)) return false;
        fence_after();
        const uint32_t k_addr = smem_u32(sm->k[st]);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          umma_ss(t_wg, tile_desc<KB>(q_addr + 32 * ks), tile_desc<KB>(k_addr + 32 * ks), idesc(BM, BN), ks);
        if (!drop_commits) umma_commit(&sm->s_full[w]);
        return true;
      };
      ok = ok && scores(0);
      for (int i = 0; ok && i < n; ++i) {
        const int st = (2 * i + w) % kStages;
        if (!kAlias && i + 1 < n) {                   // the next scores, as soon as these are in registers
          ok = mbar_wait(&sm->s_free[w], i & 1, ctl);
          if (ok) fence_after();
          ok = ok && scores(i + 1);
          if (!ok) break;
        }
        ok = mbar_wait(&sm->p_full[w], i & 1, ctl);
        if (!ok) break;
        fence_after();
        const uint32_t v_addr = smem_u32(sm->v[st]);
#pragma unroll
        for (int ks = 0; ks < BN / 16; ++ks)
          umma_ts(t_wg + kColO, t_wg + kColP + 8 * ks, tile_desc<128>(v_addr + 32 * ks), idesc(BM, DH), i > 0 || ks > 0);
        umma_commit(&sm->o_full[w]);
        umma_commit(&sm->kv_empty[st]);
        if (kAlias && i + 1 < n) {                    // P lies where the next scores go
          ok = mbar_wait(&sm->o_full[w], i & 1, ctl);
          if (ok) fence_after();
          ok = ok && scores(i + 1);
        }
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    // ------------------------- codes into operand tiles -------------------------
    const int ct = tid - 256;
    uint4 rk[KS], rv[KS];
    const auto load = [&](int j) {
      const uint4* src = reinterpret_cast<const uint4*>(codes + (size_t)(rank + j * a.splits) * (2 * kCacheBlock * DH));
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        rk[i] = src[ct + i * kConvert];
        rv[i] = src[kCacheBlock * DH / 16 + ct + i * kConvert];
      }
    };
    if (nb > 0) load(0);
    for (int j = 0; ok && j < nb; ++j) {
      const int st = j % kStages;
      if (j >= kStages) ok = __all_sync(0xffffffffu, mbar_wait(&sm->kv_empty[st], ((j / kStages) + 1) & 1, ctl));
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < KS; ++i) {                  // 16 channels of a key: two chunks
        const int u = ct + i * kConvert, r = u / KS, c = u % KS * 2;
        const uint32_t w[4] = {rk[i].x, rk[i].y, rk[i].z, rk[i].w};
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<uint4*>(sm->k[st] + swizzled<KB>(r, c + e)) =
              make_uint4(codes_to_halves(w[2 * e], false), codes_to_halves(w[2 * e], true),
                         codes_to_halves(w[2 * e + 1], false), codes_to_halves(w[2 * e + 1], true));
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {                  // 16 places of a value channel: rows 16 s + 8 h + 2 t + {0, 1}
        const int u = ct + i * kConvert, d = u / 4, t = u % 4;
        const uint32_t w[4] = {rv[i].x, rv[i].y, rv[i].z, rv[i].w};
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<uint32_t*>(sm->v[st] + swizzled<128>(d, 2 * s + e) + 4 * t) = codes_to_halves(w[s], e);
      }
      if (j + 1 < nb) load(j + 1);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&sm->kv_full[st]);
    }
  } else {
    // --------------------------------- softmax ---------------------------------
    vmax = 0.0f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) vmax = fmaxf(vmax, sm->vmax[w]);
    // a quotient by vmax as a product: both sides lifted where the scale is small
    const float big = vmax < 1.0f ? 1.152921504606846976e18f : 1.0f, vinv = vmax > 0.0f ? 1.0f / (vmax * big) : 0.0f;
    float f;
    {
      float x[DH];
#pragma unroll
      for (int i = 0; i < DH; ++i) x[i] = 0.0f;
      const int r = row0 + row;
      if (r < a.rows)
        load_elements<__nv_bfloat16, DH>(reinterpret_cast<const __nv_bfloat16*>(a.q.p) + stream_of(r) * a.q.s0 + h * a.q.s1 +
                                             query_of(r) * a.q.s2, a.vec_q, x);
      float top = 0.0f, to, back;
#pragma unroll
      for (int i = 0; i < DH; ++i) top = fmaxf(top, fabsf(x[i]));
      row_scale(top, to, back);
      f = back * fabsf(a.scale_log2);
      to = copysignf(to, a.scale_log2);
      if (wg == 0) {
#pragma unroll
        for (int c = 0; c < DH / 8; ++c) {
          uint32_t u[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i] = h2_bits(__floats2half2_rn(x[8 * c + 2 * i] * to, x[8 * c + 2 * i + 1] * to));
          *reinterpret_cast<uint4*>(sm->q + swizzled<KB>(row, c)) = make_uint4(u[0], u[1], u[2], u[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&sm->q_full);
      }
    }
    float2 next = steps > 0 ? scales[rank + wg * a.splits] : make_float2(0.0f, 0.0f);
    for (int i = 0; i < steps; ++i) {
      const int blk = rank + (2 * i + wg) * a.splits;
      const float2 sc = next;
      if (i + 1 < steps) next = scales[blk + 2 * a.splits];
      const int live = len - blk * kCacheBlock;
      float ratio = sc.y * big * vinv;
      if (ratio != ratio) poison = sc.y, ratio = 1.0f;
      ratio = fmaxf(ratio, kLeastRatio);
      const float lift = kLiftTc + __log2f(ratio), unlift = __frcp_rn(ratio);
      const float x = f * sc.x, slope = !(x <= 1e-37f) ? x : 1e-37f;
      ok = __all_sync(0xffffffffu, mbar_wait(&sm->s_full[wg], i & 1, ctl));
      if (!ok) break;
      fence_after();
      uint32_t r[32];
      float top = -CUDART_INF_F;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        tmem_ld32(t_row + 32 * c, r);
        wait_ld();
        if (live < BN) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * c + e < live) top = fmaxf(top, __uint_as_float(r[e]));
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 2) top = fmaxf(top, fmaxf(__uint_as_float(r[e]), __uint_as_float(r[e + 1])));
        }
      }
      top *= slope;
      const bool raise = !(top <= m + kLag);
      const float alpha = raise ? ex2(m - top) : 1.0f;
      if (raise) m = top;
      const float2 sl2 = make_float2(slope, slope), add2 = make_float2(lift - m, lift - m);
      float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t pk[16];
        tmem_ld32(t_row + 32 * c, r);
        wait_ld();
        if (!kAlias && c == 1) {
          fence_before();
          mbar_arrive(&sm->s_free[wg]);
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float2 y = pk_fma(make_float2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), sl2, add2);
          if (((e >> 1) & 7) < ARTAB_CACHE_POLY_OF_8)
            y = ex2_fma(y);
          else
            y = make_float2(ex2(y.x), ex2(y.y));
          if (live < BN) {
            if (32 * c + e >= live) y.x = 0.0f;
            if (32 * c + e + 1 >= live) y.y = 0.0f;
          }
          sum = pk_add(sum, y);
          pk[e >> 1] = h2_bits(__floats2half2_rn(y.x, y.y));
        }
        if (c == 0 && i > 0) {                        // the P . V before this one has read P and written O
          if (!kAlias) ok = __all_sync(0xffffffffu, mbar_wait(&sm->o_full[wg], (i - 1) & 1, ctl));
          fence_after();
          if (__any_sync(0xffffffffu, raise)) {
#pragma unroll 1
            for (int d = 0; d < DH; d += 16) {
              uint32_t o[16];
              tmem_ld16(t_row + kColO + d, o);
              wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16(t_row + kColO + d, o);
            }
          }
        }
        tmem_st16(t_row + kColP + 16 * c, pk);
      }
      l = fmaf(l, alpha, (sum.x + sum.y) * unlift);
      wait_st();
      fence_before();
      mbar_arrive(&sm->p_full[wg]);
      if (!ok) break;
    }
    if (ok && steps > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sm->o_full[wg], (steps - 1) & 1, ctl));
    fence_after();
  }

  // both warpgroups' results where the tiles were: [2][128][DH + 2]
  float* part = reinterpret_cast<float*>(sm);
  uint32_t o[DH];
  if (wg < 2) {
#pragma unroll
    for (int d = 0; d < DH; ++d) o[d] = 0u;
    if (steps > 0) {
#pragma unroll
      for (int d = 0; d < DH; d += 16) tmem_ld16(t_row + kColO + d, o + d);
      wait_ld();
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 10) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
  const bool gave_up = ctl->abort_flag != 0;
  if (wg < 2) {
    float* to = part + (wg * BM + row) * P;
#pragma unroll
    for (int d = 0; d < DH; ++d) to[d] = __uint_as_float(o[d]) * vmax + poison;
    to[DH] = m;
    to[DH + 1] = gave_up ? CUDART_NAN_F : l;
  }
  if (a.splits == 1)
    __syncthreads();
  else
    cluster_meet();
  const uint32_t base = smem_u32(part);
  const auto at = [&](int w, int i) {                 // partial result w: warpgroup w % 2 of CTA w / 2
    if (a.splits == 1) return part[(w & 1) * BM * P + i];
    return ld_cluster(base + ((w & 1) * BM * P + i) * 4, w >> 1);
  };
  merge_rows<__nv_bfloat16, DH>(a, at, 2 * a.splits, rank * kThreads + tid, a.splits * kThreads, BM, row0, h, group, kLiftTc);
  if (a.splits > 1) cluster_meet();
}

}  // namespace

template <int DH>
static int launch_tc(const AttnArgs& a, cudaStream_t s) {
  static SmemConfig config;
  static_assert(TcSmem<DH>::kFree >= 2 * BM * (DH + 2) * 4, "the merge fits where the tiles were");
  const long long limit = debug_wait_cycles() ? debug_wait_cycles() : kDefaultWaitCycles;
  return launch_attn(cache_attn_tc_kernel<DH>, config, sizeof(TcSmem<DH>) + 1024, kThreads, a, s, limit, debug_drop_score_commits());
}

int launch_cache_attn_tc(const AttnArgs& a, cudaStream_t s) {
  return a.c.head_dim == 16 ? launch_tc<16>(a, s) : a.c.head_dim == 32 ? launch_tc<32>(a, s) : launch_tc<64>(a, s);
}

}  // namespace artab
