// Attention over the 8-bit context cache for many query rows, on the 5th-generation tensor cores.
//
// The formulas are those of cache_attn.cu.  One CTA = 128 query rows of a (group, head) and a share of its blocks of 64 rows,
// 384 threads:
//   warps 0-3, 4-7   two softmax warpgroups; a thread owns one query row (TMEM lane).  Each warpgroup takes every other
//                    block, with scores, numerators and an output accumulator of its own in tensor memory, a running
//                    reference and sum in registers: the two meet only at the end, like two key splits
//   warps 8, 9       turn codes into half-precision tiles (K-major, swizzled) of a ring of four blocks (three where four do not fit)
//   warps 10, 11     issue the MMAs of one warpgroup each, by an elected lane of a warp that walks and waits as a whole
// S = Q . codes^T is M 128, N 64; O += P . codes is M 128, N = Dh with P from tensor memory.  All operands are halves:
// queries of bf16 are exact in them (scaled by a power of two per row), codes are whole numbers, numerators keep
// 11 bits.  fp32: queries and numerators in two parts of 11 bits, each product once per part into the same accumulator.  Scales of keys go into the exponent's factor, scales of values into its offset and the reference (relative to the
// largest of the context, taken out of the row sum again), so O accumulates over all blocks.
// Two CTAs share an SM (256 TMEM columns each), so four warpgroups are in different phases of their blocks.  Head size 64
// and two parts have no room for P beside S: it overwrites the scores it came from, and the next scores wait for P . V.
// Measured (B200), bf16, 8192 queries x 8192 rows x 6 heads: head size 32 174 us (296 TFLOP/s, 2.3e12 exponentials a second),
// 16 161 us, 64 220 us (468 TFLOP/s); 87 us is what the special-function units need for the exponentials.  They are 65 % busy,
// issue slots 57 % (of some 440 instructions a warp and block 160 are the 64 numerators' own), the tensor pipe 15 %.  Two
// warpgroups alone on an SM take 2200 cycles a block each, four 3400: latency of a chain of loads, exponentials, stores and
// barriers with four warps a scheduler.  What was measured on the way at head size 32: masked blocks in
// code of their own 261 -> 226 us; MMAs issued by an elected lane instead of lane 0 of a divergent warp, scores read again
// (not kept) where the reference rises, waits in a tight loop 226 -> 208; all memory asked for before the first barrier,
// both halves of a block unrolled, the next scores as soon as these are read 208 -> 176.  A share of the exponentials on the FMA
// pipe (degree four, packed pairs) cost more issue slots than it freed at every share: 242 us with none, 246 with an eighth,
// 255 with a quarter of them.
// fp32, 4096 queries x 8192 rows x 6 heads: size 32 134 us (register tiles of cache_attn.cu 227), 16 123 (164), 64 148 (380).  Two
// parts of 32 numerators beside their scores do not fit 80 registers: sizes 16 and 32 spill 80 - 88 bytes a thread, read back in 164.
// Every wait is bounded; a CTA that gives up lets its MMAs end, frees its tensor memory and writes NaN for its rows.
#include "cache_attn.cuh"

namespace artab {
namespace {

constexpr int BM = 128, BN = kCacheBlock, kAhead = 3, kThreads = 384, kConvert = 64;
constexpr uint32_t kTmemCols = 256;
// numerators are 2^6 times exp(s - reference)
constexpr float kLiftTc = 6.0f;

struct Ctl {
  int abort_flag, pad;
  long long limit;
};
// Tensor memory of a warpgroup: scores, numerators (packed halves), output.  One part of the numerators has columns of its own
// where there is room; else numerators overwrite scores, those of 32 scores the columns of these: one part of both halves the
// upper 32, two parts (fp32) the 16 + 16 columns of their own half.
template <typename T, int DH>
struct Plan {
  static constexpr int kParts = sizeof(T) == 4 ? 2 : 1;
  static constexpr bool kAlias = DH == 64 || kParts == 2;
  static constexpr uint32_t kColO = kAlias ? BN : BN + BN / 2, kColsWg = kTmemCols / 2;
  static constexpr int kStages = DH == 64 && kParts == 2 ? 3 : 4;     // two CTAs in 227 KB
  // column of part `part` of the numerators of scores 32 c ..
  static constexpr uint32_t col_p(int c, int part) { return kParts == 2 ? 32 * c + 16 * part : (kAlias ? BN / 2 : BN) + 16 * c; }
};
template <typename T, int DH>
struct __align__(1024) TcSmem {
  using Pl = Plan<T, DH>;
  uint8_t k[Pl::kStages][BN * DH * 2];       // [64 rows][DH] halves
  uint8_t v[Pl::kStages][DH * 128];          // [DH][64 rows] halves
  uint8_t q[Pl::kParts][BM * DH * 2];
  uint8_t raw[kAhead][2 * BN * DH];          // records as they are kept
  uint64_t q_full, kv_full[Pl::kStages], kv_empty[Pl::kStages];
  uint64_t s_full[2], s_free[2], p_full[2], o_full[2], drained[2];
  float vmax[kThreads / 32];
  uint32_t tmem_base;
  Ctl ctl;
  static constexpr int kFree = Pl::kStages * (BN * DH * 2 + DH * 128) + Pl::kParts * BM * DH * 2;   // bytes that the merge may use
};

__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
// one lane of a whole warp, the same one every time
__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// False when the CTA is giving up (this wait or another one ran out).  The clock and the flag are looked at now and then
// only: eight warps of an SM wait at any time, and what they issue is taken from the others.
__device__ __forceinline__ bool mbar_tries(uint32_t b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, 32;\n"
      "again:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra done;\n\t"
      "sub.u32 n, n, 1;\n\t"
      "setp.ne.u32 q, n, 0;\n\t"
      "@q bra again;\n"
      "done:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(b), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __noinline__ bool mbar_wait_long(uint32_t b, uint32_t parity, volatile Ctl* ctl) {
  const long long t0 = clock64();
  for (;;) {
    if (mbar_tries(b, parity)) return true;
    if (ctl->abort_flag) return false;
    if (clock64() - t0 > ctl->limit) {
      ctl->abort_flag = 1;
      return false;
    }
  }
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile Ctl* ctl) {
  const uint32_t b = smem_u32(bar);
  return mbar_tries(b, parity) || mbar_wait_long(b, parity, ctl);
}

// K-major tile of rows of 32, 64 or 128 bytes: swizzle of that span, groups of eight rows behind one another
template <int ROW_BYTES>
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) {   // byte offset of a 16-byte chunk
  constexpr uint32_t kMask = ROW_BYTES / 16 - 1;
  constexpr uint32_t kShift = ROW_BYTES == 128 ? 0 : ROW_BYTES == 64 ? 1 : 2;
  return row * ROW_BYTES + ((chunk ^ ((row >> kShift) & kMask)) << 4);
}
__device__ __forceinline__ void st_shared16(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void st_shared4(uint32_t at, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
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
// Numerators of 32 scores of this thread's row against the reference m: packed halves (in one part or two), and their sum.
template <bool MASKED, int PARTS>
__device__ __forceinline__ float numerators(const uint32_t (&r)[32], uint32_t (&pk)[PARTS][16], float slope, float add, int live) {
  const float2 sl2 = make_float2(slope, slope), add2 = make_float2(add, add);
  float2 sums[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    float2 y = pk_fma(make_float2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), sl2, add2);
    y = make_float2(ex2(y.x), ex2(y.y));
    if (MASKED) {
      if (e >= live) y.x = 0.0f;
      if (e + 1 >= live) y.y = 0.0f;
    }
    sums[(e >> 1) & 1] = pk_add(sums[(e >> 1) & 1], y);
    const __half2 hi = __floats2half2_rn(y.x, y.y);
    pk[0][e >> 1] = h2_bits(hi);
    if constexpr (PARTS == 2) pk[1][e >> 1] = h2_bits(__floats2half2_rn(y.x - __low2float(hi), y.y - __high2float(hi)));
  }
  return (sums[0].x + sums[1].x) + (sums[0].y + sums[1].y);
}
template <bool MASKED>
__device__ __forceinline__ float largest(const uint32_t (&r)[32], int live) {
  float top[4];                                   // four chains: one would wait for itself
#pragma unroll
  for (int e = 0; e < 4; ++e) top[e] = -CUDART_INF_F;
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (!MASKED || e < live) top[e & 3] = fmaxf(top[e & 3], __uint_as_float(r[e]));
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

// One block of a warpgroup: scores of this thread's row out of tensor memory, numerators back into it, 32 columns at a
// time, the upper ones first (where numerators overwrite scores, they overwrite those).  MASKED: the block's last rows
// are not in use.  False when a wait gave up.
//
// The scores are read once: the reference m is a score of the row's first block (plus log2 of its value scale, `lift` - kLiftTc),
// and stays until the sum of 32
// numerators shows that one may have passed the range of halves (2^10 above m).  Then, rarely on ordinary
// scores, m rises by a whole number k and all that was taken against it shrinks by 2^-k, exactly: sums, the numerators
// that are in tensor memory, the output.  The result does not depend on m.
constexpr float kMostSum = 60000.0f;
template <typename T, int DH, bool MASKED>
__device__ __forceinline__ bool softmax_block(TcSmem<T, DH>* sm, uint32_t t_row, int wg, int i, float slope, float lift,
                                              float unlift, int live, float& m, float& l) {
  using Pl = Plan<T, DH>;
  constexpr bool kAlias = Pl::kAlias;
  constexpr uint32_t kColO = Pl::kColO;
  volatile Ctl* ctl = &sm->ctl;
  bool ok = true;
  float sum = 0.0f;
#pragma unroll
  for (int c = 1; c >= 0; --c) {
    uint32_t r[32], pk[Pl::kParts][16];
    tmem_ld32(t_row + 32 * c, r);
    wait_ld();
    const int lv = live - 32 * c;
    if (!kAlias && c == 0) {                      // the next scores may come
      fence_before();
      mbar_arrive(&sm->s_free[wg]);
    }
    if (i == 0 && c == 1) m = MASKED && lv <= 0 ? m : fmaf(largest<MASKED>(r, lv), slope, lift - kLiftTc);   // no row of these in use: not yet
    if (MASKED && i == 0 && c == 0 && live <= 32) m = fmaf(largest<MASKED>(r, lv), slope, lift - kLiftTc);
    float part = numerators<MASKED, Pl::kParts>(r, pk, slope, lift - m, lv);
    if (c == 1 && i > 0) {                        // the P . V before this one has read P and written O
      if (!kAlias) ok = __all_sync(0xffffffffu, mbar_wait(&sm->o_full[wg], (i - 1) & 1, ctl));
      fence_after();
    }
    if (__any_sync(0xffffffffu, !(part < kMostSum))) {
      float k = 0.0f;
      if (kAlias || c == 1) {   // still there: scores kept in registers for this cost the common path a copy each
        tmem_ld32(t_row + 32 * c, r);
        wait_ld();
      }
      if (!(part < kMostSum)) k = fmaxf(ceilf(fmaf(largest<MASKED>(r, lv), slope, lift - kLiftTc) - m), 0.0f);
      m += k;
      const float alpha = ex2(-k);
      part = numerators<MASKED, Pl::kParts>(r, pk, slope, lift - m, lv);
      l *= alpha;
      sum *= alpha;
      if (c == 0) {                               // the other half of this block's numerators, by way of fp32: as a half, alpha is 0 from 2^-25 on
        wait_st();
#pragma unroll 1
        for (int part = 0; part < Pl::kParts; ++part) {
          uint32_t u[16];
          tmem_ld16(t_row + Pl::col_p(1, part), u);
          wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
            u[e] = h2_bits(__floats2half2_rn(y.x * alpha, y.y * alpha));
          }
          tmem_st16(t_row + Pl::col_p(1, part), u);
        }
      }
      if (i > 0) {
#pragma unroll 1
        for (int d = 0; d < DH; d += 16) {
          uint32_t o[16];
          tmem_ld16(t_row + kColO + d, o);
          wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st16(t_row + kColO + d, o);
        }
        wait_st();
      }
    }
    sum += part;
#pragma unroll
    for (int part = 0; part < Pl::kParts; ++part) tmem_st16(t_row + Pl::col_p(c, part), pk[part]);
  }
  l = fmaf(sum, unlift, l);
  wait_st();
  fence_before();
  mbar_arrive(&sm->p_full[wg]);
  return ok;
}

template <typename T, int DH>
__global__ void __launch_bounds__(kThreads, 2) cache_attn_tc_kernel(const AttnArgs a, long long wait_cycles, int drop_commits) {
  using Pl = Plan<T, DH>;
  constexpr bool kAlias = Pl::kAlias;
  constexpr int kStages = Pl::kStages;
  constexpr uint32_t kColO = Pl::kColO, kColsWg = Pl::kColsWg;
  constexpr int KS = DH / 16, P = kPartial<DH>, KB = DH * 2;
  extern __shared__ uint8_t smem_raw[];
  using S = TcSmem<T, DH>;
  S* sm = reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  // the warp's number from its first lane: what follows from it is then known to be the same for all lanes, and an MMA takes
  // its operands from uniform registers as they are
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
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
      mbar_init(&sm->drained[w], 1);
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
  // Everything that comes from memory is asked for before the first barrier.
  const int wg = warp >> 2, row = tid & (BM - 1);     // softmax threads
  const int ct = tid - 256;                           // converting threads
  // a converting thread copies the pieces that it turns itself, three blocks ahead: no other thread waits for them
  const auto fetch = [&](int j) {
    if (j < nb) {
      const uint8_t* src = codes + (size_t)(rank + j * a.splits) * (2 * kCacheBlock * DH);
      const uint32_t dst = smem_u32(sm->raw[j % kAhead]);
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) cache_cp16(dst + (ct + i * kConvert) * 16, src + (ct + i * kConvert) * 16);
    }
    cp_commit();
  };
  float f = 0.0f;
  if (wg < 2) {
    float x[DH];
#pragma unroll
    for (int i = 0; i < DH; ++i) x[i] = 0.0f;
    const int r = row0 + row;
    if (r < a.rows)
      load_elements<T, DH>(reinterpret_cast<const T*>(a.q.p) + stream_of(r) * a.q.s0 + h * a.q.s1 +
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
        uint32_t u[Pl::kParts][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = x[8 * c + 2 * i] * to, z = x[8 * c + 2 * i + 1] * to;
          const __half2 hi = __floats2half2_rn(y, z);
          u[0][i] = h2_bits(hi);
          if constexpr (Pl::kParts == 2) u[1][i] = h2_bits(__floats2half2_rn(y - __low2float(hi), z - __high2float(hi)));
        }
#pragma unroll
        for (int part = 0; part < Pl::kParts; ++part)
          *reinterpret_cast<uint4*>(sm->q[part] + swizzled<KB>(row, c)) = make_uint4(u[part][0], u[part][1], u[part][2], u[part][3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
  } else if (warp < 10) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) fetch(j);
  }
  // largest value scale of the context, and whether a scale is not a number (what attends to such a block is not, either)
  float vmax = 0.0f;
  bool bad_k = false, bad_v = false;
  for (int i = tid; i < held; i += kThreads) {
    const float2 sc = scales[i];
    vmax = fmaxf(vmax, sc.y);
    bad_k |= sc.x != sc.x;
    bad_v |= sc.y != sc.y;
  }
  vmax = warp_max(vmax);
  if (lane == 0) sm->vmax[warp] = vmax;
  fence_before();
  bad_k = __syncthreads_or(bad_k);
  bad_v = __syncthreads_or(bad_v);
  fence_after();
  const uint32_t tmem = sm->tmem_base;

  // value scales are relative to 1 / inverse_scale(), which is the largest unless that is subnormal
  const auto inverse_scale = [&]() {
    float top = 0.0f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, sm->vmax[w]);
    return fminf(1.0f / top, 3e38f);
  };

  bool ok = true;
  float m = -CUDART_INF_F, l = 0.0f;
  const uint32_t t_row = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (wg & 1) * kColsWg;
  const int steps = wg < 2 ? (nb - wg + 1) / 2 : 0;   // blocks of the warpgroup

  if (warp >= 10) {
    // ------------------------------ MMA issuers ------------------------------
    // The whole warp walks and waits, one lane issues.
    const int w = warp - 10, n = (nb - w + 1) / 2;
    const uint32_t t_wg = tmem + w * kColsWg, q_addr = smem_u32(sm->q[0]);
    const auto wait = [&](uint64_t* bar, uint32_t parity) {
      const bool done = __all_sync(0xffffffffu, mbar_wait(bar, parity, ctl));
      if (done) fence_after();
      return done;
    };
    const auto scores = [&](int i) {                  // S = Q . K^T of step i
      const int j = 2 * i + w, st = j % kStages;
      if (!wait(&sm->kv_full[st], (j / kStages) & 1)) return false;
      const uint32_t k_addr = smem_u32(sm->k[st]);
      if (elected()) {
#pragma unroll
        for (int part = 0; part < Pl::kParts; ++part)
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            umma_ss(t_wg, tile_desc<KB>(q_addr + part * BM * KB + 32 * ks), tile_desc<KB>(k_addr + 32 * ks), idesc(BM, BN),
                    part + ks);
        if (!drop_commits) umma_commit(&sm->s_full[w]);
      }
      __syncwarp();
      return true;
    };
    if (n > 0) ok = wait(&sm->q_full, 0) && scores(0);
    for (int i = 0; ok && i < n; ++i) {
      const int st = (2 * i + w) % kStages;
      if (!kAlias && i + 1 < n) {                     // the next scores, as soon as these are in registers
        ok = wait(&sm->s_free[w], i & 1) && scores(i + 1);
        if (!ok) break;
      }
      ok = wait(&sm->p_full[w], i & 1);
      if (!ok) break;
      const uint32_t v_addr = smem_u32(sm->v[st]);
      if (elected()) {
#pragma unroll
        for (int part = 0; part < Pl::kParts; ++part)
#pragma unroll
          for (int ks = 0; ks < BN / 16; ++ks)
            umma_ts(t_wg + kColO, t_wg + Pl::col_p(ks >> 1, part) + 8 * (ks & 1), tile_desc<128>(v_addr + 32 * ks), idesc(BM, DH),
                    i > 0 || part + ks > 0);
        umma_commit(&sm->o_full[w]);
        umma_commit(&sm->kv_empty[st]);
      }
      __syncwarp();
      if (kAlias && i + 1 < n)                        // P lies where the next scores go
        ok = wait(&sm->o_full[w], i & 1) && scores(i + 1);
    }
    // no MMA outlives its operands and its tensor memory, whether or not the CTA is giving up
    if (elected()) umma_commit(&sm->drained[w]);
    __syncwarp();
    const uint32_t drained = smem_u32(&sm->drained[w]);
    for (const long long t0 = clock64(); !mbar_tries(drained, 0) && clock64() - t0 < kDefaultWaitCycles;) {
    }
  } else if (warp >= 8) {
    // ------------------------- codes into operand tiles -------------------------
    uint32_t k_at[KS], v_at[KS];                      // where a thread's pieces begin in a tile
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int u = ct + i * kConvert;
      k_at[i] = swizzled<KB>(u / KS, u % KS * 2);
      v_at[i] = swizzled<128>(u / 4, 0) + 4 * (u % 4);
    }
    for (int j = 0; ok && j < nb; ++j) {
      const int st = j % kStages;
      cp_wait<kAhead - 1>();
      uint4 rk[KS], rv[KS];
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const uint4* from = reinterpret_cast<const uint4*>(sm->raw[j % kAhead]) + ct + i * kConvert;
        rk[i] = from[0];
        rv[i] = from[kCacheBlock * DH / 16];
      }
      fetch(j + kAhead);
      if (j >= kStages) ok = __all_sync(0xffffffffu, mbar_wait(&sm->kv_empty[st], ((j / kStages) + 1) & 1, ctl));
      if (!ok) break;
      // the swizzle is an exclusive or of address bits that a tile's base leaves zero
      const uint32_t k_to = smem_u32(sm->k[st]), v_to = smem_u32(sm->v[st]);
#pragma unroll
      for (int i = 0; i < KS; ++i) {                  // 16 channels of a key: two chunks
        const uint32_t w[4] = {rk[i].x, rk[i].y, rk[i].z, rk[i].w};
#pragma unroll
        for (int e = 0; e < 2; ++e)
          st_shared16((k_to + k_at[i]) ^ (16 * e),
                      make_uint4(codes_to_halves(w[2 * e], false), codes_to_halves(w[2 * e], true),
                                 codes_to_halves(w[2 * e + 1], false), codes_to_halves(w[2 * e + 1], true)));
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {                  // 16 places of a value channel: rows 16 s + 8 h + 2 t + {0, 1}
        const uint32_t w[4] = {rv[i].x, rv[i].y, rv[i].z, rv[i].w};
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e) st_shared4((v_to + v_at[i]) ^ (32 * s + 16 * e), codes_to_halves(w[s], e));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&sm->kv_full[st]);
    }
    cp_wait<0>();
  } else {
    // --------------------------------- softmax ---------------------------------
    const float vinv = inverse_scale();
    if (wg == 0) mbar_arrive(&sm->q_full);
    float2 next = steps > 0 ? scales[rank + wg * a.splits] : make_float2(0.0f, 0.0f);
    for (int i = 0; i < steps; ++i) {
      const int blk = rank + (2 * i + wg) * a.splits;
      const float2 sc = next;
      if (i + 1 < steps) next = scales[blk + 2 * a.splits];
      const int live = len - blk * kCacheBlock;
      const float ratio = fmaxf(sc.y * vinv, kLeastRatio), lift = kLiftTc + lg2(ratio), unlift = rcp(ratio);
      const float slope = fmaxf(f * sc.x, 1e-37f);    // never 0: scores that are not finite stay so
      ok = __all_sync(0xffffffffu, mbar_wait(&sm->s_full[wg], i & 1, ctl));
      if (!ok) break;
      fence_after();
      ok = live < BN ? softmax_block<T, DH, true>(sm, t_row, wg, i, slope, lift, unlift, live, m, l)
                     : softmax_block<T, DH, false>(sm, t_row, wg, i, slope, lift, unlift, BN, m, l);
      if (!ok) break;
    }
    if (ok && steps > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sm->o_full[wg], (steps - 1) & 1, ctl));
    fence_after();
  }

  // both warpgroups' results where the tiles were: [2][128][kPartial]
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
    for (int d = 0; d < DH; d += 4) *reinterpret_cast<uint4*>(to + d) = make_uint4(o[d], o[d + 1], o[d + 2], o[d + 3]);
    to[DH] = m;
    to[DH + 1] = gave_up || bad_k ? CUDART_NAN_F : l;
  }
  if (a.splits == 1)
    __syncthreads();
  else
    cluster_meet();
  const float factor = bad_k || bad_v ? CUDART_NAN_F : 1.0f / inverse_scale();
  merge_rows<T, DH>(a, smem_u32(part), 2, rank * kThreads + tid, a.splits * kThreads, BM, row0, h, group, kLiftTc, factor);
  if (a.splits > 1) cluster_meet();
}

}  // namespace

template <typename T, int DH>
static int launch_tc(const AttnArgs& a, cudaStream_t s) {
  static SmemConfig config;
  static_assert(TcSmem<T, DH>::kFree >= 2 * BM * kPartial<DH> * 4, "the merge fits where the tiles were");
  const long long limit = debug_wait_cycles() ? debug_wait_cycles() : kDefaultWaitCycles;
  return launch_attn(cache_attn_tc_kernel<T, DH>, config, sizeof(TcSmem<T, DH>) + 1024, kThreads, a, s, limit, debug_drop_score_commits());
}

template <typename T>
int launch_cache_attn_tc(const AttnArgs& a, cudaStream_t s) {
  return a.c.head_dim == 16 ? launch_tc<T, 16>(a, s) : a.c.head_dim == 32 ? launch_tc<T, 32>(a, s) : launch_tc<T, 64>(a, s);
}
template int launch_cache_attn_tc<float>(const AttnArgs&, cudaStream_t);
template int launch_cache_attn_tc<__nv_bfloat16>(const AttnArgs&, cudaStream_t);

}  // namespace artab
