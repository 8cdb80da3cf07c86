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
// and no warp waits for another until the end, where the warps of a unit and the CTAs of a cluster (up to eight
// share the rows of a context) merge maximum, sum and output through shared memory.
// Measured (B200), queries of one row each: 8 contexts x 65536 rows x 8 heads of size 64, 81 us for 537 MB, called again and again
// (6.6 TB/s, a copy's rate; half of the issue slots busy), 97 with the launch and other data in between; size 32 51 us (5.3 TB/s),
// size 16 36 us (3.8 TB/s: 16 codes a lane between two shuffles).  64 contexts x 2048 rows x 6 heads, two queries each: size 16 9.5 us,
// 32 13, 64 18.4, fp32 the same; one context of 8192 rows 7 us: a chain of loads, products and merges.
#include "cache_tile.cuh"

namespace artab {
namespace {

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

// A unit is a tile of query rows of a (group, head), or (LIST) one query with its listed blocks: a CTA of W warps, or a cluster.
template <typename T, int DH, int PARTS, bool LIST, int W>
__global__ void __launch_bounds__(W * 32) cache_attn_kernel(const AttnArgs a) {
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
  const int n = LIST ? a.n_list : held;                       // blocks of the unit
  const int32_t* list = LIST ? a.list + unit * a.n_list : nullptr;
  const size_t gh = (size_t)group * H + h;
  const uint8_t* codes = a.c.codes + gh * a.c.n_blocks * (size_t)R::kRecord;
  const float* scales = a.c.scales + gh * a.c.n_blocks * 2;

  uint8_t* ring = smem + warp * R::kBytes;
  const uint32_t ring_addr = smem_u32(ring);
  const int first = rank * W + warp, step = a.splits * W;
  // block to fetch next; -1: nothing there.  Of a list, the lanes keep 32 entries of the warp's share
  int fetched = 0, entries = -1;
  const auto next_block = [&]() {
    const int k = fetched++, i = first + k * step;
    if (!LIST) return i < n ? i : -1;
    if (k % 32 == 0) {
      const int mine = i + lane * step;
      entries = mine < n ? list[mine] : -1;
    }
    const int b = __shfl_sync(0xffffffffu, entries, k % 32);
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
    ahead[i] = next_block();
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
    const int next = next_block();
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
  float* mine = part + W * ROWS * P;
  const auto merge = [&](auto at, int count, int row, int d, float& m, float& l, float& o) {
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
  const auto store = [&](int r, int d, float m, float l, float o) {
    const int row = row0 + r;
    if (row >= n_rows) return;
    const size_t at = ((size_t)stream_of(row) * H + h) * a.n_q + query_of(row);
    reinterpret_cast<T*>(a.out)[at * DH + d] = from_f32<T>(l == 0.0f ? 0.0f : o / (kUnlift * l));
    if (d == 0) a.lse[at] = l == 0.0f ? -CUDART_INF_F : (m - kLift) * kLn2 + logf(l);
  };
  for (int e = tid; e < ROWS * DH; e += W * 32) {
    float m, l, o;
    merge([&](int w, int i) { return part[w * ROWS * P + i]; }, W, e / DH, e % DH, m, l, o);
    if (a.splits == 1) {
      store(e / DH, e % DH, m, l, o);
    } else {
      mine[e / DH * P + e % DH] = o;
      if (e % DH == 0) mine[e / DH * P + DH] = m, mine[e / DH * P + DH + 1] = l;
    }
  }
  if (a.splits == 1) return;
  cluster_meet();
  const uint32_t base = smem_u32(mine);
  for (int e = rank * W * 32 + tid; e < ROWS * DH; e += a.splits * W * 32) {
    float m, l, o;
    merge([&](int w, int i) {
      return ld_cluster(base + i * 4, w);
    }, a.splits, e / DH, e % DH, m, l, o);
    store(e / DH, e % DH, m, l, o);
  }
  cluster_meet();
}

// ---- fp32 rows, some hundreds --------------------------------------------------------------------------------
// cache_attn_rows_kernel: the queries are the 16-row operand, part p of query g of a tile in row g + 8 p.  A CTA of four
// warps owns 64 queries and walks the blocks of its share together: each warp turns a quarter of a block's codes into
// half-precision fragments in shared memory, in the order in which a lane reads them with 16-byte loads, while the
// block before is worked on; the numerators go from the accumulators of one product straight into the operand
// registers of the next.  The value scale of a block is folded into the exponent and the maximum, relative to the largest of the
// context, so that one accumulator serves all blocks.  (bf16 queries and larger jobs: cache_attn_tc.cu.)
// B200, 6 heads of size 32: 512 queries x 2000 rows 16.6 us, 512 x 8192 41 us.  Two CTAs (size 64) or three of 168 registers an
// SM; with 1024 queries x 8192 rows (62 us) the tensor pipe is 40 % busy, issue slots 40 %: latency of a block's chain (scores,
// maximum, exponentials, second product) with twelve warps to hide it.
template <int DH>
struct RowTile {
  static constexpr int MT = 2, NW = 4;                              // tiles of 8 queries a warp, warps
  static constexpr int ROWS = NW * MT * 8;
  static constexpr int kBlockBytes = 2 * kCacheBlock * DH * 2;      // keys and values as halves
  static constexpr int kSmem = 2 * kBlockBytes > ROWS * kPartial<DH> * 4 ? 2 * kBlockBytes : ROWS * kPartial<DH> * 4;
};
template <int DH>
__global__ void __launch_bounds__(128, DH == 64 ? 2 : 3) cache_attn_rows_kernel(const AttnArgs a) {
  using RT = RowTile<DH>;
  constexpr int MT = RT::MT, NW = RT::NW, KS = DH / 16, ND = DH / 8, P = kPartial<DH>;
  constexpr int KN = 8 / NW, VN = ND > NW ? ND / NW : 1;         // key and value tiles that a warp lays out
  constexpr int KQ = KS >= 2 ? KS / 2 : 1;                       // 16-byte pieces of a lane's key fragments
  constexpr size_t kRecord = 2 * kCacheBlock * DH;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_max[NW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int rank = (int)(blockIdx.x % a.splits);
  const long unit = blockIdx.x / a.splits;
  const int H = a.c.n_heads, row0 = (int)(unit % a.tiles) * RT::ROWS, h = (int)(unit / a.tiles % H);
  const int group = (int)(unit / a.tiles / H);
  const bool one = a.c.n_groups == 1;
  const auto stream_of = [&](int row) { return one ? row / a.n_q : group; };
  const auto query_of = [&](int row) { return one ? row % a.n_q : row; };
  int len = a.c.lens[group];
  const int cap = a.c.n_blocks * kCacheBlock;
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int held = (len + kCacheBlock - 1) / kCacheBlock;
  const size_t gh = (size_t)group * H + h;
  const uint8_t* codes = a.c.codes + gh * a.c.n_blocks * kRecord;
  const float2* scales = reinterpret_cast<const float2*>(a.c.scales) + gh * a.c.n_blocks;

  uint32_t rk[KN][KS];
  uint4 rv[VN];
  const auto load = [&](int blk) {                                // raw codes of this warp's tiles
    const uint8_t* rec = codes + (size_t)blk * kRecord;
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const uint8_t* p = rec + (8 * (warp + i * NW) + g) * DH + t * (DH / 4);
      if constexpr (KS == 1) rk[i][0] = *reinterpret_cast<const uint32_t*>(p);
      if constexpr (KS == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        rk[i][0] = v.x, rk[i][1] = v.y;
      }
      if constexpr (KS == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        rk[i][0] = v.x, rk[i][1] = v.y, rk[i][2] = v.z, rk[i][3] = v.w;
      }
    }
#pragma unroll
    for (int i = 0; i < VN; ++i)
      if (ND >= NW || warp < ND)
        rv[i] = *reinterpret_cast<const uint4*>(rec + kCacheBlock * DH + (8 * (warp + i * NW) + g) * kCacheBlock + 16 * t);
  };
  const auto lay_out = [&](uint8_t* to) {
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const int j = warp + i * NW;
      if constexpr (KS == 1) {
        reinterpret_cast<uint2*>(to)[j * 32 + lane] = make_uint2(codes_to_halves(rk[i][0], false), codes_to_halves(rk[i][0], true));
      } else {
#pragma unroll
        for (int q = 0; q < KQ; ++q)
          reinterpret_cast<uint4*>(to)[(j * KQ + q) * 32 + lane] =
              make_uint4(codes_to_halves(rk[i][2 * q], false), codes_to_halves(rk[i][2 * q], true),
                         codes_to_halves(rk[i][2 * q + 1], false), codes_to_halves(rk[i][2 * q + 1], true));
      }
    }
    uint4* v = reinterpret_cast<uint4*>(to + 2 * kCacheBlock * DH);
#pragma unroll
    for (int i = 0; i < VN; ++i)
      if (ND >= NW || warp < ND) {
        const int j = warp + i * NW;
        v[(j * 2 + 0) * 32 + lane] = make_uint4(codes_to_halves(rv[i].x, false), codes_to_halves(rv[i].x, true),
                                                codes_to_halves(rv[i].y, false), codes_to_halves(rv[i].y, true));
        v[(j * 2 + 1) * 32 + lane] = make_uint4(codes_to_halves(rv[i].z, false), codes_to_halves(rv[i].z, true),
                                                codes_to_halves(rv[i].w, false), codes_to_halves(rv[i].w, true));
      }
  };
  if (rank < held) load(rank);

  // largest value scale of the context (a NaN among them shows in its own block)
  float vmax = 0.0f;
  for (int i = tid; i < held; i += 32 * NW) vmax = fmaxf(vmax, scales[i].y);
  vmax = warp_max(vmax);
  if (lane == 0) s_max[warp] = vmax;

  // queries: fragments a0 .. a3 of every k step
  uint32_t q[MT][KS][4];
  float f[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    constexpr int NE = DH / 4;
    const int row = row0 + (warp * MT + mt) * 8 + g;
    float x[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) x[i] = 0.0f;
    if (row < a.rows)
      load_elements<float, NE>(reinterpret_cast<const float*>(a.q.p) + stream_of(row) * a.q.s0 + h * a.q.s1 +
                               query_of(row) * a.q.s2 + t * NE, a.vec_q, x);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i) top = fmaxf(top, fabsf(x[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float to, back;
    row_scale(top, to, back);
    f[mt] = back * fabsf(a.scale_log2);
    to = copysignf(to, a.scale_log2);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float u = x[4 * s + 2 * j] * to, w = x[4 * s + 2 * j + 1] * to;
        const __half2 hi = __floats2half2_rn(u, w);
        q[mt][s][2 * j] = h2_bits(hi);
        q[mt][s][2 * j + 1] = h2_bits(__floats2half2_rn(u - __low2float(hi), w - __high2float(hi)));
      }
    }
  float m[MT], l[MT], o[MT][ND][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -CUDART_INF_F, l[mt] = 0.0f;
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][j][e] = 0.0f;
  }
  if (rank < held) {
    lay_out(smem);
    if (rank + a.splits < held) load(rank + a.splits);
  }
  __syncthreads();
  vmax = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  float poison = 0.0f;

  int buf = 0;
  for (int blk = rank; blk < held; blk += a.splits) {
    const float2 sc = scales[blk];
    const uint8_t* kv = smem + buf * RT::kBlockBytes;
    const int live = len - blk * kCacheBlock;
    // value scale: a factor of the numerators (in the exponent) and, back, of their sum
    float ratio = vmax > 0.0f ? sc.y / vmax : 0.0f;
    if (sc.y != sc.y) poison = sc.y, ratio = 1.0f;     // a block with values that are not finite: the weights are sound
    ratio = fmaxf(ratio, kLeastRatio);
    const float part_of = __log2f(ratio), lift = kLift + part_of, unlift = 1.0f / ratio;
    float c[MT][8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t b[KS][2];
      if constexpr (KS == 1) {
        const uint2 v = reinterpret_cast<const uint2*>(kv)[j * 32 + lane];
        b[0][0] = v.x, b[0][1] = v.y;
      } else {
#pragma unroll
        for (int i = 0; i < KQ; ++i) {
          const uint4 v = reinterpret_cast<const uint4*>(kv)[(j * KQ + i) * 32 + lane];
          b[2 * i][0] = v.x, b[2 * i][1] = v.y, b[2 * i + 1][0] = v.z, b[2 * i + 1][1] = v.w;
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c[mt][j][e] = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) mma_f16(c[mt][j], q[mt][s][0], q[mt][s][1], q[mt][s][2], q[mt][s][3], b[s][0], b[s][1]);
      }
    }
    uint32_t p[MT][4][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int j = 0; j < 8; ++j) c[mt][j][0] += c[mt][j][2], c[mt][j][1] += c[mt][j][3];
      if (live < kCacheBlock)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (8 * j + 2 * t + e >= live) c[mt][j][e] = -CUDART_INF_F;
      float mx = c[mt][0][0];
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fmaxf(c[mt][j][0], c[mt][j][1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float x = f[mt] * sc.x, slope = !(x <= 1e-37f) ? x : 1e-37f;      // never 0 (a masked score stays -inf), NaN as it is
      mx = fmaxf(m[mt], fmaf(mx, slope, part_of));
      const float base = mx == -CUDART_INF_F ? 0.0f : mx, alpha = ex2(m[mt] - base), add = lift - base;
      m[mt] = mx;
      if (__any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[mt][j][e] *= alpha;
      }
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = ex2(fmaf(c[mt][j][0], slope, add)), z = ex2(fmaf(c[mt][j][1], slope, add));
        sum += y + z;
        const __half2 hi = __floats2half2_rn(y, z);
        p[mt][j >> 1][2 * (j & 1)] = h2_bits(hi);
        p[mt][j >> 1][2 * (j & 1) + 1] = h2_bits(__floats2half2_rn(y - __low2float(hi), z - __high2float(hi)));
      }
      l[mt] = fmaf(l[mt], alpha, sum * unlift);
    }
    const uint4* v = reinterpret_cast<const uint4*>(kv + 2 * kCacheBlock * DH);
#pragma unroll
    for (int j = 0; j < ND; ++j) {
      const uint4 b0 = v[(j * 2 + 0) * 32 + lane], b1 = v[(j * 2 + 1) * 32 + lane];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mma_f16(o[mt][j], p[mt][0][0], p[mt][0][1], p[mt][0][2], p[mt][0][3], b0.x, b0.y);
        mma_f16(o[mt][j], p[mt][1][0], p[mt][1][1], p[mt][1][2], p[mt][1][3], b0.z, b0.w);
        mma_f16(o[mt][j], p[mt][2][0], p[mt][2][1], p[mt][2][2], p[mt][2][3], b1.x, b1.y);
        mma_f16(o[mt][j], p[mt][3][0], p[mt][3][1], p[mt][3][2], p[mt][3][3], b1.z, b1.w);
      }
    }
    buf ^= 1;
    if (blk + a.splits < held) {
      lay_out(smem + buf * RT::kBlockBytes);      // the buffer of the block before this one: all warps are past it
      if (blk + 2 * a.splits < held) load(blk + 2 * a.splits);
    }
    __syncthreads();
  }

  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = (warp * MT + mt) * 8 + g;
    float s = l[mt];
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    s += __shfl_xor_sync(0xffffffffu, s, 2);
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) part[row * P + 8 * j + 2 * t + e] = o[mt][j][e] + o[mt][j][2 + e] + poison;
    if (t == 0) part[row * P + DH] = m[mt], part[row * P + DH + 1] = s;
  }
  if (a.splits == 1)
    __syncthreads();
  else
    cluster_meet();
  merge_rows<float, DH>(a, smem_u32(part), 1, rank * 32 * NW + tid, a.splits * 32 * NW, RT::ROWS, row0, h, group, kLift, vmax);
  if (a.splits > 1) cluster_meet();
}

// CTAs that the GPU holds, `per_sm` an SM: a cluster of more than two has to fit into a part of the GPU of some 18 SMs, one
// of which is smaller
double held_ctas(int per_sm, int splits) {
  return splits <= 2 ? kSms * per_sm : (8 * (18 * per_sm / splits) - 1) * splits;
}
// Warps of a CTA and CTAs of a unit, the few-row kernel: the least of the times, in us, that a warp's blocks take on the SM with the
// most warps.  A block takes a warp `alone` + `shared` times the warps of its SM (measured, B200, 4 - 32 warps an SM; CTAs of one
// warp a fifth more); start and merge of a round 2.5, of clusters 4, and many of these are slow to find their
// places.
// Small CTAs spread better, larger ones need fewer partial results.  64 contexts x heads of 65536 rows of size 64: 2 CTAs of eight
// warps 86 us, 8 of two 82; 160 of 8192: 46 and, 4 of two, 33; 384 of 8192 of size 32: 4 of four 43, one of four 41; 240 of 4096 of
// size 16: 8 of two 16, one of eight 12; 512 contexts x 6 heads of 256 rows of size 32: one of eight 43, one of one 13.
struct FewPlan {
  double time;
  int warps, splits;
};
template <int DH>
FewPlan plan_few(long units, long blocks) {
  constexpr double alone = DH == 16 ? 0.2 : DH == 32 ? 0.36 : 0.5, shared = DH == 16 ? 0.047 : DH == 32 ? 0.062 : 0.09;
  constexpr int kRegisters = 72, kShared = 227 * 1024;    // the instances use 50 - 80 registers
  FewPlan best = {0.0, 0, 0};
  for (int warps = 1; warps <= 8; warps *= 2) {
    const int by_shared = kShared / (warps * Ring<DH>::kBytes + 1024), by_registers = 65536 / (32 * kRegisters * warps);
    const int fit = by_shared < by_registers ? by_shared : by_registers;
    for (int s = 1; s <= (warps == 1 ? 1 : 8); s *= 2) {
      const long ctas = units * s, per_sm = (ctas + kSms - 1) / kSms, per = (long)warps * s;
      const double full = held_ctas(fit, s), quotient = (double)ctas / full;
      const double rounds = ctas <= full ? 1.0 : 0.25 * quotient + 0.75 * (double)(long)(quotient + 0.999);
      const double block = alone + shared * (warps == 1 ? 1.2 : warps) * (per_sm < fit ? per_sm : fit);
      const double t = rounds * ((double)((blocks + per - 1) / per) * block + (s > 1 ? 4.0 : 2.5)) + (s > 1 && ctas > 600 ? 0.007 * (ctas - 600) : 0.0);
      if (!best.warps || t < best.time) best = {t, warps, s};
    }
  }
  return best;
}

template <typename T, int DH, int PARTS, bool LIST, int W>
int launch(const AttnArgs& a, cudaStream_t s) {
  static SmemConfig config;
  const size_t part = (size_t)(W + 1) * partial_floats<DH, PARTS>() * sizeof(float);
  const size_t ring = (size_t)W * Ring<DH>::kBytes;
  return launch_attn(cache_attn_kernel<T, DH, PARTS, LIST, W>, config, part > ring ? part : ring, W * 32, a, s);
}
template <typename T, int DH, int PARTS, bool LIST>
int launch_few(AttnArgs& a, const FewPlan& plan, cudaStream_t s) {
  a.splits = plan.splits;
  switch (plan.warps) {
    case 1: return launch<T, DH, PARTS, LIST, 1>(a, s);
    case 2: return launch<T, DH, PARTS, LIST, 2>(a, s);
    case 4: return launch<T, DH, PARTS, LIST, 4>(a, s);
    default: return launch<T, DH, PARTS, LIST, 8>(a, s);
  }
}
template <int DH>
int launch_rows(const AttnArgs& a, cudaStream_t s) {
  static SmemConfig config;
  return launch_attn(cache_attn_rows_kernel<DH>, config, RowTile<DH>::kSmem, RowTile<DH>::NW * 32, a, s);
}

// Which kernel, and how many CTAs share a unit's blocks: the least of the times that these figures give, in us.  Measured
// (B200) over 12 - 4096 rows, 1 - 384 contexts x heads and 500 - 32768 context rows: the pick is 1 - 3 % from the fastest in the
// mean, up to 26 % where two are close (1024 fp32 rows x 500 of size 64: few rows 19.6 us, tcgen05 15.6).  Few rows: plan_few, for size
// 32 a fifth more: over 64 - 1024 bf16 rows x 500 - 8192 x 6 heads the picks are then 0.2 % from the fastest in the mean and 4 % at
// most; without it 1.5 % and 19 %.  Sizes 16 and 64 have no such factor.
//   tiles of many rows: a CTA's time for a block when it has an SM to itself and when the SM is full; start and merge in either
//   case; CTAs of an SM; rows of a tile.  Splits that fill the last round matter: 4096 bf16 queries x 8192 rows x 6 heads of
//   size 32, 192 tiles, 120 us in one piece and 98 in two; 2048 x 32768, 96 tiles, 231 in two and 180 in four.
struct TileCost {
  double alone, full, start, start_full;
  int per_sm, rows;
};
// cache_attn_tc_kernel
template <typename T, int DH>
constexpr TileCost tc_cost() {
  if (sizeof(T) == 2) return DH == 16 ? TileCost{0.53, 0.8, 6.0, 9.0, 2, 128} : DH == 32 ? TileCost{0.56, 0.87, 6.0, 9.0, 2, 128} : TileCost{0.7, 1.0, 10.5, 13.5, 2, 128};
  return DH == 16 ? TileCost{0.77, 1.03, 8.0, 13.0, 2, 128} : DH == 32 ? TileCost{0.74, 1.06, 9.6, 15.0, 2, 128} : TileCost{0.78, 1.2, 13.8, 16.0, 2, 128};
}
// cache_attn_rows_kernel.  It starts sooner and has half the rows a tile, tcgen05 is faster once it runs (6 heads of size 32: 1024 queries x
// 500 rows 11.7 and 13.3 us, x 2000 20.5 and 22.6, x 8192 62 and 44; 4096 x 8192 227 and 134).
template <int DH>
constexpr TileCost rows_cost() {
  constexpr int rows = RowTile<DH>::ROWS;
  return DH == 16 ? TileCost{0.83, 1.7, 4.0, 4.0, 3, rows} : DH == 32 ? TileCost{0.96, 2.0, 4.0, 4.0, 3, rows} : TileCost{1.3, 2.3, 5.0, 5.0, 2, rows};
}
// least time over the splits of a unit, and those splits.  Of several rounds, the last one starts before the one before it has
// ended: between the sum of the rounds and what the work alone would take, the nearer to the sum the larger the clusters.
double tiles_time(const TileCost& c, const AttnArgs& a, long blocks, int& splits) {
  const double units = (double)a.units * (double)((a.rows + c.rows - 1) / c.rows);
  double least = 0.0;
  for (const int s : {1, 2, 4, 5, 8}) {
    const double ctas = units * s, cap = held_ctas(c.per_sm, s), each = (double)((blocks + s - 1) / s), merge = 0.9 * s;
    const auto round = [&](double n) {               // n CTAs at a time
      const double crowd = n <= 0.0 ? 0.0 : (double)(long)((n + kSms - 1) / kSms - 1.0) / (c.per_sm - 1), x = crowd < 1.0 ? crowd : 1.0;
      return n <= 0.0 ? 0.0 : (c.alone + (c.full - c.alone) * x) * each + c.start + (c.start_full - c.start) * x + merge;
    };
    double t = round(ctas);
    if (ctas > cap) {
      const double whole = (double)(long)(ctas / cap), rounds = whole * round(cap) + round(ctas - whole * cap);
      const double work = ctas / cap * c.full * each + c.start_full + merge, share = s <= 2 ? 0.5 : s == 4 ? 0.7 : 0.86;
      t = share * rounds + (1.0 - share) * work;
    }
    if (s == 1 || t < 0.96 * least) least = t, splits = s;   // more partial results have to be worth it
  }
  return least;
}

template <typename T, int DH>
int by_form(AttnArgs& a, long blocks, cudaStream_t s) {
  constexpr int kParts = sizeof(T) == 2 ? 1 : 2;
  const auto tiles = [&a](int rows) { a.tiles = (a.rows + rows - 1) / rows, a.units *= a.tiles; };
  if (a.list) return launch_few<T, DH, 2, true>(a, plan_few<DH>(a.units, blocks), s);
  const int form = debug_cache_form();
  const bool eight = kParts == 1 && a.rows > 4;
  FewPlan few = plan_few<DH>(a.units * ((a.rows + (eight ? 7 : 3)) / (eight ? 8 : 4)), blocks);
  if (form >= 2 || (form == 0 && a.rows > 8)) {
    if (DH == 32) few.time *= 1.2;
    constexpr TileCost tc = tc_cost<T, DH>();
    int tc_splits = 1;
    const double tc_time = tiles_time(tc, a, blocks, tc_splits);
    if constexpr (kParts == 2) {
      constexpr TileCost rows = rows_cost<DH>();
      int splits = 1;
      const double time = tiles_time(rows, a, blocks, splits);
      if (form == 2 || (form == 0 && time < tc_time && time < few.time)) {
        tiles(rows.rows);
        a.splits = splits;
        return launch_rows<DH>(a, s);
      }
    }
    if (form >= 2 || tc_time < few.time) {
      tiles(tc.rows);
      a.splits = tc_splits;
      return launch_cache_attn_tc<T>(a, s);
    }
  }
  tiles(eight ? 8 : 4);
  return eight ? launch_few<T, DH, kParts, false>(a, few, s) : launch_few<T, DH, 2, false>(a, few, s);
}

int attention(int dtype, const void* q, const int64_t* strides, int n_streams, int n_q, const artab_cache* c,
              int max_len, const int32_t* list, int n_list, float scale, void* out, float* lse, void* workspace,
              cudaStream_t s, const char* what) {
  int rc = check_cache(c, what);
  if (rc) return rc;
  rc = check_queries(dtype, q, n_streams, n_q, c, what);
  if (rc) return rc;
  ARTAB_REQUIRE(out && lse, ARTAB_EINVAL, "%s: null pointer", what);
  ARTAB_REQUIRE(reinterpret_cast<uintptr_t>(out) % 16 == 0, ARTAB_EINVAL, "%s: the output must be 16-byte aligned", what);
  AttnArgs a;
  a.c = *c;
  a.q = row_view(q, strides, c->n_heads, n_q, c->head_dim);
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
  if (workspace) return launch_cache_by_block(dtype, a, workspace, s);
  const long blocks = list ? n_list : (max_len + kCacheBlock - 1L) / kCacheBlock;
  a.splits = 1;
  if (dtype == ARTAB_F32) {
    if (c->head_dim == 16) return by_form<float, 16>(a, blocks, s);
    if (c->head_dim == 32) return by_form<float, 32>(a, blocks, s);
    return by_form<float, 64>(a, blocks, s);
  }
  if (c->head_dim == 16) return by_form<__nv_bfloat16, 16>(a, blocks, s);
  if (c->head_dim == 32) return by_form<__nv_bfloat16, 32>(a, blocks, s);
  return by_form<__nv_bfloat16, 64>(a, blocks, s);
}

}  // namespace

int check_queries(int dtype, const void* q, int n_streams, int n_q, const artab_cache* c, const char* what) {
  ARTAB_REQUIRE(dtype == ARTAB_F32 || dtype == ARTAB_BF16, ARTAB_EINVAL, "%s: bad dtype %d", what, dtype);
  ARTAB_REQUIRE(q, ARTAB_EINVAL, "%s: null pointer", what);
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
  return attention(dtype, q, q_strides, n_streams, n_q, c, max_len, nullptr, 0, scale, out, lse, nullptr,
                   (cudaStream_t)stream, "cache_attention");
}

int64_t artab_cache_block_workspace(const artab_cache* c, int n_streams, int n_q, int n_list) {
  if (check_cache(c, "cache_block_workspace") || n_streams < 1 || n_q < 1 || n_list < 1) return 0;
  return by_block_workspace(c, n_streams, n_q, n_list);
}

int artab_cache_block_attention(int dtype, const void* q, const int64_t* q_strides, int n_streams, int n_q,
                                const artab_cache* c, const int32_t* blocks, int n_list, float scale, void* out,
                                float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  ARTAB_REQUIRE(blocks && n_list >= 1, ARTAB_EINVAL, "cache_block_attention: no blocks");
  ARTAB_REQUIRE(n_list <= kMostListed, ARTAB_EINVAL, "cache_block_attention: %d blocks a query", n_list);
  int rc = check_cache(c, "cache_block_attention");
  if (rc) return rc;
  rc = check_queries(dtype, q, n_streams, n_q, c, "cache_block_attention");
  if (rc) return rc;
  const int64_t need = by_block_workspace(c, n_streams, n_q, n_list);
  ARTAB_REQUIRE(!need || !workspace || workspace_bytes >= need, ARTAB_ECAPACITY, "cache_block_attention: workspace too small");
  ARTAB_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, ARTAB_EINVAL, "cache_block_attention: workspace must be 16-byte aligned");
  return attention(dtype, q, q_strides, n_streams, n_q, c, 0, blocks, n_list, scale, out, lse, need ? workspace : nullptr,
                   (cudaStream_t)stream, "cache_block_attention");
}

}  // extern "C"
