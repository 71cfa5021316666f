// Attention weight by key over a bf16 cache (see key_weights.cu for what is
// computed).
//
// Few query rows (single tokens and a few more): bound by reading K once, 256
// bytes a key.  few_scores_kernel keeps the rows of Q as mma fragments and
// streams the pages of a key range from global memory straight into A
// fragments: the product does not depend on the order of the 128 dimensions,
// so a lane takes whole 16-byte chunks and Q is laid out to match.  For a few
// thousand keys a cluster takes a unit, keeps its scores in shared memory and
// writes the weights: one launch.  For more, every SM takes key ranges; their
// scores (4 bytes a key and row, which stay in L2) and (m, l) go to a workspace
// and few_sum_kernel turns them into weights.
//
// More rows: tensor_pass_kernel, the same product three ways.  A CTA keeps up
// to two 128-row tiles of one operand in shared memory and streams 128-row
// tiles of the other; each 128 x 128 product goes to tensor memory (two
// buffers per resident tile) and is read by two warpgroups, thread = row of
// the product, half of the columns each, while the other buffer is filled.
//   kLse     query rows resident, keys streamed, rows = query rows: a thread
//            keeps its row's running maximum and sum.
//   kSums    keys resident, query rows streamed, rows = keys: a thread adds up
//            exp(s - lse) over its columns.
//   kStream  at most two tiles of query rows, resident, keys streamed, rows =
//            keys: the sums of a key tile are complete with it.
// So no pass exchanges anything between threads per element.  Query rows are
// packed (token, head) pairs, so a chunk of a few tokens still fills a tile.
// Bound: the exponentials, two a (query, key) pair, against 512 flops: the
// MUFU alone would take 1024 cycles an SM for a product that the tensor cores
// do in 512.  Four warpgroups keep it fed, and one pair in eight goes to a
// polynomial of the same accuracy on the FMA pipe.
// A query row's maximum and sum reach the sums as one fp32 number, -(m + log2 l):
// with m and 1 / l apart, as the few-rows kernels have them, an element would
// take a product more.  Its rounding is half a step of a number of the scores'
// size, as the score's own is: 1.4e-7 to 1.8e-7 from the exact weights (plain
// fp32: 0.4e-7 to 1.1e-7).
#include <type_traits>

#include "common.cuh"
#include "fast_math.cuh"
#include "internal.h"
#include "key_weights.h"
#include "launch.cuh"
#include "page_layout.cuh"

namespace aoh {
namespace {

// ---------------------------------------------------------------------------
// few query rows
// ---------------------------------------------------------------------------
constexpr int kFewWarps = 8;
constexpr int kMaxOne = 16;             // CTAs of a unit's cluster
constexpr int kOneSmem = 160 * 1024;    // scores of one of them

struct FewArgs {
  KeyWeightsArgs a;
  float2* part;   // [split][unit row][row]
  float* score;   // [unit row][key][stride]: q . k, -inf where a row does not see the key
  int rows, splits;
  int cols, stride;      // of a key: scores that are written (no rows behind `rows`: -inf), floats
  long long score_unit;  // floats of a unit's scores
};

// NT tiles of 8 query rows.  kOne: the ranges of a unit are the CTAs of a
// cluster, which keep their scores in shared memory, combine their (m, l)
// across it and write the weights: one launch and no workspace.
template <int NT, bool kOne>
__global__ void __launch_bounds__(kFewWarps * 32, NT == 4 ? 1 : 2) few_scores_kernel(const __grid_constant__ FewArgs f) {
  __shared__ float2 red[kFewWarps][NT * 8];
  extern __shared__ __align__(16) float own_scores[];  // kOne: [key of the range][stride]
  const KeyWeightsArgs& a = f.a;
  griddep_wait();
  if (!kOne) griddep_launch_dependents();  // the sums wait for this grid to finish
  const int r = blockIdx.y;
  const RetrievalRow info = a.rows[r];
  const int unit = info.unit, base = info.table, held = info.held;
  const int past = key_weights_past(a), len = past + a.q_len;
  if (held == 0) {  // not stored here: no weight
    if (kOne && !a.accumulate)
      for (int j = blockIdx.x * blockDim.x + threadIdx.x; j < len; j += gridDim.x * blockDim.x)
        a.out[r * a.out_stride + j] = 0.f;
    return;
  }
  const int n_pages = (len + kPage - 1) / kPage;
  const int b = (unit - a.unit0) / a.g.G, kvh = (unit - a.unit0) % a.g.G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  const int p0 = (int)((long long)n_pages * blockIdx.x / f.splits), p1 = (int)((long long)n_pages * (blockIdx.x + 1) / f.splits);

  uint4 qf[NT][4];
  int last[NT][2];  // last key that the lane's two query rows see (-1: no such row)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = n * 8 + gq;
    const uint4* src = nullptr;
    if (row < f.rows)
      src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) +
                                           (((long long)b * a.q_len + row / a.g.grp) * a.g.Hq + kvh * a.g.grp + row % a.g.grp) *
                                               kHeadDim);
#pragma unroll
    for (int i = 0; i < 4; ++i) qf[n][i] = src ? src[4 * i + tq] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = n * 8 + 2 * tq + e;
      last[n][e] = col < f.rows ? past + col / a.g.grp : -1;
    }
  }
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) m[n][e] = -INFINITY, l[n][e] = 0.f;

  const char* pool = static_cast<const char*>(a.g.pool);
  // page ids of the warp's next 32 pages, one a lane
  int ids = -1, ids_at = -32;
  auto page_id = [&](int i) {  // i: the warp's i-th page
    if (i - ids_at >= 32) {
      ids_at = i;
      const int p = p0 + warp + (i + lane) * kFewWarps;
      ids = p < p1 && p < held ? a.g.block_table[base + p] : -1;
      if (p < p1 && (ids < 0 || ids >= a.g.num_pages)) {
        atomicOr(a.g.err, kErrBadPage);
        ids = -1;
      }
    }
    return __shfl_sync(0xffffffffu, ids, i - ids_at);
  };
  // chunk 4 i + t of rows g and g + 8
  auto load_page = [&](int id, uint4 (&k)[4][2]) {
    const char* src = pool + (long long)id * kPageBf16Bytes + gq * 128;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        k[i][h] = id < 0 ? make_uint4(0u, 0u, 0u, 0u)
                         : __ldcs(reinterpret_cast<const uint4*>(src + (i >> 1) * kHalfBytes + h * 1024 +
                                                                 (((4 * (i & 1) + tq) ^ gq) << 4)));
  };
  const int mine = p1 - p0 > warp ? (p1 - p0 - warp + kFewWarps - 1) / kFewWarps : 0;
  uint4 cur[4][2], nxt[4][2];
  if (mine > 0) load_page(page_id(0), cur);
  for (int i = 0; i < mine; ++i) {
    if (i + 1 < mine) load_page(page_id(i + 1), nxt);
    float c[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t a0[4] = {cur[k][0].x, cur[k][1].x, cur[k][0].y, cur[k][1].y};
        mma_bf16_16816(c[n], a0, qf[n][k].x, qf[n][k].y);
        const uint32_t a1[4] = {cur[k][0].z, cur[k][1].z, cur[k][0].w, cur[k][1].w};
        mma_bf16_16816(c[n], a1, qf[n][k].z, qf[n][k].w);
      }
    }
    const int j0 = (p0 + warp + i * kFewWarps) * kPage + gq;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float s[2][2];  // [key j0, j0 + 8][column]
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) s[h][e] = j0 + 8 * h <= last[n][e] ? c[n][2 * h + e] : -INFINITY;
      const int col = n * 8 + 2 * tq;
      if (col < f.cols) {
        float* o = kOne ? own_scores + (j0 - p0 * kPage) * f.stride + col
                        : f.score + r * f.score_unit + (long long)j0 * f.stride + col;
        *reinterpret_cast<float2*>(o) = make_float2(s[0][0], s[0][1]);
        *reinterpret_cast<float2*>(o + 8 * f.stride) = make_float2(s[1][0], s[1][1]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // the scaling is part of the subtraction's one rounding: scaled by itself, a score of 16 is 1e-6 off
        const float mt = fmaxf(s[0][e], s[1][e]) * kScoreScale;
        if (mt > m[n][e]) {
          l[n][e] *= fast_exp2(m[n][e] - mt);
          m[n][e] = mt;
        }
        if (m[n][e] > -INFINITY)
          l[n][e] += fast_exp2(fmaf(s[0][e], kScoreScale, -m[n][e])) + fast_exp2(fmaf(s[1][e], kScoreScale, -m[n][e]));
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) cur[k][0] = nxt[k][0], cur[k][1] = nxt[k][1];
  }
  // over the 8 lanes of a column, then over the warps
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float mm = m[n][e];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
      float ll = mm > -INFINITY ? l[n][e] * fast_exp2(m[n][e] - mm) : 0.f;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) ll += __shfl_xor_sync(0xffffffffu, ll, off);
      if (gq == 0) red[warp][n * 8 + 2 * tq + e] = make_float2(mm, ll);
    }
  __syncthreads();
  if (threadIdx.x < f.rows) {
    float mm = -INFINITY, ll = 0.f;
    for (int w = 0; w < kFewWarps; ++w) mm = fmaxf(mm, red[w][threadIdx.x].x);
    for (int w = 0; w < kFewWarps; ++w) {
      const float2 v = red[w][threadIdx.x];
      if (v.y > 0.f) ll += v.y * fast_exp2(v.x - mm);
    }
    if (kOne)
      red[0][threadIdx.x] = make_float2(mm, ll);  // a thread reads its own column of red alone
    else
      f.part[((long long)blockIdx.x * a.units + r) * f.rows + threadIdx.x] = make_float2(mm, ll);
  }
  if constexpr (kOne) {
    __shared__ float2 ml[NT * 8];  // of a row: its maximum and 1 / sum
    __syncwarp();
    cluster_sync_all();
    if (threadIdx.x < f.rows) {
      float mm = -INFINITY, ll = 0.f;
      float2 v[kMaxOne];
#pragma unroll
      for (int i = 0; i < kMaxOne; ++i) {
        v[i] = make_float2(-INFINITY, 0.f);
        if (i < f.splits)
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                       : "=f"(v[i].x), "=f"(v[i].y)
                       : "r"(mapa_shared(&red[0][threadIdx.x], i)));
        mm = fmaxf(mm, v[i].x);
      }
#pragma unroll
      for (int i = 0; i < kMaxOne; ++i)
        if (v[i].y > 0.f) ll = fmaf(v[i].y, fast_exp2(v[i].x - mm), ll);
      ml[threadIdx.x] = make_float2(mm, 1.f / ll);
    }
    __syncwarp();
    cluster_arrive();  // no CTA's red is read from here on
    __syncthreads();
    const int n = min(p1 * kPage, len) - p0 * kPage;
    for (int j = threadIdx.x; j < n; j += kFewWarps * 32) {
      float w = 0.f;
      for (int row = 0; row < f.rows; row += 2) {
        const float2 x = *reinterpret_cast<const float2*>(own_scores + j * f.stride + row);
        w = fmaf(fast_exp2(fmaf(x.x, kScoreScale, -ml[row].x)), ml[row].y, w);
        if (row + 1 < f.rows) w = fmaf(fast_exp2(fmaf(x.y, kScoreScale, -ml[row + 1].x)), ml[row + 1].y, w);
      }
      float* o = a.out + r * a.out_stride + p0 * kPage + j;
      *o = a.accumulate ? *o + w : w;
    }
    __syncwarp();
    cluster_wait();
  }
}

// Weights of 1024 keys from their scores, four keys a thread, S scores a key
// (f.stride), all of whose loads are in flight at once.
constexpr int kFewKeys = 4;
template <int S>
__global__ void __launch_bounds__(256) few_sum_kernel(const __grid_constant__ FewArgs f) {
  using Vec = typename std::conditional<S == 2, float2, float4>::type;
  constexpr int V = sizeof(Vec) / 4, kRanges = 5;  // ranges of a lane whose (m, l) are loaded together
  __shared__ float2 ml[S];  // of a row: its maximum and 1 / sum (their rounded logarithm would be 1e-6 off)
  const KeyWeightsArgs& a = f.a;
  const int r = blockIdx.y;
  const bool stored = a.rows[r].held > 0;
  const int len = key_weights_past(a) + a.q_len;
  const int j0 = blockIdx.x * 256 * kFewKeys + threadIdx.x;
  griddep_wait();
  if (blockIdx.x * 256 * kFewKeys >= len) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the scores are on their way while the ranges are combined
  const float* s = f.score + r * f.score_unit;
  Vec v[kFewKeys][S / V];
#pragma unroll
  for (int k = 0; k < kFewKeys; ++k)
    if (stored && j0 + 256 * k < len) {
#pragma unroll
      for (int c = 0; c < S / V; ++c) v[k][c] = reinterpret_cast<const Vec*>(s + (long long)(j0 + 256 * k) * S)[c];
    }
  if (threadIdx.x >= f.rows && threadIdx.x < S) ml[threadIdx.x] = make_float2(0.f, 0.f);
  if (stored) {
    for (int row = warp; row < f.rows; row += 8) {
      float m = -INFINITY, l = 0.f;
      for (int i0 = lane; i0 < f.splits; i0 += 32 * kRanges) {
        float2 p[kRanges];
        float mm = m;
#pragma unroll
        for (int k = 0; k < kRanges; ++k) {
          const int i = i0 + 32 * k;
          p[k] = i < f.splits ? f.part[((long long)i * a.units + r) * f.rows + row] : make_float2(-INFINITY, 0.f);
          mm = fmaxf(mm, p[k].x);
        }
        if (l > 0.f) l *= fast_exp2(m - mm);
#pragma unroll
        for (int k = 0; k < kRanges; ++k)
          if (p[k].y > 0.f) l = fmaf(p[k].y, fast_exp2(p[k].x - mm), l);
        m = mm;
      }
      float mm = m;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
      l = m > -INFINITY ? l * fast_exp2(m - mm) : 0.f;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
      if (lane == 0) ml[row] = make_float2(mm, 1.f / l);
    }
  }
  __syncthreads();
  float w[kFewKeys] = {};
#pragma unroll
  for (int k = 0; k < kFewKeys; ++k) {
    if (!stored || j0 + 256 * k >= len) continue;
#pragma unroll
    for (int c = 0; c < S / V; ++c) {
      const float* x = reinterpret_cast<const float*>(&v[k][c]);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 m = ml[c * V + e];
        w[k] = fmaf(fast_exp2(fmaf(x[e], kScoreScale, -m.x)), m.y, w[k]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kFewKeys; ++k) {
    if (j0 + 256 * k >= len) continue;
    float* o = a.out + r * a.out_stride + j0 + 256 * k;
    *o = a.accumulate ? *o + w[k] : w[k];
  }
}

// ---------------------------------------------------------------------------
// tensor cores
// ---------------------------------------------------------------------------
constexpr int kTcThreads = 640;  // warp 0 loads, warp 1 issues, warps 4..19: two warpgroups per resident tile
constexpr int kStages = 3;
constexpr int kTileRows = 128;
constexpr int kHalfTile = kTileRows * 128;   // 64 dimensions of 128 rows
constexpr int kTileBytes = 2 * kHalfTile;    // 32 KB
constexpr int kLseBytes = kTileRows * 4;
// Slots of the streamed columns' -lse.  A warpgroup hands a product's buffer
// back before it has read that tile's slot, so the products may be two tiles
// ahead of it and the loads kStages ahead of those: a slot must outlive
// kStages + 2 tiles.
constexpr int kLseSlots = 8;
static_assert(kLseSlots > kStages + 2, "a slot of -lse would be loaded over while it is read");
constexpr int kTcSmem = (2 + kStages) * kTileBytes + kLseSlots * kLseBytes + 1024;  // + alignment
constexpr int kTmemCols = 512;

enum { kLse = 0, kSums = 1, kStream = 2 };

struct TcArgs {
  KeyWeightsArgs a;
  float2* part;    // [split][unit row][row tile * 128 + row]: (m, l) by key range (kLse; kStream reads them)
  float* neg_lse;  // [unit row][row tile * 128 + row]: -lse, -inf for rows that hold no query (kSums)
  float* sums;     // [row split][unit row][key], kSums with several row ranges
  int row_tiles, tile_tokens;
  int pairs;       // pairs of resident tiles of a unit
  int splits;      // ranges of the streamed tiles
  int lse_splits;  // ranges that part holds
  long long sums_unit;
};

// Waits for this thread's tensor-memory loads.  The registers pass through, so
// that nothing the compiler does with them moves before the wait.
__device__ __forceinline__ void tc_wait_ld32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), 
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), 
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), 
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// Exponentials of 32 scores, added to acc: 2^(s * scale + b), b per column
// pair.  One pair in eight takes the FMA pipe (none: 313 us for a pass over
// 4096 x 16K keys of 4 units, one or two: 294, three: 314, four: 339 -- the
// polynomial's twelve instructions soon cost more than the MUFU's wait); a
// masked tile's scores (-inf, whose power must be exactly 0) all take the MUFU.
template <bool kPoly, class B>
__device__ __forceinline__ void add_exp2(const uint32_t (&sv)[32], B&& b, uint64_t (&acc)[4]) {
  const uint64_t scale2 = f2_pack(kScoreScale, kScoreScale);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), scale2, b(e));
    if (kPoly && (e & 7) == 7) {
      acc[e & 3] = f2_add(acc[e & 3], exp2_poly2_f32(x2));
    } else {
      float x0, x1;
      f2_unpack(x2, x0, x1);
      acc[e & 3] = f2_add(acc[e & 3], f2_pack(fast_exp2(x0), fast_exp2(x1)));
    }
  }
}

__device__ __forceinline__ float total(const uint64_t (&acc)[4]) {
  float u[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) f2_unpack(acc[k], u[2 * k], u[2 * k + 1]);
  return ((u[0] + u[1]) + (u[2] + u[3])) + ((u[4] + u[5]) + (u[6] + u[7]));
}

// One 128 x 128 product over 128 dimensions: eight instructions of 16
// dimensions, four in each 64-dim half.  The descriptors differ from the first
// one's by their address fields (units of 16 bytes) alone, so stepping them is
// one addition each: the issuing warp shares its scheduler with four busy
// warps, and with descriptors built one by one it was late with the products.
__device__ __forceinline__ void mma_tile(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred l, no, yes;\n\t.reg .u32 lid;\n\t.reg .b64 x, y;\n\t"
      "mov.u32 lid, %%laneid;\n\tsetp.eq.u32 l, lid, 0;\n\tsetp.ne.u32 no, 0, 0;\n\tsetp.eq.u32 yes, 0, 0;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, no;\n\t"
      "add.s64 x, %1, 2;\n\tadd.s64 y, %2, 2;\n\t@l tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, yes;\n\t"
      "add.s64 x, %1, 4;\n\tadd.s64 y, %2, 4;\n\t@l tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, yes;\n\t"
      "add.s64 x, %1, 6;\n\tadd.s64 y, %2, 6;\n\t@l tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, yes;\n\t"
      "add.s64 x, %1, 1024;\n\tadd.s64 y, %2, 1024;\n\t@l tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, yes;\n\t"
      "add.s64 x, %1, 1026;\n\tadd.s64 y, %2, 1026;\n\t@l tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, yes;\n\t"
      "add.s64 x, %1, 1028;\n\tadd.s64 y, %2, 1028;\n\t@l tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, yes;\n\t"
      "add.s64 x, %1, 1030;\n\tadd.s64 y, %2, 1030;\n\t@l tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, yes;\n\t"
      "}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc)
      : "memory");
}
static_assert(kHalfTile / 16 == 1024, "descriptor step between the halves");

// (m, l) of two disjoint sets of keys as one.
__device__ __forceinline__ float2 merge_ml(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  const float la = a.y > 0.f ? a.y * fast_exp2(a.x - m) : 0.f, lb = b.y > 0.f ? b.y * fast_exp2(b.x - m) : 0.f;
  return make_float2(m, la + lb);
}

template <int kPass>
__global__ void __launch_bounds__(kTcThreads, 1)
    tensor_pass_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ TcArgs t) {
  constexpr bool kKeysStreamed = kPass != kSums;    // otherwise the query rows are
  constexpr bool kQueriesResident = kPass != kSums;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_a, bar_final, bar_full[kStages], bar_empty[kStages], bar_s_full[2][2], bar_s_empty[2][2],
      bar_lse[kLseSlots], bar_part_full[2], bar_part_empty[2];
  __shared__ float2 s_row[2][kTileRows];     // kLse, kSums: what the second half's warpgroups found
  __shared__ float s_part[2][3][kTileRows];  // kStream: sums of all but the first warpgroup, [slot][warpgroup - 1][key]
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  const KeyWeightsArgs& a = t.a;
  const CacheGeom& G = a.g;
  uint8_t* sA = smem_raw + (1024 - (smem_u32(smem_raw) & 1023)) % 1024;  // resident tiles
  uint8_t* sB = sA + 2 * kTileBytes;                                     // ring of streamed tiles
  float* sLse = reinterpret_cast<float*>(sB + kStages * kTileBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  if (kPass == kLse) griddep_wait();  // before the next pass may start: it reads the lengths without waiting itself
  if (kPass == kLse || (kPass == kSums && t.splits > 1)) griddep_launch_dependents();  // not the call's last kernel

  // this CTA's resident pair and range of streamed tiles
  const int split = blockIdx.x % t.splits;
  const int item = blockIdx.x / t.splits;
  const int r = item % a.units;
  // causal: late query rows see more keys, early keys are seen by more rows -- the long items first
  const int pair = kPass == kLse ? t.pairs - 1 - item / a.units : item / a.units;
  const RetrievalRow info = a.rows[r];
  const int unit = info.unit, base = info.table, held = info.held;
  const int past = key_weights_past(a), len = past + a.q_len;
  const int b = (unit - a.unit0) / G.G, kvh = (unit - a.unit0) % G.G;
  const int tt = t.tile_tokens;
  const int key_tiles = (len + kTileRows - 1) / kTileRows;
  const int na = min(2, (kQueriesResident ? t.row_tiles : key_tiles) - 2 * pair);  // a device length may leave none
  if (na <= 0) {
    if (kPass != kLse) griddep_wait();  // no grid ends before those in front of it
    return;
  }
  int first = 0, end;  // streamed tiles that any resident row needs
  if (kPass == kSums) {
    first = max(0, 2 * pair * kTileRows - past) / tt;
    end = t.row_tiles;
  } else {
    end = (past + min(a.q_len, (2 * pair + na) * tt) + kTileRows - 1) / kTileRows;
  }
  const int t0 = first + (int)((long long)(end - first) * split / t.splits);
  const int n = first + (int)((long long)(end - first) * (split + 1) / t.splits) - t0;
  if (held == 0) {  // not stored here: no weight
    if (kPass == kLse) return;
    griddep_wait();
    const int lo = kPass == kSums ? 2 * pair * kTileRows : t0 * kTileRows;
    const int hi = min(len, kPass == kSums ? lo + 2 * kTileRows : (t0 + n) * kTileRows);
    for (int j = lo + tid; j < hi; j += kTcThreads) {
      if (kPass == kSums && t.splits > 1)
        t.sums[((long long)split * a.units + r) * t.sums_unit + j] = 0.f;
      else if (!a.accumulate)
        a.out[r * a.out_stride + j] = 0.f;
    }
    return;
  }

  // K rows of 128 keys: lane = (page, 64-dim half), 2 KB each; the page id is not looked at until the tile's turn
  auto wanted = [&](int tile) { return lane < 16 && (tile * 8 + (lane >> 1)) * kPage < len; };
  auto fetch_id = [&](int tile) {
    const int p = tile * 8 + (lane >> 1);
    return wanted(tile) && p < held ? G.block_table[base + p] : -1;
  };
  int id_next = -1, id_second = -1;
  if (warp == 0) {
    if (kKeysStreamed) {
      if (n > 0) id_next = fetch_id(t0);
    } else {
      id_next = fetch_id(2 * pair);
      if (na > 1) id_second = fetch_id(2 * pair + 1);
    }
  }
  if (warp == 1) {
    tmem_alloc(&s_tmem, kTmemCols);
    tmem_relinquish();
  }
  if (tid == 0) {
    mbar_init(&bar_a, 1);
    mbar_init(&bar_final, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], 1);
    }
    for (int s = 0; s < kLseSlots; ++s) mbar_init(&bar_lse[s], 1);
    for (int u = 0; u < 2; ++u) {
      for (int k = 0; k < 2; ++k) {
        mbar_init(&bar_s_full[u][k], 1);
        mbar_init(&bar_s_empty[u][k], 256);
      }
      mbar_init(&bar_part_full[u], (2 * na - 1) * 128);
      mbar_init(&bar_part_empty[u], 128);
    }
    s_abort = 0;
    fence_mbar_init();
  }
  // rows of a tile of queries that no load writes: zero scores, which -lse = -inf turns to nothing
  const int q_rows = tt * G.grp;
  if (kPass != kLse) {
    uint8_t* tiles = kPass == kSums ? sB : sA;
    const int halves = kPass == kSums ? 2 * kStages : 4, tail = kTileRows - q_rows;
    for (int i = tid; i < halves * tail * 8; i += kTcThreads) {
      const int row = q_rows + (i / 8) % tail, h = i / 8 / tail;
      reinterpret_cast<uint4*>(tiles + h * kHalfTile + row * 128)[i % 8] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  float m = -INFINITY, sum = 0.f;  // of this thread's row, where it has one

  if (warp == 0) {
    // ============================ loads ============================
    const uint8_t* pool = static_cast<const uint8_t*>(G.pool);
    const uint32_t q_bytes = (uint32_t)q_rows * 256;
    auto check_id = [&](int tile, int id) {
      if (!wanted(tile) || (id >= 0 && id < G.num_pages)) return id;
      atomicOr(G.err, kErrBadPage);
      return -1;
    };
    auto copy_keys = [&](int id, uint8_t* dst, uint64_t* bar) {
      if (id >= 0)
        bulk_load(dst + (lane & 1) * kHalfTile + (lane >> 1) * kBlockBytes,
                  pool + (size_t)id * kPageBf16Bytes + (lane & 1) * kHalfBytes, kBlockBytes, bar);
    };
    // one arrival for `blocks` copies of 2 KB
    auto expect_blocks = [&](uint64_t* bar, int blocks) {
      if (lane == 0) {
        if (blocks)
          mbar_arrive_expect_tx(bar, blocks * kBlockBytes);
        else
          mbar_arrive(bar);
      }
      __syncwarp();
    };
    auto load_queries = [&](int tile, uint8_t* dst, uint64_t* bar) {
      tma_load_4d(dst, &tm_q, bar, 0, kvh * G.grp, tile * tt, b);
      tma_load_4d(dst + kHalfTile, &tm_q, bar, 64, kvh * G.grp, tile * tt, b);
    };
    if (kQueriesResident) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&bar_a, na * q_bytes);
        for (int w = 0; w < na; ++w) load_queries(2 * pair + w, sA + w * kTileBytes, &bar_a);
      }
    } else {
      const int id0 = check_id(2 * pair, id_next), id1 = na > 1 ? check_id(2 * pair + 1, id_second) : -1;
      expect_blocks(&bar_a, __popc(__ballot_sync(0xffffffffu, id0 >= 0)) + __popc(__ballot_sync(0xffffffffu, id1 >= 0)));
      copy_keys(id0, sA, &bar_a);
      copy_keys(id1, sA + kTileBytes, &bar_a);
      griddep_wait();  // the lse that the first pass found
    }
    int issued = 0;
    for (int i = 0; i < n; ++i) {
      const int s = i % kStages;
      const int id = kKeysStreamed ? check_id(t0 + i, id_next) : -1;
      if (kKeysStreamed && i + 1 < n) id_next = fetch_id(t0 + i + 1);
      // the stages of the first two tiles come free without the pass before (products 0 and 1 are all that is made
      // ahead of it); the later ones' bounded waits time this grid alone
      if (kPass == kStream && i == kStages + 2) griddep_wait();
      if (lane == 0 && i >= kStages && !s_abort) {
        if (!mbar_wait(&bar_empty[s], (i / kStages - 1) & 1, G.err)) s_abort = 1;
      }
      __syncwarp();
      if (s_abort) break;
      uint8_t* dst = sB + s * kTileBytes;
      if (kKeysStreamed) {
        expect_blocks(&bar_full[s], __popc(__ballot_sync(0xffffffffu, id >= 0)));
        copy_keys(id, dst, &bar_full[s]);
      } else if (lane == 0) {
        const int slot = i % kLseSlots;
        mbar_arrive_expect_tx(&bar_full[s], q_bytes);
        load_queries(t0 + i, dst, &bar_full[s]);
        mbar_arrive_expect_tx(&bar_lse[slot], kLseBytes);
        bulk_load(sLse + slot * kTileRows, t.neg_lse + ((long long)r * t.row_tiles + t0 + i) * kTileRows, kLseBytes,
                  &bar_lse[slot]);
      }
      issued = i + 1;
      __syncwarp();
    }
    // nothing this CTA issued may still be landing when it exits
    if (lane == 0) {
      mbar_wait(&bar_a, 0, G.err);
      for (int i = max(0, issued - kStages); i < issued; ++i) {
        mbar_wait(&bar_full[i % kStages], (i / kStages) & 1, G.err);
        if (kPass == kSums) mbar_wait(&bar_lse[i % kLseSlots], (i / kLseSlots) & 1, G.err);
      }
    }
  } else if (warp == 1) {
    // ============================ products ============================
    constexpr uint32_t kIdesc = idesc_bf16(kTileRows, kTileRows, 0, 0);
    if (kPass == kSums) griddep_wait();  // the bounded waits time this grid, not the one before
    bool ok = mbar_wait_warp(&bar_a, 0, G.err);
    tc_fence_after();
    const uint64_t res = smem_desc_sw128(smem_u32(sA), 16, 1024), str0 = smem_desc_sw128(smem_u32(sB), 16, 1024);
    uint64_t str = str0;
    int s = 0;
    uint32_t round = 0;  // of the ring: parity of bar_full[s]
    for (int i = 0; i < n && ok && !s_abort; ++i) {
      if (!(ok = mbar_wait_warp(&bar_full[s], round & 1, G.err))) break;
      const int buf = i & 1;
      for (int w = 0; w < na && ok; ++w) {
        if (kPass == kStream && i == 2 && w == 0) griddep_wait();  // as the warpgroups that give the buffers back
        if (i >= 2 && !(ok = mbar_wait_warp(&bar_s_empty[w][buf], ((i >> 1) - 1) & 1, G.err))) break;
        tc_fence_after();
        const uint64_t tile = res + w * (kTileBytes / 16);
        mma_tile(tmem + (w * 2 + buf) * kTileRows, kPass == kStream ? str : tile, kPass == kStream ? tile : str, kIdesc);
        mma_commit(&bar_s_full[w][buf]);
      }
      if (ok) mma_commit(&bar_empty[s]);
      str += kTileBytes / 16;
      if (++s == kStages) {
        s = 0;
        str = str0;
        ++round;
      }
    }
    if (!ok) s_abort = 1;
    __syncwarp();
    mma_commit(&bar_final);  // fires once every product issued above has completed
  } else if (warp >= 4 && (warp - 4) / 8 < na) {
    // ============================ exponentials ============================
    const int u = (warp - 4) / 4, w = u >> 1, h = u & 1;  // half h of the columns of resident tile w's products
    const int row = 32 * (warp & 3) + lane;
    const uint32_t s_col = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + w * 2 * kTileRows + 64 * h;
    const int tile = 2 * pair + w;
    const int last = past + tile * tt + row / G.grp;  // kLse: last key the row's query sees
    if (kPass != kLse) griddep_wait();
    if (kPass == kStream) {
      // -lse of the resident query rows from their key ranges, while the first
      // products are made: two threads a row, 20 ranges of each in flight (one
      // thread with eight at a time took 2 us more for 37 ranges)
      constexpr int kRanges = 20;
      const long long rows = (long long)a.units * t.row_tiles * kTileRows;
      const int i = (tid - 128) >> 1;  // of na * 128 rows
      const float2* p = t.part + ((long long)r * t.row_tiles + 2 * pair) * kTileRows + i;
      float mm = -INFINITY, ll = 0.f;
      for (int k0 = tid & 1; k0 < t.lse_splits; k0 += 2 * kRanges) {
        float2 v[kRanges];
        float top = mm;
#pragma unroll
        for (int k = 0; k < kRanges; ++k) {
          v[k] = k0 + 2 * k < t.lse_splits ? p[(k0 + 2 * k) * rows] : make_float2(-INFINITY, 0.f);
          top = fmaxf(top, v[k].x);
        }
        if (ll > 0.f) ll *= fast_exp2(mm - top);
#pragma unroll
        for (int k = 0; k < kRanges; ++k)
          if (v[k].y > 0.f) ll = fmaf(v[k].y, fast_exp2(v[k].x - top), ll);
        mm = top;
      }
      const float om = __shfl_xor_sync(0xffffffffu, mm, 1), ol = __shfl_xor_sync(0xffffffffu, ll, 1);
      const float2 ml = merge_ml(make_float2(mm, ll), make_float2(om, ol));
      if ((tid & 1) == 0) sLse[i] = ml.y > 0.f ? -(ml.x + log2f(ml.y)) : -INFINITY;
      named_bar_sync(1, na * 256);  // all threads of this role
    }
    uint64_t acc[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = 0;
    // 32 scores of product i, from column 64 h + c0 on, are added up
    auto add_scores = [&](int i, int c0, uint32_t (&sv)[32]) {
      // the tile of keys and the first token of the tile of queries of this product
      const int key0 = (kKeysStreamed ? t0 + i : tile) * kTileRows, tok0 = (kQueriesResident ? tile : t0 + i) * tt;
      const bool full = key0 + kTileRows - 1 <= past + tok0;  // every token sees every key
      if (!full) {
        // rows = keys: columns from the first token that sees the row's key on
        const int c_min = max(0, key0 + row - past - tok0) * G.grp - 64 * h - c0, k_max = last - key0 - 64 * h - c0;
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (kPass == kLse ? e > k_max : e < c_min) sv[e] = __float_as_uint(-INFINITY);
      }
      if (kPass == kLse) {
        float mx[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = fmaxf(__uint_as_float(sv[2 * k]), __uint_as_float(sv[2 * k + 1]));
#pragma unroll
        for (int e = 8; e < 32; e += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mx[k] = fmax3(mx[k], __uint_as_float(sv[e + 2 * k]), __uint_as_float(sv[e + 2 * k + 1]));
        const float mt = fmax3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * kScoreScale;
        if (mt > m) {
          const float f = fast_exp2(m - mt);
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[k] = f2_fma(acc[k], f2_pack(f, f), 0);
          m = mt;
        }
        const float nm = m == -INFINITY ? 0.f : -m;
        const uint64_t nm2 = f2_pack(nm, nm);
        if (full)
          add_exp2<true>(sv, [&](int) { return nm2; }, acc);
        else
          add_exp2<false>(sv, [&](int) { return nm2; }, acc);
      } else {
        const ulonglong2* nl =
            reinterpret_cast<const ulonglong2*>(sLse + (kPass == kSums ? i % kLseSlots : w) * kTileRows + 64 * h + c0);
        ulonglong2 v = make_ulonglong2(0, 0);
        auto column = [&](int e) {
          if (e % 2 == 0) v = nl[e / 2];
          return e % 2 == 0 ? v.x : v.y;
        };
        if (full)
          add_exp2<true>(sv, column, acc);
        else
          add_exp2<false>(sv, column, acc);
      }
    };
    // Each 32 columns are on their way from tensor memory while the 32 before
    // them are worked on.
    auto arrived = [&](int i) {  // product i (and its columns' -lse)
      if (kPass == kSums && !mbar_wait(&bar_lse[i % kLseSlots], (i / kLseSlots) & 1, G.err)) return false;
      if (!mbar_wait(&bar_s_full[w][i & 1], (i >> 1) & 1, G.err)) return false;
      tc_fence_after();
      return true;
    };
    uint32_t lo[32], hi[32];
    bool ok = n > 0 && arrived(0);
    if (ok) tmem_ld32(s_col, lo);
    for (int i = 0; i < n && ok; ++i) {
      const int buf = i & 1;
      tc_wait_ld32(lo);
      tmem_ld32(s_col + buf * kTileRows + 32, hi);
      add_scores(i, 0, lo);
      tc_wait_ld32(hi);
      tc_fence_before();
      mbar_arrive(&bar_s_empty[w][buf]);
      if (i + 1 < n) {
        ok = arrived(i + 1);
        if (ok) tmem_ld32(s_col + (buf ^ 1) * kTileRows, lo);
      }
      add_scores(i, 32, hi);
      if (kPass == kStream) {
        // the other warpgroups hand their columns' sums of this tile of keys to the first
        sum = total(acc);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = 0;
        const int key = (t0 + i) * kTileRows + row, ps = i & 1;
        if (u > 0) {
          if (i >= 2 && !mbar_wait(&bar_part_empty[ps], ((i >> 1) - 1) & 1, G.err)) break;
          s_part[ps][u - 1][row] = sum;
          mbar_arrive(&bar_part_full[ps]);
        } else {
          if (!mbar_wait(&bar_part_full[ps], (i >> 1) & 1, G.err)) break;
          for (int k = 0; k < 2 * na - 1; ++k) sum += s_part[ps][k][row];
          mbar_arrive(&bar_part_empty[ps]);
          if (key < len) {
            float* o = a.out + r * a.out_stride + key;
            *o = a.accumulate ? *o + sum : sum;
          }
        }
      }
    }
    if (kPass != kStream) {
      sum = total(acc);
      if (h == 1) s_row[w][row] = make_float2(m, sum);
    }
  }

  // ============================ teardown ============================
  tc_fence_before();
  __syncthreads();
  if (kPass != kStream && warp >= 4 && (warp - 4) / 8 < na && ((warp - 4) / 4 & 1) == 0) {
    // the first half's warpgroups add what the second's found
    const int w = (warp - 4) / 8, row = 32 * (warp & 3) + lane, tile = 2 * pair + w;
    const float2 other = s_row[w][row];
    if (kPass == kLse) {
      const float2 ml = merge_ml(make_float2(m, sum), other);
      const long long at = ((long long)r * t.row_tiles + tile) * kTileRows + row;
      const bool live = row < q_rows && tile * tt + row / G.grp < a.q_len;
      if (t.part)
        t.part[(long long)split * a.units * t.row_tiles * kTileRows + at] = live ? ml : make_float2(-INFINITY, 0.f);
      else
        t.neg_lse[at] = live ? -(ml.x + log2f(ml.y)) : -INFINITY;
    } else {
      const int key = tile * kTileRows + row;
      const float x = sum + other.y;
      if (key < len) {
        if (t.splits > 1) {
          t.sums[((long long)split * a.units + r) * t.sums_unit + key] = x;
        } else {
          float* o = a.out + r * a.out_stride + key;
          *o = a.accumulate ? *o + x : x;
        }
      }
    }
  }
  if (warp == 1) {
    if (lane == 0) mbar_wait(&bar_final, 0, G.err);  // every product has completed
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// -lse of every row from its key ranges: a CTA takes 32 rows, eight threads each.
__global__ void __launch_bounds__(256) combine_lse_kernel(const float2* part, float* neg_lse, long long rows, int splits) {
  __shared__ float2 s_ml[8][32];
  const int row = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const long long i = (long long)blockIdx.x * 32 + row;  // rows is a multiple of 128
  griddep_wait();
  float2 ml = make_float2(-INFINITY, 0.f);
  for (int s = sub; s < splits; s += 8) ml = merge_ml(ml, part[s * rows + i]);
  s_ml[sub][row] = ml;
  __syncthreads();
  if (sub == 0) {
    for (int k = 1; k < 8; ++k) ml = merge_ml(ml, s_ml[k][row]);
    neg_lse[i] = ml.y > 0.f ? -(ml.x + log2f(ml.y)) : -INFINITY;  // a row that holds no query adds nothing
  }
}

// The row ranges' sums, in their order.
__global__ void __launch_bounds__(256) combine_sums_kernel(const __grid_constant__ TcArgs t) {
  const KeyWeightsArgs& a = t.a;
  const int j = blockIdx.x * 256 + threadIdx.x, r = blockIdx.y;
  griddep_wait();
  if (j >= key_weights_past(a) + a.q_len) return;
  float x = 0.f;
  for (int s = 0; s < t.splits; ++s) x += t.sums[((long long)s * a.units + r) * t.sums_unit + j];
  float* o = a.out + r * a.out_stride + j;
  *o = a.accumulate ? *o + x : x;
}

int encode_queries(CUtensorMap* map, const KeyWeightsArgs& a, int tile_tokens) {
  typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                    const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                    CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qr;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr);
    return e == cudaSuccess && qr == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
  }();
  if (!fn) return fail(AOH_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  // (B, C, Hq, 128): a box is 64 dimensions of one group's heads of tile_tokens tokens; tokens behind the last read as zeros
  const cuuint64_t dims[4] = {(cuuint64_t)kHeadDim, (cuuint64_t)a.g.Hq, (cuuint64_t)a.q_len, (cuuint64_t)a.g.B};
  const cuuint64_t strides[3] = {(cuuint64_t)kHeadDim * 2, (cuuint64_t)a.g.Hq * kHeadDim * 2,
                                 (cuuint64_t)a.q_len * a.g.Hq * kHeadDim * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)a.g.grp, (cuuint32_t)tile_tokens, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(a.q), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? AOH_OK : fail(AOH_ERR_CUDA, "cuTensorMapEncodeTiled (queries) failed (%d)", (int)r);
}

int key_pairs(int max_len) { return ((max_len + kTileRows - 1) / kTileRows + 1) / 2; }
// Ranges that `items` CTAs' lists of at most `tiles` tiles are cut into, one CTA
// per SM: the fewest tile periods, a range costing its tiles and about four for
// a CTA's start and end.  Candidates: a few ranges, what fills 1 to 4 waves, and
// ranges of 1 to 8 tiles (2 items of 64 tiles: 8 ranges 21 us, 64 ranges 14 us).
// 4096 tokens over 16384 keys, 4 units: `even` lists in 1, 2, 3, 4, 7 ranges
// 311, 319, 327, 304, 335 us; uneven ones 343, 288, 296, 298, 321 us.
int plan_ranges(long long items, int tiles, int sms, bool even) {
  int best = 1;
  double least = 1e300;
  for (int k = 1; k <= 20; ++k) {
    const long long s = k <= 8 ? k : k <= 12 ? (k - 8) * (long long)sms / items : (tiles + 20 - k) / (21 - k);
    if (s < 1 || s > std::min(tiles, 256)) continue;
    const double ctas = (double)items * s / sms;
    // lists of one length end in whole waves; of uneven ones, the long ones
    // first, the waves overlap at their ends and half a range is lost
    const double waves = ctas <= 1 ? 1.0 : even ? (double)(((long long)items * s + sms - 1) / sms) : ctas + 0.5;
    const double cost = waves * ((tiles + s - 1) / s + 4);
    if (cost < least * 0.98) {
      best = (int)s;
      least = cost;
    }
  }
  return best;
}

// Most pages of a unit that a cluster takes.  On the device and from Python, one
// launch against two, 2 units: 4 rows x 4096 keys 5.4 / 9.5 us against 5.8 / 13.6,
// x 8192 7.4 / 9.5 against 6.2 / 13.7, x 16384 11.4 / 11.6 against 7.2 / 13.7; 32
// rows x 8192 keys 10.7 / 10.9 against 13.5 / 13.9 on the tensor cores.
constexpr int kOnePages = 512;
// Floats of a key's scores: in a cluster two more than are written, which keeps
// the keys of a warp on distinct banks; else 2, 4, 8 or 16, for wide loads.
int one_cols(int rows) { return (rows + 1) / 2 * 2; }
int one_stride(int rows) { return one_cols(rows) + 2; }
int few_stride(int rows) { return rows <= 2 ? 2 : rows <= 4 ? 4 : rows <= 8 ? 8 : 16; }
// bytes of the scores of one of n CTAs
size_t one_smem(int pages, int n, int rows) {
  return (size_t)((pages + n - 1) / n) * kPage * one_stride(rows) * sizeof(float);
}

// CTAs of a unit's cluster at most on `device`, 0 if that cannot be told; prepares the kernels, once.
int one_largest(int device) {
  static PerDeviceOnce once;
  static int largest[kMaxDevices];
  const int rc = once.run(device, [device] {
    int current = 0, n[3] = {};
    int e = current_device(&current);  // a plan may be asked for while another device is the current one
    if (e) return e;
    if (current != device) e = cuda_check(cudaSetDevice(device), "cudaSetDevice");
    auto ask = [&](auto kernel, int i) {
      if (!e)
        e = larger_cluster(kernel, kMaxOne, kMaxOne / 2, kFewWarps * 32, kOneSmem, "aoh_key_weights clusters", &n[i]);
    };
    ask(few_scores_kernel<1, true>, 0);
    ask(few_scores_kernel<2, true>, 1);
    ask(few_scores_kernel<4, true>, 2);
    if (current != device) cudaSetDevice(current);
    largest[device] = std::min(n[0], std::min(n[1], n[2]));
    return e;
  });
  return rc ? 0 : largest[device];
}

template <int NT>
int launch_few_one(const FewArgs& f, cudaStream_t st) {
  auto kernel = few_scores_kernel<NT, true>;
  return launch_dependent(kernel, dim3((unsigned)f.splits, (unsigned)f.a.units), f.splits, kFewWarps * 32,
                          one_smem((f.a.max_len + kPage - 1) / kPage, f.splits, f.rows), st, "aoh_key_weights launch", f);
}

}  // namespace

bool plan_key_weights_few(const aoh_kv_cache* c, int units, int max_len, KeyWeightsPlan& p) {
  p.kind = KeyWeightsKind::few;
  const int pages = (max_len + kPage - 1) / kPage;
  // A cluster a unit where its 16 CTAs read K fast enough.  More than 16 rows
  // leave an SM one CTA, and clusters of 16 of those do not fit every GPC (8
  // units of 32 rows x 4096 keys: 20 us, with 8 CTAs 11).
  const int fits = pages <= kOnePages && c->bound ? one_largest(c->device) : 0;
  const int most = std::min(fits, p.rows > kFewRows && units * kMaxOne > c->num_sms / 2 ? kMaxOne / 2 : kMaxOne);
  const int one = std::max(1, std::min(most, pages / (2 * kFewWarps)));  // at least two pages for each of a CTA's warps
  if (fits && units * one <= c->num_sms && one_smem(pages, one, p.rows) <= kOneSmem) {
    p.splits = one;
    p.one = true;
    return true;
  }
  if (p.rows > kFewRows) return false;
  // two CTAs per SM in one wave, at least two pages for each of a CTA's warps
  p.splits = std::max(1, std::min(2 * std::max(1, c->num_sms) / std::max(1, units), pages / (2 * kFewWarps)));
  p.part = 0;
  p.score = align256((size_t)p.splits * units * p.rows * sizeof(float2));
  p.bytes = p.score + (size_t)units * pages * kPage * few_stride(p.rows) * sizeof(float);
  return true;
}

int launch_key_weights_few(const aoh_kv_cache* c, const KeyWeightsArgs& a, const KeyWeightsPlan& p, char* ws,
                           cudaStream_t st) {
  FewArgs f;
  f.a = a;
  f.part = reinterpret_cast<float2*>(ws + p.part);
  f.score = reinterpret_cast<float*>(ws + p.score);
  f.rows = p.rows;
  f.splits = p.splits;
  f.cols = p.one ? one_cols(p.rows) : few_stride(p.rows);
  f.stride = p.one ? one_stride(p.rows) : f.cols;
  f.score_unit = (long long)((a.max_len + kPage - 1) / kPage) * kPage * f.stride;
  const dim3 grid(p.splits, a.units);
  int rc = AOH_OK;
  if (p.one) {
    f.part = nullptr;
    f.score = nullptr;
    return p.rows <= 8    ? launch_few_one<1>(f, st)
           : p.rows <= 16 ? launch_few_one<2>(f, st)
                          : launch_few_one<4>(f, st);
  }
  if (p.rows <= 8)
    rc = launch_dependent(few_scores_kernel<1, false>, grid, 1, kFewWarps * 32, 0, st, "aoh_key_weights scores launch", f);
  else
    rc = launch_dependent(few_scores_kernel<2, false>, grid, 1, kFewWarps * 32, 0, st, "aoh_key_weights scores launch", f);
  if (rc) return rc;
  auto sums = f.stride == 2   ? few_sum_kernel<2>
              : f.stride == 4 ? few_sum_kernel<4>
              : f.stride == 8 ? few_sum_kernel<8>
                              : few_sum_kernel<16>;
  return launch_dependent(sums, dim3((a.max_len + 256 * kFewKeys - 1) / (256 * kFewKeys), a.units), 1, 256, 0, st,
                          "aoh_key_weights sums launch", f);
}

void plan_key_weights_tensor(const aoh_kv_cache* c, int units, int max_len, int q_len, KeyWeightsPlan& p) {
  p.kind = KeyWeightsKind::tensor;
  const int grp = c->cfg.num_q_heads / c->cfg.num_kv_heads, sms = std::max(1, c->num_sms);
  p.tile_tokens = std::min(kTileRows / grp, q_len);
  p.row_tiles = (q_len + p.tile_tokens - 1) / p.tile_tokens;
  const long long lse_items = (long long)units * ((p.row_tiles + 1) / 2), sum_items = (long long)units * key_pairs(max_len);
  // Causal: the first tokens' rows have max_len - q_len keys, the last ones' max_len.  Taken as even from a quarter
  // on.  30 sizes each (1 to 12 units, 2K to 46K keys) for which the two ways give different ranges, the call's time
  // taken as even to that as uneven: cached part 0 to 0.25 of the keys 0.99, 1.00, 1.01, 1.01, 1.02, 1.00; 0.3 0.99,
  // 0.4 0.98, 0.5 to 0.7 0.97; above (10 sizes each) 0.95 to 0.98.
  p.splits = plan_ranges(lse_items, (max_len + kTileRows - 1) / kTileRows, sms, 4LL * (max_len - q_len) >= max_len);
  // up to two tiles of query rows stay resident in the second pass too, which then needs the ranges alone
  p.stream = p.row_tiles <= 2;
  p.row_splits = p.stream ? p.splits : plan_ranges(sum_items, p.row_tiles, sms, false);
  const size_t rows = (size_t)units * p.row_tiles * kTileRows;
  p.part = 0;
  p.lse = p.stream || p.splits > 1 ? align256(rows * p.splits * sizeof(float2)) : 0;
  p.sums = p.lse + (p.stream ? 0 : align256(rows * sizeof(float)));
  p.bytes = p.sums + (!p.stream && p.row_splits > 1 ? (size_t)p.row_splits * units * max_len * sizeof(float) : 0);
}

int launch_key_weights_tensor(const aoh_kv_cache* c, const KeyWeightsArgs& a, const KeyWeightsPlan& p, char* ws,
                              cudaStream_t st) {
  static PerDeviceOnce once;
  int rc = once.run(c->device, [] {
    const void* kernels[3] = {reinterpret_cast<const void*>(tensor_pass_kernel<kLse>),
                              reinterpret_cast<const void*>(tensor_pass_kernel<kSums>),
                              reinterpret_cast<const void*>(tensor_pass_kernel<kStream>)};
    int e = AOH_OK;
    for (const void* k : kernels)
      if (e == AOH_OK)
        e = cuda_check(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmem),
                       "key weights shared memory");
    return e;
  });
  if (rc) return rc;
  CUtensorMap tm;
  rc = encode_queries(&tm, a, p.tile_tokens);
  if (rc) return rc;
  TcArgs t;
  t.a = a;
  t.part = p.stream || p.splits > 1 ? reinterpret_cast<float2*>(ws + p.part) : nullptr;
  t.neg_lse = reinterpret_cast<float*>(ws + p.lse);
  t.sums = reinterpret_cast<float*>(ws + p.sums);
  t.row_tiles = p.row_tiles;
  t.tile_tokens = p.tile_tokens;
  t.sums_unit = a.max_len;
  t.pairs = (p.row_tiles + 1) / 2;
  t.splits = t.lse_splits = p.splits;
  const long long g1 = (long long)a.units * t.pairs * p.splits;
  const long long g2 = p.stream ? g1 : (long long)a.units * key_pairs(a.max_len) * p.row_splits;
  if (g1 > 0x7fffffffLL || g2 > 0x7fffffffLL) return fail(AOH_ERR_UNSUPPORTED, "aoh_key_weights: too many tiles");
  rc = launch_dependent(tensor_pass_kernel<kLse>, dim3((unsigned)g1), 1, kTcThreads, kTcSmem, st, "aoh_key_weights launch",
                        tm, t);
  if (rc) return rc;
  if (p.stream)
    return launch_dependent(tensor_pass_kernel<kStream>, dim3((unsigned)g2), 1, kTcThreads, kTcSmem, st,
                            "aoh_key_weights sums launch", tm, t);
  if (p.splits > 1) {
    const long long rows = (long long)a.units * p.row_tiles * kTileRows;
    rc = launch_dependent(combine_lse_kernel, dim3((unsigned)(rows / 32)), 1, 256, 0, st, "aoh_key_weights combine launch",
                          (const float2*)t.part, t.neg_lse, rows, p.splits);
    if (rc) return rc;
  }
  t.pairs = key_pairs(a.max_len);
  t.splits = p.row_splits;
  rc = launch_dependent(tensor_pass_kernel<kSums>, dim3((unsigned)g2), 1, kTcThreads, kTcSmem, st,
                        "aoh_key_weights sums launch", tm, t);
  if (rc || p.row_splits == 1) return rc;
  return launch_dependent(combine_sums_kernel, dim3((a.max_len + 255) / 256, a.units), 1, 256, 0, st,
                          "aoh_key_weights combine launch", t);
}

}  // namespace aoh
