// Attention weight by key: for a layer's retrieval units
//
//   W[j] (+)= sum over queries i and heads h of the unit's group of
//             softmax over j' <= past_len + i of (q_ih . k_j' / sqrt(128))  at j
//
// i.e. the column sums of the softmax matrix whose product with V the
// attention entry points compute.  A weight needs its row's maximum and sum
// over all keys first, so a call has two passes: one for every query row's
// (m, l), by key ranges that fill the GPU, one that adds up exp(s - lse) per
// key.  Each key is summed by one CTA in a fixed order, so results do not depend
// on timing.
//
// This file holds the entry point and the kernels for any type.  Their first
// pass also writes the scores, 4 bytes each, and the second reads them: 128
// products on the CUDA cores cost 3.6 ps, a write and a read of 4 bytes 1.2 ps.
// The query rows are taken in blocks whose scores fit L2, two launches a block.
// 2 x 33 tokens, 3 groups of 2 heads, over 2023 keys, fp32: 15 us a call,
// of which the scores take 10; with the scores computed again 35.
// bf16 caches run the kernels of key_weights_sm100.cu: one pass over K for few
// query rows (single tokens), tensor cores for more.
#include "common.cuh"
#include "fast_math.cuh"
#include "internal.h"
#include "key_weights.h"
#include "launch.cuh"
#include "page_layout.cuh"

namespace aoh {
namespace {

constexpr int kTile = 64;                 // query rows, and keys, of a tile
constexpr int kSumKeys = 32;              // keys of a CTA of the second pass
constexpr int kSumRows = 128;             // query rows whose maximum and sum it holds at a time
constexpr int kStride = kHeadDim + 4;     // floats of a row in shared memory: 16-byte rows on distinct banks
constexpr int any_smem(int tile_rows) { return (kTile + tile_rows) * kStride * 4; }
constexpr long long kScoreBytes = 96 << 20;  // of a block of query rows, if 16 rows need no more: three quarters of L2

// A block of query rows: rows row_base .. row_base + rows - 1 of every unit.
struct AnyArgs {
  KeyWeightsArgs a;
  float2* part;        // (key range, retrieval row, query row): maximum, sum
  float* score;        // (retrieval row, query row, key): q . k
  long long score_row; // floats of a query row's scores
  int splits, row_base, rows, tile_rows;
};

// Four dimensions of a stored row into shared memory; fp32 without a register in between.
__device__ __forceinline__ void copy4(float* dst, const float* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(float* dst, const __nv_bfloat16* src) {
  const uint2 v = *reinterpret_cast<const uint2*>(src);
  *reinterpret_cast<float4*>(dst) = make_float4(bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y));
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A warp's 8 query rows from `row` on; rows from row_end on are zero.
template <typename T>
__device__ __forceinline__ void load_queries(const KeyWeightsArgs& a, int b, int g, int row, int row_end, float* sm) {
  const int c = (threadIdx.x & 31) * 4;
  int tok = row / a.g.grp, h = row % a.g.grp;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float* dst = sm + i * kStride + c;
    if (row + i < row_end)
      copy4(dst, static_cast<const T*>(a.q) + (((long long)b * a.q_len + tok) * a.g.Hq + g * a.g.grp + h) * kHeadDim + c);
    else
      *reinterpret_cast<float4*>(dst) = make_float4(0.f, 0.f, 0.f, 0.f);
    if (++h == a.g.grp) h = 0, ++tok;
  }
}

// The page of keys j0 + 16 lane .. of a unit (lanes 0 to 3), -1 where there is none.
__device__ __forceinline__ int fetch_page(const KeyWeightsArgs& a, const RetrievalRow& info, int j0, int len) {
  const int lane = threadIdx.x & 31, p = j0 / kPage + lane;
  return lane < kTile / kPage && p * kPage < len && p < info.held ? a.g.block_table[info.table + p] : -1;
}

// 64 keys from j0 on, the warps' rows in turn; rows that are not stored are zero.
template <typename T>
__device__ __forceinline__ void load_keys(const KeyWeightsArgs& a, int my_page, int j0, int len, float* sm) {
  const int lane = threadIdx.x & 31, c = lane * 4, warps = blockDim.x >> 5;
  if (threadIdx.x < kTile / kPage && j0 + (int)threadIdx.x * kPage < len && (my_page < 0 || my_page >= a.g.num_pages))
    atomicOr(a.g.err, kErrBadPage);
#pragma unroll 8
  for (int r = threadIdx.x >> 5; r < kTile; r += warps) {
    const int page = __shfl_sync(0xffffffffu, my_page, r / kPage), slot = r % kPage;
    float* dst = sm + r * kStride + c;
    if (page >= 0 && page < a.g.num_pages && j0 + r < len) {
      const char* p = static_cast<const char*>(a.g.pool);
      p += sizeof(T) == 4 ? (long long)page * kPageF32Bytes + 4 * f32_elem_offset(0, slot, c)
                          : (long long)page * kPageBf16Bytes + 2 * bf16_elem_offset(0, slot, c);
      copy4(dst, reinterpret_cast<const T*>(p));
    } else {
      *reinterpret_cast<float4*>(dst) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
}

// s[i][j] = q . k of row 4 ty + i and key tx + 16 j, even and odd dimensions
// added apart: one packed product for two.  The scaling to the log2 domain is
// left to the subtraction of a row's maximum, one rounding for both.
__device__ __forceinline__ void tile_scores(const float* qs, const float* ks, int ty, int tx, float (&s)[4][4]) {
  uint64_t acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0;
#pragma unroll 4
  for (int d = 0; d < kHeadDim; d += 4) {
    ulonglong2 q[4], k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const ulonglong2*>(qs + (4 * ty + i) * kStride + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const ulonglong2*>(ks + (tx + 16 * j) * kStride + d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = f2_fma(q[i].y, k[j].y, f2_fma(q[i].x, k[j].x, acc[i][j]));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x, y;
      f2_unpack(acc[i][j], x, y);
      s[i][j] = x + y;
    }
}

// Keys a row may see: j <= past + token.
__device__ __forceinline__ int last_key(const KeyWeightsArgs& a, int past, int row) { return past + row / a.g.grp; }

// Scores and (m, l) of up to 64 query rows over one range of keys: a warp for 8
// rows, a thread for 4 rows and 4 keys of each tile.
template <typename T>
__global__ void __launch_bounds__(256, 3) key_lse_kernel(const __grid_constant__ AnyArgs k) {
  extern __shared__ float sm[];
  const KeyWeightsArgs& a = k.a;
  griddep_wait();
  griddep_launch_dependents();  // the sums wait for this grid to finish
  const int r = blockIdx.y;
  const RetrievalRow info = a.rows[r];
  if (info.held == 0) return;
  const int past = key_weights_past(a);
  const int row0 = k.row_base + blockIdx.z * k.tile_rows, row_end = min(row0 + k.tile_rows, k.row_base + k.rows);
  const int b = (info.unit - a.unit0) / a.g.G, g = (info.unit - a.unit0) % a.g.G;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15, warp_row = row0 + 8 * (int)(threadIdx.x >> 5);
  float *ks = sm, *qs = sm + kTile * kStride;
  // key tiles up to the last one that any row of the tile sees, split evenly
  const int len = last_key(a, past, row_end - 1) + 1;
  const int tiles = (len + kTile - 1) / kTile;
  const int t0 = (int)((long long)tiles * blockIdx.x / k.splits), t1 = (int)((long long)tiles * (blockIdx.x + 1) / k.splits);
  int page = fetch_page(a, info, t0 * kTile, len);
  if (t0 < t1) load_queries<T>(a, b, g, warp_row, row_end, qs + (threadIdx.x >> 5) * 8 * kStride);
  float m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = -INFINITY, l[i] = 0.f;
  for (int t = t0; t < t1; ++t) {
    if (t > t0) __syncthreads();
    load_keys<T>(a, page, t * kTile, len, ks);
    if (t + 1 < t1) page = fetch_page(a, info, (t + 1) * kTile, len);
    copies_wait();
    __syncthreads();
    if (warp_row >= row_end) continue;
    float s[4][4];
    tile_scores(qs, ks, ty, tx, s);
    const int key = t * kTile + tx;
    int row = row0 + 4 * ty, tok = row / a.g.grp, h = row % a.g.grp;
    float* out = k.score + ((long long)r * k.rows + (row - k.row_base)) * k.score_row + key;
#pragma unroll
    for (int i = 0; i < 4; ++i, ++row) {
      const int last = past + tok;
      float mt = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (key + 16 * j <= last) {
          if (row < row_end) out[16 * j] = s[i][j];
        } else {
          s[i][j] = -INFINITY;
        }
        mt = fmaxf(mt, s[i][j]);
      }
      out += k.score_row;
      if (++h == a.g.grp) h = 0, ++tok;
      mt *= kScoreScale;
      if (mt > m[i]) {
        l[i] *= fast_exp2(m[i] - mt);
        m[i] = mt;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (s[i][j] > -INFINITY) l[i] += fast_exp2(fmaf(s[i][j], kScoreScale, -m[i]));
    }
  }
  // the 16 threads of a row
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float mm = m[i];
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
    float ll = mm > -INFINITY ? l[i] * fast_exp2(m[i] - mm) : 0.f;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, off);
    const int row = row0 + 4 * ty + i;
    if (tx == 0 && row < row_end)
      k.part[((long long)blockIdx.x * a.units + r) * k.rows + (row - k.row_base)] = make_float2(mm, ll);
  }
}

// The weights of kSumKeys keys, a lane each, summed over the block's query
// rows: row 8 i + warp of every 128.
__global__ void __launch_bounds__(256) key_sum_kernel(const __grid_constant__ AnyArgs k) {
  constexpr int kMine = kSumRows / 8;
  __shared__ float2 ml[kSumRows];  // of a row: its maximum and 1 / sum
  __shared__ float sums[8][kSumKeys];
  const KeyWeightsArgs& a = k.a;
  const int r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  const int past = key_weights_past(a), len = past + a.q_len, j0 = (int)blockIdx.x * kSumKeys, key = j0 + lane;
  if (j0 >= len) return;
  const bool stored = a.rows[r].held > 0;
  float w = 0.f;
  // rows of the block from the first token on that sees this key (and this CTA's first key)
  const int first = max(0, key - past) * a.g.grp - k.row_base;
  for (int i0 = max(0, max(0, j0 - past) * a.g.grp - k.row_base); stored && i0 < k.rows; i0 += kSumRows) {
    float s[kMine];
    const float* score = k.score + ((long long)r * k.rows + i0 + warp) * k.score_row + key;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int row = i0 + warp + 8 * i;
      s[i] = row < k.rows && row >= first && key < len ? score[8 * i * k.score_row] : -INFINITY;
    }
    // the rows' maxima and sums from their key ranges, two threads a row
    const int mine = i0 + (threadIdx.x >> 1);
    float mm = -INFINITY, ll = 0.f;
    if (mine < k.rows) {
      const float2* p = k.part + (long long)r * k.rows + mine;
      for (int s0 = threadIdx.x & 1; s0 < k.splits; s0 += 2 * kMine) {
        float2 v[kMine];
        float top = mm;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          v[i] = s0 + 2 * i < k.splits ? p[(long long)(s0 + 2 * i) * a.units * k.rows] : make_float2(-INFINITY, 0.f);
          top = fmaxf(top, v[i].x);
        }
        if (ll > 0.f) ll *= fast_exp2(mm - top);
#pragma unroll
        for (int i = 0; i < kMine; ++i)
          if (v[i].y > 0.f) ll = fmaf(v[i].y, fast_exp2(v[i].x - top), ll);
        mm = top;
      }
    }
    const float om = __shfl_xor_sync(0xffffffffu, mm, 1), ol = __shfl_xor_sync(0xffffffffu, ll, 1), top = fmaxf(mm, om);
    ll = (ll > 0.f ? ll * fast_exp2(mm - top) : 0.f) + (ol > 0.f ? ol * fast_exp2(om - top) : 0.f);
    if (i0 > 0) __syncthreads();
    if ((threadIdx.x & 1) == 0) ml[threadIdx.x >> 1] = make_float2(top, 1.f / ll);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const float2 e = ml[warp + 8 * i];
      if (s[i] != -INFINITY) w = fmaf(fast_exp2(fmaf(s[i], kScoreScale, -e.x)), e.y, w);
    }
  }
  sums[warp][lane] = w;
  __syncthreads();
  if (warp == 0 && key < len) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x += sums[i][lane];
    float* o = a.out + r * a.out_stride + key;
    *o = a.accumulate ? *o + x : x;
  }
}

template <typename T>
int launch_any(const KeyWeightsArgs& a, const KeyWeightsPlan& p, char* ws, cudaStream_t st) {
  int dev = 0;
  int rc = current_device(&dev);
  if (rc) return rc;
  static PerDeviceOnce once;
  rc = once.run(dev, [] {
    return cuda_check(cudaFuncSetAttribute(key_lse_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, any_smem(kTile)),
                      "key_lse shared memory");
  });
  if (rc) return rc;
  if (p.row_tiles > 65535) return fail(AOH_ERR_UNSUPPORTED, "aoh_key_weights: too many queries");
  AnyArgs k;
  k.a = a;
  k.part = reinterpret_cast<float2*>(ws + p.part);
  k.score = reinterpret_cast<float*>(ws + p.score);
  k.score_row = a.max_len;
  k.splits = p.splits;
  k.tile_rows = p.tile_rows;
  const int rows = a.q_len * a.g.grp;
  for (k.row_base = 0; k.row_base < rows; k.row_base += p.rows) {
    k.rows = std::min(p.rows, rows - k.row_base);
    const int row_tiles = (k.rows + p.tile_rows - 1) / p.tile_rows;
    rc = launch_dependent(key_lse_kernel<T>, dim3(p.splits, a.units, row_tiles), 1, 4 * p.tile_rows, any_smem(p.tile_rows),
                          st, "aoh_key_weights launch", k);
    if (rc) return rc;
    rc = launch_dependent(key_sum_kernel, dim3((a.max_len + kSumKeys - 1) / kSumKeys, a.units), 1, 256, 0, st,
                          "aoh_key_weights sums launch", k);
    if (rc) return rc;
    k.a.accumulate = 1;
  }
  return AOH_OK;
}

int retrieval_heads(const aoh_kv_cache* c, int layer) {
  int n = 0;
  for (int g = 0; g < c->cfg.num_kv_heads; ++g) n += c->retrieval(layer, g);
  return n;
}

KeyWeightsPlan plan(const aoh_kv_cache* c, int layer, int max_len, int q_len) {
  KeyWeightsPlan p;
  const int units = c->cfg.batch * retrieval_heads(c, layer), grp = c->cfg.num_q_heads / c->cfg.num_kv_heads;
  p.rows = q_len * grp;
  if (c->cfg.dtype == AOH_BF16 && p.rows <= kOneRows && plan_key_weights_few(c, units, max_len, p)) return p;
  p.kind = KeyWeightsKind::any;
  if (c->cfg.dtype == AOH_BF16 && grp <= 128) {
    plan_key_weights_tensor(c, units, max_len, q_len, p);
  } else {
    // as many rows a block as have room for their scores, in whole tiles (of 16 rows at least)
    const long long row_bytes = (long long)units * max_len * sizeof(float), room = kScoreBytes / std::max(1LL, row_bytes);
    if (p.rows > room) p.rows = (int)(room >= kTile ? room / kTile * kTile : std::max(16LL, room / 16 * 16));
    const int key_tiles = (max_len + kTile - 1) / kTile;
    // Up to 64 rows a tile, or 32 where one key tile for every CTA is no more than
    // one wave: 2 x 3 units of 66 rows x 2023 keys 14.7 us, with 64 rows 15.9; 4
    // units of 400 rows x 4000 keys 87, with 64 rows 70.
    p.row_tiles = (p.rows + kTile - 1) / kTile;
    if ((long long)units * p.row_tiles * key_tiles <= 3LL * c->num_sms) p.row_tiles = (p.rows + kTile / 2 - 1) / (kTile / 2);
    p.tile_rows = ((p.rows + p.row_tiles - 1) / p.row_tiles + 7) / 8 * 8;  // tiles of like height: 66 rows = 24 + 24 + 18
    // as many CTAs as the SMs hold at a time: three of 64 rows, four of 32, five of 8
    const long long ctas = std::max(1LL, (long long)units * p.row_tiles), resident = 224 * 1024 / any_smem(p.tile_rows);
    p.splits = (int)std::max(1LL, std::min<long long>(std::min(64, key_tiles),
                                                      (resident * std::max(1, c->num_sms) + ctas - 1) / ctas));
    p.score = align256((size_t)p.splits * units * p.rows * sizeof(float2));
    p.bytes = p.score + (size_t)p.rows * row_bytes;
  }
  return p;
}

// Keys a call covers: with the device's length, every position the cache may come to hold.
int most_keys(const aoh_kv_cache* c, int32_t past_len, int32_t q_len) {
  return past_len == AOH_PAST_LEN_DEVICE ? c->cfg.max_context : past_len + q_len;
}

}  // namespace
}  // namespace aoh

using namespace aoh;

extern "C" size_t aoh_key_weights_workspace_bytes(const aoh_kv_cache* c, int32_t layer, int32_t past_len, int32_t q_len) {
  if (!c || layer < 0 || layer >= c->cfg.num_layers || past_len < AOH_PAST_LEN_DEVICE || q_len <= 0 ||
      (int64_t)past_len + q_len > c->cfg.max_context)
    return 0;
  return plan(c, layer, most_keys(c, past_len, q_len), q_len).bytes;
}

extern "C" int aoh_key_weights(aoh_kv_cache* c, int32_t layer, int32_t past_len, int32_t q_len, const void* q, float* out,
                               int64_t out_stride, int32_t accumulate, void* workspace, size_t workspace_bytes,
                               aoh_stream stream) {
  const char* who = "aoh_key_weights";
  if (!c) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null cache", who);
  const bool device_len = past_len == AOH_PAST_LEN_DEVICE;
  const int rc = check_common(c, layer, device_len ? 0 : past_len, q_len, q, q, q, nullptr, who);
  if (rc) return rc;
  const int n_ret = retrieval_heads(c, layer);
  if (n_ret == 0 || q_len == 0) return AOH_OK;
  const int max_len = most_keys(c, past_len, q_len);
  if (!out) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null tensor", who);
  if (out_stride < max_len)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: rows of %lld weights for %d keys", who, (long long)out_stride, max_len);
  KeyWeightsArgs a{};
  a.g = c->geom();
  a.units = c->cfg.batch * n_ret;
  if (a.units > 65535) return fail(AOH_ERR_UNSUPPORTED, "%s: too many units", who);
  if ((long long)q_len * a.g.grp > (1 << 30)) return fail(AOH_ERR_UNSUPPORTED, "%s: too many queries", who);
  const KeyWeightsPlan p = plan(c, layer, max_len, q_len);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes))
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, p.bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", who);
  int row0 = 0;
  for (int l = 0; l < layer; ++l) row0 += c->cfg.batch * retrieval_heads(c, l);
  a.rows = c->dev_rows + row0;
  a.unit0 = c->unit(layer, 0, 0);
  a.past_len = past_len;
  a.past_len_dev = device_len ? c->dev_err + 1 : nullptr;
  a.max_len = max_len;
  a.q_len = q_len;
  a.q = q;
  a.out = out;
  a.out_stride = out_stride;
  a.accumulate = accumulate;
  char* ws = static_cast<char*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (p.kind) {
    case KeyWeightsKind::few: return launch_key_weights_few(c, a, p, ws, st);
    case KeyWeightsKind::tensor: return launch_key_weights_tensor(c, a, p, ws, st);
    default:
      return c->cfg.dtype == AOH_BF16 ? launch_any<__nv_bfloat16>(a, p, ws, st) : launch_any<float>(a, p, ws, st);
  }
}
