// Attention weight by key: for a layer's retrieval units
//
//   W[j] (+)= sum over queries i and heads h of the unit's group of
//             softmax over j' <= past_len + i of (q_ih . k_j' / sqrt(128))  at j
//
// i.e. the column sums of the softmax matrix whose product with V the
// attention entry points compute.  A weight needs its row's maximum and sum
// over all keys first, so two passes over K: one for every query row's (m, l),
// by key ranges that fill the GPU, one that adds up exp(s - lse) per key.  Each
// key is summed by one CTA in a fixed order, so results do not depend on timing.
//
// This file holds the entry point and the kernels for any type: 64 rows x 64
// (or 32) keys per tile in fp32 on the CUDA cores, 4 x 4 products a thread.  bf16
// caches run those of key_weights_sm100.cu: one pass over K for few query rows
// (single tokens), tensor cores for more.
#include "common.cuh"
#include "internal.h"
#include "key_weights.h"
#include "page_layout.cuh"

namespace aoh {
namespace {

constexpr int kTile = 64;                 // query rows of a tile, and keys of the first pass's
constexpr int kSumKeys = 32;              // keys of the second pass's tiles: twice the CTAs, which 64 leave uneven
constexpr int kStride = kHeadDim + 4;     // floats of a row in shared memory: 16-byte rows on distinct banks
constexpr int kSmem = 2 * kTile * kStride * 4, kSumSmem = (kTile + kSumKeys) * kStride * 4;

// Four dimensions of a stored row, as loaded and as floats.
template <typename T>
struct Raw4;
template <>
struct Raw4<float> {
  float4 v;
  __device__ float4 get() const { return v; }
};
template <>
struct Raw4<__nv_bfloat16> {
  uint2 v;
  __device__ float4 get() const { return make_float4(bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y)); }
};

constexpr int kLoads = kTile * (kHeadDim / 4) / 256;  // of a thread for a tile: row 8 i + warp, dimensions 4 lane ..

// The loads of a tile are all issued before any is stored: a thread's eight
// would otherwise each wait for memory in turn.
template <typename T>
__device__ __forceinline__ void load_queries(const KeyWeightsArgs& a, int b, int g, int row0, int rows, float* sm) {
  const int r0 = threadIdx.x >> 5, c = (threadIdx.x & 31) * 4;
  Raw4<T> v[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = row0 + r0 + 8 * i;
    v[i] = Raw4<T>{};
    if (row < rows) {
      const int tok = row / a.g.grp, h = g * a.g.grp + row % a.g.grp;
      v[i] = *reinterpret_cast<const Raw4<T>*>(static_cast<const T*>(a.q) +
                                               (((long long)b * a.q_len + tok) * a.g.Hq + h) * kHeadDim + c);
    }
  }
#pragma unroll
  for (int i = 0; i < kLoads; ++i) *reinterpret_cast<float4*>(sm + (r0 + 8 * i) * kStride + c) = v[i].get();
}

// Keys [j0, j0 + KT) of a unit; rows that are not stored are zero.
template <typename T, int KT>
__device__ __forceinline__ void load_keys(const KeyWeightsArgs& a, int unit, int j0, int len, float* sm) {
  const int base = a.g.unit_offset[unit], n_pages = a.g.unit_offset[unit + 1] - base;
  const int r0 = threadIdx.x >> 5, c = (threadIdx.x & 31) * 4;
  int pages[KT / kPage];
#pragma unroll
  for (int i = 0; i < KT / kPage; ++i) {
    const int p = j0 / kPage + i;
    pages[i] = p * kPage < len && p < n_pages ? a.g.block_table[base + p] : -1;
    if (pages[i] >= a.g.num_pages) pages[i] = -1;
    if (pages[i] < 0 && p * kPage < len && threadIdx.x == 0) atomicOr(a.g.err, kErrBadPage);
  }
  Raw4<T> v[KT / 8];
#pragma unroll
  for (int i = 0; i < KT / 8; ++i) {
    const int r = r0 + 8 * i, slot = r % kPage;
    const int page = pages[8 * i / kPage];  // r0 < 8: row r is in page 8 i / 16
    v[i] = Raw4<T>{};
    if (page >= 0 && j0 + r < len) {
      const char* p = static_cast<const char*>(a.g.pool);
      p += sizeof(T) == 4 ? (long long)page * kPageF32Bytes + 4 * f32_elem_offset(0, slot, c)
                          : (long long)page * kPageBf16Bytes + 2 * bf16_elem_offset(0, slot, c);
      v[i] = *reinterpret_cast<const Raw4<T>*>(p);
    }
  }
#pragma unroll
  for (int i = 0; i < KT / 8; ++i) *reinterpret_cast<float4*>(sm + (r0 + 8 * i) * kStride + c) = v[i].get();
}

// s[i][j] = q . k of row 4 ty + i and key tx + 16 j.  The scaling to the log2
// domain is left to the subtraction of a row's maximum, one rounding for both.
template <int J>
__device__ __forceinline__ void tile_scores(const float* qs, const float* ks, int ty, int tx, float (&s)[4][J]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) s[i][j] = 0.f;
#pragma unroll 4
  for (int d = 0; d < kHeadDim; d += 4) {
    float4 q[4], k[J];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4*>(qs + (4 * ty + i) * kStride + d);
#pragma unroll
    for (int j = 0; j < J; ++j) k[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * kStride + d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        s[i][j] = fmaf(q[i].x, k[j].x, s[i][j]);
        s[i][j] = fmaf(q[i].y, k[j].y, s[i][j]);
        s[i][j] = fmaf(q[i].z, k[j].z, s[i][j]);
        s[i][j] = fmaf(q[i].w, k[j].w, s[i][j]);
      }
  }
}

// Keys a row may see: j <= past + token.
__device__ __forceinline__ int last_key(const KeyWeightsArgs& a, int past, int row) { return past + row / a.g.grp; }

// (m, l) of 64 query rows over one range of keys.
template <typename T>
__global__ void __launch_bounds__(256) key_lse_kernel(const __grid_constant__ KeyWeightsArgs a, float2* part, int splits) {
  extern __shared__ float sm[];
  const int r = blockIdx.y, unit = a.rows[r].unit;
  if (a.rows[r].held == 0) return;
  const int past = key_weights_past(a);
  const int rows = a.q_len * a.g.grp, row0 = blockIdx.z * kTile;
  const int b = (unit - a.unit0) / a.g.G, g = (unit - a.unit0) % a.g.G;
  const long long rows_total = (long long)a.units * rows;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  float *qs = sm, *ks = sm + kTile * kStride;
  load_queries<T>(a, b, g, row0, rows, qs);
  // key tiles up to the last one that any row of the tile sees, split evenly
  const int len = last_key(a, past, min(row0 + kTile, rows) - 1) + 1;
  const int tiles = (len + kTile - 1) / kTile;
  const int t0 = (int)((long long)tiles * blockIdx.x / splits), t1 = (int)((long long)tiles * (blockIdx.x + 1) / splits);
  const bool idle = row0 + 8 * (int)(threadIdx.x >> 5) >= rows;  // a warp has 8 rows: none of them is one
  float m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = -INFINITY, l[i] = 0.f;
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
    load_keys<T, kTile>(a, unit, t * kTile, len, ks);
    __syncthreads();
    if (idle) continue;
    float s[4][4];
    tile_scores(qs, ks, ty, tx, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int last = last_key(a, past, row0 + 4 * ty + i);
      float mt = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (t * kTile + tx + 16 * j > last) s[i][j] = -INFINITY;
        mt = fmaxf(mt, s[i][j]);
      }
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
    if (tx == 0 && row < rows)
      part[blockIdx.x * rows_total + (long long)r * rows + row] = make_float2(mm, ll);
  }
}

// The weights of kSumKeys keys, summed over every query row of the unit.
template <typename T>
__global__ void __launch_bounds__(256) key_sum_kernel(const __grid_constant__ KeyWeightsArgs a, float2* part, int splits) {
  extern __shared__ float sm[];
  __shared__ float2 ml[kTile];  // of a row: its maximum and 1 / sum
  const int r = blockIdx.y, unit = a.rows[r].unit;
  const int past = key_weights_past(a);
  const int len = past + a.q_len, rows = a.q_len * a.g.grp;
  const int j0 = blockIdx.x * kSumKeys;
  if (j0 >= len) return;
  const bool stored = a.rows[r].held > 0;
  const int b = (unit - a.unit0) / a.g.G, g = (unit - a.unit0) % a.g.G;
  const long long rows_total = (long long)a.units * rows;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  float *qs = sm, *ks = sm + kTile * kStride;
  constexpr int J = kSumKeys / 16;
  float w[J] = {};
  if (stored) {
    load_keys<T, kSumKeys>(a, unit, j0, len, ks);
    // the first token that sees key j0
    const int tok0 = max(0, j0 - past);
    for (int row0 = tok0 * a.g.grp; row0 < rows; row0 += kTile) {
      __syncthreads();
      load_queries<T>(a, b, g, row0, rows, qs);
      {  // the tile's rows' maxima and sums from their key ranges, four threads a row
        const int row = threadIdx.x >> 2;
        float mm = -INFINITY, ll = 0.f;
        if (row0 + row < rows) {
          const float2* p = part + (long long)r * rows + row0 + row;
#pragma unroll 8
          for (int i = threadIdx.x & 3; i < splits; i += 4) {
            const float2 v = p[i * rows_total];
            const float top = fmaxf(mm, v.x);
            if (v.y > 0.f) ll = ll * fast_exp2(mm - top) + v.y * fast_exp2(v.x - top);
            mm = top;
          }
        }
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
          const float om = __shfl_xor_sync(0xffffffffu, mm, off), ol = __shfl_xor_sync(0xffffffffu, ll, off);
          const float top = fmaxf(mm, om);
          ll = (ll > 0.f ? ll * fast_exp2(mm - top) : 0.f) + (ol > 0.f ? ol * fast_exp2(om - top) : 0.f);
          mm = top;
        }
        if ((threadIdx.x & 3) == 0) ml[row] = make_float2(mm, 1.f / ll);
      }
      __syncthreads();
      if (row0 + 8 * (int)(threadIdx.x >> 5) >= rows) continue;  // none of this warp's 8 rows is one
      float s[4][J];
      tile_scores(qs, ks, ty, tx, s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = row0 + 4 * ty + i;
        if (row >= rows) continue;
        const int last = last_key(a, past, row);
        const float2 e = ml[4 * ty + i];
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (j0 + tx + 16 * j <= last) w[j] = fmaf(fast_exp2(fmaf(s[i][j], kScoreScale, -e.x)), e.y, w[j]);
      }
    }
  }
  // over the 16 groups of rows, in their order
  __syncthreads();
#pragma unroll
  for (int j = 0; j < J; ++j) qs[ty * kSumKeys + tx + 16 * j] = w[j];
  __syncthreads();
  if (threadIdx.x < kSumKeys && j0 + threadIdx.x < len) {
    float x = 0.f;
    for (int i = 0; i < 16; ++i) x += qs[i * kSumKeys + threadIdx.x];
    float* o = a.out + r * a.out_stride + j0 + threadIdx.x;
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
    int e = cuda_check(cudaFuncSetAttribute(key_lse_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem),
                       "key_lse shared memory");
    return e ? e : cuda_check(cudaFuncSetAttribute(key_sum_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSumSmem),
                              "key_sum shared memory");
  });
  if (rc) return rc;
  const int key_tiles = (a.max_len + kSumKeys - 1) / kSumKeys;
  float2* part = reinterpret_cast<float2*>(ws + p.part);
  if (p.row_tiles > 65535) return fail(AOH_ERR_UNSUPPORTED, "aoh_key_weights: too many queries");
  key_lse_kernel<T><<<dim3(p.splits, a.units, p.row_tiles), 256, kSmem, st>>>(a, part, p.splits);
  key_sum_kernel<T><<<dim3(key_tiles, a.units), 256, kSumSmem, st>>>(a, part, p.splits);
  return cuda_check(cudaGetLastError(), "aoh_key_weights launch");
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
  if (c->cfg.dtype == AOH_BF16 && p.rows <= kFewRows) {
    plan_key_weights_few(c, units, max_len, p);
  } else if (c->cfg.dtype == AOH_BF16 && grp <= 128) {
    plan_key_weights_tensor(c, units, max_len, q_len, p);
  } else {
    p.row_tiles = (p.rows + kTile - 1) / kTile;
    const int key_tiles = (max_len + kTile - 1) / kTile;
    // enough CTAs for three per SM
    const long long ctas = std::max(1LL, (long long)units * p.row_tiles);
    p.splits = (int)std::max(1LL, std::min<long long>(std::min(64, key_tiles), (3LL * std::max(1, c->num_sms) + ctas - 1) / ctas));
    p.bytes = (size_t)p.splits * units * p.rows * sizeof(float2);
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
  if (!workspace || workspace_bytes < p.bytes)
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
