// Eviction by accumulated attention weight: which keys a retrieval head keeps,
// and the copy of the kept rows into another cache.
//
// select: of each row of n weights the first `sink` and the last `recent` keys
// and the largest of the keys between them, `keep` in all, in ascending order
// of their positions; of equal weights the lower position first.  NaN ranks
// like -inf, -0 like +0.
//   A cluster of 1 to 8 CTAs takes a row, each CTA a contiguous part of the
//   middle, which it reads from memory once and holds in registers (up to 32 a
//   thread) as 32-bit keys in the order of the weights; a part larger than that
//   is read again by each step.  Three passes over 11, 11 and 10 bits find the
//   exact bits of the smallest kept weight: every CTA counts its part, and all
//   of them add up the cluster's histograms.  A count of larger and of equal
//   keys per warp, summed over warps and CTAs, then gives every kept key its
//   place, so the output needs no sorting.
//   Bound: the latency of the passes (HBM would take 4 bytes a key in, 8 bytes a
//   kept key out).
//
// evict: retrieval units' kept rows go to positions 0..keep-1 of the other
// cache; a streaming unit's sink rows keep their place and the rows of its
// ring go to the slots of their new positions (keep - T lower).  Source and
// destination are different caches, so every row moves independently.
//   Bound: HBM, 2 x 512 bytes a row (bf16).  A warp copies 8 rows: eight lanes
//   resolve the rows' pages side by side, then each 16-byte chunk of the 8
//   rows is in flight at once.
#include "common.cuh"
#include "internal.h"
#include "launch.cuh"
#include "page_layout.cuh"

namespace aoh {
namespace {

// ---------------------------------------------------------------------------
// select
// ---------------------------------------------------------------------------
constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr int kSelMaxCluster = 8;
constexpr int kSelMaxKeys = 32;  // of a thread, in registers

struct SelectArgs {
  const float* w;
  long long w_stride;
  int n, sink, recent, take;  // take: keys chosen from the middle
  int keep;
  int cluster, part;  // CTAs of a row, keys of a part (a multiple of kSelThreads)
  int32_t* kept;
  float* kept_w;
};

// Order-preserving bits of a weight: larger weight, larger key.
__device__ __forceinline__ uint32_t weight_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// The weight of a key, unless that may be NaN (like -inf) or -0 (like +0): then as it is in memory.
__device__ __forceinline__ float key_weight(uint32_t k, const float* p) {
  constexpr uint32_t kNegInf = ~0xff800000u, kZero = 0x80000000u;
  return k == kNegInf || k == kZero ? *p : __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ uint32_t ld_dsmem_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// No memory clobber: several are in flight at once, between two cluster barriers.
__device__ __forceinline__ uint2 ld_dsmem_v2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// Keys per thread: kKeys, in registers; kKeys = 0: any number, from memory.
// Warp w has the part's keys [w * 32 * per, (w + 1) * 32 * per), 32 neighbours
// at a time, so that a ballot keeps their order.
template <int kKeys>
__global__ void __launch_bounds__(kSelThreads) select_kernel(const __grid_constant__ SelectArgs a) {
  __shared__ alignas(16) uint32_t s_hist[3][kBins];  // one a pass: the cluster reads one while the next is filled
  __shared__ uint32_t s_scan[kSelWarps], s_eq[kSelWarps];
  __shared__ uint32_t s_total[2];  // this CTA's larger and equal keys
  __shared__ uint32_t s_bin, s_above;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = a.cluster > 1 ? (int)cluster_ctarank() : 0;
  const long long row = blockIdx.x / a.cluster;
  const float* w = a.w + row * a.w_stride;
  const int mid = a.n - a.sink - a.recent;
  const int lo = rank * a.part, cnt = max(0, min(a.part, mid - lo));
  const float* wm = w + a.sink + lo;
  int32_t* kept = a.kept + row * a.keep;
  float* kept_w = a.kept_w ? a.kept_w + row * a.keep : nullptr;
  auto sync = [&] {
    if (a.cluster > 1)
      cluster_sync_all();
    else
      __syncthreads();
  };

  griddep_wait();
  if (a.take > 0) {  // the same for every CTA of the cluster
    const int per = a.part / kSelThreads;  // <= kKeys
    const int i0 = warp * 32 * per + lane;
    // Behind the last key: 0, below every weight's key.  It is counted, but the
    // `take` largest keys, among which the threshold is sought, are weights.
    uint32_t key[kKeys ? kKeys : 1];
    if constexpr (kKeys > 0) {
      float x[kKeys];
#pragma unroll
      for (int j = 0; j < kKeys; ++j) x[j] = i0 + 32 * j < cnt ? wm[i0 + 32 * j] : 0.f;
#pragma unroll
      for (int j = 0; j < kKeys; ++j) key[j] = i0 + 32 * j < cnt ? weight_key(x[j]) : 0u;
    }
    // f(key, its index) for each of the thread's keys; every lane of a warp together
    auto each = [&](auto&& f) {
      if constexpr (kKeys > 0) {
#pragma unroll
        for (int j = 0; j < kKeys; ++j)
          if (j < per) f(key[j], i0 + 32 * j);
      } else {
        for (int j = 0; j < per; ++j) f(i0 + 32 * j < cnt ? weight_key(wm[i0 + 32 * j]) : 0u, i0 + 32 * j);
      }
    };
    for (int i = tid; i < 3 * kBins / 4; i += kSelThreads) reinterpret_cast<uint4*>(s_hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();

    uint32_t prefix = 0, left = (uint32_t)a.take;  // the threshold's leading bits, keys still to take
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digit = pass == 2 ? 1023u : 2047u;
      uint32_t* hist = s_hist[pass];
      each([&](uint32_t k, int) {  // digits above this one agree with the threshold
        if (pass == 0 || k >> (pass == 2 ? 10 : 21) == prefix) atomicAdd(&hist[k >> shift & digit], 1u);
      });
      sync();
      // thread t sums the bins kBins - 1 - 2 t and the one below over the cluster
      static_assert(kBins == 2 * kSelThreads, "a thread's bins are one 8-byte load");
      const uint32_t* top = hist + kBins - 2 * (tid + 1);
      uint2 c = make_uint2(0, 0);  // y: the upper bin
      if (a.cluster > 1) {
        uint2 v[kSelMaxCluster];
#pragma unroll
        for (int r = 0; r < kSelMaxCluster; ++r) v[r] = r < a.cluster ? ld_dsmem_v2(mapa_shared(top, r)) : make_uint2(0, 0);
#pragma unroll
        for (int r = 0; r < kSelMaxCluster; ++r) {
          c.x += v[r].x;
          c.y += v[r].y;
        }
      } else {
        c = *reinterpret_cast<const uint2*>(top);
      }
      uint32_t incl = c.x + c.y;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
      }
      if (lane == 31) s_scan[warp] = incl;
      __syncthreads();
      const uint32_t before = incl - c.x - c.y + __reduce_add_sync(0xffffffffu, lane < warp ? s_scan[lane] : 0u);
      if (before < left && before + c.x + c.y >= left) {  // one thread
        const bool upper = before + c.y >= left;
        s_bin = (uint32_t)(kBins - 1 - 2 * tid - (upper ? 0 : 1));
        s_above = before + (upper ? 0 : c.y);
      }
      __syncthreads();
      prefix = pass == 0 ? s_bin : pass == 1 ? prefix << 11 | s_bin : prefix << 10 | s_bin;
      left -= s_above;
    }
    // prefix: the threshold's bits; `left` of the keys equal to it are taken
    const uint32_t thr = prefix;

    uint32_t gt = 0, eq = 0;
    each([&](uint32_t k, int) {
      gt += k > thr;
      eq += k == thr;
    });
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
      s_scan[warp] = gt;
      s_eq[warp] = eq;
    }
    __syncthreads();
    // larger / equal keys before this warp's
    uint32_t bg = __reduce_add_sync(0xffffffffu, lane < warp ? s_scan[lane] : 0u);
    uint32_t be = __reduce_add_sync(0xffffffffu, lane < warp ? s_eq[lane] : 0u);
    if (a.cluster > 1) {
      if (tid == kSelThreads - 1) {
        s_total[0] = bg + gt;
        s_total[1] = be + eq;
      }
      __syncwarp();  // the barrier is one for converged warps
      cluster_sync_all();
      uint2 v = make_uint2(0, 0);
      if (lane < rank) v = make_uint2(ld_dsmem_u32(mapa_shared(&s_total[0], lane)), ld_dsmem_u32(mapa_shared(&s_total[1], lane)));
      bg += __reduce_add_sync(0xffffffffu, v.x);
      be += __reduce_add_sync(0xffffffffu, v.y);
      cluster_arrive();  // no CTA leaves while another may still read its counts
    }
    const unsigned below = (1u << lane) - 1u;
    each([&](uint32_t k, int i) {
      const bool is_gt = k > thr, is_eq = k == thr;
      const unsigned mg = __ballot_sync(0xffffffffu, is_gt), me = __ballot_sync(0xffffffffu, is_eq);
      const uint32_t re = be + __popc(me & below);
      if (is_gt || (is_eq && re < left)) {
        const int at = a.sink + (int)(bg + __popc(mg & below) + min(re, left));
        kept[at] = a.sink + lo + i;
        if (kept_w) kept_w[at] = key_weight(k, wm + i);
      }
      bg += __popc(mg);
      be += __popc(me);
    });
  }
  // the first and the last keys are kept as they are
  for (int i = rank * kSelThreads + tid; i < a.sink + a.recent; i += a.cluster * kSelThreads) {
    const int at = i < a.sink ? i : a.keep - a.sink - a.recent + i;
    const int p = i < a.sink ? i : a.n - a.sink - a.recent + i;
    kept[at] = p;
    if (kept_w) kept_w[at] = w[p];
  }
  __syncwarp();
  if (a.take > 0 && a.cluster > 1) cluster_wait();
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------
constexpr int kEvictWarps = 8, kEvictRows = 8;  // warps of a CTA, rows of a warp

// Table entry (page index within the unit) and slot of position p in a unit that holds it.
__device__ __forceinline__ void place(const CacheGeom& g, bool retrieval, int p, int& entry, int& slot) {
  if (retrieval || p < g.sink) {
    entry = p / kPage;
    slot = p % kPage;
  } else {
    const int r = (p - g.sink) % g.ring_cap;
    entry = g.sink_pages + r / kPage;
    slot = r % kPage;
  }
}

__device__ __forceinline__ int page_of(const CacheGeom& g, int unit, int entry) {
  const int at = g.unit_offset[unit] + entry;
  if (at >= g.unit_offset[unit + 1]) return -1;
  const int p = g.block_table[at];
  return p >= 0 && p < g.num_pages ? p : -1;
}

template <bool kBf16>
__global__ void __launch_bounds__(kEvictWarps * 32)
    evict_kernel(CacheGeom src, CacheGeom dst, const int32_t* unit_row, const int32_t* kept, long long kept_stride,
                 int keep, int len, int chunks) {
  const int unit = blockIdx.x / chunks;
  griddep_wait();
  if (dst.unit_offset[unit + 1] == dst.unit_offset[unit]) return;  // not stored here
  const int row = unit_row[unit];
  const bool retrieval = row >= 0;
  // a streaming unit holds its sink and, behind it, the latest ring_cap positions
  const int sink = min(dst.sink, keep), held = max(0, min(dst.ring_cap, keep - dst.sink));
  const int rows = retrieval ? keep : sink + held;
  const int lane = threadIdx.x & 31;
  const int r0 = ((blockIdx.x % chunks) * kEvictWarps + (threadIdx.x >> 5)) * kEvictRows;
  if (r0 >= rows) return;
  // lane j resolves row r0 + j
  int from = -1, to = -1;  // page * 16 + slot
  if (lane < kEvictRows && r0 + lane < rows) {
    const int i = r0 + lane;
    const int p_dst = retrieval || i < sink ? i : keep - held + (i - sink);
    const int p_src = retrieval ? kept[row * kept_stride + i] : i < sink ? i : p_dst + len - keep;
    if (p_src >= 0 && p_src < len) {
      int e, sl;
      place(src, retrieval, p_src, e, sl);
      const int ps = page_of(src, unit, e);
      if (ps >= 0) from = ps * kPage + sl;
      place(dst, retrieval, p_dst, e, sl);
      const int pd = page_of(dst, unit, e);
      if (pd >= 0) to = pd * kPage + sl;
    }
    if (from < 0 || to < 0) {
      atomicOr(dst.err, kErrBadPage);
      to = -1;
    }
  }
  const char* sp = static_cast<const char*>(src.pool);
  char* dp = static_cast<char*>(dst.pool);
  constexpr int kRowChunks = kBf16 ? 32 : 64;  // 16-byte chunks of a row's K and V
#pragma unroll
  for (int c0 = 0; c0 < kRowChunks; c0 += 32) {
    uint4 v[kEvictRows];
    const int c = c0 + lane;
#pragma unroll
    for (int j = 0; j < kEvictRows; ++j) {
      const int f = __shfl_sync(0xffffffffu, from, j), t = __shfl_sync(0xffffffffu, to, j);
      if (t < 0) continue;
      const long long page = f / kPage;
      const int slot = f % kPage;
      v[j] = kBf16 ? *reinterpret_cast<const uint4*>(sp + page * kPageBf16Bytes + bf16_chunk_offset(c >> 4, slot, c & 15))
                   : *reinterpret_cast<const uint4*>(sp + page * kPageF32Bytes + ((c >> 5) * kPage + slot) * 512 +
                                                     (c & 31) * 16);
    }
#pragma unroll
    for (int j = 0; j < kEvictRows; ++j) {
      const int t = __shfl_sync(0xffffffffu, to, j);
      if (t < 0) continue;
      const long long page = t / kPage;
      const int slot = t % kPage;
      char* o = kBf16 ? dp + page * kPageBf16Bytes + bf16_chunk_offset(c >> 4, slot, c & 15)
                      : dp + page * kPageF32Bytes + ((c >> 5) * kPage + slot) * 512 + (c & 31) * 16;
      *reinterpret_cast<uint4*>(o) = v[j];
    }
  }
}

}  // namespace
}  // namespace aoh

using namespace aoh;

extern "C" int aoh_select_keys(const float* weights, int64_t row_stride, int32_t rows, int32_t n, int32_t keep,
                               int32_t sink, int32_t recent, int32_t* kept, float* kept_weights, aoh_stream stream) {
  const char* who = "aoh_select_keys";
  if (rows < 0 || n < 0 || sink < 0 || recent < 0) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: negative size", who);
  if (keep < 0 || keep > n) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: keep %d of %d keys", who, keep, n);
  if ((int64_t)sink + recent > keep)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: sink %d and recent %d exceed keep %d", who, sink, recent, keep);
  if (rows == 0 || keep == 0) return AOH_OK;
  if (!weights || !kept) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null tensor", who);
  if (rows > (1 << 27)) return fail(AOH_ERR_UNSUPPORTED, "%s: too many rows", who);
  int dev = 0;
  int rc = current_device(&dev);
  if (rc) return rc;
  int sms = 0;
  rc = cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
  if (rc) return rc;
  SelectArgs a{};
  a.w = weights;
  a.w_stride = row_stride;
  a.n = n;
  a.sink = sink;
  a.recent = recent;
  a.keep = keep;
  a.take = keep - sink - recent;
  const int mid = n - sink - recent;
  // A CTA for every 8192 keys of a row, 8 at most, as long as all of them are
  // one wave of the GPU (an eighth of the SMs cannot be filled with clusters of
  // 8: 18 rows of 64K took 38 us in them, 32 rows in clusters of 4 22 us); a
  // thread then has 8 keys, or more.
  a.cluster = 1;
  while (a.cluster < kSelMaxCluster && a.cluster * 8 * kSelThreads < mid &&
         ((long long)rows * a.cluster * 2 <= sms * 7 / 8 || a.cluster * kSelMaxKeys * kSelThreads < mid))
    a.cluster *= 2;
  const int64_t keys = ((int64_t)mid + a.cluster - 1) / a.cluster;  // of a CTA; mid may be the largest int
  a.part = (int)((keys + kSelThreads - 1) / kSelThreads * kSelThreads);
  const int per = a.part / kSelThreads;
  a.kept = kept;
  a.kept_w = kept_weights;
  auto kernel = per <= 2    ? select_kernel<2>
                : per <= 8  ? select_kernel<8>
                : per <= 16 ? select_kernel<16>
                : per <= kSelMaxKeys ? select_kernel<kSelMaxKeys>
                                     : select_kernel<0>;
  return launch_dependent(kernel, dim3((unsigned)(rows * a.cluster)), a.cluster, kSelThreads, 0,
                          static_cast<cudaStream_t>(stream), "aoh_select_keys launch", a);
}

extern "C" int aoh_kv_evict(aoh_kv_cache* src, aoh_kv_cache* dst, int32_t past_len, const int32_t* kept,
                            int64_t kept_stride, int32_t keep, aoh_stream stream) {
  const char* who = "aoh_kv_evict";
  if (!src || !dst) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null cache", who);
  if (src == dst) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: source and destination are the same cache", who);
  const aoh_kv_config &a = src->cfg, &b = dst->cfg;
  if (a.num_layers != b.num_layers || a.batch != b.batch || a.num_kv_heads != b.num_kv_heads || a.dtype != b.dtype ||
      a.sink_size != b.sink_size || a.recent_size != b.recent_size || src->labels != dst->labels ||
      src->owned != dst->owned)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: the caches differ in more than their length", who);
  if (keep < 0 || past_len < 0 || keep > past_len)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: keep %d of %d positions", who, keep, past_len);
  bool any_retrieval = false, any_streaming = false;
  for (uint8_t v : src->labels) (v ? any_retrieval : any_streaming) = true;
  // a streaming head attends to its sink and window after the eviction as before
  if (any_streaming && keep < past_len && (int64_t)a.sink_size + a.recent_size > keep)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: keep %d is less than the streaming heads' sink %d + recent %d", who, keep,
                a.sink_size, a.recent_size);
  if (any_retrieval && keep > 0 && !kept) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null tensor", who);
  if (!src->bound || !dst->bound) return fail(AOH_ERR_STATE, "%s: cache is not bound to device memory", who);
  if (src->device != dst->device) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: the caches are on different devices", who);
  if (src->dirty_hi > src->dirty_lo || dst->dirty_hi > dst->dirty_lo)
    return fail(AOH_ERR_STATE, "%s: block tables changed since the last aoh_kv_sync", who);
  const int need_src = (past_len + kPage - 1) / kPage, need_dst = (keep + kPage - 1) / kPage;
  for (int u = 0; u < src->n_units; ++u) {
    const int l = u / (a.batch * a.num_kv_heads), g = u % a.num_kv_heads;
    if (!src->owned[u] || !src->retrieval(l, g)) continue;
    if (src->unit_npages[u] < need_src || dst->unit_npages[u] < need_dst)
      return fail(AOH_ERR_OUT_OF_PAGES, "%s: positions < %d (source) and < %d (destination) are not reserved", who,
                  past_len, keep);
  }
  if (keep == 0) return AOH_OK;
  const int rows = std::max(any_retrieval ? keep : 0, any_streaming ? a.sink_size + dst->ring_cap : 0);
  if (rows == 0) return AOH_OK;
  const int chunks = (rows + kEvictWarps * kEvictRows - 1) / (kEvictWarps * kEvictRows);
  const long long blocks = (long long)src->n_units * chunks;
  if (blocks > 0x7fffffffLL) return fail(AOH_ERR_UNSUPPORTED, "%s: too many rows", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const CacheGeom gs = src->geom(), gd = dst->geom();
  dst->last_write_layer = kEveryLayer;
  return launch_dependent(a.dtype == AOH_BF16 ? evict_kernel<true> : evict_kernel<false>, dim3((unsigned)blocks), 1,
                          kEvictWarps * 32, 0, st, "aoh_kv_evict launch", gs, gd, (const int32_t*)src->dev_unit_row, kept,
                          (long long)kept_stride, keep, past_len, chunks);
}
