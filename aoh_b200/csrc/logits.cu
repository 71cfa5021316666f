// Logits on their way to the next token: penalties for repeated tokens, biases
// and a grammar's mask, with the greedy token of the result.
//
//   x = logits[n, t]
//   x = x > 0 ? x / repetition : x * repetition      where t is in the prompt or the output
//   x = x - frequency * count[n, t]                  count: occurrences in the output
//   x = x - presence * [count[n, t] > 0]
//   x = x + sum of the row's biases for t
//   x = -inf                                         where the grammar does not allow t
//
// each step rounded to fp32 as written (no fused multiply-add), so the result
// is the one of the same steps in elementary operations.
//
// A sequence's history is a count per token (bit 31: in the prompt) and a
// bitmap of the tokens whose count word is not zero.  The bitmap is what a
// pass reads, 1 bit a token; the count words are read for the tokens it names.
//
// Floor: logits in and fp32 out (6 bytes a token for bf16 logits, 1/4 byte for
// the two bitmaps; 64 x 128K: 7.9 us, 18.5 here).  What bounds it there is not
// HBM (22.6 MB of DRAM traffic, 13% of its peak; the output stays in L2) but
// latency: issue slots 54% and warps 40%, one wave whose listed tokens are a
// second round trip to memory behind the copy.  A cluster of up to 16
// CTAs takes a row, 8192 tokens each (or more, where 16 CTAs do not reach): a
// thread then has all its loads, four groups of 8 tokens, in flight at once.
// The CTAs take 64 tokens in turn: vocabularies are sorted by frequency, and the
// CTA of a row's first tokens would list nearly all of the row's history
// (64 x 128K: its listed tokens took 9 us of 13).  The greedy token is reduced over the cluster
// in shared memory, so one launch and no workspace.  The main pass copies and
// masks; the few tokens with a count or a bias are listed in shared memory and
// done behind it, a thread each: the division of the penalties, in every group
// that holds one such token, cost more than the copy.  A CTA's biases are
// listed in the order given, and the entries of one token linked in that order:
// their sum has a fixed order (reading the whole list for each sum took 2 us more
// with 240 biases in a CTA's part).
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "launch.cuh"

namespace aoh {
namespace {

constexpr int kMaxCluster = 16;
constexpr int kThreads = 256;
constexpr int kMaxBias = 4096;  // biases of a row (64 KB of shared memory if all fall into one slice)
constexpr int kSlice = kThreads * 32;  // tokens whose loads a CTA has in flight at once (half of them where rows are not aligned)
constexpr int kTurn = 64;              // tokens that a row's CTAs take in turn
constexpr int kMaxVocab = 1 << 21;
constexpr uint32_t kInPrompt = 0x80000000u;
// two bits a token of the largest slice, and the list of 4096 biases: 192.3 KB
constexpr int kMaxSmem = 196 * 1024;

// Entries that a list of n biases is given: whole groups of 16, with those behind the last.
__host__ __device__ constexpr int bias_room(int n) { return (n + 31) / 16 * 16; }

struct LogitsArgs {
  const void* logits;
  long long row_stride;  // elements
  int vocab;
  int cluster, cluster_log, slice;  // CTAs of a row, tokens of one CTA (a multiple of 256)
  const uint32_t *counts, *seen;
  const float *repetition, *presence, *frequency;  // per row, or null: the scalar
  float repetition_s, presence_s, frequency_s;
  const int32_t* bias_ids;
  const float* bias;
  int n_bias;
  const uint32_t* allowed;
  const int32_t* allowed_rows;
  int n_allowed;
  void* out;
  long long out_stride;
  long long* greedy;
};

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float x) { *p = __float2bfloat16(x); }

// 8 consecutive elements, 16-byte aligned, as loaded and as floats
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void get(float* x) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};
template <>
struct Raw8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float* x) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = bf16_lo(w[j]);
      x[2 * j + 1] = bf16_hi(w[j]);
    }
  }
};
template <typename T>
struct Raw1 {
  T a;
  __device__ __forceinline__ void load(const T* p) { a = *p; }
  __device__ __forceinline__ void get(float* x) const { x[0] = load1(&a); }
};
__device__ __forceinline__ void store8(float* p, const float* x) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* x) {
  uint4 a;
  a.x = pack_bf16(x[0], x[1]);
  a.y = pack_bf16(x[2], x[3]);
  a.z = pack_bf16(x[4], x[5]);
  a.w = pack_bf16(x[6], x[7]);
  *reinterpret_cast<uint4*>(p) = a;
}

struct RowPenalties {
  float rep, pres, freq;
  const uint32_t* counts;
  // w: the token's count word; 0 leaves x as it is
  __device__ __forceinline__ float apply(float x, uint32_t w) const {
    const uint32_t n = w & ~kInPrompt;
    float y = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    y = __fsub_rn(y, __fmul_rn(freq, (float)n));
    y = n ? __fsub_rn(y, pres) : y;
    return w ? y : x;
  }
};

// Larger value first, then the lower index; NaN above every number, -0 == +0.
__device__ __forceinline__ unsigned long long greedy_key(float x, int t) {
  uint32_t u = __float_as_uint(x + 0.f);
  u = x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return ((unsigned long long)u << 32) | (uint32_t)~t;
}

__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The best of a thread's tokens, seen in ascending order.  -inf gives no key:
// a row of nothing else has token 0.
struct Best {
  float x = -INFINITY;
  int t = INT_MAX, nan_t = INT_MAX;
  __device__ __forceinline__ void one(float v, int at) {
    if (v > x) {
      x = v;
      t = at;
    }
    if (v != v) nan_t = min(nan_t, at);
  }
  // v, from the last of a group to the first, of which mx (NaN if any is) is the largest
  __device__ __forceinline__ void note(float v, float mx, int at) {
    if (v == mx) {
      x = mx;
      t = at;
    }
    if (v != v) nan_t = min(nan_t, at);
  }
  __device__ __forceinline__ unsigned long long key() const {
    unsigned long long k = t == INT_MAX ? 0 : greedy_key(x, t);
    return nan_t == INT_MAX ? k : greedy_key(NAN, nan_t);
  }
};

template <typename T, typename O, bool kWide>
__global__ void __launch_bounds__(kThreads, 4) logits_kernel(const __grid_constant__ LogitsArgs a) {
  // with biases: two bits per token of the slice, then the slice's list: ids, values, next entry of the same token
  extern __shared__ __align__(16) uint32_t smem[];
  __shared__ unsigned long long best_warp[kThreads / 32];
  __shared__ unsigned long long best_cta[kMaxCluster];
  __shared__ int s_count[kThreads / 32];
  uint32_t *biased = smem, *repeated = smem + a.slice / 32;
  int* b_id = reinterpret_cast<int*>(smem + a.slice / 16);  // behind the last 16 times -1
  float* b_value = reinterpret_cast<float*>(b_id + bias_room(a.n_bias));
  int* b_next = b_id + 2 * bias_room(a.n_bias);         // INT_MAX: none
  int* b_later = b_id + 3 * bias_room(a.n_bias);        // not 0: an entry before is of the same token
  const int rank = a.cluster > 1 ? (int)cluster_ctarank() : 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / a.cluster;
  // token of the CTA's p-th place, and a token's place
  auto token = [&](int p) { return ((((p / kTurn) << a.cluster_log) + rank) * kTurn) | (p % kTurn); };
  auto place = [&](int t) { return (((t / kTurn) >> a.cluster_log) * kTurn) | (t % kTurn); };
  const int words = (a.vocab + 31) >> 5;
  const bool greedy = a.greedy != nullptr;
  // A CTA's shared memory may be reached once the CTA is known to run: all of the cluster
  // arrive here, and wait before the best keys are handed to the first one (long done by then).
  if (greedy && a.cluster > 1) cluster_arrive();
  griddep_wait();
  const T* x_row = static_cast<const T*>(a.logits) + row * a.row_stride;
  O* out = static_cast<O*>(a.out) + row * a.out_stride;
  const uint32_t* seen = a.seen ? a.seen + (long long)row * words : nullptr;
  const RowPenalties pen{a.repetition ? a.repetition[row] : a.repetition_s,
                         a.presence ? a.presence[row] : a.presence_s,
                         a.frequency ? a.frequency[row] : a.frequency_s,
                         a.seen ? a.counts + (long long)row * a.vocab : nullptr};
  const uint32_t* allowed = nullptr;
  if (a.allowed) {
    const int r = a.allowed_rows ? a.allowed_rows[row] : row;
    if (r >= 0 && r < a.n_allowed) allowed = a.allowed + (long long)r * words;
  }
  Best best;

  // A thread's tokens of one round: U units of N neighbours, a stride apart.
  // Rows that are not 16-byte aligned take single tokens, a lane each of a word.
  constexpr int N = kWide ? 8 : 1, U = kWide ? 4 : 16, kRound = U * N * kThreads;
  constexpr uint32_t kOnes = (1u << N) - 1u;
  __shared__ uint16_t s_list[kRound];  // places of tokens with a count, from the round's first on
  __shared__ int s_listed;
  using Raw = typename std::conditional<kWide, Raw8<T>, Raw1<T>>::type;
  Raw raw[U];
  // bits of a unit's tokens: a byte each (wide), or in word `lane` those of the warp's unit `lane`
  constexpr int W = kWide ? U : 1;
  uint32_t s[W], al[W];
  auto fetch = [&](int base) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = token(base + (u * kThreads + tid) * N);
      if (t < a.vocab) raw[u].load(x_row + t);
    }
#pragma unroll
    for (int u = 0; u < W; ++u) {
      const int t = token(kWide ? base + (u * kThreads + tid) * N : base + lane * kThreads + warp * 32);
      const bool in = t < a.vocab && (kWide || lane < U);
      s[u] = 0;
      al[u] = 0xffffffffu;
      if (kWide) {
        if (in && seen) s[u] = reinterpret_cast<const uint8_t*>(seen)[t / 8];
        if (in && allowed) al[u] = reinterpret_cast<const uint8_t*>(allowed)[t / 8];
      } else {
        if (in && seen) s[u] = seen[t / 32];
        if (in && allowed) al[u] = allowed[t / 32];
      }
    }
  };
  // the first biases are asked for before the logits: their list is made while those are on their way
  const int32_t* ids = a.bias_ids + (long long)row * a.n_bias;
  const float* values = a.bias + (long long)row * a.n_bias;
  int id_next = tid < a.n_bias ? ids[tid] : -1;
  float v_next = tid < a.n_bias ? values[tid] : 0.f;
  fetch(0);
  if (tid == 0) s_listed = 0;

  int n_biased = 0;
  if (a.n_bias) {
    for (int i = tid; i < a.slice / 16; i += kThreads) smem[i] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < a.n_bias; i0 += kThreads) {
      const int id = id_next, i = i0 + kThreads + tid;
      const float v = v_next;
      if (i < a.n_bias) {
        id_next = ids[i];
        v_next = values[i];
      } else {
        id_next = -1;
      }
      const bool in = id >= 0 && id < a.vocab && ((id / kTurn) & (a.cluster - 1)) == rank;
      const unsigned m = __ballot_sync(0xffffffffu, in);
      if (lane == 0) s_count[warp] = __popc(m);
      if (in) {
        const uint32_t bit = 1u << (id & 31);
        const int word = place(id) / 32;
        if (atomicOr(&biased[word], bit) & bit) atomicOr(&repeated[word], bit);
      }
      __syncthreads();
      int at = n_biased + __popc(m & ((1u << lane) - 1u));
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) at += s_count[w];
        n_biased += s_count[w];
      }
      if (in) {
        b_id[at] = id;
        b_value[at] = v;
        b_later[at] = 0;
      }
      __syncthreads();
    }
    if (tid < 16) b_id[n_biased + tid] = -1;
    __syncthreads();
    // entries of one token are linked in their order, while the logits are on their way
    for (int i0 = warp * 32; i0 < n_biased; i0 += kThreads) {
      const int i = i0 + lane, id = i < n_biased ? b_id[i] : -1;
      const bool more = id >= 0 && repeated[place(id) / 32] >> (id & 31) & 1;
      if (!__any_sync(0xffffffffu, more)) continue;
      // the first entry behind i of its token, by its place in a group of four
      int next[4] = {INT_MAX, INT_MAX, INT_MAX, INT_MAX};
      auto look = [&](int j, bool check) {  // 16 entries
        int4 o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = reinterpret_cast<const int4*>(b_id + j)[k];
#pragma unroll
        for (int k = 3; k >= 0; --k) {
          if (o[k].x == id && (!check || j + 4 * k > i)) next[0] = j + 4 * k;
          if (o[k].y == id && (!check || j + 4 * k + 1 > i)) next[1] = j + 4 * k + 1;
          if (o[k].z == id && (!check || j + 4 * k + 2 > i)) next[2] = j + 4 * k + 2;
          if (o[k].w == id && (!check || j + 4 * k + 3 > i)) next[3] = j + 4 * k + 3;
        }
      };
      int j = (n_biased - 1) / 16 * 16;
      for (; j >= i0 + 32; j -= 16) look(j, false);
      for (; j >= i0; j -= 16) look(j, true);
      const int found = min(min(next[0], next[1]), min(next[2], next[3]));
      if (more) {
        b_next[i] = found;
        if (found != INT_MAX) b_later[found] = 1;
      }
    }
  } else if (seen) {
    __syncthreads();
  }

  unsigned long long key = 0;
  auto put = [&](int t, float y) {
    if (greedy && y != -INFINITY) key = max(key, greedy_key(y, t));
    store1(out + t, y);
  };
  for (int base = 0; base < a.slice; base += kRound) {
    if (base) fetch(base);
    int n_special = 0;
    uint32_t sp[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = base + (u * kThreads + tid) * N, t = token(p);
      const uint32_t se = kWide ? s[u % W] : __shfl_sync(0xffffffffu, s[0], u) >> lane & 1u;
      const uint32_t alw = kWide ? al[u % W] & kOnes : __shfl_sync(0xffffffffu, al[0], u) >> lane & 1u;
      sp[u] = 0;
      if (t >= a.vocab) continue;
      float x[N];
      raw[u].get(x);
      if (alw != kOnes) {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = alw >> j & 1 ? x[j] : -INFINITY;
      }
      const uint32_t bi = a.n_bias ? biased[p / 32] >> (p & 31) & kOnes : 0u;
      sp[u] = se & alw & ~bi;
      n_special += __popc(sp[u]);
      // tokens that are done again below are stored as they came: in place they must stay, and they are overwritten
      if constexpr (kWide)
        store8(out + t, x);
      else
        store1(out + t, x[0]);
      if (greedy) {
        const uint32_t later = sp[u] | bi;
        if (later) {
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] = later >> j & 1 ? -INFINITY : x[j];
        }
        if constexpr (kWide) {
          const float mx = max_nan(max_nan(max_nan(x[0], x[1], x[2]), x[3], x[4]), max_nan(x[5], x[6], x[7]));
          if (!(mx <= best.x)) {  // larger, or NaN
#pragma unroll
            for (int j = N - 1; j >= 0; --j) best.note(x[j], mx, t + j);
          }
        } else {
          best.one(x[0], t);
        }
      }
    }
    if (!seen) continue;
    // the list, in any order: its tokens do not depend on one another
    if (__any_sync(0xffffffffu, n_special > 0)) {
      int incl = n_special;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
      }
      int at = 0;
      if (lane == 31) at = atomicAdd(&s_listed, incl);
      at = __shfl_sync(0xffffffffu, at, 31) + incl - n_special;
#pragma unroll
      for (int u = 0; u < U; ++u)
        for (uint32_t m = sp[u]; m; m &= m - 1) s_list[at++] = (uint16_t)((u * kThreads + tid) * N + __ffs(m) - 1);
    }
    __syncthreads();
    const int n_listed = s_listed;
    // four a thread in flight: a slice of frequent tokens lists thousands
    for (int i0 = tid; i0 < n_listed; i0 += 4 * kThreads) {
      int t[4];
      uint32_t count[4];
      float x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * kThreads;
        t[u] = i < n_listed ? token(base + s_list[i]) : -1;
        if (t[u] >= 0) {
          count[u] = pen.counts[t[u]];
          x[u] = load1(x_row + t[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (t[u] >= 0) put(t[u], pen.apply(x[u], count[u]));
    }
    if (base + kRound < a.slice) {
      __syncthreads();
      if (tid == 0) s_listed = 0;
      __syncthreads();
    }
  }
  key = max(key, best.key());

  if (n_biased) {
    if (!seen) __syncthreads();  // the main pass has stored its tokens, and the entries are linked
    for (int i = tid; i < n_biased; i += kThreads) {
      if (b_later[i]) continue;
      const int t = b_id[i];
      const uint32_t count = seen ? pen.counts[t] : 0u;
      const bool ok = !allowed || allowed[t >> 5] >> (t & 31) & 1;
      const float x = load1(x_row + t);
      float sum = b_value[i];
      // listed more than once: added up in their order
      if (repeated[place(t) / 32] >> (t & 31) & 1)
        for (int j = b_next[i]; j != INT_MAX; j = b_next[j]) sum = __fadd_rn(sum, b_value[j]);
      put(t, ok ? __fadd_rn(pen.apply(x, count), sum) : -INFINITY);
    }
  }

  if (!greedy) return;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, off));
  if (lane == 0) best_warp[warp] = key;
  __syncthreads();
  if (a.cluster > 1) cluster_wait();
  if (tid == 0) {
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) key = max(key, best_warp[i]);
    if (a.cluster > 1) {
      const uint32_t to = mapa_shared(&best_cta[rank], 0);
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(key) : "memory");
    }
  }
  if (a.cluster > 1) {
    __syncwarp();  // the barrier is one for converged warps
    cluster_sync_all();
    if (rank == 0 && tid == 0) {
      key = best_cta[0];
      for (int i = 1; i < a.cluster; ++i) key = max(key, best_cta[i]);
    }
  }
  // no key: every logit is -inf, and token 0 the first of equal ones
  if (rank == 0 && tid == 0) a.greedy[row] = key == 0 ? 0 : (long long)(uint32_t) ~(uint32_t)key;
}

// history[n, ids[n, i]]: +1 in the output, or the mark of the prompt
template <typename I>
__global__ void history_add_kernel(uint32_t* counts, uint32_t* seen, int vocab, const I* ids, long long id_stride,
                                   int per_row, const int32_t* lengths, bool prompt) {
  const int row = blockIdx.y;
  griddep_wait();
  const int n = lengths ? min(lengths[row], per_row) : per_row;
  const int words = (vocab + 31) >> 5;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
    const long long t = (long long)ids[row * id_stride + i];
    if (t < 0 || t >= vocab) continue;
    uint32_t* c = counts + (long long)row * vocab + t;
    if (prompt)
      atomicOr(c, kInPrompt);
    else
      atomicAdd(c, 1u);
    atomicOr(seen + (long long)row * words + (t >> 5), 1u << (t & 31));
  }
}

template <typename T, typename O, bool kWide>
int launch(LogitsArgs& a, int rows, cudaStream_t st) {
  auto kernel = logits_kernel<T, O, kWide>;
  int dev = 0, sms = 0;
  int rc = current_device(&dev);
  if (rc) return rc;
  static PerDeviceOnce once;
  static int largest[kMaxDevices];
  rc = once.run(dev, [&] {
    return larger_cluster(kernel, kMaxCluster, kMaxCluster / 2, kThreads, kMaxSmem, "aoh_logits_penalize clusters",
                          &largest[dev]);
  });
  if (rc) return rc;
  rc = cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
  if (rc) return rc;
  // 16 CTAs a row take the least time while all of them have an SM's third part
  // (24 rows of 128K, all features, with 16 / 8: 10.6 / 11.4 us, 32 rows 14.2 /
  // 11.7), then 8, and 4 once those are more than one wave (64 rows: 21.4 with
  // 16, 16.0 with 8, 18.1 with 4).
  const int most = std::min(largest[dev], rows * 16LL <= 3 * sms ? 16 : rows * 8LL <= 4 * sms ? 8 : 4);
  a.cluster = 1;
  a.cluster_log = 0;
  while (a.cluster < most && a.cluster * (kWide ? kSlice : kSlice / 2) < a.vocab) {
    a.cluster *= 2;
    ++a.cluster_log;
  }
  const int turns = (a.vocab + kTurn - 1) / kTurn;
  a.slice = ((turns + a.cluster - 1) / a.cluster * kTurn + 255) / 256 * 256;
  const size_t smem = a.n_bias ? (size_t)a.slice / 4 + 4 * (size_t)bias_room(a.n_bias) * sizeof(int) : 0;
  return launch_dependent(kernel, dim3((unsigned)(rows * a.cluster)), a.cluster, kThreads, smem, st,
                          "aoh_logits_penalize launch", a);
}
template <typename T, typename O>
int launch(LogitsArgs& a, int rows, bool wide, cudaStream_t st) {
  return wide ? launch<T, O, true>(a, rows, st) : launch<T, O, false>(a, rows, st);
}

}  // namespace
}  // namespace aoh

using namespace aoh;

extern "C" int aoh_logits_penalize(const aoh_logits_args* args, aoh_stream stream) {
  const char* who = "aoh_logits_penalize";
  if (!args) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null argument", who);
  const aoh_logits_args& p = *args;
  if (p.rows < 0 || p.vocab < 1 || p.n_bias < 0 || p.n_allowed < 0)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
  if (p.rows > 0 && (!p.logits || !p.out)) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null tensor", who);
  if ((p.dtype != AOH_BF16 && p.dtype != AOH_F32) || (p.out_dtype != AOH_BF16 && p.out_dtype != AOH_F32))
    return fail(AOH_ERR_UNSUPPORTED, "%s: bad dtype", who);
  if ((p.counts == nullptr) != (p.seen == nullptr))
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: a history is counts and their bitmap", who);
  if (p.n_bias > 0 && (!p.bias_ids || !p.bias)) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null biases", who);
  if (p.allowed && !p.allowed_rows && p.n_allowed < p.rows)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: %d mask rows for %d rows", who, p.n_allowed, p.rows);
  if (p.logits == p.out && (p.dtype != p.out_dtype || (p.rows > 1 && p.row_stride != p.out_stride)))
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: in place needs the same type and strides", who);
  if (p.vocab > kMaxVocab) return fail(AOH_ERR_UNSUPPORTED, "%s: vocabulary of %d", who, p.vocab);
  if (p.n_bias > kMaxBias) return fail(AOH_ERR_UNSUPPORTED, "%s: %d biases of a row, at most %d", who, p.n_bias, kMaxBias);
  if (p.rows > (1 << 26)) return fail(AOH_ERR_UNSUPPORTED, "%s: too many rows", who);
  if (p.rows == 0) return AOH_OK;
  const int vin = p.dtype == AOH_BF16 ? 8 : 4, vout = p.out_dtype == AOH_BF16 ? 8 : 4;
  const bool wide = p.vocab % 8 == 0 && (p.rows == 1 || (p.row_stride % vin == 0 && p.out_stride % vout == 0)) &&
                    reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  LogitsArgs a{};
  a.logits = p.logits;
  a.row_stride = p.row_stride;
  a.vocab = p.vocab;
  a.counts = reinterpret_cast<const uint32_t*>(p.counts);
  a.seen = reinterpret_cast<const uint32_t*>(p.seen);
  a.repetition = p.repetition;
  a.presence = p.presence;
  a.frequency = p.frequency;
  a.repetition_s = p.repetition_scalar;
  a.presence_s = p.presence_scalar;
  a.frequency_s = p.frequency_scalar;
  a.bias_ids = p.bias_ids;
  a.bias = p.bias;
  a.n_bias = p.n_bias;
  a.allowed = reinterpret_cast<const uint32_t*>(p.allowed);
  a.allowed_rows = p.allowed_rows;
  a.n_allowed = p.n_allowed;
  a.out = p.out;
  a.out_stride = p.out_stride;
  a.greedy = reinterpret_cast<long long*>(p.greedy);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.dtype == AOH_BF16)
    return p.out_dtype == AOH_BF16 ? launch<__nv_bfloat16, __nv_bfloat16>(a, p.rows, wide, st)
                                   : launch<__nv_bfloat16, float>(a, p.rows, wide, st);
  return p.out_dtype == AOH_BF16 ? launch<float, __nv_bfloat16>(a, p.rows, wide, st)
                                 : launch<float, float>(a, p.rows, wide, st);
}

extern "C" int aoh_history_add(int32_t* counts, int32_t* seen, int32_t rows, int32_t vocab, const void* ids,
                               int32_t ids_64, int64_t id_stride, int32_t per_row, const int32_t* lengths,
                               int32_t prompt, aoh_stream stream) {
  const char* who = "aoh_history_add";
  if (rows < 0 || vocab < 1 || per_row < 0) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
  if (rows > 65535) return fail(AOH_ERR_UNSUPPORTED, "%s: at most 65535 rows", who);
  if (rows == 0 || per_row == 0) return AOH_OK;
  if (!counts || !seen || !ids) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null argument", who);
  const dim3 grid((unsigned)std::min(64, (per_row + 255) / 256), (unsigned)rows);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint32_t *c = reinterpret_cast<uint32_t*>(counts), *s = reinterpret_cast<uint32_t*>(seen);
  if (ids_64)
    return launch_dependent(history_add_kernel<long long>, grid, 1, 256, 0, st, "aoh_history_add launch", c, s, vocab,
                            static_cast<const long long*>(ids), (long long)id_stride, per_row, lengths, prompt != 0);
  return launch_dependent(history_add_kernel<int>, grid, 1, 256, 0, st, "aoh_history_add launch", c, s, vocab,
                          static_cast<const int*>(ids), (long long)id_stride, per_row, lengths, prompt != 0);
}
