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
// Bound: HBM, logits in and fp32 out (6 bytes a token for bf16 logits, 1/4
// byte for the two bitmaps), and latency for a few rows.  One cluster of 8 CTAs
// takes a row, each an eighth of the vocabulary; the greedy token is reduced
// over the cluster in shared memory, so one launch and no workspace.  A thread
// has the loads of four groups of 8 tokens (or 8 single ones) in flight before
// it works on any.  A CTA's biased tokens are listed in shared memory first, in
// the order given, and marked in a bitmap there; the main pass leaves them out
// and a thread for each listed token does it alone, so that the sum over a
// token listed more than once has a fixed order.
#include <climits>

#include "common.cuh"
#include "internal.h"

namespace aoh {
namespace {

constexpr int kCluster = 8;
constexpr int kThreads = 256;
constexpr int kMaxBias = 4096;  // biases of a row (32 KB of shared memory if all fall into one slice)
constexpr uint32_t kInPrompt = 0x80000000u;

struct LogitsArgs {
  const void* logits;
  long long row_stride;  // elements
  int vocab, slice;      // tokens of one CTA, a multiple of 256
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

// 8 consecutive elements, 16-byte aligned
__device__ __forceinline__ void load8(const float* p, float* x) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* x) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = bf16_lo(w[j]);
    x[2 * j + 1] = bf16_hi(w[j]);
  }
}
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
  __device__ __forceinline__ float apply(float x, uint32_t w) const {
    x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    const uint32_t n = w & ~kInPrompt;
    x = __fsub_rn(x, __fmul_rn(freq, (float)n));
    return n ? __fsub_rn(x, pres) : x;
  }
};

// Larger value first, then the lower index; NaN above every number, -0 == +0.
__device__ __forceinline__ unsigned long long greedy_key(float x, int t) {
  uint32_t u = __float_as_uint(x + 0.f);
  u = x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return ((unsigned long long)u << 32) | (uint32_t)~t;
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
  __device__ __forceinline__ unsigned long long key() const {
    unsigned long long k = t == INT_MAX ? 0 : greedy_key(x, t);
    return nan_t == INT_MAX ? k : greedy_key(NAN, nan_t);
  }
};

template <typename T, typename O, bool kWide>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads, 4)
    logits_kernel(const __grid_constant__ LogitsArgs a) {
  extern __shared__ uint32_t smem[];  // with biases: a bit per token of the slice, then the slice's (id, value) list
  __shared__ unsigned long long best_warp[kThreads / 32];
  __shared__ unsigned long long best_cta[kCluster];
  __shared__ int s_count[kThreads / 32];
  uint32_t* biased = smem;
  int2* list = reinterpret_cast<int2*>(smem + a.slice / 32);
  const int rank = (int)cluster_ctarank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / kCluster;
  const int lo = rank * a.slice, hi = min(lo + a.slice, a.vocab);  // may be empty
  const int words = (a.vocab + 31) >> 5;
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
  const bool greedy = a.greedy != nullptr;
  Best best;

  int listed = 0;
  if (a.n_bias) {
    const int32_t* ids = a.bias_ids + (long long)row * a.n_bias;
    const float* values = a.bias + (long long)row * a.n_bias;
    for (int i = tid; i < a.slice / 32; i += kThreads) biased[i] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < a.n_bias; i0 += kThreads) {
      const int i = i0 + tid;
      const int id = i < a.n_bias ? ids[i] : -1;
      const float v = i < a.n_bias ? values[i] : 0.f;
      const bool in = id >= lo && id < hi;
      const unsigned m = __ballot_sync(0xffffffffu, in);
      if (lane == 0) s_count[warp] = __popc(m);
      if (in) atomicOr(&biased[(id - lo) >> 5], 1u << (id & 31));
      __syncthreads();
      int at = listed + __popc(m & ((1u << lane) - 1u));
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) at += s_count[w];
        listed += s_count[w];
      }
      if (in) list[at] = make_int2(id, __float_as_int(v));
      __syncthreads();
    }
  }

  if (kWide) {
    // groups of 8 tokens (vocab is a multiple of 8 here), four in flight
    constexpr int U = 4;
    for (int t0 = lo + tid * 8; t0 < hi; t0 += U * kThreads * 8) {
      float x[U][8];
      uint32_t s[U], al[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * kThreads * 8;
        s[u] = 0;
        al[u] = 0xffu;
        if (t < hi) {
          load8(x_row + t, x[u]);
          if (seen) s[u] = seen[t >> 5] >> (t & 31) & 0xffu;
          if (allowed) al[u] = allowed[t >> 5] >> (t & 31) & 0xffu;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * kThreads * 8;
        if (t >= hi) break;
        if (s[u]) {
          const uint4 c0 = reinterpret_cast<const uint4*>(pen.counts + t)[0], c1 = reinterpret_cast<const uint4*>(pen.counts + t)[1];
          const uint32_t c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (s[u] >> j & 1) x[u][j] = pen.apply(x[u][j], c[j]);
        }
        if (al[u] != 0xffu) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(al[u] >> j & 1)) x[u][j] = -INFINITY;
        }
        const uint32_t bi = a.n_bias ? biased[(t - lo) >> 5] >> (t & 31) & 0xffu : 0u;
        if (bi) {  // without the biased ones
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(bi >> j & 1)) {
              store1(out + t + j, x[u][j]);
              best.one(x[u][j], t + j);
            }
          continue;
        }
        store8(out + t, x[u]);
        if (greedy) {
          const float mx = fmaxf(fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3])),
                                 fmaxf(fmaxf(x[u][4], x[u][5]), fmaxf(x[u][6], x[u][7])));
          bool nan = false;
#pragma unroll
          for (int j = 0; j < 8; ++j) nan |= x[u][j] != x[u][j];
          if (mx > best.x || nan) {
#pragma unroll
            for (int j = 0; j < 8; ++j) best.one(x[u][j], t + j);
          }
        }
      }
    }
  } else {
    // rows that are not 16-byte aligned: a lane takes one token of the warp's word, eight words in flight
    constexpr int U = 8;
    for (int t0 = lo + tid; t0 < hi; t0 += U * kThreads) {
      float x[U];
      uint32_t s[U], al[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * kThreads;
        s[u] = 0;
        al[u] = 1;
        x[u] = 0.f;
        if (t < hi) {
          x[u] = load1(x_row + t);
          if (seen) s[u] = seen[t >> 5] >> lane & 1;
          if (allowed) al[u] = allowed[t >> 5] >> lane & 1;
        }
      }
      uint32_t c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) c[u] = s[u] ? pen.counts[t0 + u * kThreads] : 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * kThreads;
        if (t >= hi) break;
        if (s[u]) x[u] = pen.apply(x[u], c[u]);
        if (!al[u]) x[u] = -INFINITY;
        if (a.n_bias && (biased[(t - lo) >> 5] >> lane & 1)) continue;
        store1(out + t, x[u]);
        if (greedy) best.one(x[u], t);
      }
    }
  }
  unsigned long long key = best.key();

  for (int i = tid; i < listed; i += kThreads) {
    const int t = list[i].x;
    float sum = 0.f;
    int n = 0;  // how often t is listed so far
    bool first = true;
    for (int j = 0; j < listed; ++j) {
      const int2 e = list[j];
      if (e.x != t) continue;
      if (j < i) first = false;
      sum = n++ == 0 ? __int_as_float(e.y) : __fadd_rn(sum, __int_as_float(e.y));
    }
    if (!first) continue;
    float x = load1(x_row + t);
    if (seen && (seen[t >> 5] >> (t & 31) & 1)) x = pen.apply(x, pen.counts[t]);
    x = __fadd_rn(x, sum);
    if (allowed && !(allowed[t >> 5] >> (t & 31) & 1)) x = -INFINITY;
    if (greedy && x != -INFINITY) key = max(key, greedy_key(x, t));
    store1(out + t, x);
  }

  if (!greedy) return;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, off));
  if (lane == 0) best_warp[warp] = key;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) key = max(key, best_warp[i]);
    const uint32_t to = mapa_shared(&best_cta[rank], 0);
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(key) : "memory");
  }
  cluster_sync_all();
  if (rank == 0 && tid == 0) {
    key = best_cta[0];
#pragma unroll
    for (int i = 1; i < kCluster; ++i) key = max(key, best_cta[i]);
    // no key: every logit is -inf, and token 0 the first of equal ones
    a.greedy[row] = key == 0 ? 0 : (long long)(uint32_t) ~(uint32_t)key;
  }
}

// history[n, ids[n, i]]: +1 in the output, or the mark of the prompt
template <typename I>
__global__ void history_add_kernel(uint32_t* counts, uint32_t* seen, int vocab, const I* ids, long long id_stride,
                                   int per_row, const int32_t* lengths, bool prompt) {
  const int row = blockIdx.y;
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

template <typename T, typename O>
int launch(const LogitsArgs& a, int rows, bool wide, cudaStream_t st) {
  const size_t smem = a.n_bias ? (size_t)a.slice / 8 + (size_t)a.n_bias * sizeof(int2) : 0;
  auto kernel = wide ? logits_kernel<T, O, true> : logits_kernel<T, O, false>;
  if (smem > 40 * 1024) {
    // an attribute of the function and device: setting it again to the same or a smaller need is harmless
    const int rc = cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                              "aoh_logits_penalize shared memory");
    if (rc) return rc;
  }
  kernel<<<rows * kCluster, kThreads, smem, st>>>(a);
  return cuda_check(cudaGetLastError(), "aoh_logits_penalize launch");
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
  if (p.vocab > (1 << 23)) return fail(AOH_ERR_UNSUPPORTED, "%s: vocabulary of %d", who, p.vocab);
  if (p.n_bias > kMaxBias) return fail(AOH_ERR_UNSUPPORTED, "%s: %d biases of a row, at most %d", who, p.n_bias, kMaxBias);
  if (p.rows > (1 << 27)) return fail(AOH_ERR_UNSUPPORTED, "%s: too many rows", who);
  if (p.rows == 0) return AOH_OK;
  LogitsArgs a{};
  a.logits = p.logits;
  a.row_stride = p.row_stride;
  a.vocab = p.vocab;
  a.slice = ((p.vocab + kCluster - 1) / kCluster + 255) / 256 * 256;
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
  const int vin = p.dtype == AOH_BF16 ? 8 : 4, vout = p.out_dtype == AOH_BF16 ? 8 : 4;
  const bool wide = p.vocab % 8 == 0 && (p.rows == 1 || (p.row_stride % vin == 0 && p.out_stride % vout == 0)) &&
                    reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
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
    history_add_kernel<long long><<<grid, 256, 0, st>>>(c, s, vocab, static_cast<const long long*>(ids), id_stride,
                                                        per_row, lengths, prompt != 0);
  else
    history_add_kernel<int><<<grid, 256, 0, st>>>(c, s, vocab, static_cast<const int*>(ids), id_stride, per_row,
                                                  lengths, prompt != 0);
  return cuda_check(cudaGetLastError(), "aoh_history_add launch");
}
