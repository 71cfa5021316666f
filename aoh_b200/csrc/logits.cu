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
// byte for the two bitmaps).  One cluster of 8 CTAs takes a row, each an
// eighth of the vocabulary; the greedy token is reduced over the cluster in
// shared memory, so one launch and no workspace.  Biased tokens are marked in
// a shared-memory bitmap first, left out by the main pass and done one by one
// behind it: the sum over a token listed more than once has a fixed order.
#include "common.cuh"
#include "internal.h"

namespace aoh {
namespace {

constexpr int kCluster = 8;
constexpr int kThreads = 512;
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
  __device__ __forceinline__ float apply(float x, int t) const {
    const uint32_t w = counts[t];
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
__device__ __forceinline__ unsigned long long shfl_xor_u64(unsigned long long v, int off) {
  return __shfl_xor_sync(0xffffffffu, v, off);
}

template <typename T, typename O, bool kWide>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads)
    logits_kernel(const __grid_constant__ LogitsArgs a) {
  extern __shared__ uint32_t biased[];  // slice / 32 words (with biases)
  __shared__ unsigned long long best_warp[kThreads / 32];
  __shared__ unsigned long long best_cta[kCluster];
  const int rank = (int)cluster_ctarank();
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
  const int32_t* bias_ids = a.bias_ids + (long long)row * a.n_bias;
  const float* bias = a.bias + (long long)row * a.n_bias;
  unsigned long long best = 0;

  if (a.n_bias) {
    for (int i = threadIdx.x; i < a.slice / 32; i += kThreads) biased[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n_bias; i += kThreads) {
      const int t = bias_ids[i];
      if (t >= lo && t < hi) atomicOr(&biased[(t - lo) >> 5], 1u << (t & 31));
    }
    __syncthreads();
  }

  // the tokens [t, t + n) of one 32-token word, bit j of the masks is token t + j
  if (kWide) {
    // a thread takes 8 tokens at a time (vocab is a multiple of 8 here)
    for (int t = lo + threadIdx.x * 8; t < hi; t += kThreads * 8) {
      float x[8];
      load8(x_row + t, x);
      const int sh = t & 31;
      const uint32_t s = seen ? seen[t >> 5] >> sh & 0xffu : 0u;
      const uint32_t al = allowed ? allowed[t >> 5] >> sh & 0xffu : 0xffu;
      const uint32_t bi = a.n_bias ? biased[(t - lo) >> 5] >> sh & 0xffu : 0u;
      if (s) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (s >> j & 1) x[j] = pen.apply(x[j], t + j);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!(al >> j & 1)) x[j] = -INFINITY;
      if (a.greedy) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(bi >> j & 1)) best = max(best, greedy_key(x[j], t + j));
      }
      if (!bi) {
        store8(out + t, x);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(bi >> j & 1)) store1(out + t + j, x[j]);
      }
    }
  } else {
    // rows that are not 16-byte aligned: a lane takes one token of the warp's word
    const int lane = threadIdx.x & 31;
    for (int t = lo + (int)threadIdx.x; t < hi; t += kThreads) {
      float x = load1(x_row + t);
      if (seen && (seen[t >> 5] >> lane & 1)) x = pen.apply(x, t);
      if (allowed && !(allowed[t >> 5] >> lane & 1)) x = -INFINITY;
      if (a.n_bias && (biased[(t - lo) >> 5] >> lane & 1)) continue;
      if (a.greedy) best = max(best, greedy_key(x, t));
      store1(out + t, x);
    }
  }

  for (int i = threadIdx.x; i < a.n_bias; i += kThreads) {
    const int t = bias_ids[i];
    if (t < lo || t >= hi) continue;
    bool first = true;
    for (int j = 0; j < i && first; ++j) first = bias_ids[j] != t;
    if (!first) continue;
    float sum = bias[i];
    for (int j = i + 1; j < a.n_bias; ++j)
      if (bias_ids[j] == t) sum = __fadd_rn(sum, bias[j]);
    float x = load1(x_row + t);
    if (seen && (seen[t >> 5] >> (t & 31) & 1)) x = pen.apply(x, t);
    x = __fadd_rn(x, sum);
    if (allowed && !(allowed[t >> 5] >> (t & 31) & 1)) x = -INFINITY;
    if (a.greedy) best = max(best, greedy_key(x, t));
    store1(out + t, x);
  }

  if (!a.greedy) return;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) best = max(best, shfl_xor_u64(best, off));
  if ((threadIdx.x & 31) == 0) best_warp[threadIdx.x >> 5] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kThreads / 32; ++i) best = max(best, best_warp[i]);
    const uint32_t to = mapa_shared(&best_cta[rank], 0);
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(best) : "memory");
  }
  cluster_sync_all();
  if (rank == 0 && threadIdx.x == 0) {
    best = best_cta[0];
    for (int i = 1; i < kCluster; ++i) best = max(best, best_cta[i]);
    a.greedy[row] = (long long)(uint32_t) ~(uint32_t)best;
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
  const size_t smem = a.n_bias ? (size_t)a.slice / 8 : 0;
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
