// Rotary embedding by positions with several axes (time, height, width for
// images and video; one axis is the ordinary rotary embedding), with optional
// per-head RMSNorm, from strided (batch, q_len, heads, head_dim) views of q and
// k to contiguous rotated q and k.
//
//   x'  = x * rsqrt(mean(x^2) + eps) * w                          (with weights)
//   a_i = positions[axis(i)] * inv_freq[i],   i < half = rotary_dim / 2
//   y_i        = (x'_i cos a_i - x'_{i+half} sin a_i) * scaling
//   y_{i+half} = (x'_{i+half} cos a_i + x'_i sin a_i) * scaling
//   dimensions from rotary_dim on pass through (normed, not rotated)
//
// Unlike aoh_rope_qk, which follows the rounding steps of the bf16 torch ops on
// given bf16 cos / sin, everything here is computed in fp32 from the positions
// and rounded once, when y is stored.  The angle of a far position needs more
// bits than a float has (at 10^6 radians an fp32 ulp is 0.06): the product and
// the reduction to one turn are done in fp64, the sine and cosine of the
// remainder in fp32 (their error is a few 2^-24).
//
// Bound: HBM, each of q and k read and written once.  A CTA computes the
// half x tokens sine / cosine pairs of its tokens once into shared memory and
// all its heads use them; a row is held by `lanes` (a power of two) threads
// with 16-byte loads of both members of each rotated pair.
#include "common.cuh"
#include "internal.h"

namespace aoh {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;  // rotary_dim <= head_dim <= 256
constexpr int kMaxAxes = 8;
constexpr int kMaxTokens = 4;  // tokens of one CTA

struct RopeAxesArgs {
  const void *q, *k, *qw, *kw;
  void *q_out, *k_out;
  const void* pos;
  const float* inv_freq;
  long long qs[3], ks[3], ps[3];  // strides in elements: batch, token, head / axis, batch, token
  long long n_tokens;
  int q_len, hq, g, d, half;
  int tokens, heads;  // of one CTA
  int lanes_log2;
  float eps, scaling;
  bool pos64;
  uint8_t axis[kMaxHalf];
};

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f(float x) { return x; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16(x); }

// VEC consecutive elements (16 bytes, or one).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void load(const T* p, float* x) {
  const Pack<T, VEC> r = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
  for (int j = 0; j < VEC; ++j) x[j] = to_f(r.v[j]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float* x) {
  Pack<T, VEC> r;
#pragma unroll
  for (int j = 0; j < VEC; ++j) r.v[j] = from_f<T>(x[j]);
  *reinterpret_cast<Pack<T, VEC>*>(p) = r;
}

// An item is VEC rotated pairs (i.., i + half..) or, behind them, up to
// 2 * VEC dimensions that pass through.
template <typename T, int VEC, int ITEMS>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ RopeAxesArgs a) {
  __shared__ float2 cs[kMaxTokens * kMaxHalf];
  const int half = a.half, lanes = 1 << a.lanes_log2;
  const long long tok0 = (long long)blockIdx.x * a.tokens;
  const int ntok = (int)min((long long)a.tokens, a.n_tokens - tok0);
  const int head0 = blockIdx.y * a.heads;
  const int nh = min(a.heads, a.hq + a.g - head0);
  const int lane = threadIdx.x & (lanes - 1);
  const int groups = kThreads >> a.lanes_log2;
  const int pairs = half / VEC;
  const int rest = (a.d - 2 * half) / VEC;  // chunks of VEC behind the rotated dimensions
  const int items = pairs + (rest + 1) / 2;

  float x[ITEMS][2][VEC];
  const T* src = nullptr;
  T* dst = nullptr;
  const T* w = nullptr;
  int tok = 0;
  auto locate = [&](int row) {
    tok = row / nh;
    const int h = head0 + row % nh;
    const long long t = tok0 + tok, b = t / a.q_len, c = t % a.q_len;
    if (h < a.hq) {
      src = static_cast<const T*>(a.q) + b * a.qs[0] + c * a.qs[1] + h * a.qs[2];
      dst = static_cast<T*>(a.q_out) + (t * a.hq + h) * a.d;
      w = static_cast<const T*>(a.qw);
    } else {
      src = static_cast<const T*>(a.k) + b * a.ks[0] + c * a.ks[1] + (h - a.hq) * a.ks[2];
      dst = static_cast<T*>(a.k_out) + (t * a.g + (h - a.hq)) * a.d;
      w = static_cast<const T*>(a.kw);
    }
  };
  // offsets of an item's two chunks (the second -1 where there is none)
  auto chunks = [&](int it, int& o0, int& o1) {
    if (it < pairs) {
      o0 = it * VEC;
      o1 = half + o0;
    } else {
      const int c = 2 * (it - pairs);
      o0 = 2 * half + c * VEC;
      o1 = c + 1 < rest ? o0 + VEC : -1;
    }
  };
  auto fetch = [&]() {
#pragma unroll
    for (int n = 0; n < ITEMS; ++n) {
      const int it = lane + (n << a.lanes_log2);
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[n][0][j] = x[n][1][j] = 0.f;
      if (it < items) {
        int o0, o1;
        chunks(it, o0, o1);
        load<T, VEC>(src + o0, x[n][0]);
        if (o1 >= 0) load<T, VEC>(src + o1, x[n][1]);
      }
    }
  };

  int row = threadIdx.x >> a.lanes_log2;
  const int rows = ntok * nh;
  // the first row is on its way while the sines and cosines are computed
  if (row < rows) {
    locate(row);
    fetch();
  }
  for (int e = threadIdx.x; e < ntok * half; e += kThreads) {
    const int t = e / half, i = e % half;
    const long long n = tok0 + t;
    const long long at = a.axis[i] * a.ps[0] + (n / a.q_len) * a.ps[1] + (n % a.q_len) * a.ps[2];
    const double p = a.pos64 ? (double)static_cast<const long long*>(a.pos)[at]
                             : (double)static_cast<const int*>(a.pos)[at];
    const double turns = p * (double)a.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[e] = make_float2(c * a.scaling, s * a.scaling);
  }
  __syncthreads();

  // the loop runs as often for every thread of a warp, which shuffles below
  const int rounds = (rows + groups - 1) / groups;
  for (int r = 0; r < rounds; ++r) {
    const bool live = row < rows;
    if (live && w) {
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < ITEMS; ++n)
#pragma unroll
        for (int j = 0; j < VEC; ++j) ss += x[n][0][j] * x[n][0][j] + x[n][1][j] * x[n][1][j];
      const unsigned mask = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u) << (threadIdx.x & 31 & ~(lanes - 1));
      for (int off = lanes >> 1; off > 0; off >>= 1) ss += __shfl_xor_sync(mask, ss, off);
      const float inv = rsqrtf(ss / (float)a.d + a.eps);
#pragma unroll
      for (int n = 0; n < ITEMS; ++n) {
        const int it = lane + (n << a.lanes_log2);
        if (it >= items) continue;
        int o0, o1;
        chunks(it, o0, o1);
        float w0[VEC], w1[VEC];
        load<T, VEC>(w + o0, w0);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[n][0][j] *= inv * w0[j];
        if (o1 >= 0) {
          load<T, VEC>(w + o1, w1);
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[n][1][j] *= inv * w1[j];
        }
      }
    }
    if (live) {
#pragma unroll
      for (int n = 0; n < ITEMS; ++n) {
        const int it = lane + (n << a.lanes_log2);
        if (it >= items) continue;
        int o0, o1;
        chunks(it, o0, o1);
        if (it < pairs) {
          const float2* row_cs = cs + tok * half + o0;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float2 t = row_cs[j];
            const float u = x[n][0][j], v = x[n][1][j];
            x[n][0][j] = u * t.x - v * t.y;
            x[n][1][j] = v * t.x + u * t.y;
          }
        }
        store<T, VEC>(dst + o0, x[n][0]);
        if (o1 >= 0) store<T, VEC>(dst + o1, x[n][1]);
      }
    }
    row += groups;
    if (row < rows) {
      locate(row);
      fetch();
    }
  }
}

template <typename T, int VEC>
int launch(RopeAxesArgs& a, int num_sms, cudaStream_t st) {
  const int items = a.half / VEC + ((a.d - 2 * a.half) / VEC + 1) / 2;
  a.lanes_log2 = 0;
  while ((1 << a.lanes_log2) < items && a.lanes_log2 < 5) ++a.lanes_log2;
  const int per_lane = (items + (1 << a.lanes_log2) - 1) >> a.lanes_log2;
  const int groups = kThreads >> a.lanes_log2, heads = a.hq + a.g;
  // Few rows: a CTA takes one round of rows of one token, so that the rows
  // spread over the SMs (the sines are computed by each of them).  Many: four
  // tokens and all their heads.
  if (a.n_tokens * heads <= 4LL * num_sms * groups) {
    a.tokens = 1;
    a.heads = std::min(heads, groups);
  } else {
    a.tokens = kMaxTokens;
    a.heads = heads;
  }
  const long long gx = (a.n_tokens + a.tokens - 1) / a.tokens;
  if (gx > 0x7fffffffLL) return fail(AOH_ERR_UNSUPPORTED, "aoh_rope_axes_qk: too many tokens");
  const dim3 grid((unsigned)gx, (unsigned)((heads + a.heads - 1) / a.heads));
  if (grid.y > 65535) return fail(AOH_ERR_UNSUPPORTED, "aoh_rope_axes_qk: too many heads");
  if (per_lane == 1)
    rope_axes_kernel<T, VEC, 1><<<grid, kThreads, 0, st>>>(a);
  else if (per_lane == 2)
    rope_axes_kernel<T, VEC, 2><<<grid, kThreads, 0, st>>>(a);
  else  // scalar items of up to 256 dimensions: at most 128 over 32 lanes
    rope_axes_kernel<T, VEC, 4><<<grid, kThreads, 0, st>>>(a);
  return cuda_check(cudaGetLastError(), "aoh_rope_axes_qk launch");
}

}  // namespace
}  // namespace aoh

using namespace aoh;

extern "C" int aoh_rope_axes_qk(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                int32_t dtype, const void* positions, int32_t positions_64,
                                const int64_t* position_strides, const float* inv_freq, const int32_t* sections,
                                int32_t n_axes, int32_t interleaved, const void* q_norm_weight,
                                const void* k_norm_weight, float eps, float scaling, int32_t batch, int32_t q_len,
                                int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, void* q_out, void* k_out,
                                aoh_stream stream) {
  const char* who = "aoh_rope_axes_qk";
  if (!q || !k || !q_strides || !k_strides || !positions || !position_strides || !inv_freq || !sections || !q_out ||
      !k_out)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null argument", who);
  if (dtype != AOH_BF16 && dtype != AOH_F32) return fail(AOH_ERR_UNSUPPORTED, "%s: bad dtype %d", who, dtype);
  if (batch < 0 || q_len < 0 || num_q_heads <= 0 || num_kv_heads <= 0)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
  if (head_dim <= 0 || head_dim > 2 * kMaxHalf || head_dim % 2)
    return fail(AOH_ERR_UNSUPPORTED, "%s: head_dim must be even and at most %d (got %d)", who, 2 * kMaxHalf, head_dim);
  if (n_axes < 1 || n_axes > kMaxAxes)
    return fail(AOH_ERR_UNSUPPORTED, "%s: 1 to %d position axes (got %d)", who, kMaxAxes, n_axes);
  if ((q_norm_weight == nullptr) != (k_norm_weight == nullptr))
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: give both norm weights or neither", who);
  if (q == q_out || k == k_out) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: outputs must not alias inputs", who);
  long long half = 0;
  for (int i = 0; i < n_axes; ++i) {
    if (sections[i] < 0) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: negative section", who);
    half += sections[i];
  }
  if (half < 1 || 2 * half > head_dim)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: the sections sum to %lld, not to 1..%d", who, half, head_dim / 2);
  RopeAxesArgs a{};
  if (interleaved) {
    for (int i = 0; i < half; ++i) {
      const int ax = i % n_axes;
      a.axis[i] = (uint8_t)(i < n_axes * (long long)sections[ax] ? ax : 0);
    }
    for (int ax = 1; ax < n_axes; ++ax)
      if (sections[ax] > 0 && (long long)(sections[ax] - 1) * n_axes + ax >= half)
        return fail(AOH_ERR_INVALID_ARGUMENT, "%s: section %d does not fit %lld interleaved frequencies", who, ax, half);
  } else {
    int i = 0;
    for (int ax = 0; ax < n_axes; ++ax)
      for (int j = 0; j < sections[ax]; ++j) a.axis[i++] = (uint8_t)ax;
  }
  a.n_tokens = (long long)batch * q_len;
  if (a.n_tokens == 0) return AOH_OK;
  int dev = 0, sms = 0;
  int rc = current_device(&dev);
  if (rc) return rc;
  rc = cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
  if (rc) return rc;
  a.q = q;
  a.k = k;
  a.qw = q_norm_weight;
  a.kw = k_norm_weight;
  a.q_out = q_out;
  a.k_out = k_out;
  a.pos = positions;
  a.pos64 = positions_64 != 0;
  a.inv_freq = inv_freq;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i];
    a.ks[i] = k_strides[i];
    a.ps[i] = position_strides[i];
  }
  a.q_len = q_len;
  a.hq = num_q_heads;
  a.g = num_kv_heads;
  a.d = head_dim;
  a.half = (int)half;
  a.eps = eps;
  a.scaling = scaling;
  // 16-byte accesses where every row, both halves and the weights allow them
  const int es = dtype == AOH_BF16 ? 2 : 4, vec = 16 / es;
  bool wide = half % vec == 0 && head_dim % vec == 0;
  const void* ptrs[6] = {q, k, q_norm_weight, k_norm_weight, q_out, k_out};
  for (const void* p : ptrs) wide = wide && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int i = 0; i < 3; ++i) wide = wide && q_strides[i] % vec == 0 && k_strides[i] % vec == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == AOH_BF16)
    return wide ? launch<__nv_bfloat16, 8>(a, sms, st) : launch<__nv_bfloat16, 1>(a, sms, st);
  return wide ? launch<float, 4>(a, sms, st) : launch<float, 1>(a, sms, st);
}
