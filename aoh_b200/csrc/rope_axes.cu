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
// Floor: each of q and k read and written once (4096 tokens of 32 bf16 heads of
// 128: 10.3 us at the copy rate, 14.3 here).  What bounds it there is not HBM --
// it moves 34 MB, a quarter of its peak, the output stays in L2 -- but the issue
// slots, 74% busy with two-element arithmetic and addresses.  A CTA computes the
// sines and cosines of its tokens once into shared memory and all its rows use them
// (eight of them in every thread's registers took 128 registers a thread and
// was slower); a row is held by `lanes` (a power of two) threads with 16-byte
// loads of both members of each rotated pair, which are under way while the
// sines are computed.  Two rows a thread and five CTAs an SM keep enough loads
// in flight.
#include "common.cuh"
#include "internal.h"
#include "launch.cuh"

namespace aoh {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;  // rotary_dim <= head_dim <= 256
constexpr int kMaxTokens = 4;  // tokens of one CTA

struct RopeAxesArgs {
  const void *q, *k, *qw, *kw;
  void *q_out, *k_out;
  const void* pos;
  const float* inv_freq;
  long long qs[3], ks[3], ps[3];  // strides in elements: batch, token, head / axis, batch, token
  int qn[3], kn[3], pn[3];        // the same, where no offset leaves 31 bits
  bool narrow;
  long long n_tokens;
  int q_len, hq, g, d, half;
  int tokens, heads;     // of one CTA
  // floor(2^32 / x) + 1: n / x is the high word of n * magic for the few n of a CTA
  uint32_t heads_magic, half_magic;
  int lanes_log2;
  float eps, scaling;
  bool pos64, norm_f32;
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
struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& r, float* x) {
  if constexpr (sizeof(T) == 2 && VEC == 8) {  // two at a time
    const uint4 u = *reinterpret_cast<const uint4*>(&r);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = bf16_lo(w[j]);
      x[2 * j + 1] = bf16_hi(w[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = to_f(r.v[j]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float* x) {
  if constexpr (sizeof(T) == 2 && VEC == 8) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  } else {
    Pack<T, VEC> r;
#pragma unroll
    for (int j = 0; j < VEC; ++j) r.v[j] = from_f<T>(x[j]);
    *reinterpret_cast<Pack<T, VEC>*>(p) = r;
  }
}

// An item is VEC rotated pairs (i.., i + half..) or, behind them, up to
// 2 * VEC dimensions that pass through.  A thread has ITEMS items of each of
// ROWS rows.
template <typename T, int VEC, int ITEMS, int ROWS>
__global__ void __launch_bounds__(kThreads, ITEMS > 1 || ROWS > 2 ? 3 : 5)
    rope_axes_kernel(const __grid_constant__ RopeAxesArgs a) {
  __shared__ alignas(16) float s_cos[kMaxTokens * kMaxHalf], s_sin[kMaxTokens * kMaxHalf];
  const int half = a.half, lanes = 1 << a.lanes_log2;
  const unsigned tok0 = blockIdx.x * (unsigned)a.tokens;
  const int ntok = (int)min((unsigned)a.tokens, (unsigned)a.n_tokens - tok0);
  const int head0 = blockIdx.y * a.heads;
  const int nh = min(a.heads, a.hq + a.g - head0);
  const int lane = threadIdx.x & (lanes - 1);
  const int groups = kThreads >> a.lanes_log2, group = threadIdx.x >> a.lanes_log2;
  const int rows = ntok * a.heads;  // at most ROWS * groups; the last of a token's CTAs may leave some out
  const int pairs = half / VEC;
  const int rest = (a.d - 2 * half) / VEC;  // chunks of VEC behind the rotated dimensions
  const int items = pairs + (rest + 1) / 2;
  // (batch, token) of the CTA's first token; the few behind it are counted on
  const unsigned b0 = tok0 / (unsigned)a.q_len, c0 = tok0 - b0 * (unsigned)a.q_len;
  auto locate = [&](int tok, int& b, int& c) {
    b = (int)b0;
    c = (int)c0 + tok;
    while (c >= a.q_len) {
      c -= a.q_len;
      ++b;
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
  int toks[ROWS], hs[ROWS];  // -1: no such row
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = group + r * groups;
    toks[r] = (int)__umulhi((unsigned)row, a.heads_magic);
    const int h = row - toks[r] * a.heads;
    hs[r] = row < rows && h < nh ? head0 + h : -1;
  }
  griddep_wait();
  Pack<T, VEC> raw[ROWS][ITEMS][2];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int h = hs[r];
    if (h < 0) continue;
    int b, c;
    locate(toks[r], b, c);
    long long off;
    if (a.narrow)
      off = h < a.hq ? b * a.qn[0] + c * a.qn[1] + h * a.qn[2] : b * a.kn[0] + c * a.kn[1] + (h - a.hq) * a.kn[2];
    else
      off = h < a.hq ? b * a.qs[0] + c * a.qs[1] + h * a.qs[2] : b * a.ks[0] + c * a.ks[1] + (h - a.hq) * a.ks[2];
    const T* src = static_cast<const T*>(h < a.hq ? a.q : a.k) + off;
#pragma unroll
    for (int n = 0; n < ITEMS; ++n) {
      const int it = lane + (n << a.lanes_log2);
      raw[r][n][0] = raw[r][n][1] = Pack<T, VEC>{};
      if (it < items) {
        int o0, o1;
        chunks(it, o0, o1);
        raw[r][n][0] = *reinterpret_cast<const Pack<T, VEC>*>(src + o0);
        if (o1 >= 0) raw[r][n][1] = *reinterpret_cast<const Pack<T, VEC>*>(src + o1);
      }
    }
  }
  for (int e = threadIdx.x; e < ntok * half; e += kThreads) {
    const int t = half > 1 ? (int)__umulhi((unsigned)e, a.half_magic) : e, i = e - t * half;
    int b, c;
    locate(t, b, c);
    const long long at = a.narrow ? a.axis[i] * a.pn[0] + b * a.pn[1] + c * a.pn[2]
                                  : a.axis[i] * a.ps[0] + b * a.ps[1] + c * a.ps[2];
    const double p = a.pos64 ? (double)static_cast<const long long*>(a.pos)[at]
                             : (double)static_cast<const int*>(a.pos)[at];
    const double turns = p * (double)a.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
    float s, co;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &co);
    s_cos[e] = co * a.scaling;
    s_sin[e] = s * a.scaling;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int tok = toks[r], h = hs[r];
    if (h < 0) continue;  // a row's lanes together
    const long long t = (long long)tok0 + tok;
    const bool is_q = h < a.hq;
    T* dst = is_q ? static_cast<T*>(a.q_out) + (t * a.hq + h) * a.d : static_cast<T*>(a.k_out) + (t * a.g + (h - a.hq)) * a.d;
    const T* w = static_cast<const T*>(is_q ? a.qw : a.kw);
    float inv = 1.f;
    if (w) {
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < ITEMS; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x[VEC];
          unpack<T, VEC>(raw[r][n][e], x);
#pragma unroll
          for (int j = 0; j < VEC; ++j) ss += x[j] * x[j];
        }
      // the row's lanes are consecutive, and take this branch together
      const unsigned mask = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u) << (threadIdx.x & 31 & ~(lanes - 1));
      for (int off = lanes >> 1; off > 0; off >>= 1) ss += __shfl_xor_sync(mask, ss, off);
      inv = rsqrtf(ss / (float)a.d + a.eps);
    }
#pragma unroll
    for (int n = 0; n < ITEMS; ++n) {
      const int it = lane + (n << a.lanes_log2);
      if (it >= items) continue;
      int o0, o1;
      chunks(it, o0, o1);
      float x[2][VEC];
      unpack<T, VEC>(raw[r][n][0], x[0]);
      unpack<T, VEC>(raw[r][n][1], x[1]);
      if (w) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int o = e ? o1 : o0;
          if (o < 0) continue;
          float v[VEC];
          if (sizeof(T) == 2 && a.norm_f32)
            unpack<float, VEC>(*reinterpret_cast<const Pack<float, VEC>*>(reinterpret_cast<const float*>(w) + o), v);
          else
            unpack<T, VEC>(*reinterpret_cast<const Pack<T, VEC>*>(w + o), v);
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[e][j] *= inv * v[j];
        }
      }
      if (it < pairs) {
        // 16-byte items: half and o0 are multiples of VEC, so these are 16-byte loads too
        const Pack<float, VEC> c = *reinterpret_cast<const Pack<float, VEC>*>(s_cos + tok * half + o0);
        const Pack<float, VEC> d = *reinterpret_cast<const Pack<float, VEC>*>(s_sin + tok * half + o0);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float u = x[0][j], v = x[1][j];
          x[0][j] = u * c.v[j] - v * d.v[j];
          x[1][j] = v * c.v[j] + u * d.v[j];
        }
      }
      store<T, VEC>(dst + o0, x[0]);
      if (o1 >= 0) store<T, VEC>(dst + o1, x[1]);
    }
  }
}

template <typename T, int VEC, int ITEMS, int ROWS>
int launch_rows(RopeAxesArgs& a, cudaStream_t st) {
  const int heads = a.hq + a.g, most = ROWS * (kThreads >> a.lanes_log2);
  a.heads = std::min(heads, most);
  a.tokens = std::max(1, std::min(kMaxTokens, most / heads));
  a.heads_magic = (uint32_t)((1ULL << 32) / a.heads + 1);  // a q and a k head at least
  a.half_magic = (uint32_t)((1ULL << 32) / a.half + 1);    // not used with half 1
  const long long gx = (a.n_tokens + a.tokens - 1) / a.tokens;
  const int gy = (heads + a.heads - 1) / a.heads;
  if (a.n_tokens > 0x7fffffffLL || gy > 65535) return fail(AOH_ERR_UNSUPPORTED, "aoh_rope_axes_qk: too many rows");
  return launch_dependent(rope_axes_kernel<T, VEC, ITEMS, ROWS>, dim3((unsigned)gx, (unsigned)gy), 1, kThreads, 0, st,
                          "aoh_rope_axes_qk launch", a);
}

template <typename T, int VEC>
int launch(RopeAxesArgs& a, int num_sms, cudaStream_t st) {
  const int items = a.half / VEC + ((a.d - 2 * a.half) / VEC + 1) / 2;
  a.lanes_log2 = 0;
  while ((1 << a.lanes_log2) < items && a.lanes_log2 < 5) ++a.lanes_log2;
  const int per_lane = (items + (1 << a.lanes_log2) - 1) >> a.lanes_log2;
  // Few rows: one a thread, so that they spread over the SMs (the sines are
  // computed by each of a token's CTAs).  Many: two.
  const bool few = a.n_tokens * (a.hq + a.g) <= 4LL * num_sms * (kThreads >> a.lanes_log2);
  if constexpr (VEC > 1) {
    // 16-byte items of at most 256 dimensions: at most 32, one a lane
    return few ? launch_rows<T, VEC, 1, 1>(a, st) : launch_rows<T, VEC, 1, 2>(a, st);
  } else {
    if (per_lane == 1) return few ? launch_rows<T, VEC, 1, 1>(a, st) : launch_rows<T, VEC, 1, 2>(a, st);
    if (per_lane == 2) return launch_rows<T, VEC, 2, 1>(a, st);
    return launch_rows<T, VEC, 4, 1>(a, st);  // at most 128 items over 32 lanes
  }
}

}  // namespace
}  // namespace aoh

using namespace aoh;

extern "C" int aoh_rope_axes_qk(const aoh_rope_axes_args* args, aoh_stream stream) {
  const char* who = "aoh_rope_axes_qk";
  if (!args) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null argument", who);
  const aoh_rope_axes_args& p = *args;
  if (!p.q || !p.k || !p.positions || !p.inv_freq || !p.q_out || !p.k_out)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: null tensor", who);
  if (p.dtype != AOH_BF16 && p.dtype != AOH_F32) return fail(AOH_ERR_UNSUPPORTED, "%s: bad dtype %d", who, p.dtype);
  if (p.batch < 0 || p.q_len < 0 || p.num_q_heads <= 0 || p.num_kv_heads <= 0)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
  if (p.head_dim <= 0 || p.head_dim > 2 * kMaxHalf || p.head_dim % 2)
    return fail(AOH_ERR_UNSUPPORTED, "%s: head_dim must be even and at most %d (got %d)", who, 2 * kMaxHalf, p.head_dim);
  if (p.n_axes < 1 || p.n_axes > AOH_ROPE_MAX_AXES)
    return fail(AOH_ERR_UNSUPPORTED, "%s: 1 to %d position axes (got %d)", who, AOH_ROPE_MAX_AXES, p.n_axes);
  if ((p.q_norm_weight == nullptr) != (p.k_norm_weight == nullptr))
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: give both norm weights or neither", who);
  if (p.q == p.q_out || p.k == p.k_out) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: outputs must not alias inputs", who);
  const int n_axes = p.n_axes;
  const int32_t* sections = p.sections;
  long long half = 0;
  for (int i = 0; i < n_axes; ++i) {
    if (sections[i] < 0) return fail(AOH_ERR_INVALID_ARGUMENT, "%s: negative section", who);
    half += sections[i];
  }
  if (half < 1 || 2 * half > p.head_dim)
    return fail(AOH_ERR_INVALID_ARGUMENT, "%s: the sections sum to %lld, not to 1..%d", who, half, p.head_dim / 2);
  RopeAxesArgs a{};
  if (p.interleaved) {
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
  a.n_tokens = (long long)p.batch * p.q_len;
  if (a.n_tokens == 0) return AOH_OK;
  int dev = 0, sms = 0;
  int rc = current_device(&dev);
  if (rc) return rc;
  rc = cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
  if (rc) return rc;
  a.q = p.q;
  a.k = p.k;
  a.qw = p.q_norm_weight;
  a.kw = p.k_norm_weight;
  a.q_out = p.q_out;
  a.k_out = p.k_out;
  a.pos = p.positions;
  a.pos64 = p.positions_64 != 0;
  a.norm_f32 = p.norm_f32 != 0;
  a.inv_freq = p.inv_freq;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = p.q_strides[i];
    a.ks[i] = p.k_strides[i];
    a.ps[i] = p.position_strides[i];
  }
  // 32-bit offsets, a third of the integer work of 64-bit ones, where the farthest element allows them
  auto farthest = [](const int64_t* s, int64_t n0, int64_t n1, int64_t n2) {
    return (n0 - 1) * std::abs(s[0]) + (n1 - 1) * std::abs(s[1]) + (n2 - 1) * std::abs(s[2]);
  };
  const int64_t limit = 1LL << 30;
  a.narrow = true;
  for (int i = 0; i < 3; ++i) {
    a.narrow = a.narrow && std::abs(p.q_strides[i]) < limit && std::abs(p.k_strides[i]) < limit &&
               std::abs(p.position_strides[i]) < limit;
    a.qn[i] = (int)p.q_strides[i];
    a.kn[i] = (int)p.k_strides[i];
    a.pn[i] = (int)p.position_strides[i];
  }
  a.narrow = a.narrow && farthest(p.q_strides, p.batch, p.q_len, p.num_q_heads) < limit &&
             farthest(p.k_strides, p.batch, p.q_len, p.num_kv_heads) < limit &&
             farthest(p.position_strides, n_axes, p.batch, p.q_len) < limit;
  a.q_len = p.q_len;
  a.hq = p.num_q_heads;
  a.g = p.num_kv_heads;
  a.d = p.head_dim;
  a.half = (int)half;
  a.eps = p.eps;
  a.scaling = p.scaling;
  // 16-byte accesses where every row, both halves and the weights allow them
  const int es = p.dtype == AOH_BF16 ? 2 : 4, vec = 16 / es;
  bool wide = half % vec == 0 && p.head_dim % vec == 0;
  const void* ptrs[6] = {p.q, p.k, p.q_norm_weight, p.k_norm_weight, p.q_out, p.k_out};
  for (const void* x : ptrs) wide = wide && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  for (int i = 0; i < 3; ++i) wide = wide && p.q_strides[i] % vec == 0 && p.k_strides[i] % vec == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.dtype == AOH_BF16)
    return wide ? launch<__nv_bfloat16, 8>(a, sms, st) : launch<__nv_bfloat16, 1>(a, sms, st);
  return wide ? launch<float, 4>(a, sms, st) : launch<float, 1>(a, sms, st);
}
