// Rotary positions with several axes (time, height, width), computed from the
// positions themselves, with the Q/K RMSNorm that precedes them:
//
//   x <- x * rsqrt(mean(x^2) + eps) * w                    (per head, optional)
//   (a, b) <- (a cos t - b sin t, b cos t + a sin t),      t = pos[axis(i)] * freq(i)
//
// for every pair i of the rotated channels: (i, i + R/2) or, interleaved,
// (2i, 2i + 1). Angles: pos * freq reaches 1e5 radians, where a 32-bit angle
// is wrong in its third digit, so the product is formed in 64 bits in turns
// (freq / 2 pi comes in from the host), the whole turns are dropped (exact),
// and only the fraction is rounded to 32 bits for sincospif. Everything after
// that is 32-bit, rounded once to the tensor's type.
//
// Bound by HBM: Q and K once in, once out. In the vector form a thread owns 16
// channels (two 16-byte pieces holding 8 whole pairs) of one token and keeps
// their cos/sin in registers while it walks over the token's heads of Q and K,
// so a token's angles are computed once, not once a head.
#include <algorithm>

#include "xgb_common.cuh"

namespace xgb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxWidth = 512;
constexpr int kMaxPairs = kMaxWidth / 2;
constexpr int kMaxAxes = 8;

// The rotation, by value in the launch: turns per unit of position and axis
// of every pair.
struct Turns {
  double per_unit[kMaxPairs];
  uint8_t axis[kMaxPairs];
};

struct Params {
  const void* src[2];  // query, key
  void* dst[2];
  const void* weight[2];  // null: no norm
  float eps[2];
  int64_t sb[2], ss[2], sh[2];  // element strides of batch, token, head
  int heads[2];
  const void* positions;
  int64_t pb, ps;  // element strides of batch (0: shared by the batch) and token
  int pos_type;    // 0 int32, 1 int64, 2 float, 3 double
  int axes;
  int64_t tokens;  // batch * seq
  int64_t seq;
  int width, rotary;
};

__device__ __forceinline__ double load_position(const Params& p, int64_t at) {
  switch (p.pos_type) {
    case 0: return static_cast<double>(__ldg(static_cast<const int32_t*>(p.positions) + at));
    case 1: return static_cast<double>(__ldg(static_cast<const long long*>(p.positions) + at));
    case 2: return static_cast<double>(__ldg(static_cast<const float*>(p.positions) + at));
    default: return __ldg(static_cast<const double*>(p.positions) + at);
  }
}

__device__ __forceinline__ float2 cos_sin(const Params& p, int64_t token, double per_unit, int axis) {
  const int64_t b = token / p.seq, s = token - b * p.seq;
  const double turns = load_position(p, b * p.pb + s * p.ps + axis) * per_unit;
  float sn, cs;
  sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn, &cs);
  return make_float2(cs, sn);
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Scalar form for any width, pairing and alignment: one warp per head row,
// lane l owns pairs l, l + 32, ... and the unrotated channels likewise.
template <typename T>
__global__ void __launch_bounds__(kThreads) rope_axes_scalar_kernel(const Params p, const __grid_constant__ Turns turns,
                                                                    bool interleaved) {
  const int lane = threadIdx.x & 31;
  const int heads = p.heads[0] + p.heads[1];
  const int64_t rows = p.tokens * heads;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); row < rows;
       row += static_cast<int64_t>(gridDim.x) * (kThreads / 32)) {
    const int64_t token = row / heads;
    int h = static_cast<int>(row - token * heads);
    const int which = h >= p.heads[0];
    if (which) h -= p.heads[0];
    const int64_t b = token / p.seq, s = token - b * p.seq;
    const T* src = static_cast<const T*>(p.src[which]) + b * p.sb[which] + s * p.ss[which] + h * p.sh[which];
    T* dst = static_cast<T*>(p.dst[which]) + (token * p.heads[which] + h) * p.width;
    const T* w = static_cast<const T*>(p.weight[which]);
    float rstd = 1.f;
    if (w) {
      float sq = 0.f;
      for (int c = lane; c < p.width; c += 32) {
        const float v = to_float(src[c]);
        sq = fmaf(v, v, sq);
      }
      rstd = rsqrtf(warp_sum(sq) / p.width + p.eps[which]);
    }
    const int half = p.rotary / 2;
    for (int i = lane; i < half; i += 32) {
      const float2 cs = cos_sin(p, token, turns.per_unit[i], turns.axis[i]);
      const int ca = interleaved ? 2 * i : i, cb = interleaved ? 2 * i + 1 : i + half;
      float a = to_float(src[ca]), d = to_float(src[cb]);
      if (w) {
        a *= rstd * to_float(w[ca]);
        d *= rstd * to_float(w[cb]);
      }
      put(dst + ca, a * cs.x - d * cs.y);
      put(dst + cb, d * cs.x + a * cs.y);
    }
    for (int c = p.rotary + lane; c < p.width; c += 32) {
      float v = to_float(src[c]);
      if (w) v *= rstd * to_float(w[c]);
      put(dst + c, v);
    }
  }
}

// Eight consecutive channels.
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) {
  unpack_bf16x8(__ldg(reinterpret_cast<const uint4*>(p)), f);
}
__device__ __forceinline__ void load8(const __half* p, float (&f)[8]) {
  const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(round_bf16x2(f[0], f[1]), round_bf16x2(f[2], f[3]), round_bf16x2(f[4], f[5]),
                                            round_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void store8(__half* p, const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Vector form: width and rotary multiples of 16, 16-byte aligned rows. Threads
// are (token, head step, lane): 2^lane_bits lanes a head, 2^head_bits heads at
// a time, the rest of the 256 threads tokens. A block walks over groups of
// tokens; a group's cos/sin go through one of two shared buffers, so one
// barrier a group is enough.
template <typename T, bool kInterleaved, bool kNorm>
__global__ void __launch_bounds__(kThreads) rope_axes_vec_kernel(const Params p, const __grid_constant__ Turns turns,
                                                                 int lane_bits, int head_bits) {
  __shared__ double per_unit[kMaxPairs];
  __shared__ uint8_t axis[kMaxPairs];
  // at most 256 / lanes tokens of 8 * lanes pairs each
  __shared__ __align__(16) float cos_buf[2][kThreads * 8];
  __shared__ __align__(16) float sin_buf[2][kThreads * 8];
  const int pairs = p.rotary / 2;
  for (int i = threadIdx.x; i < pairs; i += kThreads) {
    per_unit[i] = turns.per_unit[i];
    axis[i] = turns.axis[i];
  }
  __syncthreads();
  const int j = threadIdx.x & ((1 << lane_bits) - 1);
  const int first_head = (threadIdx.x >> lane_bits) & ((1 << head_bits) - 1);
  const int t = threadIdx.x >> (lane_bits + head_bits);
  const int per_group = kThreads >> (lane_bits + head_bits);
  const int heads = p.heads[0] + p.heads[1];
  const bool active = j < p.width / 16, turned = j < p.rotary / 16;
  const int ca = kInterleaved || !turned ? 16 * j : 8 * j;
  const int cb = kInterleaved || !turned ? ca + 8 : ca + pairs;
  const int64_t groups = (p.tokens + per_group - 1) / per_group;
  int buf = 0;
  for (int64_t group = blockIdx.x; group < groups; group += gridDim.x, buf ^= 1) {
    const int64_t first = group * per_group;
    for (int i = threadIdx.x; i < per_group * pairs; i += kThreads) {
      const int tt = i / pairs, pair = i - tt * pairs;
      if (first + tt < p.tokens) {
        const float2 cs = cos_sin(p, first + tt, per_unit[pair], axis[pair]);
        cos_buf[buf][i] = cs.x;
        sin_buf[buf][i] = cs.y;
      }
    }
    __syncthreads();
    const int64_t token = first + t;
    const bool here = active && token < p.tokens;
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = 1.f;
      s[i] = 0.f;
    }
    if (here && turned) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 cv = *reinterpret_cast<const float4*>(&cos_buf[buf][t * pairs + 8 * j + i]);
        const float4 sv = *reinterpret_cast<const float4*>(&sin_buf[buf][t * pairs + 8 * j + i]);
        c[i] = cv.x; c[i + 1] = cv.y; c[i + 2] = cv.z; c[i + 3] = cv.w;
        s[i] = sv.x; s[i + 1] = sv.y; s[i + 2] = sv.z; s[i + 3] = sv.w;
      }
    }
    const int64_t b = token / p.seq, at = token - b * p.seq;
#pragma unroll 2
    for (int h0 = 0; h0 < heads; h0 += 1 << head_bits) {
      int h = h0 + first_head;
      const bool go = here && h < heads;
      const int which = h >= p.heads[0];
      if (which) h -= p.heads[0];
      float x[8], y[8];
      if (go) {
        const T* src = static_cast<const T*>(p.src[which]) + b * p.sb[which] + at * p.ss[which] + h * p.sh[which];
        load8(src + ca, x);
        load8(src + cb, y);
      }
      if constexpr (kNorm) {
        // every lane takes part; a tensor without a norm keeps its values
        float sq = 0.f;
        if (go) {
#pragma unroll
          for (int i = 0; i < 8; ++i) sq = fmaf(x[i], x[i], fmaf(y[i], y[i], sq));
        }
        for (int o = (1 << lane_bits) >> 1; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        const T* w = static_cast<const T*>(p.weight[which]);
        if (go && w) {
          const float rstd = rsqrtf(sq / p.width + p.eps[which]);
          float wa[8], wb[8];
          load8(w + ca, wa);
          load8(w + cb, wb);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] *= rstd * wa[i];
            y[i] *= rstd * wb[i];
          }
        }
      }
      if (go) {
        T* dst = static_cast<T*>(p.dst[which]) + (token * p.heads[which] + h) * p.width;
        if constexpr (kInterleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = x[2 * i], d = y[2 * i];
            x[2 * i] = a * c[i] - x[2 * i + 1] * s[i];
            x[2 * i + 1] = x[2 * i + 1] * c[i] + a * s[i];
            y[2 * i] = d * c[4 + i] - y[2 * i + 1] * s[4 + i];
            y[2 * i + 1] = y[2 * i + 1] * c[4 + i] + d * s[4 + i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = x[i];
            x[i] = a * c[i] - y[i] * s[i];
            y[i] = y[i] * c[i] + a * s[i];
          }
        }
        store8(dst + ca, x);
        store8(dst + cb, y);
      }
    }
  }
}

int bits_for(int n) {  // smallest b with 2^b >= n
  int b = 0;
  while ((1 << b) < n) ++b;
  return b;
}

template <typename T>
int launch(const Params& p, const Turns& turns, bool interleaved, cudaStream_t st) {
  const int heads = p.heads[0] + p.heads[1];
  bool vec = p.width % 16 == 0 && p.rotary % 16 == 0;
  for (int i = 0; i < 2 && vec; ++i) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.src[i]) | reinterpret_cast<uintptr_t>(p.dst[i]) |
                         reinterpret_cast<uintptr_t>(p.weight[i]);
    const int64_t strides = p.sb[i] | p.ss[i] | p.sh[i];
    vec = at % 16 == 0 && strides * static_cast<int64_t>(sizeof(T)) % 16 == 0;
  }
  if (!vec) {
    const int64_t blocks = std::min<int64_t>(cdiv(p.tokens * heads, kThreads / 32), 148 * 64);
    rope_axes_scalar_kernel<T><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(p, turns, interleaved);
    return launch_status();
  }
  const int lane_bits = bits_for(p.width / 16);
  // Few tokens: all heads of a token at once, so that more blocks have work.
  // Many: 8 heads at a time, so that a group has enough angles for its threads.
  const int most = p.tokens <= 2 * 148 ? 8 - lane_bits : std::min(3, 8 - lane_bits);
  const int head_bits = std::min(bits_for(heads), most);
  const int64_t groups = cdiv(p.tokens, kThreads >> (lane_bits + head_bits));
  const int64_t blocks = std::min<int64_t>(groups, 148 * 8);
  const bool norm = p.weight[0] || p.weight[1];
  auto run = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(p, turns, lane_bits, head_bits);
    return launch_status();
  };
  if (interleaved) return norm ? run(rope_axes_vec_kernel<T, true, true>) : run(rope_axes_vec_kernel<T, true, false>);
  return norm ? run(rope_axes_vec_kernel<T, false, true>) : run(rope_axes_vec_kernel<T, false, false>);
}

}  // namespace
}  // namespace xgb

using namespace xgb;

XGB_API int xgb_rope_axes(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype,
                          int64_t batch, int64_t seq, int64_t q_heads, int64_t k_heads, int64_t width,
                          const void* positions, int position_type, int64_t position_batch_stride,
                          int64_t position_stride, int64_t axes, const int64_t* axis_channels, const double* thetas,
                          int interleaved, const void* q_weight, const void* k_weight, float q_eps, float k_eps,
                          void* q_out, void* k_out, void* stream) {
  if (!q || !q_strides || !q_out || !positions || !axis_channels || !thetas) return XGB_ERR_ARG;
  if ((k == nullptr) != (k_out == nullptr) || (k && !k_strides)) return XGB_ERR_ARG;
  if (dtype < XGB_BF16 || dtype > XGB_F32 || position_type < 0 || position_type > 3) return XGB_ERR_ARG;
  if (batch < 0 || seq < 0 || q_heads <= 0 || (k && k_heads <= 0) || width <= 0 || width > kMaxWidth || axes <= 0 ||
      axes > kMaxAxes || q_heads > 65535 || k_heads > 65535)
    return XGB_ERR_SHAPE;
  if ((q_weight && !(q_eps >= 0.f)) || (k_weight && !(k_eps >= 0.f))) return XGB_ERR_ARG;
  Turns turns;
  int pairs = 0;
  constexpr double kTwoPi = 6.283185307179586476925286766559;
  for (int64_t a = 0; a < axes; ++a) {
    const int64_t d = axis_channels[a];
    if (d <= 0 || d % 2 || 2 * pairs + d > width) return XGB_ERR_SHAPE;
    if (!(thetas[a] > 0.0)) return XGB_ERR_ARG;
    for (int64_t i = 0; i < d / 2; ++i, ++pairs) {
      turns.per_unit[pairs] = pow(thetas[a], -2.0 * static_cast<double>(i) / static_cast<double>(d)) / kTwoPi;
      turns.axis[pairs] = static_cast<uint8_t>(a);
    }
  }
  if (batch == 0 || seq == 0) return XGB_OK;
  Params p{};
  const void* src[2] = {q, k};
  void* dst[2] = {q_out, k_out};
  const void* weight[2] = {q_weight, k_weight};
  const int64_t* strides[2] = {q_strides, k_strides};
  for (int i = 0; i < 2; ++i) {
    p.src[i] = src[i];
    p.dst[i] = dst[i];
    p.weight[i] = weight[i];
    if (src[i]) {
      p.sb[i] = strides[i][0];
      p.ss[i] = strides[i][1];
      p.sh[i] = strides[i][2];
    }
  }
  p.eps[0] = q_eps;
  p.eps[1] = k_eps;
  p.heads[0] = static_cast<int>(q_heads);
  p.heads[1] = k ? static_cast<int>(k_heads) : 0;
  p.positions = positions;
  p.pb = position_batch_stride;
  p.ps = position_stride;
  p.pos_type = position_type;
  p.axes = static_cast<int>(axes);
  p.tokens = batch * seq;
  p.seq = seq;
  p.width = static_cast<int>(width);
  p.rotary = 2 * pairs;
  cudaStream_t st = as_stream(stream);
  if (dtype == XGB_BF16) return launch<__nv_bfloat16>(p, turns, interleaved != 0, st);
  if (dtype == XGB_F16) return launch<__half>(p, turns, interleaved != 0, st);
  return launch<float>(p, turns, interleaved != 0, st);
}
