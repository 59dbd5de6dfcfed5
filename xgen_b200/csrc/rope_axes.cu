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
// Bound by HBM: Q and K once in, once out. A token's cos/sin (R/2 pairs) are
// computed once into shared memory and used by all of its heads, so the 64-bit
// work is 1/96th of the elements at 48 heads of 128.
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
  int per_block;  // tokens of one step of a block
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

template <typename T>
int launch(const Params& p, const Turns& turns, bool interleaved, cudaStream_t st) {
  const int64_t rows = p.tokens * (p.heads[0] + p.heads[1]);
  const int64_t blocks = std::min<int64_t>(cdiv(rows, kThreads / 32), 148 * 64);
  rope_axes_scalar_kernel<T><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(p, turns, interleaved);
  return launch_status();
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
