// The end of one DiT branch and the start of the next in one pass over a row:
//
//   x' = x + r * gate[idx] * post(y)         post = norm of the branch's output
//   h  = pre(x') * (1 + scale[idx]) + shift[idx]
//
// post and pre are each RMSNorm or LayerNorm times an optional weight, or
// nothing; gate and modulation are optional. x' and h are stored in the
// tensors' type, or h as int8 / e4m3 codes with one 32-bit scale a row,
// max(amax / 127 or 448, FLT_MIN): what the next 8-bit linear reads.
// Statistics, x' and h are 32-bit in registers; each stored value is rounded
// once, and h is computed from the x' before its rounding. Variances are sums
// of squared differences from the mean, so a mean far from zero costs no
// digits.
//
// Bound by HBM: y and x in, x' and h out. The two norms of the unfused form
// would read x' twice more and write and read post(y).
#include <math_constants.h>

#include <cfloat>
#include <algorithm>

#include "xgb_common.cuh"

namespace xgb {
namespace {

constexpr int kMaxWidth = 16384;

enum Norm : int { kNone = 0, kLayer = 1, kRms = 2 };
enum Quant : int { kPlain = 0, kInt8 = 1, kE4m3 = 2 };

struct Params {
  const void* y;
  const void* x;
  int64_t yb, ys, xb, xs;  // element strides of batch and token
  int64_t seq;
  int width;
  int post, pre;
  const void* post_weight;
  const void* pre_weight;
  float eps;
  float residual_scale;
  const void* gate;
  const void* scale;
  const void* shift;
  int64_t ldg, lds, ldsh;
  const int64_t* idx;
  int64_t idx_batch;  // element stride of the index between batches (0: shared)
  int64_t table_rows;
  void* x_out;
  void* h_out;
  uint8_t* codes;
  float* code_scale;
  int quant;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <int kThreads>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  if constexpr (kThreads > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) v += red[i];
    __syncthreads();
  }
  return v;
}

// Maximum of |h| by the bits of its absolute value, so that a NaN stays one.
template <int kThreads>
__device__ __forceinline__ float block_amax(uint32_t bits, uint32_t* red) {
  bits = __reduce_max_sync(0xffffffffu, bits);
  if constexpr (kThreads > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = bits;
    __syncthreads();
    bits = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) bits = max(bits, red[i]);
    __syncthreads();
  }
  return __uint_as_float(bits);
}

__device__ __forceinline__ float code_scale_of(float amax, int quant) {
  const float s = __fdiv_rn(amax, quant == kInt8 ? 127.0f : 448.0f);
  return s < FLT_MIN ? FLT_MIN : s;  // a NaN stays one
}

__device__ __forceinline__ uint8_t code_of(float h, float s, int quant) {
  const float v = __fdiv_rn(h, s);
  if (quant == kInt8) return static_cast<uint8_t>(__float2int_rn(fminf(fmaxf(v, -127.f), 127.f)));
  return f32_to_e4m3(fminf(fmaxf(v, -448.f), 448.f));
}

// Scalar form for any width, stride and alignment: one block a row, the row in
// shared memory.
constexpr int kScalarThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kScalarThreads) sandwich_norm_scalar_kernel(const Params p) {
  extern __shared__ float row[];
  __shared__ float red[kScalarThreads / 32];
  const int64_t r = blockIdx.x, b = r / p.seq, s = r - b * p.seq;
  const T* y = static_cast<const T*>(p.y) + b * p.yb + s * p.ys;
  const T* x = static_cast<const T*>(p.x) + b * p.xb + s * p.xs;
  int64_t t = 0;
  bool known = true;
  if (p.idx) {
    t = p.idx[b * p.idx_batch + s];
    known = t >= 0 && t < p.table_rows;
    if (!known) t = 0;
  }
  // (mean, 1 / deviation) of the values in `row`, which this thread wrote at
  // its own places
  auto stats = [&](int kind, float& mean, float& rstd) {
    mean = 0.f;
    rstd = 1.f;
    if (kind == kNone) return;
    float acc = 0.f;
    if (kind == kLayer) {
      for (int c = threadIdx.x; c < p.width; c += kScalarThreads) acc += row[c];
      mean = block_sum<kScalarThreads>(acc, red) / p.width;
      acc = 0.f;
    }
    for (int c = threadIdx.x; c < p.width; c += kScalarThreads) {
      const float d = row[c] - mean;
      acc = fmaf(d, d, acc);
    }
    rstd = rsqrtf(block_sum<kScalarThreads>(acc, red) / p.width + p.eps);
  };
  for (int c = threadIdx.x; c < p.width; c += kScalarThreads) row[c] = to_float(y[c]);
  float mean, rstd;
  stats(p.post, mean, rstd);
  for (int c = threadIdx.x; c < p.width; c += kScalarThreads) {
    float v = (row[c] - mean) * rstd;
    if (p.post_weight) v *= to_float(static_cast<const T*>(p.post_weight)[c]);
    if (p.gate) v *= known ? to_float(static_cast<const T*>(p.gate)[t * p.ldg + c]) : CUDART_NAN_F;
    v = fmaf(p.residual_scale, v, to_float(x[c]));
    row[c] = v;
    put(static_cast<T*>(p.x_out) + r * p.width + c, v);
  }
  if (!p.h_out && !p.codes) return;
  stats(p.pre, mean, rstd);
  uint32_t top = 0;
  for (int c = threadIdx.x; c < p.width; c += kScalarThreads) {
    float v = (row[c] - mean) * rstd;
    if (p.pre_weight) v *= to_float(static_cast<const T*>(p.pre_weight)[c]);
    if (p.scale) {
      const float sc = known ? to_float(static_cast<const T*>(p.scale)[t * p.lds + c]) : CUDART_NAN_F;
      v = fmaf(v, 1.0f + sc, to_float(static_cast<const T*>(p.shift)[t * p.ldsh + c]));
    }
    row[c] = v;
    top = max(top, __float_as_uint(v) & 0x7FFFFFFFu);
    if (p.h_out) put(static_cast<T*>(p.h_out) + r * p.width + c, v);
  }
  if (!p.codes) return;
  const float sc = code_scale_of(block_amax<kScalarThreads>(top, reinterpret_cast<uint32_t*>(red)), p.quant);
  if (threadIdx.x == 0) p.code_scale[r] = sc;
  for (int c = threadIdx.x; c < p.width; c += kScalarThreads) p.codes[r * p.width + c] = code_of(row[c], sc, p.quant);
}

template <typename T>
int launch(const Params& p, int64_t rows, cudaStream_t st) {
  auto kernel = sandwich_norm_scalar_kernel<T>;
  const size_t smem = static_cast<size_t>(p.width) * sizeof(float);
  if (smem > 40 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxWidth * sizeof(float)) != cudaSuccess)
    return XGB_ERR_LAUNCH;
  kernel<<<static_cast<unsigned>(rows), kScalarThreads, smem, st>>>(p);
  return launch_status();
}

}  // namespace
}  // namespace xgb

using namespace xgb;

XGB_API int xgb_sandwich_norm(const void* y, const int64_t* y_strides, const void* x, const int64_t* x_strides, int dtype,
                              int64_t batch, int64_t seq, int64_t width, int post_norm, const void* post_weight,
                              int pre_norm, const void* pre_weight, float eps, const void* gate, int64_t ldg,
                              float residual_scale, const void* scale, int64_t lds, const void* shift, int64_t ldsh,
                              const int64_t* indices, int64_t index_batch_stride, int64_t table_rows, void* x_out,
                              void* h_out, int quant, uint8_t* codes, float* code_scale, void* stream) {
  if (!y || !x || !y_strides || !x_strides || !x_out) return XGB_ERR_ARG;
  if (dtype < XGB_BF16 || dtype > XGB_F32 || post_norm < kNone || post_norm > kRms || pre_norm < kNone || pre_norm > kRms ||
      quant < kPlain || quant > kE4m3)
    return XGB_ERR_ARG;
  if ((quant == kPlain) != (codes == nullptr) || (codes == nullptr) != (code_scale == nullptr)) return XGB_ERR_ARG;
  if ((scale == nullptr) != (shift == nullptr)) return XGB_ERR_ARG;
  if ((gate || scale) != (indices != nullptr) || (indices && table_rows <= 0)) return XGB_ERR_ARG;
  if (!(eps >= 0.f)) return XGB_ERR_ARG;
  if (batch < 0 || seq < 0 || width <= 0 || width > kMaxWidth) return XGB_ERR_SHAPE;
  if ((gate && ldg < width) || (scale && (lds < width || ldsh < width))) return XGB_ERR_STRIDE;
  const int64_t rows = batch * seq;
  if (rows > INT32_MAX) return XGB_ERR_SHAPE;
  if (rows == 0) return XGB_OK;
  Params p{};
  p.y = y;
  p.x = x;
  p.yb = y_strides[0];
  p.ys = y_strides[1];
  p.xb = x_strides[0];
  p.xs = x_strides[1];
  p.seq = seq;
  p.width = static_cast<int>(width);
  p.post = post_norm;
  p.pre = pre_norm;
  p.post_weight = post_weight;
  p.pre_weight = pre_weight;
  p.eps = eps;
  p.residual_scale = residual_scale;
  p.gate = gate;
  p.scale = scale;
  p.shift = shift;
  p.ldg = ldg;
  p.lds = lds;
  p.ldsh = ldsh;
  p.idx = indices;
  p.idx_batch = index_batch_stride;
  p.table_rows = table_rows;
  p.x_out = x_out;
  p.h_out = h_out;
  p.codes = codes;
  p.code_scale = code_scale;
  p.quant = quant;
  cudaStream_t st = as_stream(stream);
  if (dtype == XGB_BF16) return launch<__nv_bfloat16>(p, rows, st);
  if (dtype == XGB_F16) return launch<__half>(p, rows, st);
  return launch<float>(p, rows, st);
}
