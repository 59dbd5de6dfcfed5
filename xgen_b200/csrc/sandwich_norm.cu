// The end of one DiT branch and the start of the next in one pass over a row:
//
//   x' = x + r * gate[idx] * post(y)         post = norm of the branch's output
//   h  = pre(x') * (1 + scale[idx]) + shift[idx]
//
// post and pre are each RMSNorm or LayerNorm times an optional weight, or
// nothing; gate and modulation are optional. x' and h are stored in the
// tensors' type, h instead or as well as int8 / e4m3 codes with one 32-bit scale
// a row, max(amax / 127 or 448, FLT_MIN): what the next 8-bit linear reads.
// Statistics, x' and h are 32-bit in registers; each stored value is rounded
// once, and h is computed from the x' before its rounding. A LayerNorm takes
// the mean off first; the differences are summed along with their squares, and
// what their sum shows of the mean's own rounding is taken off as well. So a
// mean far from zero costs no digits, and a constant row gives zeros to 2^-38
// of its value over sqrt(eps). 32-bit rows with codes are computed in 64 bits
// (below).
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
// shared memory, one value an access. 8,704 rows of 1001 in bf16 take 63 us, of
// 1000, in the vector form, 17; of 100 29 us, which is what a block a row costs.
// (32-bit rows with codes go to a form of their own, in 64 bits.)
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
  // (what is left of the mean, 1 / deviation) of the values in `row`, which this
  // thread wrote at its own places; a LayerNorm's are made differences from
  // their mean
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
    float off = 0.f;
    for (int c = threadIdx.x; c < p.width; c += kScalarThreads) {
      const float d = row[c] - mean;
      if (kind == kLayer) row[c] = d;
      off += d;
      acc = fmaf(d, d, acc);
    }
    mean = kind == kLayer ? block_sum<kScalarThreads>(off, red) / p.width : 0.f;
    rstd = rsqrtf(fmaxf(block_sum<kScalarThreads>(acc, red) / p.width - mean * mean, 0.f) + p.eps);
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
  if (sizeof(T) == 4 || !p.codes) return;
  const float sc = code_scale_of(block_amax<kScalarThreads>(top, reinterpret_cast<uint32_t*>(red)), p.quant);
  if (threadIdx.x == 0) p.code_scale[r] = sc;
  for (int c = threadIdx.x; c < p.width; c += kScalarThreads) p.codes[r * p.width + c] = code_of(row[c], sc, p.quant);
}

// Eight channels as they lie in memory, and as four pairs of 32-bit values:
// the arithmetic below is packed (two values an instruction), because at two
// bytes a value the instructions are as near to their limit as the bytes.
template <typename T>
struct Raw {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* p) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
__device__ __forceinline__ void unpack(const Raw<float>& r, float2 (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[2 * i] = make_float2(__uint_as_float(r.w[i].x), __uint_as_float(r.w[i].y));
    f[2 * i + 1] = make_float2(__uint_as_float(r.w[i].z), __uint_as_float(r.w[i].w));
  }
}
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16>& r, float2 (&f)[4]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}
__device__ __forceinline__ void unpack(const Raw<__half>& r, float2 (&f)[4]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}
__device__ __forceinline__ void store8(float* p, const float2 (&f)[4]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float2 (&f)[4]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(round_bf16x2(f[0].x, f[0].y), round_bf16x2(f[1].x, f[1].y), round_bf16x2(f[2].x, f[2].y), round_bf16x2(f[3].x, f[3].y));
}
__device__ __forceinline__ void store8(__half* p, const float2 (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __floats2half2_rn(f[i].x, f[i].y);
    w[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Vector form: 16-byte aligned rows of a multiple of 8 channels. kThreads
// threads hold a row, kChunks pieces of 8 channels each, so that its sums are
// short and, up to 1024 channels, need no barrier. The thread count is a
// constant because every address is then a base and an immediate: with both
// as run-time values the addresses, index divisions and joins of the sums took
// more instructions than the arithmetic (55 a channel at width 5120).
// At two bytes a value 64 registers a thread, 32 warps an SM, hold a row's
// loads and hide the joins of its sums (256 and 512 threads a row spill 16
// bytes): 31,689 rows of 5120 take 216 us (6.0 TB/s), with a LayerNorm 225 us;
// with as many registers as the compiler likes 15% more, with 51 18%. At four
// bytes the loads need the registers (44 us either way for 8,704 rows of 1536).
template <int kThreads>
constexpr int kRowsOf = kThreads == 32 ? 4 : 1;  // rows of a block
template <typename T, int kThreads>
constexpr int kBlocksOf = sizeof(T) == 2 && kThreads <= 512 ? 1024 / (kThreads * kRowsOf<kThreads>) : 1;

template <typename T, int kThreads, int kChunks>
__global__ void __launch_bounds__(kThreads * kRowsOf<kThreads>, kBlocksOf<T, kThreads>)
    sandwich_norm_vec_kernel(const Params p, uint32_t rows, FastDiv div_seq) {
  constexpr int kWarps = kThreads / 32;
  __shared__ float red[3][kWarps];
  __shared__ float2 red2[2][kWarps];
  const uint32_t r = kWarps == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (kWarps == 1 && r >= rows) return;
  const uint32_t b = fast_div(r, div_seq), s = r - b * div_seq.d;
  const int lane = kWarps == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int left = (p.width >> 3) - lane;  // piece j exists while j * kThreads < left
  const T* y = static_cast<const T*>(p.y) + b * p.yb + s * p.ys + lane * 8;
  const T* x = static_cast<const T*>(p.x) + b * p.xb + s * p.xs + lane * 8;
  Raw<T> yr[kChunks], xr[kChunks];
#pragma unroll
  for (int j = 0; j < kChunks; ++j)
    if (j * kThreads < left) {
      yr[j] = load_raw(y + j * kThreads * 8);
      xr[j] = load_raw(x + j * kThreads * 8);
    }
  int64_t t = 0;
  bool known = true;
  if (p.idx) {
    t = __ldg(p.idx + b * p.idx_batch + s);
    known = t >= 0 && t < p.table_rows;
    if (!known) t = 0;
  }
  const T* gate = static_cast<const T*>(p.gate) + t * p.ldg + lane * 8;
  const T* post_weight = static_cast<const T*>(p.post_weight) + lane * 8;
  const float inv_width = 1.0f / p.width;
  // every reduction has its own slots, so one barrier each is enough
  auto sum = [&](float v, int slot) {
    v = warp_sum(v);
    if constexpr (kWarps > 1) {
      if ((threadIdx.x & 31) == 0) red[slot][threadIdx.x >> 5] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) v += red[slot][i];
    }
    return v;
  };
  // Two at once: each half of a warp goes on with one of them.
  auto two_sums = [&](float a, float c, float2* slots) {
    const bool upper = threadIdx.x & 16;
    float v = upper ? c : a;
    v += __shfl_xor_sync(0xffffffffu, upper ? a : c, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (kWarps > 1) {
      if ((threadIdx.x & 15) == 0) reinterpret_cast<float*>(slots + (threadIdx.x >> 5))[upper] = v;
      __syncthreads();
      float2 both_sums = both(0.f);
#pragma unroll
      for (int i = 0; i < kWarps; ++i) both_sums = __fadd2_rn(both_sums, slots[i]);
      return both_sums;
    }
    return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
  };
  float2 v[kChunks][4];
  // The norm as v * rstd + shift, of a LayerNorm's values less their mean.
  auto stats = [&](int kind, int slot, float& rstd, float& shift) {
    rstd = 1.f;
    shift = 0.f;
    if (kind == kNone) return;
    float2 acc = both(0.f);
    if (kind == kLayer) {
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
        if (j * kThreads < left)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc = __fadd2_rn(acc, v[j][e]);
      const float2 minus = both(-sum(acc.x + acc.y, slot) * inv_width);
      acc = both(0.f);
      float2 off = both(0.f);
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
        if (j * kThreads < left)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[j][e] = __fadd2_rn(v[j][e], minus);
            off = __fadd2_rn(off, v[j][e]);
            acc = __ffma2_rn(v[j][e], v[j][e], acc);
          }
      const float2 sums = two_sums(acc.x + acc.y, off.x + off.y, red2[slot]);
      const float rest = sums.y * inv_width;
      rstd = rsqrtf(fmaxf(fmaf(sums.x, inv_width, -rest * rest), 0.f) + p.eps);
      shift = -rest * rstd;
    } else {
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
        if (j * kThreads < left)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc = __ffma2_rn(v[j][e], v[j][e], acc);
      rstd = rsqrtf(fmaf(sum(acc.x + acc.y, slot), inv_width, p.eps));
    }
  };
#pragma unroll
  for (int j = 0; j < kChunks; ++j)
    if (j * kThreads < left) unpack(yr[j], v[j]);
  float rstd, shift;
  stats(p.post, 0, rstd, shift);
  // a row whose index is outside the table becomes NaN through its factor
  if (p.gate && !known) rstd = CUDART_NAN_F;
  T* x_out = static_cast<T*>(p.x_out) + static_cast<int64_t>(r) * p.width + lane * 8;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    if (j * kThreads >= left) continue;
    float2 f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[j][e] = __ffma2_rn(v[j][e], both(rstd), both(shift));
    if (p.post_weight) {
      unpack(load_raw(post_weight + j * kThreads * 8), f);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = __fmul2_rn(v[j][e], f[e]);
    }
    if (p.gate) {
      unpack(load_raw(gate + j * kThreads * 8), f);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = __fmul2_rn(v[j][e], f[e]);
    }
    unpack(xr[j], f);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[j][e] = __ffma2_rn(v[j][e], both(p.residual_scale), f[e]);
    store8(x_out + j * kThreads * 8, v[j]);
  }
  if (!p.h_out && !p.codes) return;
  stats(p.pre, 1, rstd, shift);
  if (p.scale && !known) rstd = CUDART_NAN_F;
  const T* pre_weight = static_cast<const T*>(p.pre_weight) + lane * 8;
  const T* mod_scale = static_cast<const T*>(p.scale) + t * p.lds + lane * 8;
  const T* mod_shift = static_cast<const T*>(p.shift) + t * p.ldsh + lane * 8;
  T* h_out = static_cast<T*>(p.h_out) + static_cast<int64_t>(r) * p.width + lane * 8;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    if (j * kThreads >= left) continue;
    float2 f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[j][e] = __ffma2_rn(v[j][e], both(rstd), both(shift));
    if (p.pre_weight) {
      unpack(load_raw(pre_weight + j * kThreads * 8), f);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = __fmul2_rn(v[j][e], f[e]);
    }
    if (p.scale) {
      float2 g[4];
      unpack(load_raw(mod_scale + j * kThreads * 8), f);
      unpack(load_raw(mod_shift + j * kThreads * 8), g);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = __ffma2_rn(v[j][e], __fadd2_rn(f[e], both(1.f)), g[e]);
    }
    if (p.h_out) store8(h_out + j * kThreads * 8, v[j]);
    if (sizeof(T) == 2 && p.codes) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        top = max(max(top, __float_as_uint(v[j][e].x) & 0x7FFFFFFFu), __float_as_uint(v[j][e].y) & 0x7FFFFFFFu);
    }
  }
  if (sizeof(T) == 4 || !p.codes) return;
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (kWarps > 1) {
    if ((threadIdx.x & 31) == 0) red[2][threadIdx.x >> 5] = __uint_as_float(top);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) top = max(top, __float_as_uint(red[2][i]));
  }
  const float sc = code_scale_of(__uint_as_float(top), p.quant);
  const float inv = __frcp_rn(sc);
  if (lane == 0) p.code_scale[r] = sc;
  uint8_t* codes = p.codes + static_cast<int64_t>(r) * p.width + lane * 8;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    if (j * kThreads >= left) continue;
    uint32_t lo, hi;
    // the correctly rounded quotient (div_by, two at a time)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 q = __fmul2_rn(v[j][e], both(inv));
      v[j][e] = __ffma2_rn(__ffma2_rn(q, both(-sc), v[j][e]), both(inv), q);
    }
    if (p.quant == kInt8) {
      // |q| <= 127 and a rounding: 1.5 * 2^23 + q has the nearest even integer
      // in its low bits
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = __fadd2_rn(v[j][e], both(12582912.0f));
      lo = __byte_perm(__byte_perm(__float_as_uint(v[j][0].x), __float_as_uint(v[j][0].y), 0x0040),
                       __byte_perm(__float_as_uint(v[j][1].x), __float_as_uint(v[j][1].y), 0x0040), 0x5410);
      hi = __byte_perm(__byte_perm(__float_as_uint(v[j][2].x), __float_as_uint(v[j][2].y), 0x0040),
                       __byte_perm(__float_as_uint(v[j][3].x), __float_as_uint(v[j][3].y), 0x0040), 0x5410);
    } else {
      lo = e4m3x2(v[j][0].x, v[j][0].y) | (e4m3x2(v[j][1].x, v[j][1].y) << 16);
      hi = e4m3x2(v[j][2].x, v[j][2].y) | (e4m3x2(v[j][3].x, v[j][3].y) << 16);
    }
    *reinterpret_cast<uint2*>(codes + j * kThreads * 8) = make_uint2(lo, hi);
  }
}

// 32-bit rows with codes, in 64 bits. A code whose quotient lies next to the
// border between two codes goes by its last bits: in 32 bits one to four of a
// million fall on the other side, and what such a code stands for is then off
// by a whole code, 2e-5 to 1.2e-4 of the tensor's norm. (16-bit rows keep 32
// bits: there that is far below the rounding of what the codes stand for.) In
// 64 bits only a quotient within some 2^-50 of a border can differ from the
// definition's. An e4m3 code is that of the quotient rounded to 32 bits.
//
// Values c, c + kThreads, .. of a row are a thread's, so any stride and
// alignment will do. Bound by chains of 64-bit arithmetic, with about 120
// instructions a value (46% of the issue slots; 36% of the conversions' pipe, 9 a
// value; 14% of the 64-bit units; DRAM 16%): 8,704 rows of 1536 to int8 take 103
// us (41 us in 32 bits), 16,384 of 336 45 us, one row 9 us. At 64 registers wide
// rows fill the SM: 15,844 of 5120 take 714 us, with x requested ahead of its
// use and 96 registers 1,025 us.
template <int kThreads, int kValues>
__global__ void __launch_bounds__(kThreads * kRowsOf<kThreads>, 1024 / (kThreads * kRowsOf<kThreads>)) sandwich_norm_codes64_kernel(const Params p, int64_t rows, double inv_width) {
  constexpr int kWarps = kThreads / 32;
  __shared__ double red[5][kWarps];
  const int64_t r = kWarps == 1 ? blockIdx.x * static_cast<int64_t>(kRowsOf<kThreads>) + (threadIdx.x >> 5) : blockIdx.x;
  if (kWarps == 1 && r >= rows) return;
  const int64_t b = r / p.seq, s = r - b * p.seq;
  const int lane = kWarps == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int left = p.width - lane;  // value j exists while j * kThreads < left
  const float* y = static_cast<const float*>(p.y) + b * p.yb + s * p.ys + lane;
  const float* x = static_cast<const float*>(p.x) + b * p.xb + s * p.xs + lane;
  double v[kValues];
#pragma unroll
  for (int j = 0; j < kValues; ++j) {
    v[j] = j * kThreads < left ? __ldg(y + j * kThreads) : 0.f;
  }
  int64_t t = 0;
  bool known = true;
  if (p.idx) {
    t = __ldg(p.idx + b * p.idx_batch + s);
    known = t >= 0 && t < p.table_rows;
    if (!known) t = 0;
  }
  const float* gate = static_cast<const float*>(p.gate) + t * p.ldg + lane;
  const float* scale = static_cast<const float*>(p.scale) + t * p.lds + lane;
  const float* shift = static_cast<const float*>(p.shift) + t * p.ldsh + lane;
  // every reduction has its own slots, as in the vector form
  auto sum = [&](double a, int slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if constexpr (kWarps > 1) {
      if ((threadIdx.x & 31) == 0) red[slot][threadIdx.x >> 5] = a;
      __syncthreads();
      a = 0.0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) a += red[slot][i];
    }
    return a;
  };
  // The norm without its last factor, which it returns: 1 / deviation.
  auto centred = [&](int kind, int slot) {
    if (kind == kNone) return 1.0;
    double acc = 0.0;
    if (kind == kLayer) {
#pragma unroll
      for (int j = 0; j < kValues; ++j)
        if (j * kThreads < left) acc += v[j];
      const double mean = sum(acc, slot) * inv_width;
      acc = 0.0;
#pragma unroll
      for (int j = 0; j < kValues; ++j) v[j] -= mean;
    }
#pragma unroll
    for (int j = 0; j < kValues; ++j)
      if (j * kThreads < left) acc = fma(v[j], v[j], acc);
    return rsqrt(fma(sum(acc, slot + 1), inv_width, static_cast<double>(p.eps)));
  };
  double rstd = centred(p.post, 0);
  if (p.gate && !known) rstd = CUDART_NAN;
  float* x_out = static_cast<float*>(p.x_out) + r * p.width + lane;
#pragma unroll
  for (int j = 0; j < kValues; ++j) {
    if (j * kThreads >= left) continue;
    v[j] *= rstd;
    if (p.post_weight) v[j] *= __ldg(static_cast<const float*>(p.post_weight) + lane + j * kThreads);
    if (p.gate) v[j] *= __ldg(gate + j * kThreads);
    v[j] = fma(static_cast<double>(p.residual_scale), v[j], static_cast<double>(__ldg(x + j * kThreads)));
    x_out[j * kThreads] = static_cast<float>(v[j]);
  }
  rstd = centred(p.pre, 2);
  if (p.scale && !known) rstd = CUDART_NAN;
  unsigned long long top = 0;  // bits of the largest magnitude, so that a NaN stays one
#pragma unroll
  for (int j = 0; j < kValues; ++j) {
    if (j * kThreads >= left) continue;
    v[j] *= rstd;
    if (p.pre_weight) v[j] *= __ldg(static_cast<const float*>(p.pre_weight) + lane + j * kThreads);
    if (p.scale) v[j] = fma(v[j], 1.0 + __ldg(scale + j * kThreads), static_cast<double>(__ldg(shift + j * kThreads)));
    if (p.h_out) static_cast<float*>(p.h_out)[r * p.width + lane + j * kThreads] = static_cast<float>(v[j]);
    top = max(top, static_cast<unsigned long long>(__double_as_longlong(fabs(v[j]))));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if constexpr (kWarps > 1) {
    if ((threadIdx.x & 31) == 0) red[4][threadIdx.x >> 5] = __longlong_as_double(static_cast<long long>(top));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) top = max(top, static_cast<unsigned long long>(__double_as_longlong(red[4][i])));
  }
  const double most = p.quant == kInt8 ? 127.0 : 448.0;
  double sc = __longlong_as_double(static_cast<long long>(top)) / most;
  if (sc < FLT_MIN) sc = FLT_MIN;  // a NaN stays one
  const double inv = __drcp_rn(sc);
  if (lane == 0) p.code_scale[r] = static_cast<float>(sc);
  uint8_t* codes = p.codes + r * p.width + lane;
#pragma unroll
  for (int j = 0; j < kValues; ++j) {
    if (j * kThreads >= left) continue;
    // the correctly rounded quotient, as div_by; of at most `most` and a rounding
    double q = v[j] * inv;
    q = fma(fma(q, -sc, v[j]), inv, q);
    codes[j * kThreads] = p.quant == kInt8 ? static_cast<uint8_t>(__double2int_rn(q)) : f32_to_e4m3(static_cast<float>(q));
  }
}

template <int kThreads, int kValues>
int launch_codes64(const Params& p, int64_t rows, cudaStream_t st) {
  constexpr int kBlockRows = kRowsOf<kThreads>;
  sandwich_norm_codes64_kernel<kThreads, kValues>
      <<<static_cast<unsigned>(cdiv(rows, kBlockRows)), kThreads * kBlockRows, 0, st>>>(p, rows, 1.0 / p.width);
  return launch_status();
}

int pick_codes64(const Params& p, int64_t rows, cudaStream_t st) {
  if (p.width <= 256) return launch_codes64<32, 8>(p, rows, st);
  if (p.width <= 512) return launch_codes64<32, 16>(p, rows, st);
  if (p.width <= 1024) return launch_codes64<64, 16>(p, rows, st);
  if (p.width <= 2048) return launch_codes64<128, 16>(p, rows, st);
  if (p.width <= 4096) return launch_codes64<256, 16>(p, rows, st);
  if (p.width <= 8192) return launch_codes64<512, 16>(p, rows, st);
  return launch_codes64<1024, 16>(p, rows, st);
}

template <typename T, int kThreads, int kChunks>
int launch_vec(const Params& p, int64_t rows, cudaStream_t st) {
  constexpr int kBlockRows = kRowsOf<kThreads>;
  sandwich_norm_vec_kernel<T, kThreads, kChunks><<<static_cast<unsigned>(cdiv(rows, kBlockRows)), kThreads * kBlockRows, 0, st>>>(
      p, static_cast<uint32_t>(rows), make_fastdiv(static_cast<uint32_t>(p.seq)));
  return launch_status();
}

// The fewest threads that hold a row at up to four pieces a thread. Few rows,
// which leave the GPU's threads idle: a piece a thread (64 rows of 1536: 3.6
// us, with three pieces 5.3 us; at 8,704 rows 25 and 21 us).
template <typename T>
int pick_vec(const Params& p, int64_t rows, cudaStream_t st) {
  const int chunks = p.width / 8;
  if (rows <= 2 * 148 && chunks > 32 && chunks <= 1024) {
    if (chunks <= 64) return launch_vec<T, 64, 1>(p, rows, st);
    if (chunks <= 128) return launch_vec<T, 128, 1>(p, rows, st);
    if (chunks <= 192) return launch_vec<T, 192, 1>(p, rows, st);
    if (chunks <= 256) return launch_vec<T, 256, 1>(p, rows, st);
    if (chunks <= 384) return launch_vec<T, 384, 1>(p, rows, st);
    if (chunks <= 640) return launch_vec<T, 640, 1>(p, rows, st);
    return launch_vec<T, 1024, 1>(p, rows, st);
  }
  if (chunks <= 32) return launch_vec<T, 32, 1>(p, rows, st);
  if (chunks <= 64) return launch_vec<T, 32, 2>(p, rows, st);
  if (chunks <= 128) return launch_vec<T, 32, 4>(p, rows, st);
  if (chunks <= 192) return launch_vec<T, 64, 3>(p, rows, st);
  if (chunks <= 256) return launch_vec<T, 64, 4>(p, rows, st);
  if (chunks <= 384) return launch_vec<T, 96, 4>(p, rows, st);
  if (chunks <= 512) return launch_vec<T, 128, 4>(p, rows, st);
  if (chunks <= 640) return launch_vec<T, 160, 4>(p, rows, st);
  if (chunks <= 768) return launch_vec<T, 192, 4>(p, rows, st);
  if (chunks <= 1024) return launch_vec<T, 256, 4>(p, rows, st);
  if (chunks <= 1536) return launch_vec<T, 384, 4>(p, rows, st);
  return launch_vec<T, 512, 4>(p, rows, st);
}

template <typename T>
int launch(const Params& p, int64_t rows, cudaStream_t st) {
  if (sizeof(T) == 4 && p.codes) return pick_codes64(p, rows, st);
  const auto whole = [](const void* q, int64_t strides) {  // 16-byte pieces
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && strides * static_cast<int64_t>(sizeof(T)) % 16 == 0;
  };
  if (p.width % 8 == 0 && whole(p.y, p.yb | p.ys) && whole(p.x, p.xb | p.xs) && whole(p.post_weight, 0) &&
      whole(p.pre_weight, 0) && whole(p.gate, p.ldg) && whole(p.scale, p.lds) && whole(p.shift, p.ldsh) &&
      whole(p.x_out, 0) && whole(p.h_out, 0) && whole(p.codes, 0))
    return pick_vec<T>(p, rows, st);
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
