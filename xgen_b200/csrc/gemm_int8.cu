// Linear layer in 8-bit integers on sm_100a tensor cores, scales for each
// token and output channel:
//
//   y[m, n]  = (sum_k a[m, k] w[n, k]) * (sa[m] * sw[n]) + bias[n]
//   out      = y | gelu(y) | silu(y[:, :N/2]) * y[:, N/2:] | residual + gate[idx[m]] * y
//
// a [M, K] and w [N, K] int8 row-major. The sum is exact (tcgen05 kind::i8,
// 32-bit integers: K <= 131056 keeps 128 * 128 * K below 2^31); it becomes a
// 32-bit float once, the epilogue stays in 32 bits and the output is rounded
// once to bf16 or fp16.
//
// Persistent kernel, one CTA per SM, tiles of 128 x 256 (M x N), K blocks of
// 128 bytes:
//   warp 0     TMA producer (A 16 KB + W 32 KB per stage, 4 stages)
//   warp 1     TMEM allocator + MMA issuer (4 x M128 N256 K32 per stage)
//   warps 2-9  epilogue: one thread per output row (TMEM lane) and column half
// Two TMEM accumulators (2 x 256 columns) let the epilogue of one tile run
// under the MMAs of the next. A W tile is loaded as two boxes of 128 rows, so
// the gate and value rows of one SwiGLU tile come from their two places in a
// plain [gate | value] weight. Every mbarrier wait is bounded.
//
// The quantiser reads a row once into registers, takes its largest magnitude
// and divides by the scale with one rounding; it is bound by HBM.
#include <math_constants.h>

#include <algorithm>
#include <cfloat>

#include "sm100.cuh"
#include "tma_host.h"

namespace xgb {
namespace int8 {

using namespace sm100;

constexpr int kBM = 128;
constexpr int kBN = 256;
constexpr int kBK = 128;  // bytes of K per stage
constexpr int kStages = 4;
constexpr int kThreads = 320;
constexpr int kEpiThreads = 256;
constexpr int kABytes = kBM * kBK;
constexpr int kBBytes = kBN * kBK;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kBarOff = kStages * kStageBytes;
constexpr int kSmem = kBarOff + 256 + 1024;
constexpr uint32_t kIdesc = instr_desc(2, 1, 1, false, false, kBM, kBN);
constexpr int64_t kMaxK = 131056;

enum Epilogue : int { kPlain = 0, kGeluErf = 1, kGeluTanh = 2, kSwiGLU = 3, kGated = 4 };

__device__ __forceinline__ float gelu_erf(float y) { return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f)); }
__device__ __forceinline__ float gelu_tanh(float y) {
  return 0.5f * y * (1.0f + tanhf(0.79788456080286536f * (y + 0.044715f * y * y * y)));
}
__device__ __forceinline__ float swiglu(float g, float v) { return __fdividef(g, 1.0f + __expf(-g)) * v; }

template <typename T>
struct Params {
  int M, N, K;
  const float* sa;
  const float* sw;
  const T* bias;  // may be null
  T* out;
  int64_t ldo;
  // gated epilogue
  const T* gate;
  int64_t ldg;
  const int64_t* idx;  // table row of each output row, repeated every idx_rows
  int idx_rows;
  int64_t table_rows;
  const T* residual;
  int64_t ldr;
  int* err;
  bool vec;  // bias, gate and residual may be read 16 bytes at a time (host-checked)
};

struct Barriers {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t end;
  uint32_t tmem_base;
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void unpack8(const __nv_bfloat16*, const uint4& raw, float (&f)[8]) { unpack_bf16x8(raw, f); }
__device__ __forceinline__ void unpack8(const __half*, const uint4& raw, float (&f)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
// Eight entries of a row of the tensor's type; `vec` says that the place is
// 16-byte aligned, `left` how many exist.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int left, float (&f)[8]) {
  if (vec && left >= 8) {
    unpack8(p, __ldg(reinterpret_cast<const uint4*>(p)), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < left ? load_as_float(p + i) : 0.f;
  }
}
__device__ __forceinline__ void load8(const float* p, int left, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = i < left ? __ldg(p + i) : 0.f;
}
template <typename T>
__device__ __forceinline__ void scaled8(const Params<T>& p, const uint32_t* acc, float sa, int n, int left, float (&y)[8]) {
  float sw[8], bias[8];
  load8(p.sw + n, left, sw);
  if (p.bias) {
    load8(p.bias + n, p.vec, left, bias);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) bias[i] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fmaf(__int2float_rn(static_cast<int>(acc[i])), sa * sw[i], bias[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* dst, int left, const float (&y)[8]) {
  const uint32_t w[4] = {pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7])};
  if (left >= 8) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    const T* wb = reinterpret_cast<const T*>(w);
    for (int i = 0; i < left; ++i) dst[i] = wb[i];
  }
}

// One accumulator tile's epilogue for the output row `m` this thread owns and
// the column half `half`; n0 = first W row of the tile (SwiGLU: first gate row
// and output column, its values N/2 further).
template <typename T, int kEpi>
__device__ __forceinline__ void epilogue_tile(const Params<T>& p, uint32_t acc, int m, int n0, int half) {
  const bool row_ok = m < p.M;
  const float sa = row_ok ? p.sa[m] : 0.f;
  const int width = kEpi == kSwiGLU ? p.N / 2 : p.N;
  int64_t grow = 0;
  bool known = true;
  if (kEpi == kGated && row_ok) {
    grow = p.idx[m % p.idx_rows];
    known = grow >= 0 && grow < p.table_rows;
    if (!known) grow = 0;
  }
  T* dst = p.out + static_cast<int64_t>(m) * p.ldo;
  constexpr int kChunks = kEpi == kSwiGLU ? 2 : 4;  // 32 output columns each
#pragma unroll 1
  for (int c = half * kChunks; c < (half + 1) * kChunks; ++c) {
    uint32_t r[32], rv[kEpi == kSwiGLU ? 32 : 1];
    tmem_ld32(acc + c * 32, r);
    if constexpr (kEpi == kSwiGLU) tmem_ld32(acc + kBN / 2 + c * 32, rv);
    tmem_ld_wait();
    if (!row_ok) continue;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int n = n0 + c * 32 + g * 8;
      const int left = width - n;
      if (left <= 0) break;
      float y[8];
      scaled8(p, r + 8 * g, sa, n, left, y);
      if constexpr (kEpi == kSwiGLU) {
        float v[8];
        scaled8(p, rv + 8 * g, sa, n + width, left, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = swiglu(y[i], v[i]);
      }
      if constexpr (kEpi == kGated) {
        float gt[8], res[8];
        load8(p.gate + grow * p.ldg + n, p.vec, left, gt);
        load8(p.residual + static_cast<int64_t>(m) * p.ldr + n, p.vec, left, res);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = fmaf(known ? gt[i] : CUDART_NAN_F, y[i], res[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kEpi == kGeluErf) y[i] = gelu_erf(y[i]);
        if constexpr (kEpi == kGeluTanh) y[i] = gelu_tanh(y[i]);
      }
      store8(dst + n, left, y);
    }
  }
}

template <typename T, int kEpi>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_int8_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const Params<T> p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Barriers* bars = reinterpret_cast<Barriers*>(smem + kBarOff);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // W rows of a tile: two boxes of 128; SwiGLU tiles cover 128 gate rows and
  // their 128 value rows.
  constexpr int kCols = kEpi == kSwiGLU ? kBN / 2 : kBN;
  const int width = kEpi == kSwiGLU ? p.N / 2 : p.N;
  const int second = kEpi == kSwiGLU ? width : kBN / 2;
  const int m_tiles = (p.M + kBM - 1) / kBM;
  const int n_tiles = (width + kCols - 1) / kCols;
  const int64_t tiles = static_cast<int64_t>(m_tiles) * n_tiles;
  const int k_blocks = (p.K + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&bars->acc_full[a], 1);
      mbar_init(&bars->acc_empty[a], kEpiThreads);
    }
    mbar_init(&bars->end, 1);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc<512>(&bars->tmem_base);
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&a_map);
    prefetch_tmap(&b_map);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      bool ok = true;
      int it = 0;
      for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const int m0 = static_cast<int>(t / n_tiles) * kBM;
        const int n0 = static_cast<int>(t % n_tiles) * kCols;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % kStages;
          if (it >= kStages) ok = mbar_wait(&bars->empty[s], ((it / kStages) - 1) & 1, p.err);
          if (!ok) break;
          uint8_t* st = smem + s * kStageBytes;
          mbar_arrive_expect_tx(&bars->full[s], kStageBytes);
          tma_load_2d(st, &a_map, &bars->full[s], kb * kBK, m0);
          tma_load_2d(st + kABytes, &b_map, &bars->full[s], kb * kBK, n0);
          tma_load_2d(st + kABytes + kBBytes / 2, &b_map, &bars->full[s], kb * kBK, n0 + second);
        }
      }
      // the last stages' copies must land before the CTA exits
      for (int j = max(0, it - kStages); j < it; ++j)
        mbar_wait(&bars->full[j % kStages], (j / kStages) & 1, p.err, 100000000ull);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      bool ok = true;
      int it = 0, lt = 0;
      for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++lt) {
        const int a = lt & 1;
        if (lt >= 2) ok = mbar_wait(&bars->acc_empty[a], ((lt >> 1) - 1) & 1, p.err);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + a * kBN;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % kStages;
          ok = mbar_wait(&bars->full[s], (it / kStages) & 1, p.err);
          if (!ok) break;
          tc_fence_after();
          const uint32_t as = smem_u32(smem + s * kStageBytes);
          const uint32_t bs = as + kABytes;
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k)
            mma_ss<Kind::kI8>(d, smem_desc_sw128(as + k * 32, 16, 1024), smem_desc_sw128(bs + k * 32, 16, 1024), kIdesc,
                              kb > 0 || k > 0);
          tc_commit(&bars->empty[s]);
        }
        if (!ok) break;
        tc_commit(&bars->acc_full[a]);
      }
      tc_commit(&bars->end);
      mbar_wait(&bars->end, 0, p.err, 100000000ull);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;      // TMEM lane quarter this warp may access
    const int half = (warp - 2) >> 2;  // column half of the tile
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    int lt = 0;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, ++lt) {
      const int a = lt & 1;
      const bool ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_full[a], (lt >> 1) & 1, p.err));
      if (!ok) break;
      tc_fence_after();
      const int m = static_cast<int>(t / n_tiles) * kBM + quarter * 32 + lane;
      const int n0 = static_cast<int>(t % n_tiles) * kCols;
      epilogue_tile<T, kEpi>(p, lane_addr + a * kBN, m, n0, half);
      tc_fence_before();
      mbar_arrive(&bars->acc_empty[a]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<512>(tmem);
  }
}

int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

template <typename T, int kEpi>
int launch(const void* a, const void* w, const Params<T>& p, cudaStream_t st) {
  CUtensorMap am, bm;
  const uint64_t adims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(p.M)};
  const uint64_t str[1] = {static_cast<uint64_t>(p.K)};
  const uint32_t box[2] = {kBK, 128};
  const uint64_t bdims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(p.N)};
  if (!make_tensor_map(&am, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, a, adims, str, box) ||
      !make_tensor_map(&bm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, w, bdims, str, box))
    return XGB_ERR_ALIGN;
  auto kernel = gemm_int8_kernel<T, kEpi>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
    return XGB_ERR_LAUNCH;
  const int cols = kEpi == kSwiGLU ? kBN / 2 : kBN;
  const int width = kEpi == kSwiGLU ? p.N / 2 : p.N;
  const int64_t tiles = cdiv(p.M, kBM) * cdiv(width, cols);
  const int grid = static_cast<int>(std::min<int64_t>(tiles, sm_count()));
  kernel<<<grid, kThreads, kSmem, st>>>(am, bm, p);
  return launch_status();
}

template <typename T>
int pick(int epilogue, const void* a, const void* w, const Params<T>& p, cudaStream_t st) {
  switch (epilogue) {
    case kPlain: return launch<T, kPlain>(a, w, p, st);
    case kGeluErf: return launch<T, kGeluErf>(a, w, p, st);
    case kGeluTanh: return launch<T, kGeluTanh>(a, w, p, st);
    case kSwiGLU: return launch<T, kSwiGLU>(a, w, p, st);
    default: return launch<T, kGated>(a, w, p, st);
  }
}

// ---------------------------------------------------------------- quantiser
// One block per row; the scale is max(amax / 127, FLT_MIN) and the codes the
// correctly rounded quotients, rounded to the nearest even integer. A row with
// a NaN or an infinity gets a scale that is not finite. The largest magnitude
// is the largest bit pattern without its sign, so a NaN is found too.
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float s = __fdiv_rn(__uint_as_float(top), 127.0f);
  return s < FLT_MIN ? FLT_MIN : s;
}
__device__ __forceinline__ uint32_t code_of(float v, float s, float inv) {
  return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(div_by(v, s, inv), -127.f), 127.f))) & 0xFFu;
}
__device__ __forceinline__ uint2 codes8(const float (&f)[8], float s, float inv) {
  uint32_t q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = code_of(f[e], s, inv);
  return make_uint2(q[0] | (q[1] << 8) | (q[2] << 16) | (q[3] << 24), q[4] | (q[5] << 8) | (q[6] << 16) | (q[7] << 24));
}

constexpr int kQuantThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_int8_kernel(const T* __restrict__ x, int64_t ldx, int cols,
                                                                      int8_t* __restrict__ out, float* __restrict__ scales) {
  __shared__ uint32_t red[kQuantThreads / 32];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  uint32_t top = 0;
  for (int c = threadIdx.x; c < cols; c += kQuantThreads) top = max(top, __float_as_uint(load_as_float(xr + c)) & 0x7FFFFFFFu);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  top = 0;
#pragma unroll
  for (int i = 0; i < kQuantThreads / 32; ++i) top = max(top, red[i]);
  const float s = scale_of(top), inv = __frcp_rn(s);
  if (threadIdx.x == 0) scales[row] = s;
  for (int c = threadIdx.x; c < cols; c += kQuantThreads)
    out[row * cols + c] = static_cast<int8_t>(code_of(load_as_float(xr + c), s, inv));
}

// Rows of 16-byte pieces that fit a block's registers (kChunks a thread): one
// read.
constexpr int kQuantVecThreads = 512;
template <typename T, int kChunks>
__global__ void __launch_bounds__(kQuantVecThreads) quantize_int8_vec_kernel(const T* __restrict__ x, int64_t ldx, int cols,
                                                                             int8_t* __restrict__ out,
                                                                             float* __restrict__ scales) {
  __shared__ uint32_t red[kQuantVecThreads / 32];
  const int64_t row = blockIdx.x;
  const uint4* xr = reinterpret_cast<const uint4*>(x + row * ldx);
  const int chunks = cols >> 3, warps = blockDim.x >> 5;
  uint4 raw[kChunks];
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int c = threadIdx.x + j * blockDim.x;
    raw[j] = c < chunks ? __ldg(xr + c) : make_uint4(0, 0, 0, 0);
  }
  // both types order their magnitudes as their bits
  uint32_t top2 = 0;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top2 = __vmaxu2(top2, w[i] & 0x7FFF7FFFu);
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, max(top2 & 0xFFFFu, top2 >> 16));
  if (warps > 1) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int i = 0; i < warps; ++i) top = max(top, red[i]);
  }
  const uint16_t bits = static_cast<uint16_t>(top);
  const float s = scale_of(__float_as_uint(load_as_float(reinterpret_cast<const T*>(&bits)))), inv = __frcp_rn(s);
  if (threadIdx.x == 0) scales[row] = s;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int c = threadIdx.x + j * blockDim.x;
    if (c >= chunks) continue;
    float f[8];
    unpack8(static_cast<const T*>(nullptr), raw[j], f);
    reinterpret_cast<uint2*>(out + row * cols)[c] = codes8(f, s, inv);
  }
}

template <typename T>
int quantize(const T* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* out, float* scales, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>(rows);
  const int n = static_cast<int>(cols);
  if (cols % 8 == 0 && cols <= kQuantVecThreads * 8 * 4 && ldx % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
      reinterpret_cast<uintptr_t>(out) % 8 == 0) {
    const int chunks = n / 8, k = chunks > 1024 ? 4 : chunks > 32 ? 2 : 1;
    const unsigned threads = static_cast<unsigned>(cdiv(cdiv(chunks, k), 32) * 32);
    if (k == 4) quantize_int8_vec_kernel<T, 4><<<grid, threads, 0, st>>>(x, ldx, n, out, scales);
    else if (k == 2) quantize_int8_vec_kernel<T, 2><<<grid, threads, 0, st>>>(x, ldx, n, out, scales);
    else quantize_int8_vec_kernel<T, 1><<<grid, threads, 0, st>>>(x, ldx, n, out, scales);
  } else {
    quantize_int8_kernel<<<grid, kQuantThreads, 0, st>>>(x, ldx, n, out, scales);
  }
  return launch_status();
}

}  // namespace int8
}  // namespace xgb

using namespace xgb;

XGB_API int xgb_int8_quantize_per_token(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                        int8_t* out, float* scales, void* stream) {
  if (!x || !out || !scales) return XGB_ERR_ARG;
  if (dtype != XGB_BF16 && dtype != XGB_F16) return XGB_ERR_ARG;
  if (rows < 0 || rows > INT32_MAX || cols <= 0 || cols > INT32_MAX) return XGB_ERR_SHAPE;
  if (rows > 1 && row_stride < cols) return XGB_ERR_STRIDE;
  if (rows == 0) return XGB_OK;
  cudaStream_t st = as_stream(stream);
  return dtype == XGB_BF16
             ? int8::quantize(static_cast<const __nv_bfloat16*>(x), row_stride, rows, cols, out, scales, st)
             : int8::quantize(static_cast<const __half*>(x), row_stride, rows, cols, out, scales, st);
}

template <typename T>
static int run_int8_gemm(const int8_t* a, const int8_t* w, int64_t M, int64_t N, int64_t K, const float* scale_a,
                         const float* scale_w, const void* bias, int epilogue, void* out, int64_t ldo, const void* gate,
                         int64_t ldg, const int64_t* gate_index, int64_t index_rows, int64_t table_rows,
                         const void* residual, int64_t ldr, int* error_flag, cudaStream_t st) {
  int8::Params<T> p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.sa = scale_a;
  p.sw = scale_w;
  p.bias = static_cast<const T*>(bias);
  p.out = static_cast<T*>(out);
  p.ldo = ldo;
  p.gate = static_cast<const T*>(gate);
  p.ldg = ldg;
  p.idx = gate_index;
  p.idx_rows = static_cast<int>(index_rows);
  p.table_rows = table_rows;
  p.residual = static_cast<const T*>(residual);
  p.ldr = ldr;
  p.err = error_flag;
  const auto a16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
  p.vec = (!bias || a16(bias)) && (!gate || (a16(gate) && a16(residual) && ldg % 8 == 0 && ldr % 8 == 0));
  return int8::pick<T>(epilogue, a, w, p, st);
}

XGB_API int xgb_int8_gemm(const int8_t* a, const int8_t* w, int64_t M, int64_t N, int64_t K, const float* scale_a,
                          const float* scale_w, int dtype, const void* bias, int activation, void* out, int64_t ldo,
                          const void* gate, int64_t ldg, const int64_t* gate_index, int64_t index_rows, int64_t table_rows,
                          const void* residual, int64_t ldr, int* error_flag, void* stream) {
  if (!a || !w || !scale_a || !scale_w || !out) return XGB_ERR_ARG;
  if (dtype != XGB_BF16 && dtype != XGB_F16) return XGB_ERR_ARG;
  if (M <= 0 || N <= 0 || K <= 0 || M > INT32_MAX - 256 || N > INT32_MAX - 512 || K > int8::kMaxK) return XGB_ERR_SHAPE;
  if (K % 16 || N % 16) return XGB_ERR_SHAPE;  // 16-byte TMA rows and output vectors
  if (activation < 0 || activation > 3) return XGB_ERR_ARG;
  const bool swiglu = activation == 3, gated = gate != nullptr;
  if (gated && (activation != 0 || !gate_index || !residual || index_rows <= 0 || index_rows > INT32_MAX ||
                M % index_rows || table_rows <= 0))
    return XGB_ERR_ARG;
  if (ldo < (swiglu ? N / 2 : N) || ldo % 8 || (gated && (ldg < N || ldr < N))) return XGB_ERR_STRIDE;
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) & 15u)
    return XGB_ERR_ALIGN;
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10)
    return XGB_ERR_DEVICE;
  const int epilogue = gated ? int8::kGated : activation;
  const auto run = dtype == XGB_BF16 ? run_int8_gemm<__nv_bfloat16> : run_int8_gemm<__half>;
  return run(a, w, M, N, K, scale_a, scale_w, bias, epilogue, out, ldo, gate, ldg, gate_index, index_rows, table_rows,
             residual, ldr, error_flag, as_stream(stream));
}
