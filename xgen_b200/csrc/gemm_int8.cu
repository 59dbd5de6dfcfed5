// Linear layer in 8-bit integers on sm_100a tensor cores, scales for each
// token and output channel:
//
//   y[m, n]  = (sum_k a[m, k] w[n, k]) * (sa[m] * sw[n]) + bias[n]
//   out      = y | gelu(y) | silu(y[:, :N/2]) * y[:, N/2:] | residual + gate[idx[m]] * y
//
// a [M, K] and w [N, K] int8 row-major. The sum is exact (32-bit integers:
// K <= 131056 keeps 128 * 128 * K below 2^31); it becomes a 32-bit float once,
// the epilogue stays in 32 bits and the output is rounded once to bf16 or fp16.
//
// Three forms, picked by sizes (see pick_form and run_few):
//   few tokens   bound by reading w once: warp-level products, below
//   CTA pairs    bound by the tensor cores: tcgen05 kind::i8, 256 x kBN tiles
//   single CTAs  tiles of 128 x kBN, where they fill the SMs better
// The tiled kernels are persistent, K blocks of 128 bytes:
//   warp 0     TMA producer
//   warp 1     TMEM allocator + MMA issuer (of rank 0 in a pair)
//   warps 2-9  epilogue: one thread per output row (TMEM lane); warps 2-5 and
//              6-9 each half of a tile's columns, or every other narrow tile
// Two TMEM accumulators let the epilogue of one tile run under the MMAs of the
// next. A thread's row is 64 columns of shared memory at a time: the residual
// comes in there by TMA ahead of the accumulators, the result takes its place
// and leaves by TMA. (With rows read and written by their threads directly,
// 32 lanes on 32 lines each, the gated epilogue took 98 us at 15845 x 2048 x
// 2048 where the products need 40.) A W tile is two boxes of kBN/2 rows (in a pair, one of each CTA), so
// the gate and value rows of a SwiGLU tile come from their two places in a
// plain [gate | value] weight. Every mbarrier wait is bounded.
//
// The quantiser reads a row once into registers, takes its largest magnitude
// and divides by the scale with one rounding; it is bound by HBM.
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <type_traits>

#include "sm100.cuh"
#include "tma_host.h"

namespace xgb {
namespace int8 {

using namespace sm100;

constexpr int kBM = 128;  // A rows of a CTA
constexpr int kBK = 128;  // bytes of K per stage
constexpr int kThreads = 320;
constexpr int kEpiThreads = 256;
constexpr int kABytes = kBM * kBK;
constexpr int64_t kMaxK = 131056;
constexpr int kRaster = 8;  // row tiles that a group of consecutive tiles shares

constexpr int kChunk = 64;                    // output columns of a step of the epilogue
constexpr int kChunkBytes = 32 * kChunk * 2;  // a warp's 32 rows of them
constexpr int kOutBytes = kEpiThreads / 32 * 2 * kChunkBytes;  // two steps of every epilogue warp
constexpr int kGroupCols = 128;                  // accumulator columns that a warpgroup takes of a tile, at most
constexpr int kColBytes = kGroupCols * (4 + 2);  // their scales and biases
constexpr int kGroupBar = 1;                     // named barriers 1, 2: an epilogue warpgroup

// Shared memory of a CTA: per stage 128 rows of A and kBN (single) or kBN/2
// (pair) rows of W; as many stages as fit.
template <int kBN, bool kPair>
struct Cfg {
  static constexpr int kBoxRows = kBN / 2;
  static constexpr int kBoxBytes = kBoxRows * kBK;
  static constexpr int kStageBytes = kABytes + (kPair ? 1 : 2) * kBoxBytes;
  static constexpr int kStages = (224 * 1024 - kOutBytes) / kStageBytes < 8 ? (224 * 1024 - kOutBytes) / kStageBytes : 8;
  static constexpr int kOutOff = kStages * kStageBytes;
  static constexpr int kColOff = kOutOff + kOutBytes;
  static constexpr int kBarOff = kColOff + 2 * kColBytes;
  static constexpr int kSmem = kBarOff + 512 + 1024;
  static constexpr uint32_t kIdesc = instr_desc(2, 1, 1, false, false, kPair ? 2 * kBM : kBM, kBN);
  static constexpr uint32_t kTmemCols = 2 * kBN;
};

enum Epilogue : int { kPlain = 0, kGeluErf = 1, kGeluTanh = 2, kSwiGLU = 3, kGated = 4 };

__device__ __forceinline__ float gelu_erf(float y) { return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f)); }
// 0.5 (1 + tanh u) = 1 / (1 + e^-2u)
__device__ __forceinline__ float gelu_tanh(float y) {
  return __fdividef(y, 1.0f + __expf(-1.5957691216057308f * (y + 0.044715f * y * y * y)));
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
  bool vec;  // gate and residual may be read 16 bytes at a time (host-checked)
  bool behind_quantiser;  // launched behind the quantiser of its codes (see wait_for_quantiser)
};

struct Barriers {
  uint64_t full[8];
  uint64_t empty[8];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t end;
  uint64_t residual[kEpiThreads / 32][2];
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
// Eight entries of a row of the tensor's type (widths are multiples of 8);
// `vec` says that the place is 16-byte aligned.
template <typename T>
__device__ __forceinline__ uint4 load_raw8(const T* p, bool vec) {
  if (vec) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = __ldg(reinterpret_cast<const uint16_t*>(p) + 2 * i);
    w[i] = lo | static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(p) + 2 * i + 1)) << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Scaled and biased values of eight columns, whose scales and biases a
// warpgroup keeps in shared memory (every thread reads the same ones).
template <typename T>
__device__ __forceinline__ void scaled8(const uint32_t* acc, float sa, const float* sw, const T* bias, float (&y)[8]) {
  float s[8], b[8];
  const float4 lo = reinterpret_cast<const float4*>(sw)[0], hi = reinterpret_cast<const float4*>(sw)[1];
  s[0] = lo.x; s[1] = lo.y; s[2] = lo.z; s[3] = lo.w;
  s[4] = hi.x; s[5] = hi.y; s[6] = hi.z; s[7] = hi.w;
  unpack8(bias, *reinterpret_cast<const uint4*>(bias), b);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fmaf(__int2float_rn(static_cast<int>(acc[i])), sa * s[i], b[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&y)[8]) {
  return make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7]));
}

// Gate values of a thread's row for one step, requested ahead of it.
template <int kEpi>
struct Gates {
  uint4 raw[kEpi == kGated ? kChunk / 8 : 1];
  template <typename T>
  __device__ __forceinline__ void load(const Params<T>& p, const T* gate, int n1, int width) {
    if constexpr (kEpi == kGated) {
#pragma unroll
      for (int g = 0; g < kChunk / 8; ++g)
        if (n1 + 8 * g < width) raw[g] = load_raw8(gate + n1 + 8 * g, p.vec);
    }
  }
};

// An epilogue warp's walk over its steps of 32 rows x 64 columns.
template <typename T, int kBN, int kEpi>
struct Steps {
  static constexpr int kCols = kEpi == kSwiGLU ? kBN / 2 : kBN;
  static constexpr bool kHalves = kCols >= 2 * kChunk;  // both warpgroups on each tile; else on every other one
  static constexpr int kSteps = kHalves ? kCols / 2 / kChunk : 1;

  const Params<T>& p;
  const CUtensorMap* out_map;
  const CUtensorMap* res_map;
  uint8_t* buf;       // two steps
  uint64_t* arrived;  // residual of each
  const float* sw;    // scales and biases of the group's columns (SwiGLU: 64 gate, 64 value)
  const T* bias;
  int lane;
  int used = 0;     // steps so far
  int fetched = 0;  // of them requested

  __device__ __forceinline__ int width() const { return kEpi == kSwiGLU ? p.N / 2 : p.N; }

  // Requests the residual of a tile's steps, n1 = first column, m1 = first row.
  __device__ __forceinline__ void fetch(int n1, int m1) {
    if constexpr (kEpi == kGated) {
      if (!p.vec || lane != 0) return;
      bulk_wait_read<0>();  // earlier results have left the buffers
      for (int i = 0; i < kSteps && n1 + i * kChunk < width(); ++i, ++fetched) {
        const int b = fetched & 1;
        mbar_arrive_expect_tx(&arrived[b], kChunkBytes);
        tma_load_2d(buf + b * kChunkBytes, res_map, &arrived[b], n1 + i * kChunk, m1);
      }
    }
  }

  // After a failed wait: requested residuals still land before the CTA exits.
  __device__ __forceinline__ void drain() {
    for (; used < fetched; ++used) mbar_wait(&arrived[used & 1], (used >> 1) & 1, p.err, 100000000ull);
  }

  // One step: accumulators at `acc`, output columns n1.., rows m1 + lane.
  // `free` is called when the accumulators have been read.
  // `c` is the step's first column of the group, `gates` its gate values on
  // entry and the next step's on return.
  template <typename Free>
  __device__ __forceinline__ bool step(uint32_t acc, int c, int n1, int m1, float sa, const T* gate, bool known,
                                       Gates<kEpi>& gates, Free free) {
    // SwiGLU takes its two accumulators 32 columns at a time, for registers (168;
    // pairs still spill 4 bytes, single CTAs 28)
    uint32_t r[2][32], rv[kEpi == kSwiGLU ? 32 : 1];
    if constexpr (kEpi == kSwiGLU) {
      tmem_ld32(acc, r[0]);
      tmem_ld32(acc + kBN / 2, rv);
    } else {
      tmem_ld64(acc, r);
    }
    const int b = used & 1, m = m1 + lane;
    uint8_t* row = buf + b * kChunkBytes + lane * kChunk * 2;
    bool ok = true;
    if constexpr (kEpi == kGated) {
      if (p.vec) {
        ok = __all_sync(0xffffffffu, mbar_wait(&arrived[b], (used >> 1) & 1, p.err));
      } else {
        if (lane == 0) bulk_wait_read<1>();
        __syncwarp();
      }
    } else {
      if (lane == 0) bulk_wait_read<1>();
      __syncwarp();
    }
    ++used;
    tmem_ld_wait();
    if (kEpi != kSwiGLU) free();
    if (!ok) return false;
#pragma unroll
    for (int g = 0; g < kChunk / 8; ++g) {
      if (kEpi == kSwiGLU && g == 4) {
        tmem_ld32(acc + 32, r[0]);
        if constexpr (kEpi == kSwiGLU) tmem_ld32(acc + kBN / 2 + 32, rv);
        tmem_ld_wait();
        free();
      }
      const int n = n1 + g * 8;
      if (n >= width()) continue;
      uint4* place = reinterpret_cast<uint4*>(row + ((g ^ (lane & 7)) << 4));  // 128-byte swizzle
      float y[8];
      scaled8<T>(&r[kEpi == kSwiGLU ? 0 : g >> 2][(g & 3) * 8], sa, sw + c + 8 * g, bias + c + 8 * g, y);
      if constexpr (kEpi == kSwiGLU) {
        float v[8];
        scaled8<T>(&rv[(g & 3) * 8], sa, sw + kChunk + 8 * g, bias + kChunk + 8 * g, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = swiglu(y[e], v[e]);
      }
      if constexpr (kEpi == kGated) {
        float gt[8], res[8];
        unpack8(p.gate, gates.raw[g], gt);
        if (p.vec) unpack8(p.gate, *place, res);
        else unpack8(p.gate, load_raw8(p.residual + static_cast<int64_t>(min(m, p.M - 1)) * p.ldr + n, false), res);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(known ? gt[e] : CUDART_NAN_F, y[e], res[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (kEpi == kGeluErf) y[e] = gelu_erf(y[e]);
        if constexpr (kEpi == kGeluTanh) y[e] = gelu_tanh(y[e]);
      }
      *place = pack8<T>(y);
    }
    if (kSteps > 1) gates.load(p, gate, n1 + kChunk, width());
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(out_map, buf + b * kChunkBytes, n1, m1);
      bulk_commit();
    }
    return true;
  }
};

// The quantiser lets the product's kernel start once its last blocks run; the
// product sets up its barriers and TMEM meanwhile and waits here until the
// codes are complete. (No wait behind any other kernel.) Codes and scales are
// written while the product's kernel is there, so they are not read-only for it:
// they come by TMA and by plain loads, never by __ldg or a restrict pointer. 1.0
// to 1.5 us less at 16 to 300 tokens of 1536 channels.
__device__ __forceinline__ void wait_for_quantiser() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_product_start() { asm volatile("griddepcontrol.launch_dependents;"); }
inline void start_behind_quantiser(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr) {
  attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
}

// Tile t of the walk: groups of kRaster row tiles, columns within a group, so
// that tiles in flight share rows of A and of W in L2.
struct Walk {
  int m_tiles, n_tiles;
  __device__ __forceinline__ void at(int64_t t, int& m, int& n) const {
    const int64_t per_group = static_cast<int64_t>(kRaster) * n_tiles;
    const int64_t g = t / per_group;
    const int in = static_cast<int>(t - g * per_group);
    const int rows = min(kRaster, m_tiles - static_cast<int>(g) * kRaster);
    m = static_cast<int>(g) * kRaster + in % rows;
    n = in / rows;
  }
};

template <typename T, int kBN, int kEpi, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_int8_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map,
                     const __grid_constant__ CUtensorMap out_map, const __grid_constant__ CUtensorMap res_map,
                     const Params<T> p) {
  using C = Cfg<kBN, kPair>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Barriers* bars = reinterpret_cast<Barriers*>(smem + C::kBarOff);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = kPair ? static_cast<int>(cluster_rank()) : 0;
  const int64_t first = kPair ? blockIdx.x >> 1 : blockIdx.x, step = kPair ? gridDim.x >> 1 : gridDim.x;
  constexpr int kCols = Steps<T, kBN, kEpi>::kCols;  // output columns of a tile
  constexpr int kRowsOfTile = kPair ? 2 * kBM : kBM;
  const int width = kEpi == kSwiGLU ? p.N / 2 : p.N;
  const int second = kEpi == kSwiGLU ? width : kBN / 2;  // W rows from the first box to the second
  const Walk walk{(p.M + kRowsOfTile - 1) / kRowsOfTile, (width + kCols - 1) / kCols};
  const int64_t tiles = static_cast<int64_t>(walk.m_tiles) * walk.n_tiles;
  const int k_blocks = (p.K + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&bars->acc_full[a], 1);
      // every epilogue warp that reads the tile, of both CTAs of a pair
      mbar_init(&bars->acc_empty[a], (kPair ? 2 : 1) * (Steps<T, kBN, kEpi>::kHalves ? 8 : 4));
    }
    for (int e = 0; e < kEpiThreads / 32; ++e)
      for (int b = 0; b < 2; ++b) mbar_init(&bars->residual[e][b], 1);
    mbar_init(&bars->end, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (kPair) tmem_alloc_pair<C::kTmemCols>(&bars->tmem_base);
    else tmem_alloc<C::kTmemCols>(&bars->tmem_base);
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&a_map);
    prefetch_tmap(&b_map);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) cluster_sync();  // both CTAs' barriers exist
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  wait_for_quantiser();

  if (warp == 0) {
    // ------------------------------------------------------------ producer (each CTA its own rows)
    if (lane == 0) {
      bool ok = true;
      int it = 0;
      for (int64_t t = first; t < tiles && ok; t += step) {
        int mt, nt;
        walk.at(t, mt, nt);
        const int m0 = mt * kRowsOfTile + rank * kBM, n0 = nt * kCols;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % kStages;
          if (it >= kStages) ok = mbar_wait(&bars->empty[s], ((it / kStages) - 1) & 1, p.err);
          if (!ok) break;
          uint8_t* st = smem + s * C::kStageBytes;
          if constexpr (kPair) {
            // both CTAs' bytes are counted on rank 0's barrier
            const uint32_t full0 = map_to_rank(&bars->full[s], 0);
            if (rank == 0) mbar_arrive_expect_tx(&bars->full[s], 2 * C::kStageBytes);
            tma_load_2d_pair(st, &a_map, full0, kb * kBK, m0);
            tma_load_2d_pair(st + kABytes, &b_map, full0, kb * kBK, n0 + rank * second);
          } else {
            mbar_arrive_expect_tx(&bars->full[s], C::kStageBytes);
            tma_load_2d(st, &a_map, &bars->full[s], kb * kBK, m0);
            tma_load_2d(st + kABytes, &b_map, &bars->full[s], kb * kBK, n0);
            tma_load_2d(st + kABytes + C::kBoxBytes, &b_map, &bars->full[s], kb * kBK, n0 + second);
          }
        }
      }
      // The armed stages' copies must land before the CTA (the pair: rank 0's
      // barrier counts both CTAs' loads) exits.
      if (!kPair || rank == 0)
        for (int j = max(0, it - kStages); j < it; ++j)
          mbar_wait(&bars->full[j % kStages], (j / kStages) & 1, p.err, 100000000ull);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (rank 0)
    if (lane == 0 && rank == 0) {
      auto commit = [&](uint64_t* bar) {
        if constexpr (kPair) {
          tc_commit_pair(map_to_rank(bar, 0));
          tc_commit_pair(map_to_rank(bar, 1));
        } else {
          tc_commit(bar);
        }
      };
      bool ok = true;
      int it = 0, lt = 0;
      for (int64_t t = first; t < tiles && ok; t += step, ++lt) {
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
          const uint32_t as = smem_u32(smem + s * C::kStageBytes), bs = as + kABytes;
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k) {
            const uint64_t da = smem_desc_sw128(as + k * 32, 16, 1024), db = smem_desc_sw128(bs + k * 32, 16, 1024);
            if constexpr (kPair) mma_pair_i8(d, da, db, C::kIdesc, kb > 0 || k > 0);
            else mma_ss<Kind::kI8>(d, da, db, C::kIdesc, kb > 0 || k > 0);
          }
          commit(&bars->empty[s]);
        }
        if (!ok) break;
        commit(&bars->acc_full[a]);
      }
      commit(&bars->end);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    using S = Steps<T, kBN, kEpi>;
    const int quarter = warp & 3;       // TMEM lane quarter this warp may access
    const int group = (warp - 2) >> 2;  // column half, or parity of the tiles
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    float* sw = reinterpret_cast<float*>(smem + C::kColOff + group * kColBytes);
    T* bias = reinterpret_cast<T*>(sw + kGroupCols);
    S steps{p, &out_map, &res_map, smem + C::kOutOff + (warp - 2) * 2 * kChunkBytes, bars->residual[warp - 2], sw, bias, lane};
    // This thread's column of the group, of a tile; loaded a tile ahead.
    const int mine = threadIdx.x - 64 - group * 128;
    float next_sw = 0.f;
    T next_bias = T(0.f);
    auto load_column = [&](int64_t t) {
      if (t >= tiles) return;
      int mt, nt;
      walk.at(t, mt, nt);
      int n = nt * kCols + (S::kHalves ? group * (kCols / 2) : 0) + mine;
      bool there = n < width;
      if constexpr (kEpi == kSwiGLU) {  // 64 gate columns, then their values
        n -= mine & kChunk;
        there = n < width;
        n += mine & kChunk ? width : 0;
      }
      next_sw = there ? __ldg(p.sw + n) : 0.f;
      next_bias = there && p.bias ? p.bias[n] : T(0.f);
    };
    const int64_t skip = S::kHalves ? step : 2 * step, start = S::kHalves ? first : first + group * step;
    load_column(start);
    bool ok = true;
    int lt = S::kHalves ? 0 : group;
    for (int64_t t = start; t < tiles; t += skip, lt += S::kHalves ? 1 : 2) {
      const int a = lt & 1;
      int mt, nt;
      walk.at(t, mt, nt);
      const int c0 = S::kHalves ? group * (kCols / 2) : 0;  // column of the tile
      const int n1 = nt * kCols + c0, m1 = mt * kRowsOfTile + rank * kBM + quarter * 32, m = m1 + lane;
      named_sync(kGroupBar + group, 128);  // the last tile's columns have been used
      sw[mine] = next_sw;
      bias[mine] = next_bias;
      load_column(t + skip);
      named_sync(kGroupBar + group, 128);
      // After a failed wait the warps stay in step for these barriers and do
      // nothing else.
      if (!ok) continue;
      steps.fetch(n1, m1);
      const float sa = m < p.M ? p.sa[m] : 0.f;
      const T* gate = p.gate;
      bool known = true;
      Gates<kEpi> gates;
      if constexpr (kEpi == kGated) {
        const int64_t at = __ldg(p.idx + min(m, p.M - 1) % p.idx_rows);
        known = at >= 0 && at < p.table_rows;
        gate += (known ? at : 0) * p.ldg;
        gates.load(p, gate, n1, width);
      }
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_full[a], (lt >> 1) & 1, p.err));
      if (!ok) continue;
      tc_fence_after();
      // the last step that has columns frees the accumulators
      const int last = min(S::kSteps, (width - n1 + kChunk - 1) / kChunk) - 1;
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair) mbar_arrive_cluster(map_to_rank(&bars->acc_empty[a], 0));
          else mbar_arrive(&bars->acc_empty[a]);
        }
      };
      if (last < 0) release();  // this half lies outside the matrix
#pragma unroll 1
      for (int i = 0; i <= last && ok; ++i)
        ok = steps.step(lane_addr + a * kBN + c0 + i * kChunk, i * kChunk, n1 + i * kChunk, m1, sa, gate, known, gates, [&]() {
          if (i == last) release();
        });
    }
    if (lane == 0) {
      steps.drain();
      bulk_wait_all();  // the results have left
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    // every MMA, which in a pair reads both CTAs' shared memory, has ended
    mbar_wait(&bars->end, 0, p.err, 100000000ull);
    tc_fence_after();
    if constexpr (kPair) tmem_dealloc_pair<C::kTmemCols>(tmem);
    else tmem_dealloc<C::kTmemCols>(tmem);
  }
  if constexpr (kPair) cluster_sync();
}

int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

// Pairs that can be resident at once, measured once per kernel and device
// (stored as pairs + 1): a walk over more of them would wait for another pair
// to end.
template <typename Kernel>
int pair_slots(Kernel kernel, std::atomic<int>* cached, const cudaLaunchConfig_t& like, int sms) {
  constexpr int kMaxDevices = 64;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return sms / 2;
  const int known = cached[dev].load(std::memory_order_relaxed);
  if (known > 0) return known - 1;
  cudaLaunchConfig_t cfg = like;
  cfg.gridDim = dim3(2 * static_cast<unsigned>(sms));
  int pairs = 0;
  if (cudaOccupancyMaxActiveClusters(&pairs, kernel, &cfg) != cudaSuccess || pairs <= 0) {
    cudaGetLastError();
    return sms / 2;
  }
  pairs = std::min(pairs, sms / 2);
  cached[dev].store(pairs + 1, std::memory_order_relaxed);
  return pairs;
}

template <typename T, int kBN, int kEpi, bool kPair>
int launch(const void* a, const void* w, const Params<T>& p, cudaStream_t st) {
  using C = Cfg<kBN, kPair>;
  CUtensorMap am, bm;
  const uint64_t adims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(p.M)};
  const uint64_t str[1] = {static_cast<uint64_t>(p.K)};
  const uint32_t abox[2] = {kBK, kBM}, bbox[2] = {kBK, C::kBoxRows};
  const uint64_t bdims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(p.N)};
  if (!make_tensor_map(&am, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, a, adims, str, abox) ||
      !make_tensor_map(&bm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, w, bdims, str, bbox))
    return XGB_ERR_ALIGN;
  const int width = kEpi == kSwiGLU ? p.N / 2 : p.N;
  constexpr auto kType = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                                 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap om, rm;
  const uint64_t odims[2] = {static_cast<uint64_t>(width), static_cast<uint64_t>(p.M)};
  const uint32_t obox[2] = {kChunk, 32};
  const uint64_t ostr[1] = {static_cast<uint64_t>(p.ldo) * 2};
  if (!make_tensor_map(&om, kType, 2, p.out, odims, ostr, obox)) return XGB_ERR_ALIGN;
  rm = om;
  if (kEpi == kGated && p.vec) {
    const uint64_t rstr[1] = {static_cast<uint64_t>(p.ldr) * 2};
    if (!make_tensor_map(&rm, kType, 2, p.residual, odims, rstr, obox)) return XGB_ERR_ALIGN;
  }
  auto kernel = gemm_int8_kernel<T, kBN, kEpi, kPair>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess)
    return XGB_ERR_LAUNCH;
  const int cols = kEpi == kSwiGLU ? kBN / 2 : kBN, rows = kPair ? 2 * kBM : kBM;
  const int64_t tiles = cdiv(p.M, rows) * cdiv(width, cols);
  const int sms = sm_count();
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if constexpr (kPair) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
    static std::atomic<int> cached[64];
    cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<int64_t>(tiles, pair_slots(kernel, cached, cfg, sms))));
  } else {
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(tiles, sms)));
  }
  if (p.behind_quantiser) start_behind_quantiser(cfg, attr);
  if (cudaLaunchKernelEx(&cfg, kernel, am, bm, om, rm, p) != cudaSuccess) {
    cudaGetLastError();
    return XGB_ERR_LAUNCH;
  }
  return launch_status();
}

// The tile shape whose estimate is least: rounds of tiles over the SMs, each
// K block of a round, and what a launch and every further round add. The
// constants are fits to measured times on B200 (us; products alone), where
// the shapes take turns by size:
//                       pair 256x256   128x128   128x64
//   300 x 1600 x 256         7.5          5.1       4.4
//   1024 x 1536 x 1536      10.7          8.3      11.2
//   4352 x 1536 x 1536      15.9         17.1      26.6
//   128 x 16384 x 4096      17.5         14.5      22.6
//   15845 x 2048 x 2048     52.2         75.3     132.3
// An epilogue that does more than scale adds to a launch and to every round,
// most to the pairs, whose warps take 128 columns each.
// (Pairs on 256 x 128 tiles were slower than one of these at every size.)
enum Form { kPair256, kSingle128, kSingle64 };
inline Form pick_form(int64_t m, int64_t width, int64_t k, int epilogue, int sms) {
  struct Candidate {
    Form form;
    int rows, cols, slots;
    double start, block, round;
    double gated_start, gated_round, act_start, act_round;
  };
  const bool swiglu = epilogue == kSwiGLU;
  const int half = swiglu ? 2 : 1;  // a SwiGLU tile has half as many output columns
  const Candidate all[3] = {{kPair256, 256, 256 / half, sms / 2, 6.9, 0.31, 1.6, 4.5, 2.3, 2.8, 0.8},
                            {kSingle128, 128, 128 / half, sms, 4.5, 0.29, 1.0, 1.3, 0.0, 1.3, 0.4},
                            {kSingle64, 128, 64, sms, 3.8, 0.276, 0.6, 1.4, 0.3, 1.5, 0.4}};
  Form best = kSingle128;
  double least = 1e300;
  for (const Candidate& c : all) {
    if (c.form == kSingle64 && swiglu) continue;
    const double rounds = static_cast<double>(cdiv(cdiv(m, c.rows) * cdiv(width, c.cols), c.slots));
    double cost = c.start + rounds * cdiv(k, kBK) * c.block + (rounds - 1) * c.round;
    if (epilogue == kGated) cost += c.gated_start + (rounds - 1) * c.gated_round;
    else if (epilogue != kPlain) cost += c.act_start + (rounds - 1) * c.act_round;
    if (cost < least) {
      least = cost;
      best = c.form;
    }
  }
  return best;
}

template <typename T, int kEpi>
int launch_form(const void* a, const void* w, const Params<T>& p, cudaStream_t st) {
  const Form f = pick_form(p.M, kEpi == kSwiGLU ? p.N / 2 : p.N, p.K, kEpi, sm_count());
  if (f == kPair256) return launch<T, 256, kEpi, true>(a, w, p, st);
  if constexpr (kEpi != kSwiGLU)
    if (f == kSingle64) return launch<T, 64, kEpi, false>(a, w, p, st);
  return launch<T, 128, kEpi, false>(a, w, p, st);
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
// Eight codes, two values an instruction; |q| <= 127 and a rounding, and
// 1.5 * 2^23 + q has the nearest even integer in its low bits.
__device__ __forceinline__ uint2 codes8(const float (&f)[8], float s, float inv) {
  const float2 inv2 = make_float2(inv, inv), minus = make_float2(-s, -s), shift = make_float2(12582912.0f, 12582912.0f);
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = make_float2(f[2 * i], f[2 * i + 1]), q = __fmul2_rn(v, inv2);
    const float2 d = __fadd2_rn(__ffma2_rn(__ffma2_rn(q, minus, v), inv2, q), shift);
    h[i] = __byte_perm(__float_as_uint(d.x), __float_as_uint(d.y), 0x0040);
  }
  return make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
}

// ---------------------------------------------------------------- few tokens
// Up to 32 tokens: the time is that of reading w once, and a 128-row tile would
// be mostly empty. A CTA takes 16 rows of w (SwiGLU: 8 gate and their 8 value
// rows) for all tokens, its 8 warps share K in pieces of 64 bytes. A lane loads
// 16-byte pieces of rows g and g + 8 (g = lane / 4) straight into the fragments
// of the warp-level 16 x 8 x 32 products; their inner index is any order of k
// as long as the tokens' codes follow the same one, so the pieces need no
// rearranging. The integer sums of the warps meet in shared memory: the result
// does not depend on how K is shared. With kFused every CTA first quantises
// the tokens itself, a few thousand values, while its first rows of w are on
// their way: one launch instead of two; a warp a token (8 x 1536 -> 4608: 5.2
// us, with the whole CTA on each token in turn 8.4), up to 3 tokens the CTA.
constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewAhead = 3;        // pieces of a warp in flight
constexpr int kFewMost = 32;        // tokens
constexpr int64_t kFusedMost = 24576;  // values that every CTA quantises for itself

__device__ __forceinline__ void mma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// x: the tokens of a fused launch (rows ldx apart, 16-byte aligned pieces).
template <typename T, int kEpi, int kTokenTiles, bool kFused>
__global__ void __launch_bounds__(kFewThreads) few_int8_kernel(const int8_t* a, const int8_t* __restrict__ w,
                                                               const Params<T> p, const T* __restrict__ x, int64_t ldx) {
  constexpr int kTokens = 8 * kTokenTiles;
  __shared__ int part[kFewWarps][16][kTokens + 1];
  __shared__ uint32_t red[kFewWarps];
  __shared__ float scales[kTokens];
  extern __shared__ __align__(16) int8_t codes[];  // fused: [M][K + 64]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int width = kEpi == kSwiGLU ? p.N / 2 : p.N;
  const int n0 = blockIdx.x * (kEpi == kSwiGLU ? 8 : 16);
  // w rows of this lane; the last tile's missing ones read a row that exists
  const int8_t* w0 = w + static_cast<int64_t>(min(n0 + g, width - 1)) * p.K + 16 * c;
  const int8_t* w1 = w + static_cast<int64_t>(kEpi == kSwiGLU ? width + min(n0 + g, width - 1) : min(n0 + g + 8, width - 1)) * p.K + 16 * c;
  const int pieces = (p.K + 63) / 64;
  auto piece = [&](const int8_t* row, int j) {
    return 64 * j + 16 * c < p.K ? __ldg(reinterpret_cast<const uint4*>(row + 64 * j)) : make_uint4(0, 0, 0, 0);
  };
  uint4 r0[kFewAhead], r1[kFewAhead];
#pragma unroll
  for (int i = 0; i < kFewAhead; ++i) {
    const int j = warp + i * kFewWarps;
    r0[i] = j < pieces ? piece(w0, j) : make_uint4(0, 0, 0, 0);
    r1[i] = j < pieces ? piece(w1, j) : make_uint4(0, 0, 0, 0);
  }
  const int stride = p.K + 64;
  if constexpr (!kFused) {
    wait_for_quantiser();
  } else {
    if (p.M > 3) {  // a warp a token
      const int left = p.K / 8;
      for (int m = warp; m < p.M; m += kFewWarps) {
        const T* xr = x + m * ldx;
        uint32_t top = 0;
#pragma unroll 4
        for (int k = lane; k < left; k += 32) {
          float f[8];
          unpack8(xr, __ldg(reinterpret_cast<const uint4*>(xr) + k), f);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7FFFFFFFu);
        }
        const float s = scale_of(__reduce_max_sync(0xffffffffu, top)), inv = __frcp_rn(s);
        if (lane == 0) scales[m] = s;
#pragma unroll 4
        for (int k = lane; k < left; k += 32) {
          float f[8];
          unpack8(xr, __ldg(reinterpret_cast<const uint4*>(xr) + k), f);
          *reinterpret_cast<uint2*>(codes + m * stride + 8 * k) = codes8(f, s, inv);
        }
      }
      __syncthreads();
    } else {
      for (int m = 0; m < p.M; ++m) {
        const T* xr = x + m * ldx;
        uint32_t top = 0;
        for (int k = threadIdx.x; k < p.K / 8; k += kFewThreads) {
          float f[8];
          unpack8(xr, __ldg(reinterpret_cast<const uint4*>(xr) + k), f);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7FFFFFFFu);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) red[warp] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kFewWarps; ++i) top = max(top, red[i]);
        const float s = scale_of(top), inv = __frcp_rn(s);
        if (threadIdx.x == 0) scales[m] = s;
        for (int k = threadIdx.x; k < p.K / 8; k += kFewThreads) {
          float f[8];
          unpack8(xr, __ldg(reinterpret_cast<const uint4*>(xr) + k), f);
          *reinterpret_cast<uint2*>(codes + m * stride + 8 * k) = codes8(f, s, inv);
        }
        __syncthreads();
      }
    }
  }
  // codes of piece j, of token g of tile t
  auto of_token = [&](int j, int t) {
    const int m = 8 * t + g;
    if (m >= p.M || 64 * j + 16 * c >= p.K) return make_uint4(0, 0, 0, 0);
    return *reinterpret_cast<const uint4*>(kFused ? codes + m * stride + 64 * j + 16 * c
                                                  : a + static_cast<int64_t>(m) * p.K + 64 * j + 16 * c);
  };
  // From global memory they come a step ahead: 32 x 4096 -> 16384 28.5 us (in
  // their own step 44 us; as far ahead as w's, with 182 registers, 43 us).
  uint4 rb[kFused ? 1 : kTokenTiles];
  if constexpr (!kFused) {
#pragma unroll
    for (int t = 0; t < kTokenTiles; ++t) rb[t] = of_token(warp, t);
  }
  int acc[kTokenTiles][4] = {};
  for (int j0 = warp; j0 < pieces; j0 += kFewAhead * kFewWarps) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int j = j0 + i * kFewWarps;
      if (j >= pieces) break;
      const uint4 u = r0[i], v = r1[i];
      const int next = j + kFewAhead * kFewWarps;
      if (next < pieces) {
        r0[i] = piece(w0, next);
        r1[i] = piece(w1, next);
      }
#pragma unroll
      for (int t = 0; t < kTokenTiles; ++t) {
        uint4 b;
        if constexpr (kFused) {
          b = of_token(j, t);
        } else {
          b = rb[t];
          rb[t] = of_token(j + kFewWarps, t);
        }
        mma16832(acc[t], u.x, v.x, u.y, v.y, b.x, b.y);
        mma16832(acc[t], u.z, v.z, u.w, v.w, b.z, b.w);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kTokenTiles; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[warp][g + 8 * (e >> 1)][8 * t + 2 * c + (e & 1)] = acc[t][e];
  __syncthreads();
  constexpr int kOut = kEpi == kSwiGLU ? 8 : 16;  // output columns of the CTA
  for (int e = threadIdx.x; e < kOut * kTokens; e += kFewThreads) {
    const int m = e / kOut, r = e % kOut, n = n0 + r;
    if (m >= p.M || n >= width) continue;
    const float sa = kFused ? scales[m] : p.sa[m];
    auto value = [&](int row, int col) {
      int sum = 0;
#pragma unroll
      for (int i = 0; i < kFewWarps; ++i) sum += part[i][row][m];
      return fmaf(__int2float_rn(sum), sa * __ldg(p.sw + col), p.bias ? load_as_float(p.bias + col) : 0.f);
    };
    float y = value(r, n);
    if constexpr (kEpi == kGeluErf) y = gelu_erf(y);
    if constexpr (kEpi == kGeluTanh) y = gelu_tanh(y);
    if constexpr (kEpi == kSwiGLU) y = swiglu(y, value(r + 8, n + width));
    if constexpr (kEpi == kGated) {
      const int64_t at = __ldg(p.idx + m % p.idx_rows);
      const bool known = at >= 0 && at < p.table_rows;
      const float gt = known ? load_as_float(p.gate + at * p.ldg + n) : CUDART_NAN_F;
      y = fmaf(gt, y, load_as_float(p.residual + m * p.ldr + n));
    }
    const uint32_t packed = pack2<T>(y, 0.f);
    p.out[m * p.ldo + n] = *reinterpret_cast<const T*>(&packed);
  }
}

template <typename T, int kEpi, bool kFused>
int launch_few(const void* a, const void* w, const Params<T>& p, const T* x, int64_t ldx, cudaStream_t st) {
  const int8_t* ap = static_cast<const int8_t*>(a);
  const int8_t* wp = static_cast<const int8_t*>(w);
  const unsigned grid = static_cast<unsigned>(kEpi == kSwiGLU ? cdiv(p.N / 2, 8) : cdiv(p.N, 16));
  const size_t smem = kFused ? static_cast<size_t>(p.M) * (p.K + 64) : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  if (p.behind_quantiser) start_behind_quantiser(cfg, attr);
  const cudaError_t rc = p.M <= 8    ? cudaLaunchKernelEx(&cfg, few_int8_kernel<T, kEpi, 1, kFused>, ap, wp, p, x, ldx)
                         : p.M <= 16 ? cudaLaunchKernelEx(&cfg, few_int8_kernel<T, kEpi, 2, kFused>, ap, wp, p, x, ldx)
                                     : cudaLaunchKernelEx(&cfg, few_int8_kernel<T, kEpi, 4, kFused>, ap, wp, p, x, ldx);
  if (rc != cudaSuccess) {
    cudaGetLastError();
    return XGB_ERR_LAUNCH;
  }
  return launch_status();
}

// Tokens that a call may quantise within the product: little work, and codes
// (M * (K + 64) bytes, 26 KB at most) that fit beside the sums. One launch /
// two, in a graph and in an eager loop: 8 x 1536 -> 4608 5.2 / 4.7 us and 11.9
// / 16.7 us, 16 x 1536 -> 4608 7.4 / 5.2 and 11.8 / 16.7, 12 x 2048 -> 2048
// 6.5 / 5.3 and 11.9 / 16.7, 18 x 1280 -> 8192 12.9 / 8.5 and 14.4 / 16.6.
inline bool fuses(int64_t m, int64_t k) { return m <= kFewMost && m * k <= kFusedMost; }

// x: the tokens to quantise within the product (null: `a` and p.sa hold their
// codes and scales).
template <typename T, int kEpi>
int run(const void* a, const void* w, const Params<T>& p, const T* x, int64_t ldx, cudaStream_t st) {
  if (x) return launch_few<T, kEpi, true>(a, w, p, x, ldx, st);
  if (p.M <= kFewMost) return launch_few<T, kEpi, false>(a, w, p, x, ldx, st);
  return launch_form<T, kEpi>(a, w, p, st);
}

template <typename T>
int pick(int epilogue, const void* a, const void* w, const Params<T>& p, const T* x, int64_t ldx, cudaStream_t st) {
  switch (epilogue) {
    case kPlain: return run<T, kPlain>(a, w, p, x, ldx, st);
    case kGeluErf: return run<T, kGeluErf>(a, w, p, x, ldx, st);
    case kGeluTanh: return run<T, kGeluTanh>(a, w, p, x, ldx, st);
    case kSwiGLU: return run<T, kSwiGLU>(a, w, p, x, ldx, st);
    default: return run<T, kGated>(a, w, p, x, ldx, st);
  }
}

constexpr int kQuantThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_int8_kernel(const T* __restrict__ x, int64_t ldx, int cols,
                                                                      int8_t* __restrict__ out, float* __restrict__ scales) {
  __shared__ uint32_t red[kQuantThreads / 32];
  let_product_start();
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
  let_product_start();
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

namespace {

struct Call {
  const int8_t* a;
  const int8_t* w;
  int64_t M, N, K;
  const float* scale_a;
  const float* scale_w;
  int dtype;
  const void* bias;
  int activation;
  void* out;
  int64_t ldo;
  const void* gate;
  int64_t ldg;
  const int64_t* gate_index;
  int64_t index_rows, table_rows;
  const void* residual;
  int64_t ldr;
  int* error_flag;
  cudaStream_t st;
  bool behind_quantiser = false;
};

inline bool a16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

int check(const Call& c) {
  if (!c.w || !c.scale_w || !c.out) return XGB_ERR_ARG;
  if (c.dtype != XGB_BF16 && c.dtype != XGB_F16) return XGB_ERR_ARG;
  if (c.M <= 0 || c.N <= 0 || c.K <= 0 || c.M > INT32_MAX - 256 || c.N > INT32_MAX - 512 || c.K > int8::kMaxK)
    return XGB_ERR_SHAPE;
  if (c.K % 16 || c.N % 16) return XGB_ERR_SHAPE;  // 16-byte TMA rows and output vectors
  if (c.activation < 0 || c.activation > 3) return XGB_ERR_ARG;
  const bool gated = c.gate != nullptr;
  if (gated && (c.activation != 0 || !c.gate_index || !c.residual || c.index_rows <= 0 || c.index_rows > INT32_MAX ||
                c.M % c.index_rows || c.table_rows <= 0))
    return XGB_ERR_ARG;
  if (c.ldo < (c.activation == 3 ? c.N / 2 : c.N) || c.ldo % 8 || (gated && (c.ldg < c.N || c.ldr < c.N)))
    return XGB_ERR_STRIDE;
  if (!a16(c.w) || !a16(c.out)) return XGB_ERR_ALIGN;
  return XGB_OK;
}

int check_device() {
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10)
    return XGB_ERR_DEVICE;
  return XGB_OK;
}

template <typename T>
int product(const Call& c, const void* x, int64_t ldx) {
  int8::Params<T> p{};
  p.M = static_cast<int>(c.M);
  p.N = static_cast<int>(c.N);
  p.K = static_cast<int>(c.K);
  p.sa = c.scale_a;
  p.sw = c.scale_w;
  p.bias = static_cast<const T*>(c.bias);
  p.out = static_cast<T*>(c.out);
  p.ldo = c.ldo;
  p.gate = static_cast<const T*>(c.gate);
  p.ldg = c.ldg;
  p.idx = c.gate_index;
  p.idx_rows = static_cast<int>(c.index_rows);
  p.table_rows = c.table_rows;
  p.residual = static_cast<const T*>(c.residual);
  p.ldr = c.ldr;
  p.err = c.error_flag;
  p.behind_quantiser = c.behind_quantiser;
  p.vec = c.gate && a16(c.gate) && a16(c.residual) && c.ldg % 8 == 0 && c.ldr % 8 == 0;
  return int8::pick<T>(c.gate ? int8::kGated : c.activation, c.a, c.w, p, static_cast<const T*>(x), ldx, c.st);
}

}  // namespace

XGB_API int xgb_int8_gemm(const int8_t* a, const int8_t* w, int64_t M, int64_t N, int64_t K, const float* scale_a,
                          const float* scale_w, int dtype, const void* bias, int activation, void* out, int64_t ldo,
                          const void* gate, int64_t ldg, const int64_t* gate_index, int64_t index_rows, int64_t table_rows,
                          const void* residual, int64_t ldr, int* error_flag, void* stream) {
  const Call c{a, w, M, N, K, scale_a, scale_w, dtype, bias, activation, out, ldo, gate, ldg, gate_index, index_rows,
               table_rows, residual, ldr, error_flag, as_stream(stream)};
  if (!a || !scale_a) return XGB_ERR_ARG;
  int rc = check(c);
  if (rc) return rc;
  if (!a16(a)) return XGB_ERR_ALIGN;
  if ((rc = check_device())) return rc;
  return dtype == XGB_BF16 ? product<__nv_bfloat16>(c, nullptr, 0) : product<__half>(c, nullptr, 0);
}

static bool fused(const void* x, int64_t ldx, int64_t M, int64_t K) {
  return int8::fuses(M, K) && a16(x) && (M == 1 || ldx % 8 == 0);
}

XGB_API int64_t xgb_int8_linear_workspace(const void* x, int64_t ldx, int64_t M, int64_t K) {
  if (M <= 0 || K <= 0 || fused(x, ldx, M, K)) return 0;
  return cdiv(M * K, 16) * 16 + M * static_cast<int64_t>(sizeof(float));
}

XGB_API int xgb_int8_linear(const void* x, int64_t ldx, const int8_t* w, int64_t M, int64_t N, int64_t K,
                            const float* scale_w, int dtype, const void* bias, int activation, void* out, int64_t ldo,
                            const void* gate, int64_t ldg, const int64_t* gate_index, int64_t index_rows,
                            int64_t table_rows, const void* residual, int64_t ldr, void* workspace, int64_t workspace_bytes,
                            int* error_flag, void* stream) {
  Call c{nullptr, w, M, N, K, nullptr, scale_w, dtype, bias, activation, out, ldo, gate, ldg, gate_index, index_rows,
         table_rows, residual, ldr, error_flag, as_stream(stream)};
  if (!x) return XGB_ERR_ARG;
  int rc = check(c);
  if (rc) return rc;
  if (M > 1 && ldx < K) return XGB_ERR_STRIDE;
  const int64_t need = xgb_int8_linear_workspace(x, ldx, M, K);
  if (need && (!workspace || workspace_bytes < need)) return XGB_ERR_WORKSPACE;
  if (need && !a16(workspace)) return XGB_ERR_ALIGN;
  if ((rc = check_device())) return rc;
  const bool bf16 = dtype == XGB_BF16;
  if (!need)
    return bf16 ? product<__nv_bfloat16>(c, x, ldx) : product<__half>(c, x, ldx);
  int8_t* codes = static_cast<int8_t*>(workspace);
  float* scales = reinterpret_cast<float*>(codes + cdiv(M * K, 16) * 16);
  rc = bf16 ? int8::quantize(static_cast<const __nv_bfloat16*>(x), ldx, M, K, codes, scales, c.st)
            : int8::quantize(static_cast<const __half*>(x), ldx, M, K, codes, scales, c.st);
  if (rc) return rc;
  c.a = codes;
  c.scale_a = scales;
  c.behind_quantiser = true;
  return bf16 ? product<__nv_bfloat16>(c, nullptr, 0) : product<__half>(c, nullptr, 0);
}
