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
#include <type_traits>

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

// `at`: where the token's positions start.
__device__ __forceinline__ float2 cos_sin(const Params& p, int64_t at, double per_unit, int axis) {
  const double turns = load_position(p, at + axis) * per_unit;
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
// lane l owns pairs l, l + 32, ... and the unrotated channels likewise. It forms
// the angles for every head anew: 8,000 tokens of 12 + 12 heads of 64, 40 of
// them rotated, take 89 us, with all of them, in the vector form, 11.
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
      const float2 cs = cos_sin(p, b * p.pb + s * p.ps, turns.per_unit[i], turns.axis[i]);
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

constexpr int kN = 8;  // channels of a piece, pairs of a thread

// A piece as it lies in memory.
template <typename T>
struct Raw {
  static constexpr int kWords = kN * static_cast<int>(sizeof(T)) / 4;
  uint32_t w[kWords];
};
template <typename T>
__device__ __forceinline__ void load(const T* p, Raw<T>& r) {
#pragma unroll
  for (int i = 0; i < Raw<T>::kWords; i += 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
    r.w[i] = v.x;
    r.w[i + 1] = v.y;
    r.w[i + 2] = v.z;
    r.w[i + 3] = v.w;
  }
}
__device__ __forceinline__ void unpack(const Raw<float>& r, float (&f)[kN]) {
#pragma unroll
  for (int i = 0; i < kN; ++i) f[i] = __uint_as_float(r.w[i]);
}
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16>& r, float (&f)[kN]) {
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
    f[2 * i] = __uint_as_float(r.w[i] << 16);
    f[2 * i + 1] = __uint_as_float(r.w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack(const Raw<__half>& r, float (&f)[kN]) {
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ void pack(const float (&f)[kN], Raw<float>& r) {
#pragma unroll
  for (int i = 0; i < kN; ++i) r.w[i] = __float_as_uint(f[i]);
}
__device__ __forceinline__ void pack(const float (&f)[kN], Raw<__nv_bfloat16>& r) {
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) r.w[i] = round_bf16x2(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ void pack(const float (&f)[kN], Raw<__half>& r) {
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
    const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    r.w[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <typename T>
__device__ __forceinline__ void store(T* p, const Raw<T>& r) {
#pragma unroll
  for (int i = 0; i < Raw<T>::kWords; i += 4)
    reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
}

// Two pieces of kN channels as kN pairs (a, d), two pairs a register pair:
// channel i of both pieces, or neighbours when interleaved.
template <bool kInterleaved, typename T>
__device__ __forceinline__ void to_pairs(const Raw<T> (&r)[2], float2 (&a)[kN / 2], float2 (&d)[kN / 2]) {
  float f[2][kN];
  unpack(r[0], f[0]);
  unpack(r[1], f[1]);
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
    if constexpr (kInterleaved) {
      const int at = i / (kN / 4), o = 4 * (i % (kN / 4));
      a[i] = make_float2(f[at][o], f[at][o + 2]);
      d[i] = make_float2(f[at][o + 1], f[at][o + 3]);
    } else {
      a[i] = make_float2(f[0][2 * i], f[0][2 * i + 1]);
      d[i] = make_float2(f[1][2 * i], f[1][2 * i + 1]);
    }
  }
}
template <bool kInterleaved, typename T>
__device__ __forceinline__ void from_pairs(const float2 (&a)[kN / 2], const float2 (&d)[kN / 2], Raw<T> (&r)[2]) {
  float f[2][kN];
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
    if constexpr (kInterleaved) {
      const int at = i / (kN / 4), o = 4 * (i % (kN / 4));
      f[at][o] = a[i].x;
      f[at][o + 1] = d[i].x;
      f[at][o + 2] = a[i].y;
      f[at][o + 3] = d[i].y;
    } else {
      f[0][2 * i] = a[i].x;
      f[0][2 * i + 1] = a[i].y;
      f[1][2 * i] = d[i].x;
      f[1][2 * i + 1] = d[i].y;
    }
  }
  pack(f[0], r[0]);
  pack(f[1], r[1]);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 minus(float2 v) { return make_float2(-v.x, -v.y); }

// Vector form: width and rotary multiples of 16, 16-byte aligned rows. Threads
// are (token, head step, lane): 2^lane_bits lanes a head, 2^head_bits heads at
// a time, the rest of the 256 threads tokens. A block walks over groups of
// tokens; a group's cos/sin go through one of two shared buffers, so one
// barrier a group is enough. With a norm the instructions weigh as much as the
// bytes, so the arithmetic is packed (two values an instruction) and nothing
// is divided in the walk; 64 registers keep 32 warps on an SM, whose loads are
// what hides the sum between a head's loads and its stores (85 registers and
// 24 warps: a sixth slower; factors with the weights multiplied in, held in 118
// registers: a third). fp32 with a norm spills 8 to 16 bytes there, except for
// halves with all channels rotated. 126,754 tokens, Q and K of 24 heads of 128
// in bf16: 491 us (6.3 TB/s), with the norms 568 us; 40,000 tokens in fp32: 355
// us (halves, 5.5 TB/s) and 332 us (neighbours), with the norms 311 and 470 us.
// kPartial: not all channels are rotated. The others are left as they are:
// turned by an angle of zero, an infinity would make its neighbour a NaN. (The
// branch in every call: 1% slower where all are rotated.)
template <typename T, bool kInterleaved, bool kNorm, bool kPartial>
__global__ void __launch_bounds__(kThreads, 4) rope_axes_vec_kernel(const Params p, const __grid_constant__ Turns turns,
                                                                 int lane_bits, int head_bits, FastDiv div_seq,
                                                                 FastDiv div_pairs) {
  __shared__ double per_unit[kMaxPairs];
  __shared__ uint8_t axis[kMaxPairs];
  // at most 256 / lanes tokens of kN * lanes pairs each
  __shared__ __align__(16) float cos_buf[2][kThreads * kN];
  __shared__ __align__(16) float sin_buf[2][kThreads * kN];
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
  const bool active = 2 * kN * j < p.width, turned = !kPartial || 2 * kN * j < p.rotary;
  const int ca = kInterleaved || !turned ? 2 * kN * j : kN * j;
  const int cb = kInterleaved || !turned ? ca + kN : ca + pairs;
  const float inv_width = 1.f / p.width;
  const uint32_t tokens = static_cast<uint32_t>(p.tokens), step = per_group * gridDim.x;
  int buf = 0;
  for (uint32_t first = blockIdx.x * per_group; first < tokens; first += step, buf ^= 1) {
    for (uint32_t i = threadIdx.x; i < per_group * pairs; i += kThreads) {
      const uint32_t tt = fast_div(i, div_pairs), pair = i - tt * pairs;
      if (first + tt < tokens) {
        const uint32_t b = fast_div(first + tt, div_seq), at = first + tt - b * div_seq.d;
        const float2 cs = cos_sin(p, b * p.pb + at * p.ps, per_unit[pair], axis[pair]);
        cos_buf[buf][i] = cs.x;
        sin_buf[buf][i] = cs.y;
      }
    }
    __syncthreads();
    const uint32_t token = first + t;
    const bool here = active && token < tokens;
    const uint32_t b = fast_div(token, div_seq), at = token - b * div_seq.d;
    float2 c[kN / 2], s[kN / 2];
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      c[i] = both(1.f);
      s[i] = both(0.f);
    }
    if (here && turned) {
#pragma unroll
      for (int i = 0; i < kN / 2; i += 2) {
        const float4 cv = *reinterpret_cast<const float4*>(&cos_buf[buf][t * pairs + kN * j + 2 * i]);
        const float4 sv = *reinterpret_cast<const float4*>(&sin_buf[buf][t * pairs + kN * j + 2 * i]);
        c[i] = make_float2(cv.x, cv.y);
        c[i + 1] = make_float2(cv.z, cv.w);
        s[i] = make_float2(sv.x, sv.y);
        s[i + 1] = make_float2(sv.z, sv.w);
      }
    }
    const T* q_src = static_cast<const T*>(p.src[0]) + b * p.sb[0] + at * p.ss[0];
    const T* k_src = static_cast<const T*>(p.src[1]) + b * p.sb[1] + at * p.ss[1];
    T* q_dst = static_cast<T*>(p.dst[0]) + static_cast<int64_t>(token) * (p.heads[0] * p.width);
    T* k_dst = static_cast<T*>(p.dst[1]) + static_cast<int64_t>(token) * (p.heads[1] * p.width);
    const int heads = p.heads[0] + p.heads[1];
    constexpr int kUnroll = kNorm ? 3 : 2;  // 2 with a norm: 2% slower
#pragma unroll kUnroll
    for (int h0 = 0; h0 < heads; h0 += 1 << head_bits) {
      int h = h0 + first_head;
      const bool go = here && h < heads;
      const bool key = h >= p.heads[0];
      if (key) h -= p.heads[0];
      const T* src = key ? k_src + h * p.sh[1] : q_src + h * p.sh[0];
      Raw<T> raw[2];
      float2 a[kN / 2], d[kN / 2];
      if (go) {
        load(src + ca, raw[0]);
        load(src + cb, raw[1]);
        to_pairs<kInterleaved>(raw, a, d);
      }
      if constexpr (kNorm) {
        const T* w = static_cast<const T*>(key ? p.weight[1] : p.weight[0]);
        // every lane takes part; a tensor without a norm keeps its values
        float2 sq = both(0.f);
        if (go) {
#pragma unroll
          for (int i = 0; i < kN / 2; ++i) sq = __ffma2_rn(a[i], a[i], __ffma2_rn(d[i], d[i], sq));
        }
        float sum = sq.x + sq.y;
        for (int o = (1 << lane_bits) >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (go && w) {
          const float2 r = both(rsqrtf(fmaf(sum, inv_width, key ? p.eps[1] : p.eps[0])));
          Raw<T> wr[2];
          float2 wa[kN / 2], wd[kN / 2];
          load(w + ca, wr[0]);
          load(w + cb, wr[1]);
          to_pairs<kInterleaved>(wr, wa, wd);
#pragma unroll
          for (int i = 0; i < kN / 2; ++i) {
            a[i] = __fmul2_rn(a[i], __fmul2_rn(wa[i], r));
            d[i] = __fmul2_rn(d[i], __fmul2_rn(wd[i], r));
          }
        }
      }
      if (go) {
#pragma unroll
        for (int i = 0; turned && i < kN / 2; ++i) {
          const float2 turned_a = __ffma2_rn(a[i], c[i], __fmul2_rn(d[i], minus(s[i])));
          d[i] = __ffma2_rn(d[i], c[i], __fmul2_rn(a[i], s[i]));
          a[i] = turned_a;
        }
        from_pairs<kInterleaved>(a, d, raw);
        T* dst = (key ? k_dst : q_dst) + h * p.width;
        store(dst + ca, raw[0]);
        store(dst + cb, raw[1]);
      }
    }
  }
}

// The turns of these axes. A thread keeps those of its last axes: 64 powers
// take about 2 us, as long as the launch.
const Turns& turns_of(int axes, const int64_t* channels, const double* thetas) {
  struct Last {
    int axes = 0;
    int64_t channels[kMaxAxes];
    double thetas[kMaxAxes];
    Turns turns;
  };
  static thread_local Last last;
  if (last.axes == axes && std::equal(channels, channels + axes, last.channels) &&
      std::equal(thetas, thetas + axes, last.thetas))
    return last.turns;
  constexpr double kTwoPi = 6.283185307179586476925286766559;
  int pairs = 0;
  for (int a = 0; a < axes; ++a)
    for (int64_t i = 0; i < channels[a] / 2; ++i, ++pairs) {
      last.turns.per_unit[pairs] = pow(thetas[a], -2.0 * static_cast<double>(i) / static_cast<double>(channels[a])) / kTwoPi;
      last.turns.axis[pairs] = static_cast<uint8_t>(a);
    }
  std::copy(channels, channels + axes, last.channels);
  std::copy(thetas, thetas + axes, last.thetas);
  last.axes = axes;
  return last.turns;
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
  const int lane_bits = bits_for(p.width / (2 * kN));
  // Few tokens: all heads of a token at once, so that more blocks have work.
  // Many: up to 8 heads at a time, 4 where 8 would leave more than an eighth
  // of the threads without a head.
  const bool few = p.tokens <= 2 * 148;
  int head_bits = std::min(bits_for(heads), few ? 8 - lane_bits : std::min(3, 8 - lane_bits));
  if (!few && head_bits == 3 && (cdiv(heads, 8) * 8 - heads) * 8 > heads) head_bits = 2;
  const int64_t groups = cdiv(p.tokens, kThreads >> (lane_bits + head_bits));
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(groups, 148 * 8));
  const FastDiv div_seq = make_fastdiv(static_cast<uint32_t>(p.seq)), div_pairs = make_fastdiv(static_cast<uint32_t>(p.rotary / 2));
  auto run = [&](auto kernel) {
    kernel<<<grid, kThreads, 0, st>>>(p, turns, lane_bits, head_bits, div_seq, div_pairs);
    return launch_status();
  };
  auto pick = [&](auto interleave, auto norm) {
    constexpr bool kInterleaved = decltype(interleave)::value, kNorm = decltype(norm)::value;
    if (p.rotary < p.width) return run(rope_axes_vec_kernel<T, kInterleaved, kNorm, true>);
    return run(rope_axes_vec_kernel<T, kInterleaved, kNorm, false>);
  };
  const std::true_type yes{};
  const std::false_type no{};
  if (p.weight[0] || p.weight[1]) return interleaved ? pick(yes, yes) : pick(no, yes);
  return interleaved ? pick(yes, no) : pick(no, no);
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
  int64_t rotary = 0;
  for (int64_t a = 0; a < axes; ++a) {
    if (axis_channels[a] <= 0 || axis_channels[a] % 2 || axis_channels[a] > width - rotary) return XGB_ERR_SHAPE;
    if (!(thetas[a] > 0.0)) return XGB_ERR_ARG;
    rotary += axis_channels[a];
  }
  if (batch == 0 || seq == 0) return XGB_OK;
  if (seq > INT32_MAX || batch > INT32_MAX / seq) return XGB_ERR_SHAPE;
  const Turns& turns = turns_of(static_cast<int>(axes), axis_channels, thetas);
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
  p.rotary = static_cast<int>(rotary);
  cudaStream_t st = as_stream(stream);
  if (dtype == XGB_BF16) return launch<__nv_bfloat16>(p, turns, interleaved != 0, st);
  if (dtype == XGB_F16) return launch<__half>(p, turns, interleaved != 0, st);
  return launch<float>(p, turns, interleaved != 0, st);
}
