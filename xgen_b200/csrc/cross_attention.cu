// Cross attention on sm_100a tensor cores: queries of one sequence against the
// keys and values of another (an encoder's states), with a key count for each
// sample, shared key heads, head dims 64 and 128, bf16 or fp16:
//
//   o[b, h, s] = sum_j p_j v[b, h', j] / sum_j p_j,  j < len[b],  h' = h / (H / H')
//   p_j = 2^(scale log2(e) q.k_j - m),  m a value for each row, see below
//
// A sample without keys gives rows of zeros. Keys and values at j >= len[b]
// are not read as numbers: their scores are overwritten with -inf and their
// value rows with zeros (a NaN times a probability of zero would be NaN).
//
// Encoder sequences are short (64 to a few hundred keys), so a query tile is
// done after 4 to 8 key tiles, and what an own CTA for each would spend on
// starting and ending (TMEM, barriers, first loads, last stores) is a large
// part of its time. The kernel is therefore persistent, one CTA per SM over a
// list of units; a unit is 256 query rows (two tiles of 128) of one (batch,
// head) and, when there are fewer of those than SMs, one part of its keys. All
// roles run through the list on their own, coupled by mbarriers only, so the
// loads and first scores of the next unit overlap the last tiles and the
// epilogue of this one:
//   warps 0-3, 4-7  softmax and epilogue of query tile 0, 1 (a thread a row)
//   warp 8          TMA producer: Q tiles, a ring of 64-key K tiles, one of V tiles
//   warps 9, 10     MMA issuers of query tile 0, 1
//   warp 11         clears the value rows behind the last key of a sample
// TMEM (512 columns): two S buffers of 64 fp32 columns for each query tile
// (P overwrites its S), O0, O1. Shared memory at D = 128: three 32 KB places
// for query tiles, so that the next unit's first one is there long before its
// scores are due and its second one two key tiles before, two K and V tiles (a
// third gave nothing), and 8 KB a softmax warp in which its output rows wait
// for their TMA store (with 4 KB, half of the channels after the other,
// 124,992 x 77 takes 8% longer). 124,992 rows, 24 heads of 128, replayed from a
// graph: 681 to 691 us with 512 keys, 269 us with 77; called in a loop, at the
// clocks of the power cap, 807 us with 512.
//
// What bounds a step of 64 keys for both query tiles is the tensor pipe and
// the threads that feed it. Measured back to back on one SM: a 128 x 64 x 16
// product from shared memory takes 49 cycles (its 6 KB of operands at 128 bytes
// a cycle; the arithmetic alone 32), a 128 x 128 x 16 one with P from TMEM 64,
// and one thread sends out at most one product in 51 cycles: 16 x 49 + 8 x 64 =
// 1,296 cycles a step. (The one product in 51 cycles holds for a thread picked
// as lane 0; one picked by elect.sync sends out one in 16, its operands being
// uniform for the compiler.) So an issuer has nothing to compute between the last
// probabilities of a tile and its products: descriptors, flags and the waits
// that can be early are behind it, indexes are kept by increments, and warps,
// not threads, arrive.
//
// Softmax in the exp2 domain with 32-bit sums. The reference value m of a row
// comes from its first key tile. Being larger or smaller than others costs a
// probability no digits, so later tiles take no maximum: the tile's own sum
// shows whether one came near a limit, and only then is the maximum taken, O
// rescaled and the tile repeated. Without the maximum's instructions and their
// place in the chain from scores to probabilities a step is a third shorter.
//   bf16: m = the largest score + 24, sums up to 2^8. A later probability may be
//     2^32 times the first tile's before a tile is repeated. O stays finite for
//     values below 2^126 / seq_kv in magnitude (each tile of 64 keys adds at
//     most 2^8 of them; with the row's largest score for m: 2^128 / seq_kv), and
//     keeps its digits for values from 2^-80. (m = the largest score, sums up to
//     2^40: infinities from values of 2^88. Sums up to 2^8: 43% slower where
//     scores have a deviation of 4.)
//   fp16: m = the largest score, sums up to 2^15, which P can hold; values up to
//     2^16 cannot overflow O.
// P is rounded to the type of V for the second product, which takes 16-bit
// operands of one type: up to half a step of every probability, in the result
// about as much as its own rounding (bf16: 2.3e-3 from 64 bits in place of
// 1.7e-3, relative). Exponentials are the SFU's, 2^-22.
//
// Parts of a unit leave 32-bit O, m and l rows in a workspace of the call;
// a second small kernel joins them.
#include <algorithm>
#include <type_traits>

#include "sm100.cuh"
#include "tma_host.h"

namespace xgb {
namespace cross {

using namespace sm100;

constexpr int kBM = 128;   // rows per query tile
constexpr int kRows = 256;  // rows per unit
constexpr int kBN = 64;    // keys per tile
constexpr int kThreads = 384;
constexpr int kTmaWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kFixWarp = 11;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kTurnBar = 1;  // named barriers 1, 2: the exponentials' turn of query tile 0, 1

constexpr int kQPlaces = 3;
constexpr int kOutBytes = 32 * 128;  // 32 rows x 64 channels of a softmax warp

template <typename T, int kD>
struct Cfg {
  static constexpr int kSubs = kD / 64;                // 128-byte-wide sub-tiles of a row
  static constexpr int kQSub = kBM * 128;
  static constexpr int kQBytes = kSubs * kQSub;
  static constexpr int kKVSub = kBN * 128;
  static constexpr int kKVBytes = kSubs * kKVSub;
  static constexpr int kStages = kD == 128 ? 2 : 4;
  static constexpr int kKOff = kQPlaces * kQBytes;
  static constexpr int kVOff = kKOff + kStages * kKVBytes;
  static constexpr int kOutOff = kVOff + kStages * kKVBytes;
  static constexpr int kBarOff = kOutOff + 8 * kSubs * kOutBytes;
  static constexpr int kSmem = kBarOff + 512 + 1024;  // + barriers + alignment slack
  static constexpr uint32_t kFmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  static constexpr uint32_t kIdescQK = instr_desc(1, kFmt, kFmt, false, false, kBM, 0);  // + keys
  // How far a row's reference value is above its largest score, and the sum of a
  // tile's probabilities above which the largest score is looked for anew.
  static constexpr float kAbove = std::is_same<T, __nv_bfloat16>::value ? 24.f : 0.f;
  static constexpr float kLimit = std::is_same<T, __nv_bfloat16>::value ? 256.f : 32768.f;
  static constexpr uint32_t kIdescPV = instr_desc(1, kFmt, kFmt, false, true, kBM, kD);
};

struct Params {
  int heads, group;  // query heads, query heads of one key head
  int seq_q, seq_kv;
  const int* lens;  // [batch], null: seq_kv
  float scale_log2;
  void* out;
  int64_t osb, osh, oss;
  // coordinate factors: 0 for a dimension that is broadcast
  int qb, qh, kb, kh, vb, vh;
  int n_qt;      // units of 256 rows of a (batch, head)
  int splits;    // parts of a unit's keys
  uint32_t units;  // batch * heads * n_qt * splits, below 2^31
  FastDiv div_splits, div_qt, div_heads, div_group;
  int part_rows;  // rows of a part in the workspace
  float* part_o;  // [units][part_rows][D]
  float2* part_ml;  // [units][part_rows]
  int* err;
};

struct Barriers {
  // Query tiles 2n + i go round the places; the barriers go round twice as many
  // tiles, so that each is only ever waited for by one query tile's issuer, a
  // phase after the other.
  uint64_t q_full[2 * kQPlaces], q_empty[2 * kQPlaces];
  // V(g) and K(g + 2) come and go together: an issuer uses them in one step.
  uint64_t kv_full[6], v_ready[6], kv_empty[6];
  uint64_t first_full[2], first_empty[2];  // K(0), K(1)
  uint64_t s_full[2][2], p_full[2][2];
  uint64_t o_full[2], o_empty[2];
  uint64_t end[2];
  uint32_t tmem_base;
};

// A unit of a CTA's walk. Every role finds its units by itself, some of them
// on one thread in the products' critical path, so the divisions are 32-bit
// multiplications.
struct Unit {
  uint32_t id;
  int b, h, m0;
  int kv0, n_kv;  // key tiles [kv0, kv0 + n_kv)
  int len;
};

__device__ __forceinline__ Unit unit_at(const Params& p, uint32_t id) {
  Unit u;
  u.id = id;
  const uint32_t item = fast_div(id, p.div_splits), bh = fast_div(item, p.div_qt), b = fast_div(bh, p.div_heads);
  const int part = static_cast<int>(id - item * p.div_splits.d);
  u.m0 = static_cast<int>(item - bh * p.div_qt.d) * kRows;
  u.b = static_cast<int>(b);
  u.h = static_cast<int>(bh - b * p.div_heads.d);
  u.len = p.lens ? min(max(__ldg(p.lens + u.b), 0), p.seq_kv) : p.seq_kv;
  const int n_all = (u.len + kBN - 1) / kBN;
  const int per = static_cast<int>(fast_div(n_all + p.splits - 1, p.div_splits));
  u.kv0 = min(part * per, n_all);
  u.n_kv = min(per, n_all - u.kv0);
  return u;
}

// Position in the stream of key tiles that the CTA's non-empty units make up
// (units without keys are visited by the softmax warps only).
struct Cursor {
  Unit u;
  int t;  // tile within the unit
  int n;  // non-empty units before this one
  bool more;
  __device__ __forceinline__ void seek(const Params& p, uint32_t id) {
    more = false;
    for (; id < p.units; id += gridDim.x) {
      u = unit_at(p, id);
      if (u.n_kv > 0) {
        more = true;
        break;
      }
    }
    t = 0;
  }
  __device__ __forceinline__ void start(const Params& p) {
    n = 0;
    seek(p, blockIdx.x);
  }
  __device__ __forceinline__ bool last() const { return t == u.n_kv - 1; }
  __device__ __forceinline__ int keys() const { return min(kBN, u.len - (u.kv0 + t) * kBN); }
  __device__ __forceinline__ void next(const Params& p) {
    if (++t == u.n_kv) {
      ++n;
      seek(p, u.id + gridDim.x);
    }
  }
};

// Place of tile g in a ring of kStages: g % kStages and the parity of g / kStages.
template <int kStages>
struct Ring {
  int stage = 0;
  uint32_t lap = 0;
  __device__ __forceinline__ void next() {
    if (++stage == kStages) {
      stage = 0;
      lap ^= 1;
    }
  }
};

__device__ __forceinline__ uint32_t s_col(int i, int b) { return static_cast<uint32_t>(i * 128 + b * 64); }
__device__ __forceinline__ uint32_t o_col(int i) { return static_cast<uint32_t>(256 + i * 128); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, int kD>
__global__ void __launch_bounds__(kThreads, 1)
    cross_attention_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                           const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap o_map,
                           const Params p) {
  using C = Cfg<T, kD>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Barriers* bars = reinterpret_cast<Barriers*>(smem + C::kBarOff);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // the same register for the warp
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->kv_full[s], 1);
      mbar_init(&bars->v_ready[s], 1);
      mbar_init(&bars->kv_empty[s], 2);  // released by both issuers
    }
    for (int e = 0; e < 2 * kQPlaces; ++e) {
      mbar_init(&bars->q_full[e], 1);
      mbar_init(&bars->q_empty[e], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->first_full[i], 1);
      mbar_init(&bars->first_empty[i], 2);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bars->s_full[i][b], 1);
        mbar_init(&bars->p_full[i][b], 4);  // one arrival a warp: 32 lanes' would queue
      }
      mbar_init(&bars->o_full[i], 1);
      mbar_init(&bars->o_empty[i], 4);
      mbar_init(&bars->end[i], 1);
    }
    fence_barrier_init();
  }
  if (warp == kMmaWarp) tmem_alloc<512>(&bars->tmem_base);
  if (warp == kTmaWarp && lane == 0) {
    prefetch_tmap(&q_map);
    prefetch_tmap(&k_map);
    prefetch_tmap(&v_map);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == kTmaWarp) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      // K runs two tiles ahead of V, as the scores do of the second product.
      bool ok = true;
      int k_loaded = 0, v_loaded = 0, q_loaded = 0;
      Cursor kc, vc;
      kc.start(p);
      vc = kc;
      auto load_q = [&]() {  // a unit's two query tiles, with its first keys
        const Unit& u = kc.u;
        for (int i = 0; i < 2; ++i, ++q_loaded) {
          const int place = q_loaded % kQPlaces, before = q_loaded - kQPlaces;  // the place's last tile
          if (before >= 0)
            ok = ok && mbar_wait(&bars->q_empty[before % (2 * kQPlaces)], (before / (2 * kQPlaces)) & 1, p.err);
          if (!ok) return;
          uint64_t* bar = &bars->q_full[q_loaded % (2 * kQPlaces)];
          mbar_arrive_expect_tx(bar, C::kQBytes);
          for (int j = 0; j < C::kSubs; ++j)
            tma_load_4d(smem + place * C::kQBytes + j * C::kQSub, &q_map, bar, j * 64, u.m0 + i * kBM, u.h * p.qh, u.b * p.qb);
        }
      };
      auto load_k = [&](uint64_t* bar, int stage) {
        const Unit& u = kc.u;
        const int kvh = static_cast<int>(fast_div(u.h, p.div_group));
        for (int j = 0; j < C::kSubs; ++j)
          tma_load_4d(smem + C::kKOff + stage * C::kKVBytes + j * C::kKVSub, &k_map, bar, j * 64, (u.kv0 + kc.t) * kBN,
                      kvh * p.kh, u.b * p.kb);
        ++k_loaded;
      };
      for (int e = 0; e < 2 && kc.more && ok; ++e) {
        if (kc.t == 0) load_q();
        if (!ok) break;
        mbar_arrive_expect_tx(&bars->first_full[e], C::kKVBytes);
        load_k(&bars->first_full[e], e);
        kc.next(p);
      }
      Ring<kStages> ring;
      int k_stage = 2 % kStages;
      while (vc.more && ok) {
        if (v_loaded >= kStages) ok = mbar_wait(&bars->kv_empty[ring.stage], ring.lap ^ 1, p.err);
        // the first keys' places become free by their own barriers
        else if (kc.more && v_loaded + 2 >= kStages)
          ok = mbar_wait(&bars->first_empty[v_loaded + 2 - kStages], 0, p.err);
        if (!ok) break;
        uint64_t* bar = &bars->kv_full[ring.stage];
        mbar_arrive_expect_tx(bar, kc.more ? 2 * C::kKVBytes : C::kKVBytes);
        const Unit& u = vc.u;
        const int kvh = static_cast<int>(fast_div(u.h, p.div_group));
        for (int j = 0; j < C::kSubs; ++j)
          tma_load_4d(smem + C::kVOff + ring.stage * C::kKVBytes + j * C::kKVSub, &v_map, bar, j * 64,
                      (u.kv0 + vc.t) * kBN, kvh * p.vh, u.b * p.vb);
        ++v_loaded;
        vc.next(p);
        ring.next();
        if (kc.more) {
          load_k(bar, k_stage);
          k_stage = k_stage + 1 == kStages ? 0 : k_stage + 1;
          if (kc.t == 0) load_q();
          if (!ok) break;
          kc.next(p);
        }
      }
      // Never leave with copies in flight: wait (bounded) for the last ones.
      for (int g = 0; g < min(2, k_loaded); ++g) mbar_wait(&bars->first_full[g], 0, p.err, 100000000ull);
      for (int g = max(0, v_loaded - kStages); g < v_loaded; ++g)
        mbar_wait(&bars->kv_full[g % kStages], (g / kStages) & 1, p.err, 100000000ull);
      for (int n = max(0, q_loaded - kQPlaces); n < q_loaded; ++n)
        mbar_wait(&bars->q_full[n % (2 * kQPlaces)], (n / (2 * kQPlaces)) & 1, p.err, 100000000ull);
    }
  } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    // ------------------------------------------------------------ MMA issuers
    const int i = warp - kMmaWarp;
    if (elect_one()) {
      // Descriptors differ in their address alone (in 16-byte units, from bit 0).
      const uint64_t q_desc = smem_desc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(smem_u32(smem + C::kKOff), 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(smem_u32(smem + C::kVOff), C::kKVSub, 1024);
      uint64_t* kv_bar = p.lens ? bars->v_ready : bars->kv_full;
      bool ok = true;
      Cursor sc;  // tile of the next scores, two ahead of the second product's
      sc.start(p);
      // What the second product of a tile has to know: products' key extents are
      // multiples of 16.
      struct Tile {
        int steps, n;
        bool there, first, last;
      };
      auto tile = [&]() { return Tile{(sc.keys() + 15) >> 4, sc.n, sc.more, sc.t == 0, sc.last()}; };
      int k_stage = 0;
      Ring<2 * kQPlaces> q_ring;  // of query tiles i, i + 2, ...
      if (i == 1) q_ring.next();
      auto issue_s = [&](int steps, int buffer, bool last) {
        const int place = q_ring.stage >= kQPlaces ? q_ring.stage - kQPlaces : q_ring.stage;
        const uint64_t qa = q_desc + place * (C::kQBytes / 16), ka = k_desc + k_stage * (C::kKVBytes / 16);
        // keys: N >> 3 at bit 17 of the descriptor
        const uint32_t idesc = C::kIdescQK | static_cast<uint32_t>(steps * 2) << 17;
#pragma unroll
        for (int k = 0; k < kD / 16; ++k)
          mma_ss<Kind::kF16>(tmem + s_col(i, buffer), qa + ((k >> 2) * C::kQSub + (k & 3) * 32) / 16,
                             ka + ((k >> 2) * C::kKVSub + (k & 3) * 32) / 16, idesc, k > 0);
        tc_commit(&bars->s_full[i][buffer]);
        if (last) {
          tc_commit(&bars->q_empty[q_ring.stage]);
          q_ring.next();
          q_ring.next();
        }
        k_stage = k_stage + 1 == kStages ? 0 : k_stage + 1;
      };
      Tile now{0, 0, false, false, false}, after = now;
      for (int e = 0; e < 2; ++e) {
        const Tile t = tile();
        if (t.there && ok) {
          if (t.first) ok = mbar_wait(&bars->q_full[q_ring.stage], q_ring.lap, p.err);
          ok = ok && mbar_wait(&bars->first_full[e], 0, p.err);
          if (ok) {
            tc_fence_after();
            issue_s(t.steps, e, t.last);
            tc_commit(&bars->first_empty[e]);
            sc.next(p);
          }
        }
        (e == 0 ? now : after) = t;
      }
      Ring<kStages> ring;
      for (int buffer = 0, lap = 0; now.there && ok; buffer ^= 1, lap ^= buffer ^ 1) {
        const Tile next = tile();
        const uint64_t va = v_desc + ring.stage * (C::kKVBytes / 16);
        const uint32_t s_tmem = tmem + s_col(i, buffer);
        ok = mbar_wait(&kv_bar[ring.stage], ring.lap, p.err);
        if (ok && now.first && now.n > 0) ok = mbar_wait(&bars->o_empty[i], (now.n - 1) & 1, p.err);
        ok = ok && mbar_wait(&bars->p_full[i][buffer], lap, p.err);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < kBN / 16; ++k)
          if (k < now.steps)
            mma_ts<Kind::kF16>(tmem + o_col(i), s_tmem + k * 8, va + k * 16 * 128 / 16, C::kIdescPV, !now.first || k > 0);
        if (now.last) tc_commit(&bars->o_full[i]);
        if (next.there) {
          // a unit's queries may wait for what this product sets free
          if (next.first) {
            ok = mbar_wait(&bars->q_full[q_ring.stage], q_ring.lap, p.err);
            if (!ok) break;
            tc_fence_after();
          }
          issue_s(next.steps, buffer, next.last);
        } else {
          tc_commit(&bars->s_full[i][buffer]);  // the two phases behind the last scores still end
        }
        tc_commit(&bars->kv_empty[ring.stage]);
        if (next.there) sc.next(p);
        ring.next();
        now = after;
        after = next;
      }
      tc_commit(&bars->end[i]);
      mbar_wait(&bars->end[i], 0, p.err, 100000000ull);
    }
  } else if (warp == kFixWarp) {
    // ------------------------------------------------------------ value rows behind the last key
    if (p.lens) {
      Cursor c;
      Ring<kStages> ring;
      for (c.start(p); c.more; c.next(p), ring.next()) {
        const int s = ring.stage;
        if (!__all_sync(0xffffffffu, mbar_wait(&bars->kv_full[s], ring.lap, p.err))) break;
        const int valid = c.keys(), read = (valid + 15) / 16 * 16;
        if (valid < read) {
          // rows of 128 bytes; the swizzle moves 16-byte pieces within a row
          for (int j = 0; j < C::kSubs; ++j) {
            uint4* rows = reinterpret_cast<uint4*>(smem + C::kVOff + s * C::kKVBytes + j * C::kKVSub);
            for (int e = valid * 8 + lane; e < read * 8; e += 32) rows[e] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->v_ready[s]);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int i = warp >> 2;
    const int lane_base = (warp & 3) * 32;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(lane_base) << 16);
    const uint32_t o_addr = lane_addr + o_col(i);
    const int r = i * kBM + lane_base + lane;  // row within the unit
    const float comb = p.scale_log2;
    bool ok = true;
    int g = 0, n = 0;
    // The two query tiles take turns with the exponentials. Without, both run
    // in step: 64 exponentials a row take 1,150 cycles for the two of them at
    // once, the SFU's rate, and what comes before and after, 700 cycles, leaves
    // it idle. A turn passes half way through a tile (at its end: 2 to 3%
    // slower), by named barriers: one wait and one arrival for each tile, tile 1
    // hands tile 0 the first turn and tile 0 takes the last. (A share of the
    // exponentials by polynomials in packed arithmetic made a step longer, with
    // a sixth of them 6 to 17% and with half 20%: a turn is a chain of one warp
    // on each scheduler.) A step of 1,490 cycles at D = 64: 800 for the
    // exponentials, half of them beside the other tile's, 172 until the scores
    // are seen, 134 for their load, 136 for the last sums and the vote.
    const int own_turn = kTurnBar + i, other_turn = kTurnBar + (i ^ 1);
    int turns = 0;
    if (i == 1) named_arrive(other_turn, 2 * kBM);
    // A unit's epilogue runs behind the first tile of the next one, whose scores
    // are there before this one's last product has ended.
    struct Pending {
      Unit u;
      float m, l;
      int n;  // -1: none
    } done;
    done.n = -1;
    auto epilogue = [&]() {
      const Unit& v = done.u;
      const int row = v.m0 + r;
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_full[i], done.n & 1, p.err));
      done.n = -1;
      if (!ok) return;
      tc_fence_after();
      if (p.splits > 1) {
        const int64_t part = static_cast<int64_t>(v.id) * p.part_rows + r;
#pragma unroll 1
        for (int c = 0; c < kD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + c * 32, o);
          tmem_ld_wait();
          if (row >= p.seq_q) continue;
          float4* po = reinterpret_cast<float4*>(p.part_o + part * kD) + c * 8;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            po[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]),
                                __uint_as_float(o[4 * e + 3]));
        }
        if (row < p.seq_q) p.part_ml[part] = make_float2(done.m, done.l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->o_empty[i]);
        return;
      }
      // Through shared memory, so that rows leave as whole lines by TMA, which
      // does not write rows behind the last query.
      const float inv_l = done.l != 0.f ? 1.0f / done.l : 0.f;
      uint8_t* stage = smem + C::kOutOff + warp * C::kSubs * kOutBytes;
      uint32_t o[C::kSubs][2][32];
#pragma unroll
      for (int c = 0; c < C::kSubs; ++c) tmem_ld64(o_addr + c * 64, o[c]);
      if (lane == 0) bulk_wait_read<0>();  // the last unit's stores have left the buffer
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->o_empty[i]);
#pragma unroll
      for (int c = 0; c < C::kSubs; ++c) {
        uint4 w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t* y = &o[c][e >> 2][(e & 3) * 8];
          auto two = [&](int k) { return pack2<T>(__uint_as_float(y[2 * k]) * inv_l, __uint_as_float(y[2 * k + 1]) * inv_l); };
          w[e] = make_uint4(two(0), two(1), two(2), two(3));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) *reinterpret_cast<uint4*>(stage + c * kOutBytes + lane * 128 + ((e ^ (lane & 7)) << 4)) = w[e];
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_4d(&o_map, stage + c * kOutBytes, c * 64, v.m0 + i * kBM + lane_base, v.h, v.b);
          bulk_commit();
        }
      }
    };
    for (uint32_t id = blockIdx.x; id < p.units && ok; id += gridDim.x) {
      const Unit u = unit_at(p, id);
      if (u.n_kv == 0) {
        const int row = u.m0 + r;
        if (row < p.seq_q) {
          if (p.splits > 1) {
            p.part_ml[static_cast<int64_t>(id) * p.part_rows + r] = make_float2(kNegInf, 0.f);
          } else {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + u.b * p.osb + u.h * p.osh + row * p.oss);
#pragma unroll
            for (int c = 0; c < kD / 8; ++c) dst[c] = make_uint4(0, 0, 0, 0);
          }
        }
        continue;
      }
      float m_used = kNegInf;
      float sum[2] = {0.f, 0.f};
      for (int t = 0; t < u.n_kv; ++t, ++g) {
        const uint32_t s_addr = lane_addr + s_col(i, g & 1);
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[i][g & 1], (g >> 1) & 1, p.err));
        if (!ok) break;
        tc_fence_after();
        uint32_t x[2][32];
        tmem_ld64(s_addr, x);
        tmem_ld_wait();
        const int valid = u.len - (u.kv0 + t) * kBN;
        if (valid < kBN) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e >= valid) x[c][e] = 0xFF800000u;
        }
        auto tile_max = [&]() {
          float m4[4];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            m4[2 * c] = fmax3(__uint_as_float(x[c][0]), __uint_as_float(x[c][1]), __uint_as_float(x[c][2]));
            m4[2 * c + 1] = fmax3(__uint_as_float(x[c][3]), __uint_as_float(x[c][4]), __uint_as_float(x[c][5]));
#pragma unroll
            for (int e = 6; e < 30; e += 4) {
              m4[2 * c] = fmax3(m4[2 * c], __uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1]));
              m4[2 * c + 1] = fmax3(m4[2 * c + 1], __uint_as_float(x[c][e + 2]), __uint_as_float(x[c][e + 3]));
            }
            m4[2 * c] = fmax3(m4[2 * c], __uint_as_float(x[c][30]), __uint_as_float(x[c][31]));
          }
          return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * comb;
        };
        // P = 2^(comb s - m_used - kAbove) over the S buffer; returns its sum in
        // two lanes. (kAbove in m_used itself: 4% slower at D = 64.)
        auto probabilities = [&](float (&ts)[2], bool pass_turn) {
          // a row whose scores are all -inf has its maximum there: p = 2^-inf
          const float off = m_used == kNegInf ? 0.f : -C::kAbove - m_used;
          float ra[4] = {0.f, 0.f, 0.f, 0.f}, rb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t packed[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float a, b;
              ffma2(a, b, __uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1]), comb, comb, off, off);
              a = ex2_approx(a);
              b = ex2_approx(b);
              const int ch = (e / 2) & 3;
              if (c == 0 && e < 8) {
                ra[ch] = a;
                rb[ch] = b;
              } else {
                fadd2(ra[ch], rb[ch], ra[ch], rb[ch], a, b);
              }
              packed[e / 2] = pack2<T>(a, b);
            }
            tmem_st16(s_addr + c * 16, packed);
            if (c == 0 && pass_turn) named_arrive(other_turn, 2 * kBM);
          }
          fadd2(ra[0], rb[0], ra[0], rb[0], ra[1], rb[1]);
          fadd2(ra[2], rb[2], ra[2], rb[2], ra[3], rb[3]);
          fadd2(ts[0], ts[1], ra[0], rb[0], ra[2], rb[2]);
        };
        if (t == 0) m_used = tile_max();
        float ts[2];
        named_sync(own_turn, 2 * kBM);
        probabilities(ts, true);
        ++turns;
        if (t > 0 && __any_sync(0xffffffffu, !(ts[0] + ts[1] <= C::kLimit) || m_used == kNegInf)) {
          // Too large, not a number, or no finite score so far: take the
          // maximum after all, with O (complete up to the tile before) rescaled.
          const float m_new = fmaxf(m_used, tile_max());
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[i][(g + 1) & 1], ((g + 1) >> 1) & 1, p.err));
          if (!ok) break;
          tc_fence_after();
          const float alpha = m_new > m_used ? ex2_approx(m_used - m_new) : 1.0f;
          m_used = m_new;
          sum[0] *= alpha;
          sum[1] *= alpha;
#pragma unroll 1
          for (int c = 0; c < kD / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(o_addr + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16(o_addr + c * 16, o);
          }
          probabilities(ts, false);
        }
        fadd2(sum[0], sum[1], sum[0], sum[1], ts[0], ts[1]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[i][g & 1]);
        if (t == 0 && done.n >= 0) epilogue();
        if (!ok) break;
      }
      if (!ok) break;
      done.u = u;
      done.m = m_used;
      done.l = sum[0] + sum[1];
      done.n = n++;
    }
    if (!ok) {
      // After a failed wait the other tile still gets its turns.
      int all = 0;
      for (uint32_t id = blockIdx.x; id < p.units; id += gridDim.x) all += unit_at(p, id).n_kv;
      for (; turns < all; ++turns) {
        named_sync(own_turn, 2 * kBM);
        named_arrive(other_turn, 2 * kBM);
      }
    }
    if (i == 0) named_sync(own_turn, 2 * kBM);
    if (ok && done.n >= 0) epilogue();
    if (lane == 0) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc<512>(tmem);
  }
}

// ---------------------------------------------------------------- few query rows
// One token, or a few, for each sample: the query rows of one key head (its
// H/H' query heads times Sq) fit a tile of 8, a 128-row tensor-core tile would
// be empty, and the time is that of reading K and V once. Warps take 16 keys
// at a time straight from global memory into the fragments of the warp-level
// 16x8x16 products, with no shared memory on the way:
//   S^T [16 keys x 8 rows] = K Q^T: a lane loads 16-byte pieces of the rows of
//     keys g and g + 8 (g = lane / 4); the products' inner index is any order
//     of d as long as Q's is the same one, so the pieces are the fragments.
//   O^T [D x 8 rows] += V^T P^T: the same pieces of V, transposed 8 x 8 by
//     movmatrix; the order of d that comes out is undone when O is written.
// Each warp keeps its own running maximum and O; the warps of a CTA join in
// shared memory. The CTAs of a unit (parts of its keys) are a cluster of up to
// 8, whose members each join some of the rows over distributed shared memory;
// only few units with many keys need more parts than that, and join in the
// second kernel.
// Keys behind a sample's last one are not loaded: zeros, with scores of -inf.
constexpr int kFewRows = 8;
constexpr int kFewWarps = 4;
constexpr int kFewKeys = 16;  // keys of a warp's step

struct FewParams {
  const void* q;
  const void* k;
  const void* v;
  int64_t qsb, qsh, qss, ksb, ksh, kss, vsb, vsh, vss;
  const uint8_t* mask;  // [batch, seq_kv] bytes, null: none
  int64_t msb, mss;
  int kv_heads, tiles;  // row tiles of 8 of a key head
  int clustered;        // a unit's parts are a cluster
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 tile of 16-bit values spread over the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// The 16-byte pieces 8c.. of every 32 channels of one row.
template <int kChunks>
__device__ __forceinline__ void load_row(const void* base, int64_t at, bool go, uint4 (&r)[kChunks]) {
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
#pragma unroll
  for (int j = 0; j < kChunks; ++j) r[j] = go ? __ldg(src + 4 * j) : make_uint4(0, 0, 0, 0);
}

template <typename T, int kD>
__global__ void __launch_bounds__(kFewWarps * 32) cross_few_kernel(const Params p, const FewParams f) {
  constexpr int kChunks = kD / 32;
  __shared__ float so[kFewWarps][kFewRows][kD];
  __shared__ float2 sml[kFewWarps][kFewRows];
  __shared__ float2 part_ml[kFewRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint32_t unit = blockIdx.x / p.splits;  // (batch, key head, row tile)
  const int part = static_cast<int>(blockIdx.x - unit * p.splits);
  const uint32_t bh = unit / f.tiles;
  const int first_row = static_cast<int>(unit - bh * f.tiles) * kFewRows;
  const int b = static_cast<int>(bh / f.kv_heads), hk = static_cast<int>(bh) - b * f.kv_heads;
  const int rows = p.group * p.seq_q;
  const int len = p.lens ? min(max(__ldg(p.lens + b), 0), p.seq_kv) : p.seq_kv;
  const int steps_all = (len + kFewKeys - 1) / kFewKeys;
  const int per = (steps_all + p.splits - 1) / p.splits;
  const int step0 = min(part * per, steps_all), step1 = min(step0 + per, steps_all);

  // query row g of the tile, as the second operand of S^T
  uint4 q[kChunks];
  {
    const int r = first_row + g;
    const int h = hk * p.group + r / p.seq_q, s = r % p.seq_q;
    load_row<kChunks>(f.q, b * f.qsb + h * f.qsh + s * f.qss + 8 * c, r < rows, q);
  }
  const int64_t kbase = b * f.ksb + hk * f.ksh + 8 * c, vbase = b * f.vsb + hk * f.vsh + 8 * c;
  auto unmasked = [&](int key) { return !f.mask || (key < len && __ldg(f.mask + b * f.msb + key * f.mss) != 0); };

  float o[2 * kChunks][4] = {};
  float m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};  // rows 2c, 2c + 1
  // Keys and values of this step and the next: both are requested a step ahead,
  // so that a step costs its arithmetic, not a memory access. One token of 4
  // samples with 24 / 8 heads against 4,099 keys each: 14.6 us (4.6 TB/s).
  uint4 k0[kChunks], k1[kChunks], v0[kChunks], v1[kChunks], vn0[kChunks], vn1[kChunks];
  bool keep0 = false, keep1 = false, next0 = false, next1 = false;
  auto request = [&](int at) {
    const int64_t key = static_cast<int64_t>(at) * kFewKeys + g;
    const bool in0 = at < step1 && key < len, in1 = at < step1 && key + 8 < len;
    load_row<kChunks>(f.k, kbase + key * f.kss, in0, k0);
    load_row<kChunks>(f.k, kbase + (key + 8) * f.kss, in1, k1);
    load_row<kChunks>(f.v, vbase + key * f.vss, in0, vn0);
    load_row<kChunks>(f.v, vbase + (key + 8) * f.vss, in1, vn1);
    next0 = in0 && unmasked(static_cast<int>(key));
    next1 = in1 && unmasked(static_cast<int>(key) + 8);
  };
  int step = step0 + warp;
  if (step < step1) request(step);
  for (; step < step1; step += kFewWarps) {
    keep0 = next0;
    keep1 = next1;
    const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {  // what a mask leaves out may hold anything
      v0[j] = keep0 ? vn0[j] : none;
      v1[j] = keep1 ? vn1[j] : none;
    }
    float st[4] = {0.f, 0.f, 0.f, 0.f};  // keys g (0, 1) and g + 8 (2, 3), rows 2c, 2c + 1
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      mma16816<T>(st, k0[j].x, k1[j].x, k0[j].y, k1[j].y, q[j].x, q[j].y);
      mma16816<T>(st, k0[j].z, k1[j].z, k0[j].w, k1[j].w, q[j].z, q[j].w);
    }
    request(step + kFewWarps);
    float pr[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float a = keep0 ? st[e] * p.scale_log2 : kNegInf, d = keep1 ? st[e + 2] * p.scale_log2 : kNegInf;
      float top = fmaxf(a, d);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      const float m_new = fmaxf(m[e], top);
      const float base = m_new == kNegInf ? 0.f : m_new;
      const float alpha = ex2_approx(m[e] - base);
      m[e] = m_new;
      pr[e] = ex2_approx(a - base);
      pr[e + 2] = ex2_approx(d - base);
      l[e] = fmaf(l[e], alpha, pr[e] + pr[e + 2]);
#pragma unroll
      for (int n = 0; n < 2 * kChunks; ++n) {
        o[n][e] *= alpha;
        o[n][e + 2] *= alpha;
      }
    }
    // P^T: keys (2c, 2c + 1) of row g, for the two halves of the 16 keys
    const uint32_t p0 = transpose8x8(pack2<T>(pr[0], pr[1])), p1 = transpose8x8(pack2<T>(pr[2], pr[3]));
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      mma16816<T>(o[2 * j], transpose8x8(v0[j].x), transpose8x8(v0[j].y), transpose8x8(v1[j].x), transpose8x8(v1[j].y), p0, p1);
      mma16816<T>(o[2 * j + 1], transpose8x8(v0[j].z), transpose8x8(v0[j].w), transpose8x8(v1[j].z), transpose8x8(v1[j].w), p0,
                  p1);
    }
  }
  // l over the keys of the warp
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int x = 4; x <= 16; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
    if (g == 0) sml[warp][2 * c + e] = make_float2(m[e], l[e]);
  }
  // o[2j + u]: channels 32 j + 8 (g / 2) + g % 2 + 4 u (values 0, 1) and + 2 (values 2, 3)
#pragma unroll
  for (int n = 0; n < 2 * kChunks; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      so[warp][2 * c + (e & 1)][32 * (n >> 1) + 8 * (g >> 1) + (g & 1) + 4 * (n & 1) + 2 * (e >> 1)] = o[n][e];
  __syncthreads();
  // The CTA's part of each value: thread t takes channels t of all rows, so it
  // is the only one that touches them in the warps' tiles.
  for (int at = threadIdx.x; at < kFewRows * kD; at += kFewWarps * 32) {
    const int r = at / kD, d = at % kD;
    float mx = kNegInf;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) mx = fmaxf(mx, sml[w][r].x);
    const float base = mx == kNegInf ? 0.f : mx;
    float lsum = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float wt = ex2_approx(sml[w][r].x - base);
      lsum = fmaf(wt, sml[w][r].y, lsum);
      sum = fmaf(wt, so[w][r][d], sum);
    }
    so[0][r][d] = sum;
    if (d == 0) part_ml[r] = make_float2(mx, lsum);
  }
  __syncthreads();
  const bool clustered = f.clustered != 0;
  if (clustered) cluster_sync();
  // Rows of this CTA: all of a unit's only part or of a part for the second
  // kernel, every splits-th one in a cluster.
  const int row_step = clustered ? p.splits : 1;
  for (int e = threadIdx.x; e < kFewRows * kD; e += kFewWarps * 32) {
    const int r = e / kD, d = e % kD, row = first_row + r;
    if (row >= rows) break;
    if (clustered && r % row_step != part) continue;
    float sum = so[0][r][d], lsum = part_ml[r].y;
    if (clustered) {
      float mx = kNegInf;
      for (int q = 0; q < p.splits; ++q) mx = fmaxf(mx, ld_cluster_f32(map_to_rank(&part_ml[r].x, q)));
      const float base = mx == kNegInf ? 0.f : mx;
      sum = lsum = 0.f;
      for (int q = 0; q < p.splits; ++q) {
        const float wt = ex2_approx(ld_cluster_f32(map_to_rank(&part_ml[r].x, q)) - base);
        lsum = fmaf(wt, ld_cluster_f32(map_to_rank(&part_ml[r].y, q)), lsum);
        sum = fmaf(wt, ld_cluster_f32(map_to_rank(&so[0][r][d], q)), sum);
      }
    } else if (p.splits > 1) {
      const int64_t slot = (static_cast<int64_t>(unit) * p.splits + part) * kFewRows + r;
      p.part_o[slot * kD + d] = sum;
      if (d == 0) p.part_ml[slot] = part_ml[r];
      continue;
    }
    const int h = hk * p.group + row / p.seq_q, s = row % p.seq_q;
    const float v = lsum != 0.f ? sum / lsum : 0.f;
    T* dst = static_cast<T*>(p.out) + b * p.osb + h * p.osh + s * p.oss + d;
    if constexpr (std::is_same<T, __half>::value) *dst = __float2half_rn(v);
    else *dst = __float2bfloat16_rn(v);
  }
  if (clustered) cluster_sync();  // nobody leaves while its part is read
}

// Joins the parts of a row: M = max m, o = sum 2^(m - M) O / sum 2^(m - M) l.
// A block a row; its warps share the parts, of which there may be hundreds. A
// part without keys (l = 0) left no O.
constexpr int kMostParts = 512;
template <typename T, int kD, int kJoinWarps>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const Params p, int few_tiles) {
  __shared__ float so[kJoinWarps][kD], sl[kJoinWarps], sm[kJoinWarps], weight[kMostParts];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bh = blockIdx.x / static_cast<uint32_t>(p.seq_q);  // (batch, head)
  const int row = static_cast<int>(blockIdx.x - bh * p.seq_q);
  const int b = static_cast<int>(bh / p.heads), h = static_cast<int>(bh) - b * p.heads;
  int64_t item = static_cast<int64_t>(bh) * p.n_qt + row / kRows;
  int r = row % kRows;
  if (few_tiles) {  // rows of a key head in tiles of 8
    const int in_head = h % p.group * p.seq_q + row;
    item = (static_cast<int64_t>(b) * (p.heads / p.group) + h / p.group) * few_tiles + in_head / kFewRows;
    r = in_head % kFewRows;
  }
  const int64_t first = item * p.splits * p.part_rows + r;
  auto at = [&](int q) { return first + static_cast<int64_t>(q) * p.part_rows; };
  float mx = kNegInf;
  for (int q = threadIdx.x; q < p.splits; q += kJoinWarps * 32) mx = fmaxf(mx, __ldg(&p.part_ml[at(q)]).x);
  mx = warp_max(mx);
  if (lane == 0) sm[warp] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) mx = fmaxf(mx, sm[w]);
  const float base = mx == kNegInf ? 0.f : mx;
  float l = 0.f;
  for (int q = threadIdx.x; q < p.splits; q += kJoinWarps * 32) {
    const float2 ml = __ldg(&p.part_ml[at(q)]);
    const float w = ml.y != 0.f ? ex2_approx(ml.x - base) : 0.f;
    weight[q] = ml.y != 0.f ? w : -1.f;  // no O to read
    l = fmaf(w, ml.y, l);
  }
  l = warp_sum(l);
  __syncthreads();
  // predicated loads, so that eight parts are on their way at once
  float o[kD / 32] = {};
#pragma unroll 8
  for (int q = warp; q < p.splits; q += kJoinWarps) {
    const float w = weight[q];
    const float* po = p.part_o + at(q) * kD + lane;
#pragma unroll
    for (int c = 0; c < kD / 32; ++c) o[c] = fmaf(w, w != -1.f ? __ldg(po + c * 32) : 0.f, o[c]);
  }
#pragma unroll
  for (int c = 0; c < kD / 32; ++c) so[warp][c * 32 + lane] = o[c];
  if (lane == 0) sl[warp] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) l += sl[w];
  const float inv_l = l != 0.f ? 1.0f / l : 0.f;
  T* dst = static_cast<T*>(p.out) + b * p.osb + h * p.osh + row * p.oss;
  for (int d = threadIdx.x; d < kD; d += kJoinWarps * 32) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) v += so[w][d];
    if constexpr (std::is_same<T, __half>::value) dst[d] = __float2half_rn(v * inv_l);
    else dst[d] = __float2bfloat16_rn(v * inv_l);
  }
}

// 4 warps a row, 16 where there are more parts than those take at once (444
// parts: 29 us with 4 warps, 12 us with 16).
template <typename T, int kD>
int join(const Params& p, int64_t rows, int few_tiles, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>(rows);
  if (p.splits > 64) join_kernel<T, kD, 16><<<grid, 512, 0, st>>>(p, few_tiles);
  else join_kernel<T, kD, 4><<<grid, 128, 0, st>>>(p, few_tiles);
  return launch_status();
}

int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

// How a call is laid out. The few-row form takes up to 8 query rows of a key
// head; up to 24 where several query heads share long keys, which the tiled
// kernel would read once for each of them. Measured, few / tiled, D = 128:
//   24 heads, rows 8, 512 keys: 6 / 10 us       rows 16: 13.8 / 10.4 us
//   rows 16, 4,096 keys, own keys: 28 / 19 us
//   rows 12 of 3 shared heads, batch 4: 512 keys 16 / 12 us, 4,096 keys 37 / 57 us
//   rows 30 of 3 shared heads, batch 4, 4,096 keys: 61 / 56 us
inline bool takes_few(int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_kv) {
  const int64_t rows = heads / kv_heads * seq_q;
  return rows <= kFewRows || (heads > kv_heads && rows <= 3 * kFewRows && seq_kv >= 1024);
}
struct Plan {
  bool few;
  int tiles;  // few: row tiles of a key head
  int64_t items;
  int splits;
  bool clustered;
  int64_t part_rows;
};
inline Plan plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_kv, int sms) {
  Plan n{};
  const int64_t rows = heads / kv_heads * seq_q;
  n.few = takes_few(heads, kv_heads, seq_q, seq_kv);
  if (n.few) {
    n.tiles = static_cast<int>(cdiv(rows, kFewRows));
    n.items = batch * kv_heads * n.tiles;
    // Two CTAs an SM (as many as are resident at D = 128), each with a step for
    // each of its warps. A cluster of up to 8 parts needs no second kernel; it
    // is taken as soon as it gives every SM a CTA. With one, two and three CTAs
    // an SM: 100,000 keys of one head 17, 19 and 25 us, 16,384 of 8 heads 18,
    // 17 and 22 us, 512 of 24 heads 7.4, 6.5 and 6.6 us.
    const int64_t most = cdiv(seq_kv, kFewKeys * kFewWarps);
    n.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({2 * sms / n.items, most, kMostParts})));
    n.clustered = n.splits > 1 && (n.splits <= 8 || n.items * 8 >= sms);
    if (n.clustered) n.splits = std::min(n.splits, 8);
    n.part_rows = kFewRows;
    return n;
  }
  n.items = batch * heads * cdiv(seq_q, kRows);
  n.splits = 1;
  // parts only where whole units would leave more than half of the SMs idle
  if (n.items * 2 <= sms) n.splits = static_cast<int>(std::min<int64_t>({sms / n.items, cdiv(seq_kv, kBN), kMostParts}));
  n.part_rows = std::min<int64_t>(seq_q, kRows);
  return n;
}

template <typename T, int kD>
int launch(const CUtensorMap (&map)[4], const Params& p, int64_t batch, int sms, cudaStream_t st) {
  using C = Cfg<T, kD>;
  auto kernel = cross_attention_kernel<T, kD>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess)
    return XGB_ERR_LAUNCH;
  const int grid = std::min(static_cast<int>(p.units), sms);
  kernel<<<grid, kThreads, C::kSmem, st>>>(map[0], map[1], map[2], map[3], p);
  const int rc = launch_status();
  if (rc || p.splits == 1) return rc;
  return join<T, kD>(p, batch * p.heads * p.seq_q, 0, st);
}

template <typename T, int kD>
int launch_few(const Params& p, const FewParams& f, int64_t items, int64_t batch, cudaStream_t st) {
  const int64_t grid = items * p.splits;
  if (grid > INT32_MAX) return XGB_ERR_SHAPE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kFewWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(f.clustered ? p.splits : 1);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, cross_few_kernel<T, kD>, p, f) != cudaSuccess) {
    cudaGetLastError();
    return XGB_ERR_LAUNCH;
  }
  const int rc = launch_status();
  if (rc || p.splits == 1 || f.clustered) return rc;
  return join<T, kD>(p, batch * p.heads * p.seq_q, f.tiles, st);
}

// ---------------------------------------------------------------- masked keys
// Gathers the keys and values that a mask keeps to the front of packed
// [batch, heads, seq_kv, D] tensors, in order, and counts them; what lies
// behind the count is not written. A block takes 64 keys of one sample and
// counts the kept ones before its own.
template <int kWords>
__global__ void __launch_bounds__(256) pack_keys_kernel(const uint8_t* __restrict__ mask, int64_t msb, int64_t mss,
                                                        const uint4* __restrict__ k, int64_t ksb, int64_t ksh, int64_t kss,
                                                        const uint4* __restrict__ v, int64_t vsb, int64_t vsh, int64_t vss,
                                                        int heads, int seq, uint4* __restrict__ k_out,
                                                        uint4* __restrict__ v_out, int* __restrict__ counts) {
  __shared__ int red[8];
  __shared__ int place[kBN];
  const int b = blockIdx.y, first = blockIdx.x * kBN;
  const uint8_t* row = mask + b * msb;
  int before = 0;
  for (int j = threadIdx.x; j < first; j += 256) before += row[j * mss] != 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) before += red[w];
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int at = before;
    for (int c = 0; c < kBN / 32; ++c) {
      const int j = first + c * 32 + lane;
      const bool keep = j < seq && row[j * mss] != 0;
      const uint32_t kept = __ballot_sync(0xffffffffu, keep);
      place[c * 32 + lane] = keep ? at + __popc(kept & ((1u << lane) - 1)) : -1;
      at += __popc(kept);
    }
    if (lane == 0 && first + kBN >= seq && blockIdx.z == 0) counts[b] = at;
  }
  __syncthreads();
  // kWords pieces of 16 bytes a row; a block's heads are blockIdx.z, + gridDim.z, ..
  const int w = threadIdx.x % kWords;
  for (int h = blockIdx.z; h < heads; h += gridDim.z) {
#pragma unroll
    for (int j = threadIdx.x / kWords; j < kBN; j += 256 / kWords) {
      const int to = place[j];
      if (to < 0) continue;
      const int64_t dst = ((static_cast<int64_t>(b) * heads + h) * seq + to) * kWords + w;
      const uint4 kw = __ldg(k + b * ksb + h * ksh + (first + j) * kss + w);
      const uint4 vw = __ldg(v + b * vsb + h * vsh + (first + j) * vss + w);
      k_out[dst] = kw;
      v_out[dst] = vw;
    }
  }
}

inline bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

}  // namespace cross
}  // namespace xgb

using namespace xgb;

XGB_API int xgb_pack_keys(const uint8_t* mask, int64_t mask_batch_stride, int64_t mask_stride, const void* k,
                          const int64_t* k_strides, const void* v, const int64_t* v_strides, int64_t batch, int64_t heads,
                          int64_t seq, int64_t head_dim, void* k_out, void* v_out, int* counts, void* stream) {
  if (!mask || !k || !v || !k_strides || !v_strides || !k_out || !v_out || !counts) return XGB_ERR_ARG;
  if (batch <= 0 || batch > 65535 || heads <= 0 || heads > 65535 || seq <= 0 || seq > (1 << 30) ||
      (head_dim != 64 && head_dim != 128))
    return XGB_ERR_SHAPE;
  const int64_t extent[3] = {batch, heads, seq};
  for (int d = 0; d < 3; ++d)
    if (extent[d] > 1 && (k_strides[d] % 8 || v_strides[d] % 8)) return XGB_ERR_STRIDE;
  if (k_strides[3] != 1 || v_strides[3] != 1) return XGB_ERR_STRIDE;
  if (!cross::aligned16(k) || !cross::aligned16(v) || !cross::aligned16(k_out) || !cross::aligned16(v_out))
    return XGB_ERR_ALIGN;
  // enough blocks to fill the GPU a few times; further heads in a loop
  const int64_t tiles = cdiv(seq, cross::kBN) * batch;
  const dim3 grid(static_cast<unsigned>(cdiv(seq, cross::kBN)), static_cast<unsigned>(batch),
                  static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(heads, 148 * 8 / tiles))));
  auto run = [&](auto kernel) {
    kernel<<<grid, 256, 0, as_stream(stream)>>>(
        mask, mask_batch_stride, mask_stride, static_cast<const uint4*>(k), k_strides[0] / 8, k_strides[1] / 8,
        k_strides[2] / 8, static_cast<const uint4*>(v), v_strides[0] / 8, v_strides[1] / 8, v_strides[2] / 8,
        static_cast<int>(heads), static_cast<int>(seq), static_cast<uint4*>(k_out), static_cast<uint4*>(v_out), counts);
    return launch_status();
  };
  return head_dim == 64 ? run(cross::pack_keys_kernel<8>) : run(cross::pack_keys_kernel<16>);
}

XGB_API int64_t xgb_cross_attention_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_kv,
                                              int64_t head_dim) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || seq_q <= 0 || seq_kv <= 0) return 0;
  const cross::Plan n = cross::plan(batch, heads, kv_heads, seq_q, seq_kv, cross::sm_count());
  if (n.splits <= 1 || n.clustered) return 0;
  return n.items * n.splits * n.part_rows * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

XGB_API int xgb_cross_attention_takes_mask(int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_kv) {
  return heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && seq_q > 0 && seq_kv > 0 &&
         cross::takes_few(heads, kv_heads, seq_q, seq_kv);
}

XGB_API int xgb_cross_attention(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                const void* v, const int64_t* v_strides, int dtype, int64_t batch, int64_t heads,
                                int64_t kv_heads, int64_t seq_q, int64_t seq_kv, int64_t head_dim, const int* kv_lens,
                                const uint8_t* mask, int64_t mask_batch_stride, int64_t mask_stride, float sm_scale,
                                void* out, const int64_t* out_strides, void* workspace, int64_t workspace_bytes,
                                int* error_flag, void* stream) {
  if (!q || !k || !v || !out || !q_strides || !k_strides || !v_strides || !out_strides) return XGB_ERR_ARG;
  if (dtype != XGB_BF16 && dtype != XGB_F16) return XGB_ERR_ARG;
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || seq_q <= 0 || seq_kv <= 0 || seq_q > (1 << 30) ||
      seq_kv > (1 << 30) || batch > 65535 || heads > 65535 || (head_dim != 64 && head_dim != 128))
    return XGB_ERR_SHAPE;
  if (!(sm_scale > 0.f)) return XGB_ERR_ARG;
  const int64_t* all[4] = {q_strides, k_strides, v_strides, out_strides};
  for (int t = 0; t < 4; ++t) {
    const int64_t extent[3] = {batch, t == 1 || t == 2 ? kv_heads : heads, t == 1 || t == 2 ? seq_kv : seq_q};
    if (all[t][3] != 1) return XGB_ERR_STRIDE;
    for (int d = 0; d < 3; ++d) {
      if (extent[d] == 1) continue;  // never stepped over
      // inputs may be broadcast over the batch and the heads
      if (all[t][d] % 8 || all[t][d] < 0 || (all[t][d] == 0 && (t == 3 || d == 2))) return XGB_ERR_STRIDE;
    }
  }
  if (!cross::aligned16(q) || !cross::aligned16(k) || !cross::aligned16(v) || !cross::aligned16(out)) return XGB_ERR_ALIGN;
  if (mask && !xgb_cross_attention_takes_mask(heads, kv_heads, seq_q, seq_kv)) return XGB_ERR_SHAPE;
  const int sms = cross::sm_count();
  const cross::Plan n = cross::plan(batch, heads, kv_heads, seq_q, seq_kv, sms);
  const int64_t need = xgb_cross_attention_workspace(batch, heads, kv_heads, seq_q, seq_kv, head_dim);
  if (need && (!workspace || workspace_bytes < need)) return XGB_ERR_WORKSPACE;
  if (need && !cross::aligned16(workspace)) return XGB_ERR_ALIGN;
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10)
    return XGB_ERR_DEVICE;
  cross::Params p{};
  p.heads = static_cast<int>(heads);
  p.group = static_cast<int>(heads / kv_heads);
  p.seq_q = static_cast<int>(seq_q);
  p.seq_kv = static_cast<int>(seq_kv);
  p.lens = kv_lens;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.out = out;
  p.osb = out_strides[0];
  p.osh = out_strides[1];
  p.oss = out_strides[2];
  p.n_qt = static_cast<int>(cdiv(seq_q, cross::kRows));
  p.splits = n.splits;
  if (n.items * n.splits > INT32_MAX - 65536) return XGB_ERR_SHAPE;  // room for a walk's last step
  p.units = static_cast<uint32_t>(n.items * n.splits);
  p.div_splits = make_fastdiv(static_cast<uint32_t>(n.splits));
  p.div_qt = make_fastdiv(static_cast<uint32_t>(p.n_qt));
  p.div_heads = make_fastdiv(static_cast<uint32_t>(heads));
  p.div_group = make_fastdiv(static_cast<uint32_t>(p.group));
  p.part_rows = static_cast<int>(n.part_rows);
  if (need) {
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + n.items * n.splits * p.part_rows * head_dim);
  }
  p.err = error_flag;
  cudaStream_t st = as_stream(stream);
  const bool bf16 = dtype == XGB_BF16;
  if (n.few) {
    cross::FewParams f{};
    f.q = q;
    f.k = k;
    f.v = v;
    f.qsb = q_strides[0];
    f.qsh = q_strides[1];
    f.qss = q_strides[2];
    f.ksb = k_strides[0];
    f.ksh = k_strides[1];
    f.kss = k_strides[2];
    f.vsb = v_strides[0];
    f.vsh = v_strides[1];
    f.vss = v_strides[2];
    f.mask = mask;
    f.msb = mask_batch_stride;
    f.mss = mask_stride;
    f.kv_heads = static_cast<int>(kv_heads);
    f.tiles = n.tiles;
    f.clustered = n.clustered;
    if (bf16)
      return head_dim == 128 ? cross::launch_few<__nv_bfloat16, 128>(p, f, n.items, batch, st)
                             : cross::launch_few<__nv_bfloat16, 64>(p, f, n.items, batch, st);
    return head_dim == 128 ? cross::launch_few<__half, 128>(p, f, n.items, batch, st)
                           : cross::launch_few<__half, 64>(p, f, n.items, batch, st);
  }
  CUtensorMap map[4];
  const void* base[4] = {q, k, v, out};
  int factor[4][2];  // batch, head
  for (int t = 0; t < 4; ++t) {
    const bool rows = t == 0 || t == 3;
    const int64_t* s = all[t];
    const int64_t seq = rows ? seq_q : seq_kv, hh = rows ? heads : kv_heads;
    // a dimension of one entry, or a broadcast one, is one entry of the map
    const int64_t ext[3] = {seq, hh > 1 && s[1] ? hh : 1, batch > 1 && s[0] ? batch : 1};
    factor[t][0] = ext[2] > 1;
    factor[t][1] = ext[1] > 1;
    const uint64_t dims[4] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(ext[0]), static_cast<uint64_t>(ext[1]),
                              static_cast<uint64_t>(ext[2])};
    const uint64_t row = static_cast<uint64_t>(head_dim) * 2;
    const uint64_t strides[3] = {ext[0] > 1 ? static_cast<uint64_t>(s[2]) * 2 : row,
                                 ext[1] > 1 ? static_cast<uint64_t>(s[1]) * 2 : row,
                                 ext[2] > 1 ? static_cast<uint64_t>(s[0]) * 2 : row};
    const uint32_t box[4] = {64, static_cast<uint32_t>(t == 0 ? cross::kBM : t == 3 ? 32 : cross::kBN), 1, 1};
    if (!make_tensor_map(&map[t], bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         base[t], dims, strides, box))
      return XGB_ERR_ALIGN;
  }
  p.qb = factor[0][0];
  p.qh = factor[0][1];
  p.kb = factor[1][0];
  p.kh = factor[1][1];
  p.vb = factor[2][0];
  p.vh = factor[2][1];
  if (bf16)
    return head_dim == 128 ? cross::launch<__nv_bfloat16, 128>(map, p, batch, sms, st)
                           : cross::launch<__nv_bfloat16, 64>(map, p, batch, sms, st);
  return head_dim == 128 ? cross::launch<__half, 128>(map, p, batch, sms, st)
                         : cross::launch<__half, 64>(map, p, batch, sms, st);
}
