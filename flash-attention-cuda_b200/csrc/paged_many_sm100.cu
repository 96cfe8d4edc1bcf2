// Attention of many new tokens per sequence over a paged K/V cache: prompt
// chunks, alone or with sequences in generation beside them
// (fa_attend_paged).
//
//   o_i = sum_j exp(scale q_i k_j - m_i) v_j / l_i,  j over the rows that
//   token i sees, m_i and l_i the running maximum and sum.
//
// Bound: the tensor cores at head_dim 128, the exponentials at 64. An item
// is two 128-row tiles of query rows (new token, head of the group) against
// the key tiles of one K/V head, each tile of keys loaded once for both:
// S_t = Q_t K^T and O_t += P_t V_t by tcgen05, S and O in tensor memory, P
// written over S as 16-bit values. The two tiles take turns, so the tensor
// cores work on one while the other's softmax runs. One CTA per SM walks its
// piece of the step (paged_sm100.cuh); nothing of it starts over between
// items: the next item's queries and keys load while this one ends.
//
// CTA = 12 warps:
//   0-3 / 4-7  softmax of query tile 0 / 1 (thread = row = TMEM lane)
//   8          TMA producer: lane j loads page j of a key tile
//   9          MMA issuer (one elected thread); owns the TMEM allocation
//   10-11      idle (they give their registers to the softmax warps)
//
// Shared memory: Q_t (128 rows x D), then a ring of key tiles (K and V, 128
// rows x D each: 2 at D 128, 5 at 64), rows as 128-byte-swizzled halves of
// 64 dims. Tensor memory: S_t at 128 t (P_t over its first 64 columns), O_t
// at 256 + D t.

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "fa_kernels.h"
#include "fa_sm100.cuh"
#include "paged_sm100.cuh"

namespace fa {
namespace paged {
namespace many {

constexpr int kRows = 128;  // query rows of a tile
constexpr int kThreads = 384;
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kCtrlRegs = 24;
constexpr int kSoftmaxRegs = 240;
static_assert(128 * kCtrlRegs + 256 * kSoftmaxRegs <= kThreads * 168,
              "register split exceeds the launch allocation");
// O is rescaled only when a row's maximum has grown by more than this (in
// log2 units): P stays below 2^8, in range of both 16-bit types.
constexpr float kRescaleThreshold = 8.0f;

template <int D>
struct Cfg {
  static constexpr uint32_t kHalf = kTileRows * 128;  // 64 dims of 128 rows
  static constexpr uint32_t kTile = D / 64 * kHalf;   // Q_t, K or V
  static constexpr uint32_t kStage = 2 * kTile;
  static constexpr int kStages = D == 128 ? 2 : 5;
  static constexpr uint32_t kQOff = 0;
  static constexpr uint32_t kRingOff = 2 * kTile;
  static constexpr uint32_t kBarOff = kRingOff + kStages * kStage;
  static constexpr int kFull = 0;                    // + stage
  static constexpr int kEmpty = kFull + kStages;     // + stage
  static constexpr int kTail = kEmpty + kStages;     // a tile past the end
  static constexpr int kQFull = kTail + 1;           // + tile
  static constexpr int kQEmpty = kQFull + 2;         // + tile
  static constexpr int kSFull = kQEmpty + 2;         // + tile
  static constexpr int kPFull = kSFull + 2;          // + tile
  static constexpr int kODone = kPFull + 2;          // + tile
  static constexpr int kJoin = kODone + 2;           // + tile
  static constexpr int kDrain = kJoin + 2;
  static constexpr int kBars = kDrain + 1;
  static constexpr uint32_t kMiscOff = kBarOff + kBars * 8;
  // plan, TMEM address, abort flag, per-tile join flags
  static constexpr uint32_t kSmemBytes = kMiscOff + sizeof(PlanSmem) + 32;
  static_assert(kSmemBytes + 1024 <= 228 * 1024, "above the SM's shared memory");
  static constexpr uint32_t kTmemO = 256;  // + D * tile
  // a partial of one tile: O as [D / 4][row] float4, then m and l per row
  static constexpr int kSlotFloats = kRows * (D + 2);
};

template <typename Dt>
constexpr uint32_t kIdescS = idesc_f16_f32(kRows, kTileRows, false, Dt::kFmt);
template <int D, typename Dt>
constexpr uint32_t kIdescPV = idesc_f16_f32(kRows, D, true, Dt::kFmt);

// S = Q K^T of one tile: D / 16 MMAs.
template <int D, typename Dt>
__device__ __forceinline__ void issue_s(uint32_t d, uint64_t q, uint64_t k) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint64_t off = (kk >> 2) * (Cfg<D>::kHalf >> 4) + 2 * (kk & 3);
    mma_f16_ss(d, q + off, k + off, kIdescS<Dt>, kk > 0 ? 1u : 0u);
  }
}

// O (+)= P V of one tile: 8 MMAs of 16 keys each.
template <int D, typename Dt>
__device__ __forceinline__ void issue_pv(uint32_t d, uint32_t p, uint64_t v,
                                         bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < kTileRows / 16; ++kk)
    mma_f16_ts(d, p + 8 * kk, v + 128 * kk, kIdescPV<D, Dt>,
               accumulate || kk > 0 ? 1u : 0u);
}

// V's descriptor: its 64-dim halves are kHalf bytes apart (leading offset).
template <int D>
__device__ __forceinline__ uint64_t v_desc(uint32_t addr) {
  return (sw128_desc(addr) & ~(0x3FFFull << 16)) |
         (static_cast<uint64_t>(Cfg<D>::kHalf >> 4) << 16);
}

// Tokens of a tile, and the end of tile t's key tiles within a part (its
// start if the tile has no token or no key there).
__device__ __forceinline__ int tile_tokens(const PagedArgs &a) {
  return a.item_tokens / 2;
}
__device__ __forceinline__ int tile_end(const PagedArgs &a, const Part &it, int t) {
  const int first = it.token + t * tile_tokens(a);
  const int last = min(first + tile_tokens(a), it.seq.n) - 1;
  if (last < first) return it.t0;
  const int tiles = (rows_seen(a, it.seq, last) + a.tile_keys - 1) / a.tile_keys;
  return max(it.t0, min(it.t1, tiles));
}

struct Ctrl {
  uint32_t tmem;
  volatile uint32_t abort;
  uint32_t join[2];
};

template <int D>
__device__ void produce(const PagedArgs &a, Walk &walk, uint8_t *smem,
                        uint64_t *bars, Ctrl *ctrl, const CUtensorMap *tm_q,
                        const CUtensorMap *tm_k, const CUtensorMap *tm_v) {
  using C = Cfg<D>;
  const int lane = threadIdx.x & 31;
  const int group = a.H / a.H_kv;
  const int box = min(a.page_rows, kTileRows);
  int pos = 0, q_used[2] = {0, 0};
  uint32_t tail_phase = 0;
  bool ok = true;
  Part it;
  while (ok && walk.next(a, it)) {
    int page = it.t0 < it.t1 ? tile_page(a, it.b, it.keys, it.t0, lane) : -1;
    for (int t = 0; ok && t < 2; ++t) {
      if (tile_end(a, it, t) <= it.t0) continue;
      if (q_used[t] > 0 && !mbar_wait(&bars[C::kQEmpty + t], (q_used[t] - 1) & 1)) {
        ok = false;
        break;
      }
      ++q_used[t];
      if (lane == 0) {
        uint64_t *bar = &bars[C::kQFull + t];
        mbar_arrive_expect_tx(bar, tile_tokens(a) * group * 128 * (D / 64));
        for (int h = 0; h < D / 64; ++h)
          tma_load_4d(smem + C::kQOff + t * C::kTile + h * C::kHalf, tm_q, bar,
                      64 * h, 0, it.h, it.seq.lo + it.token + t * tile_tokens(a));
      }
    }
    for (int i = it.t0; ok && i < it.t1; ++i, ++pos) {
      const int next = i + 1 < it.t1 ? tile_page(a, it.b, it.keys, i + 1, lane) : -1;
      const int slot = pos % C::kStages, use = pos / C::kStages;
      if (ctrl->abort ||
          (use > 0 && !mbar_wait(&bars[C::kEmpty + slot], (use - 1) & 1))) {
        ok = false;
        break;
      }
      // A tile that reaches past the sequence's rows goes through a barrier
      // of its own: its V rows there may hold anything, NaN included, and are
      // cleared before the tile is handed on (P is zero there, and zero times
      // NaN is not).
      const int valid = it.keys - i * a.tile_keys;
      const bool tail = valid < a.tile_keys;
      uint64_t *bar = &bars[tail ? C::kTail : C::kFull + slot];
      const uint32_t pages = __ballot_sync(0xffffffffu, page >= 0);
      if (lane == 0)
        mbar_arrive_expect_tx(bar, __popc(pages) * box * 128 * (D / 64) * 2);
      __syncwarp();
      uint8_t *stage = smem + C::kRingOff + slot * C::kStage;
      if (page >= 0) {
        const int row = a.page_rows < kTileRows ? 0 : i * a.tile_keys % a.page_rows;
        uint8_t *to = stage + lane * box * 128;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          tma_load_4d(to + h * C::kHalf, tm_k, bar, 64 * h, row, it.h, page);
          tma_load_4d(to + C::kTile + h * C::kHalf, tm_v, bar, 64 * h, row, it.h, page);
        }
      }
      if (tail) {
        ok = mbar_wait(bar, tail_phase);
        tail_phase ^= 1;
        for (int h = 0; h < D / 64; ++h)
          for (int e = valid * 8 + lane; e < a.tile_keys * 8; e += 32)
            *reinterpret_cast<uint4 *>(stage + C::kTile + h * C::kHalf + 16 * e) =
                make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[C::kFull + slot]);
      }
      page = next;
    }
  }
  if (!ok) {
    ctrl->abort = 1;
    // no copy of ours may still be landing when the CTA exits
    for (int t = 0; t < 2; ++t)
      if (q_used[t] > 0) mbar_wait(&bars[C::kQFull + t], (q_used[t] - 1) & 1);
    for (int p = pos > C::kStages ? pos - C::kStages : 0; p < pos; ++p)
      mbar_wait(&bars[C::kFull + p % C::kStages], (p / C::kStages) & 1);
  }
}

template <int D, typename Dt>
__device__ void issue(const PagedArgs &a, Walk &walk, uint8_t *smem,
                      uint64_t *bars, Ctrl *ctrl) {
  using C = Cfg<D>;
  const bool leader = elect_one();
  const uint32_t tmem = __shfl_sync(0xffffffffu, ctrl->tmem, 0);
  const uint32_t sbase = smem_u32(smem);
  const uint64_t desc0 = sw128_desc(sbase);
  const uint64_t vdesc0 = v_desc<D>(sbase);
  auto s_tile = [&](int t, int pos) {
    if (leader) {
      issue_s<D, Dt>(tmem + 128 * t, desc0 + ((C::kQOff + t * C::kTile) >> 4),
                     desc0 + ((C::kRingOff + pos % C::kStages * C::kStage) >> 4));
      mma_commit(&bars[C::kSFull + t]);
    }
    __syncwarp();
  };
  int pos = 0;                // ring position of the part's first tile
  int q_used[2] = {0, 0};     // queries taken
  int done[2] = {0, 0};       // P V products issued
  bool ok = true;
  Part it;
  while (ok && walk.next(a, it)) {
    if (it.t0 >= it.t1) continue;
    const int end[2] = {tile_end(a, it, 0), tile_end(a, it, 1)};
    // first S of each tile; its tensor memory was P of the last item
    for (int t = 0; ok && t < 2; ++t) {
      if (end[t] <= it.t0) continue;
      ok = mbar_wait(&bars[C::kQFull + t], q_used[t] & 1) &&
           mbar_wait(&bars[C::kFull + pos % C::kStages], (pos / C::kStages) & 1) &&
           (done[t] == 0 || mbar_wait(&bars[C::kODone + t], (done[t] - 1) & 1));
      if (!ok) break;
      ++q_used[t];
      tc_fence_after();
      s_tile(t, pos);
      if (leader && end[t] == it.t0 + 1) mma_commit(&bars[C::kQEmpty + t]);
      __syncwarp();
    }
    for (int j = it.t0; ok && j < it.t1; ++j, ++pos) {
      if (ctrl->abort) {
        ok = false;
        break;
      }
      const int slot = pos % C::kStages;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!ok || j >= end[t]) continue;
        if (!mbar_wait(&bars[C::kPFull + t], done[t] & 1)) {
          ok = false;
          continue;
        }
        tc_fence_after();
        if (leader) {
          issue_pv<D, Dt>(tmem + C::kTmemO + D * t, tmem + 128 * t,
                          vdesc0 + ((C::kRingOff + slot * C::kStage + C::kTile) >> 4),
                          j > it.t0);
          mma_commit(&bars[C::kODone + t]);
          // the last product of the key tile frees its stage
          if (t == 1 || j >= end[1]) mma_commit(&bars[C::kEmpty + slot]);
        }
        __syncwarp();
        ++done[t];
        if (j + 1 < end[t]) {
          // S(j + 1) is written over P(j): P V(j) has to be done
          const int p1 = pos + 1;
          if (!mbar_wait(&bars[C::kFull + p1 % C::kStages], (p1 / C::kStages) & 1) ||
              !mbar_wait(&bars[C::kODone + t], (done[t] - 1) & 1)) {
            ok = false;
            continue;
          }
          tc_fence_after();
          s_tile(t, p1);
          if (leader && j + 2 == end[t]) mma_commit(&bars[C::kQEmpty + t]);
          __syncwarp();
        }
      }
    }
  }
  if (!ok && leader) ctrl->abort = 1;
  if (leader) mma_commit(&bars[C::kDrain]);
  __syncwarp();
  mbar_wait(&bars[C::kDrain], 0);
}

// Maximum of a row's 128 scores, NaN if one is (three inputs a step, eight
// chains).
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float row_max_nan(const float (&s)[128]) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = s[i];
#pragma unroll
  for (int c = 8; c + 16 <= 128; c += 16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = max3_nan(x[i], s[c + i], s[c + 8 + i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = max3_nan(x[i], s[120 + i], s[120 + i]);
  return max3_nan(max3_nan(x[0], x[1], x[2]), max3_nan(x[3], x[4], x[5]),
                  max3_nan(x[6], x[7], x[7]));
}

// 32 dims of a row (fp32 words) scaled to the output.
template <int D, typename Dt>
__device__ __forceinline__ void store_dims(__half *dst, const uint32_t (&o)[32],
                                           float inv) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t *s = &o[8 * c];
    uint4 v;
    v.x = Dt::pack2(__uint_as_float(s[0]) * inv, __uint_as_float(s[1]) * inv);
    v.y = Dt::pack2(__uint_as_float(s[2]) * inv, __uint_as_float(s[3]) * inv);
    v.z = Dt::pack2(__uint_as_float(s[4]) * inv, __uint_as_float(s[5]) * inv);
    v.w = Dt::pack2(__uint_as_float(s[6]) * inv, __uint_as_float(s[7]) * inv);
    reinterpret_cast<uint4 *>(dst)[c] = v;
  }
}

template <int D, typename Dt>
__device__ void soften(const PagedArgs &a, const Division &d, Walk &walk,
                       uint64_t *bars, Ctrl *ctrl) {
  using C = Cfg<D>;
  const int warp = threadIdx.x >> 5;
  const int t = warp >> 2;
  const int row = threadIdx.x & 127;
  const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const uint32_t tS = ctrl->tmem + lane_addr + 128 * t;
  const uint32_t tO = ctrl->tmem + lane_addr + C::kTmemO + D * t;
  const int group = a.H / a.H_kv;
  const int tok = row / group;  // token of this row within its tile
  int done = 0;                 // key tiles of this query tile so far
  uint32_t met = 0;
  Part it;
  while (walk.next(a, it)) {
    const int token = it.token + t * tile_tokens(a) + tok;
    const bool real = tok < tile_tokens(a) && token < it.seq.n;
    const int seen = real ? rows_seen(a, it.seq, token) : 0;
    const int end = tile_end(a, it, t);
    // a warp without a row only keeps the tile's barriers going
    const bool idle = !__any_sync(0xffffffffu, real);
    // keys that every row of the tile sees
    const int all_see = rows_seen(a, it.seq, it.token + t * tile_tokens(a));
    float m = -INFINITY, l = 0.f;

    for (int j = it.t0; j < end; ++j, ++done) {
      if (ctrl->abort || !mbar_wait(&bars[C::kSFull + t], done & 1)) {
        ctrl->abort = 1;
        return;
      }
      if (idle) {
        mbar_arrive(&bars[C::kPFull + t]);
        continue;
      }
      tc_fence_after();
      uint32_t sr[4][32];
      tmem_ld32(tS + 0, sr[0]);
      tmem_ld32(tS + 32, sr[1]);
      tmem_ld32(tS + 64, sr[2]);
      tmem_ld32(tS + 96, sr[3]);
      tmem_wait_ld();
      float s[128];
#pragma unroll
      for (int c = 0; c < 128; ++c) s[c] = __uint_as_float(sr[c >> 5][c & 31]);
      float sl = a.scale_log2;
      if (sl <= 0.f) {
#pragma unroll
        for (int c = 0; c < 128; ++c) s[c] *= a.scale_log2;
        sl = 1.f;
      }
      const int base = j * a.tile_keys;
      if (base + kTileRows > all_see || a.tile_keys < kTileRows) {
        const int lim = min(seen - base, a.tile_keys);
#pragma unroll
        for (int c = 0; c < 128; ++c) s[c] = c < lim ? s[c] : -INFINITY;
      }
      float corr = 1.f;
      bool rescale = false;
      const float mt = row_max_nan(s) * sl;
      if (mt > m + kRescaleThreshold) {
        corr = fast_exp2(m - mt);  // 0 on the first keys of a row
        m = mt;
        rescale = true;
      }
      uint32_t pk[2][32];
      // a row that has seen nothing yet keeps P at 2^-126 and less, which
      // the next rescaling (by zero) removes from l and O
      float sum = exp_row<Dt>(s, sl, m == -INFINITY ? 0.f : m, pk);
      // exp_row's polynomial takes NaN for the smallest exponent: a row with
      // a NaN or infinite score is NaN
      if (!(mt < INFINITY)) sum = NAN;
      l = m == -INFINITY && mt < INFINITY ? 0.f : fmaf(l, corr, sum);
      // P V of the tile before has completed: S was issued after it
      if (j > it.t0 && __any_sync(0xffffffffu, rescale)) {
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
          uint32_t o[32];
          tmem_ld32(tO + 32 * h, o);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c)
            o[c] = __float_as_uint(__uint_as_float(o[c]) * corr);
          tmem_st32(tO + 32 * h, o);
        }
      }
      tmem_st32(tS, pk[0]);
      tmem_st32(tS + 32, pk[1]);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bars[C::kPFull + t]);
    }

    const bool any = end > it.t0;  // O_t holds something of this part
    if (any) {
      if (!mbar_wait(&bars[C::kODone + t], (done - 1) & 1)) {
        ctrl->abort = 1;
        return;
      }
      tc_fence_after();
    }
    const size_t out_row =
        static_cast<size_t>(it.seq.lo + token) * a.H + it.h * group + row - tok * group;
    __half *dst = a.out + out_row * D;
    if (it.whole()) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int h = 0; h < D / 32; ++h) {
        uint32_t o[32];
        if (any && !idle) {
          tmem_ld32(tO + 32 * h, o);
          tmem_wait_ld();
        }
        // a row without keys: zeros, whatever its lane of O holds
        if (l == 0.f) {
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = 0;
        }
        if (real) store_dims<D, Dt>(dst + 32 * h, o, inv);
      }
      if (real && a.lse)
        a.lse[out_row] = l == 0.f ? -INFINITY : 0.69314718055994531f * (m + log2f(l));
      continue;
    }

    // ---- a part: kept, and joined with the others by the last to finish
    auto slot = [&](int c, int t0) {
      return a.partials +
             ((2 * static_cast<size_t>(c) + slot_of(t0)) * 2 + t) * C::kSlotFloats;
    };
    float *mine = slot(blockIdx.x, it.t0);
#pragma unroll
    for (int h = 0; h < D / 32; ++h) {
      uint32_t o[32];
      if (any && !idle) {
        tmem_ld32(tO + 32 * h, o);
        tmem_wait_ld();
      }
      if (real && l != 0.f) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<uint4 *>(mine + ((8 * h + c) * kRows + row) * 4) =
              make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
      }
    }
    mine[D * kRows + row] = m;
    mine[(D + 1) * kRows + row] = l;
    __threadfence();
    // the tile's 128 threads meet (bounded, like every wait here)
    auto meet = [&]() {
      mbar_arrive(&bars[C::kJoin + t]);
      const bool ok = mbar_wait(&bars[C::kJoin + t], met & 1);
      ++met;
      if (!ok) ctrl->abort = 1;
      return ok;
    };
    if (!meet()) return;
    if (row == 0) {
      uint32_t *counter = a.counters + 2 * d.owner(it.at) + t;
      const uint32_t had = atomicAdd(counter, it.t1 - it.t0);
      ctrl->join[t] = had + (it.t1 - it.t0) == static_cast<uint32_t>(it.tiles);
      if (ctrl->join[t]) *counter = 0;
      __threadfence();
    }
    if (!meet()) return;
    if (!ctrl->join[t] || !real) continue;
    const int c0 = d.owner(it.at), c1 = d.owner(it.at + it.cost - 1);
    float M = -INFINITY;
    for (int c = c0; c <= c1; ++c) {
      int t0, t1;
      tiles_of_cta(a, d, it, c, t0, t1);
      if (t0 >= t1) continue;
      const float *p = slot(c, t0);
      if (__ldcg(p + (D + 1) * kRows + row) != 0.f)
        M = fmaxf(M, __ldcg(p + D * kRows + row));
    }
    float L = 0.f;
#pragma unroll
    for (int h = 0; h < D / 32; ++h) {
      float acc[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) acc[c] = 0.f;
      for (int c = c0; c <= c1; ++c) {
        int t0, t1;
        tiles_of_cta(a, d, it, c, t0, t1);
        if (t0 >= t1) continue;
        const float *p = slot(c, t0);
        const float lc = __ldcg(p + (D + 1) * kRows + row);
        if (lc == 0.f) continue;  // saw nothing
        const float w = fast_exp2(__ldcg(p + D * kRows + row) - M);
        if (h == 0) L = fmaf(lc, w, L);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float4 v = __ldcg(reinterpret_cast<const float4 *>(p) +
                                  (8 * h + k) * kRows + row);
          acc[4 * k] = fmaf(v.x, w, acc[4 * k]);
          acc[4 * k + 1] = fmaf(v.y, w, acc[4 * k + 1]);
          acc[4 * k + 2] = fmaf(v.z, w, acc[4 * k + 2]);
          acc[4 * k + 3] = fmaf(v.w, w, acc[4 * k + 3]);
        }
      }
      uint32_t o[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(acc[c]);
      store_dims<D, Dt>(dst + 32 * h, o, L == 0.f ? 0.f : 1.f / L);
    }
    if (a.lse)
      a.lse[out_row] = L == 0.f ? -INFINITY : 0.69314718055994531f * (M + log2f(L));
  }
}

template <int D, typename Dt>
__global__ void __launch_bounds__(kThreads, 1)
    attend_many_kernel(const PagedArgs a, const __grid_constant__ CUtensorMap tm_q,
                       const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kBarOff);
  PlanSmem *ps = reinterpret_cast<PlanSmem *>(smem + C::kMiscOff);
  Ctrl *ctrl = reinterpret_cast<Ctrl *>(smem + C::kMiscOff + sizeof(PlanSmem));
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) record_error(FA_ERR_SMEM_ALIGN);
    return;
  }
  if (warp == kProducerWarp && lane == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&bars[C::kFull + s], 1);
      mbar_init(&bars[C::kEmpty + s], 1);
    }
    mbar_init(&bars[C::kTail], 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars[C::kQFull + t], 1);
      mbar_init(&bars[C::kQEmpty + t], 1);
      mbar_init(&bars[C::kSFull + t], 1);
      mbar_init(&bars[C::kPFull + t], 128);
      mbar_init(&bars[C::kODone + t], 1);
      mbar_init(&bars[C::kJoin + t], 128);
    }
    mbar_init(&bars[C::kDrain], 1);
    fence_barrier_init();
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
    ctrl->abort = device_failed() ? 1u : 0u;
  }
  // Pages that do not fill a tile leave its last rows unwritten: V is zero
  // there (and K's scores are masked).
  if (a.tile_keys < kTileRows) {
    const int chunks = (kTileRows - a.tile_keys) * 8;
    for (int i = threadIdx.x; i < C::kStages * (D / 64) * chunks; i += kThreads) {
      const int half = i / chunks, e = a.tile_keys * 8 + i % chunks;
      *reinterpret_cast<uint4 *>(smem + C::kRingOff + half / (D / 64) * C::kStage +
                                 C::kTile + half % (D / 64) * C::kHalf + 16 * e) =
          make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
  }
  Division d;
  Walk walk;
  if (!plan<kThreads>(a, *ps, d, walk)) return;  // synchronises the CTA
  if (ctrl->abort) return;
  if (warp == kMmaWarp) {
    tmem_alloc(&ctrl->tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (warp >= kProducerWarp) {
    setmaxnreg_dec<kCtrlRegs>();
    if (warp == kProducerWarp)
      produce<D>(a, walk, smem, bars, ctrl, &tm_q, &tm_k, &tm_v);
    else if (warp == kMmaWarp)
      issue<D, Dt>(a, walk, smem, bars, ctrl);
  } else {
    setmaxnreg_inc<kSoftmaxRegs>();
    soften<D, Dt>(a, d, walk, bars, ctrl);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(ctrl->tmem, 512);
  }
}

}  // namespace many
}  // namespace paged
}  // namespace fa
