// Rotary positions (fa_rope) and the append of new rows to a paged K/V cache
// with the rotation on the way (fa_append_paged).
//
// Mathematics: pair (x0, x1) of a row at position p becomes
//   (x0 c - x1 s, x1 c + x0 s) * amplitude,  (c, s) = cos, sin of p * freq.
// p * freq is formed in 64 bits and reduced to a fraction of a turn there,
// so the fp32 sine and cosine see an exact argument at any position (in fp32
// the product alone would be 0.004 rad off at position 100000).
//
// Bound: HBM for long inputs (each element is read and written once), launch
// latency for a generation step. A block takes a few tokens, forms their
// cosines and sines once in shared memory (every head of a token shares
// them) and streams the heads' rows through 16-byte accesses.

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "fa_kernels.h"
#include "fa_sm100.cuh"

namespace fa {
namespace rope {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 4;    // tokens of a block
constexpr int kMaxPairs = 512;   // rotary_dim / 2 at head_dim 1024

struct Smem {
  float2 turn[kMaxTokens * kMaxPairs];  // (cos, sin) * amplitude
  double position[kMaxTokens];
  long long k_at[kMaxTokens];  // element offset of the cache row, -1: none
  long long v_at[kMaxTokens];
  int in_step[kMaxTokens];  // the token belongs to a sequence
};

// V consecutive 16-bit elements (16 bytes, or one).
template <int V>
struct Pack;
template <>
struct Pack<8> {
  using T = uint4;
};
template <>
struct Pack<1> {
  using T = __half;
};

template <typename Dt, int V>
__device__ __forceinline__ void to_float(const typename Pack<V>::T &x,
                                         float (&f)[V]) {
  if constexpr (V == 8) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = Dt::unpack2(w[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  } else {
    f[0] = Dt::unpack2(static_cast<uint32_t>(__half_as_ushort(x))).x;
  }
}

template <typename Dt, int V>
__device__ __forceinline__ typename Pack<V>::T from_float(const float (&f)[V]) {
  if constexpr (V == 8) {
    return make_uint4(Dt::pack2(f[0], f[1]), Dt::pack2(f[2], f[3]),
                      Dt::pack2(f[4], f[5]), Dt::pack2(f[6], f[7]));
  } else {
    return store_elem(f[0], Dt::kDtype);
  }
}

// One unit of a row: V elements of each half of the rotated part, V
// neighbouring elements of it (at least one pair) with kInterleaved, or V
// copied elements after it.
template <typename Dt, int V, bool kInterleaved>
__device__ __forceinline__ void move_unit(const __half *src, __half *dst,
                                          int u, int rot, const float2 *turn) {
  using T = typename Pack<V>::T;
  constexpr int kPairStep = kInterleaved ? (V == 1 ? 2 : V) : V;
  const int n_pair_units = kInterleaved ? rot / kPairStep : rot / (2 * V);
  if (u >= n_pair_units) {
    const int e = rot + (u - n_pair_units) * V;
    *reinterpret_cast<T *>(dst + e) = *reinterpret_cast<const T *>(src + e);
    return;
  }
  const int e = u * kPairStep;
  if constexpr (kInterleaved && V == 1) {
    float a[1], b[1];
    to_float<Dt, 1>(src[e], a);
    to_float<Dt, 1>(src[e + 1], b);
    const float2 t = turn[u];
    const float y0[1] = {a[0] * t.x - b[0] * t.y};
    const float y1[1] = {b[0] * t.x + a[0] * t.y};
    dst[e] = from_float<Dt, 1>(y0);
    dst[e + 1] = from_float<Dt, 1>(y1);
  } else if constexpr (kInterleaved) {
    float f[V], y[V];
    to_float<Dt, V>(*reinterpret_cast<const T *>(src + e), f);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 t = turn[e / 2 + i];
      y[2 * i] = f[2 * i] * t.x - f[2 * i + 1] * t.y;
      y[2 * i + 1] = f[2 * i + 1] * t.x + f[2 * i] * t.y;
    }
    *reinterpret_cast<T *>(dst + e) = from_float<Dt, V>(y);
  } else {
    const int half = rot / 2;
    float a[V], b[V], y0[V], y1[V];
    to_float<Dt, V>(*reinterpret_cast<const T *>(src + e), a);
    to_float<Dt, V>(*reinterpret_cast<const T *>(src + half + e), b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 t = turn[e + i];
      y0[i] = a[i] * t.x - b[i] * t.y;
      y1[i] = b[i] * t.x + a[i] * t.y;
    }
    *reinterpret_cast<T *>(dst + e) = from_float<Dt, V>(y0);
    *reinterpret_cast<T *>(dst + half + e) = from_float<Dt, V>(y1);
  }
}

// Where token t of a step is: its row in its sequence's cache (and through
// the page table, the element offsets of that row). Called by a whole warp.
__device__ __forceinline__ void place_token(const RopeArgs &a, int t, int slot,
                                            Smem &s) {
  const int lane = threadIdx.x & 31;
  // the sequences that end at or before t come before t's own
  int seq = 0;
  for (int b = lane; b < a.batch; b += 32) seq += a.starts[b + 1] <= t;
  seq = __reduce_add_sync(0xffffffffu, seq);
  if (lane != 0) return;
  s.k_at[slot] = s.v_at[slot] = -1;
  s.in_step[slot] = seq < a.batch;
  s.position[slot] = 0.;
  if (seq >= a.batch) return;
  const long long row =
      static_cast<long long>(a.seq_lens[seq]) - a.starts[seq + 1] + t;
  s.position[slot] = a.positions ? static_cast<double>(a.positions[t])
                                 : static_cast<double>(row);
  if (row < 0 || row >= static_cast<long long>(a.table_width) * a.page_rows)
    return;
  const int page = a.page_table[seq * a.table_stride + row / a.page_rows];
  if (page < 0 || page >= a.num_pages) {
    record_error(FA_ERR_PAGE);
    return;
  }
  const long long r = row % a.page_rows;
  s.k_at[slot] = page * a.kp_sp + r * a.kp_sr;
  s.v_at[slot] = page * a.vp_sp + r * a.vp_sr;
}

// Block (x, y): tokens [x * tokens_per_block, ...), rows (heads of q, then k,
// then v) [y * rows_per_block, ...).
template <typename Dt, int V, bool kInterleaved, bool kAppend>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeArgs a) {
  __shared__ Smem s;
  const int t0 = static_cast<int>(blockIdx.x) * a.tokens_per_block;
  const int n_tok = min(a.tokens_per_block, a.tokens - t0);
  const int pairs = a.rot / 2;
  if (kAppend) {
    for (int i = threadIdx.x >> 5; i < n_tok; i += kThreads / 32)
      place_token(a, t0 + i, i, s);
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n_tok * pairs; i += kThreads) {
    const int tok = i / pairs;
    double p;
    if (kAppend) {
      p = s.position[tok];
    } else {
      const int t = t0 + tok;
      p = a.positions[(t / a.N) * a.position_stride + t % a.N];
    }
    double turns = p * a.freqs[i - tok * pairs] * 0.15915494309189533577;
    turns -= rint(turns);
    float sn, cs;
    sincospif(static_cast<float>(2. * turns), &sn, &cs);
    s.turn[i] = make_float2(cs * a.amplitude, sn * a.amplitude * a.sign);
  }
  __syncthreads();

  const int pair_units = kInterleaved ? a.rot / (V == 1 ? 2 : V) : a.rot / (2 * V);
  const int units = pair_units + (a.D - a.rot) / V;
  const int all_rows = a.H + a.H_kv + (kAppend ? a.H_kv : 0);
  const int row0 = static_cast<int>(blockIdx.y) * a.rows_per_block;
  const int n_rows = min(a.rows_per_block, all_rows - row0);
  for (int i = threadIdx.x; i < n_tok * n_rows * units; i += kThreads) {
    const int u = i % units;
    const int rest = i / units;
    const int tok = rest / n_rows;
    const int row = row0 + rest - tok * n_rows;
    const int t = t0 + tok;
    const int b = kAppend ? 0 : t / a.N;
    const int n = kAppend ? t : t - b * a.N;
    if (kAppend && !s.in_step[tok]) continue;
    const __half *src;
    __half *dst;
    if (row < a.H) {
      src = a.q + b * a.q_sb + row * a.q_sh + n * a.q_sn;
      dst = a.q_out + b * a.qo_sb + row * a.qo_sh + n * a.qo_sn;
    } else if (row < a.H + a.H_kv) {
      const int h = row - a.H;
      src = a.k + b * a.k_sb + h * a.k_sh + n * a.k_sn;
      if (kAppend) {
        if (s.k_at[tok] < 0) continue;
        dst = a.k_out + s.k_at[tok] + h * a.kp_sh;
      } else {
        dst = a.k_out + b * a.ko_sb + h * a.ko_sh + n * a.ko_sn;
      }
    } else {
      const int h = row - a.H - a.H_kv;
      if (s.v_at[tok] < 0) continue;
      src = a.v + h * a.v_sh + n * a.v_sn;
      dst = a.v_out + s.v_at[tok] + h * a.vp_sh;
    }
    if (kAppend && row >= a.H + a.H_kv) {
      // V rows are copied: the same units, unrotated
      using T = typename Pack<V>::T;
      if constexpr (kInterleaved && V == 1) {
        if (u < pair_units) {
          dst[2 * u] = src[2 * u];
          dst[2 * u + 1] = src[2 * u + 1];
          continue;
        }
      }
      const int e = kInterleaved || u < pair_units
                        ? u * V
                        : a.rot + (u - pair_units) * V;
      if constexpr (kInterleaved && V == 1) {
        dst[a.rot + u - pair_units] = src[a.rot + u - pair_units];
      } else {
        *reinterpret_cast<T *>(dst + e) = *reinterpret_cast<const T *>(src + e);
        if (!kInterleaved && u < pair_units)
          *reinterpret_cast<T *>(dst + a.rot / 2 + e) =
              *reinterpret_cast<const T *>(src + a.rot / 2 + e);
      }
      continue;
    }
    move_unit<Dt, V, kInterleaved>(src, dst, u, a.rot,
                                   s.turn + tok * pairs);
  }
}

template <typename Dt, int V, bool kInterleaved, bool kAppend>
cudaError_t launch(const RopeArgs &args, cudaStream_t stream) {
  RopeArgs a = args;
  const int rows = a.H + a.H_kv + (kAppend ? a.H_kv : 0);
  a.tokens_per_block = a.tokens > 4 * 148 ? kMaxTokens : 1;
  a.rows_per_block = rows;
  const int units = a.D / V;
  if (a.tokens_per_block == 1) {
    a.rows_per_block = kThreads / units > 0 ? kThreads / units : 1;
    if (a.rows_per_block > rows) a.rows_per_block = rows;
  }
  const dim3 grid((a.tokens + a.tokens_per_block - 1) / a.tokens_per_block,
                  (rows + a.rows_per_block - 1) / a.rows_per_block);
  rope_kernel<Dt, V, kInterleaved, kAppend><<<grid, kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename Dt, int V>
cudaError_t pick(const RopeArgs &a, bool interleaved, bool append,
                 cudaStream_t stream) {
  if (interleaved)
    return append ? launch<Dt, V, true, true>(a, stream)
                  : launch<Dt, V, true, false>(a, stream);
  return append ? launch<Dt, V, false, true>(a, stream)
                : launch<Dt, V, false, false>(a, stream);
}

}  // namespace rope

cudaError_t launch_rope_kernel(const RopeArgs &a, bool interleaved,
                               bool append, bool vector, int dtype,
                               cudaStream_t stream) {
  if (dtype == FA_DTYPE_BF16)
    return vector ? rope::pick<BF16, 8>(a, interleaved, append, stream)
                  : rope::pick<BF16, 1>(a, interleaved, append, stream);
  return vector ? rope::pick<F16, 8>(a, interleaved, append, stream)
                : rope::pick<F16, 1>(a, interleaved, append, stream);
}

}  // namespace fa
