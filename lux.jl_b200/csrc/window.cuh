// Windowed attention: what its kernels share. Which keys a query sees, the bias of a relative position, and the rows that are
// computed again one key at a time where an infinity or NaN was met.
//
// Query l and key s (positions of one sequence of n tokens, n = lengths[b] or all) see each other when
//   l < n, s < n,  s <= l if causal,  |l - s| < window or s < sinks.
// z[s, l] = scale * k_s . q_l + table[h, bucket(s - l)],  p = softmax of z over the visible s (nothing visible: all zero).
#pragma once
#include <algorithm>

#include "common.cuh"

namespace lb2 {

int32_t check_rel_buckets(const lb2_rel_buckets* t);   // relpos.cu

constexpr int kWinMaxBuckets = LB2_MAX_REL_BUCKETS;   // per side

struct WinParams {
  const void *q, *k, *v, *table;
  const int32_t* lengths;
  int D, E, H, Hkv, rep, L, S, B;
  int window, sinks, causal;
  float scale, scale2;        // of the logits; scale2 = scale * log2(e)
  lb2_rel_buckets buckets;    // count = 0: no bias
};

// Logits are kept times log2(e): p = 2^((z2 - m2) - log2(sum)). A finite bias stays finite: the type's lowest value is a mask
// whose rows still have a softmax.
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float win_bias2(float b) { return isinf(b) ? b : fminf(fmaxf(b * kLog2e, -3.402823466e38f), 3.402823466e38f); }

__device__ __forceinline__ int win_tokens(const WinParams& p, int b, int n) {
  return p.lengths == nullptr ? n : max(0, min(n, p.lengths[b]));
}
// The keys that some query of [l0, l1) sees: [0, sinks) and [lo, hi), lo >= sinks.
__device__ __forceinline__ void win_key_range(const WinParams& p, int l0, int l1, int keys, int* sinks, int* lo, int* hi) {
  *hi = p.causal ? min(keys, l1) : keys;
  *sinks = min(p.sinks, *hi);
  if (!p.causal) *hi = min(keys, l1 - 1 + p.window);
  *lo = max(*sinks, l0 - p.window + 1);
}
// The queries that see some key of [s0, s1).
__device__ __forceinline__ void win_query_range(const WinParams& p, int s0, int s1, int queries, int* lo, int* hi) {
  *lo = p.causal ? s0 : (s0 < p.sinks ? 0 : max(0, s0 - p.window + 1));
  *hi = s0 < p.sinks ? queries : min(queries, s1 - 1 + p.window);
}
__device__ __forceinline__ bool win_sees(const WinParams& p, int l, int s) {
  if (p.causal && s > l) return false;
  return abs(l - s) < p.window || s < p.sinks;
}
// the keys of [0, keys) that query l sees are not none
__device__ __forceinline__ bool win_any(const WinParams& p, int l, int keys) {
  int sinks, lo, hi;
  win_key_range(p, l, l + 1, keys, &sinks, &lo, &hi);
  return sinks > 0 || lo < hi;
}

// Query l sees one key alone: its weight is 1 whatever its logit, so the logit's gradient p (dp - delta) is dp - dp, not the difference
// of two sums in different orders.
__device__ __forceinline__ bool win_single(const WinParams& p, int l, int keys) {
  int sinks, lo, hi;
  win_key_range(p, l, l + 1, keys, &sinks, &lo, &hi);
  return sinks + max(0, hi - lo) == 1;
}

// bucket of the relative position rel = s - l: the last one that starts at or below the distance. `first` is t.first, or a copy of it
// in shared memory: lanes that look in different places of the parameters are served one by one.
__device__ __forceinline__ int win_bucket(const lb2_rel_buckets& t, const int32_t* first, int rel) {
  const int dist = t.bidirectional ? abs(rel) : max(-rel, 0);
  int lo = 0, n = t.count;                  // invariant: first[lo] <= dist, the answer lies in [lo, lo + n)
  while (n > 1) {
    const int half = n >> 1;
    if (first[lo + half] <= dist) { lo += half; n -= half; } else { n = half; }
  }
  return lo + (t.bidirectional && rel > 0 ? t.count : 0);
}
__device__ __forceinline__ int win_bucket(const lb2_rel_buckets& t, int rel) { return win_bucket(t, t.first, rel); }
// what rounding took from a value; nothing where it is infinite
__device__ __forceinline__ float win_rest(float a, float rounded) { return isinf(rounded) ? 0.f : a - rounded; }
template <typename T> __device__ __forceinline__ float win_bias(const WinParams& p, int h, int rel) {
  return win_bias2(to_f32(static_cast<const T*>(p.table)[h + (int64_t)p.H * win_bucket(p.buckets, rel)]));
}
template <typename T> __device__ __forceinline__ float win_bias(const WinParams& p, const int32_t* first, int h, int rel) {
  return win_bias2(to_f32(static_cast<const T*>(p.table)[h + (int64_t)p.H * win_bucket(p.buckets, first, rel)]));
}

// 16 bytes into shared memory, zeros in their place if not `real`
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, bool real = true) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
// dtable[h, bucket]: the blocks' sums [n][head][bucket], 64 bits, a warp per entry
template <typename T>
__global__ void __launch_bounds__(256) win_dtable_kernel(T* __restrict__ dtable, const float* __restrict__ partial, int H, int columns, int64_t n) {
  const int lane = threadIdx.x & 31, i = blockIdx.x * 8 + (threadIdx.x >> 5);     // h + H * bucket
  if (i >= H * columns) return;
  const int h = i % H, c = i / H;
  double s = 0.0;
  for (int64_t j = lane; j < n; j += 32) s += partial[(j * H + h) * columns + c];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) dtable[i] = from_f32<T>((float)s);
}

// The tiles of keys that hold sinks, and by how many blocks each is shared in dk, dv: a block walks no more tiles of queries than an
// ordinary one or, if that is more, half an SM's share of the whole. 8192 tokens, 32 heads on 8, window 1024, 4 sinks: 4 blocks, 450 us
// where one block for the sinks took 995.
struct WinSinkPlan { int tiles, splits; };
inline WinSinkPlan win_sink_plan(int tile, int64_t queries, int64_t keys, int64_t window, int64_t sinks, int64_t rep, int64_t groups) {
  auto tiles = [&](int64_t n) { return (n + tile - 1) / tile; };
  const int64_t nsink = tiles(std::min(sinks, keys)), usual = std::min(tiles(queries), tiles(window) + 1) * rep;
  const int64_t all = groups * ((tiles(keys) - nsink) * usual + nsink * tiles(queries) * rep), share = std::max(usual, all / (2 * sm_count()) + 1);
  const int64_t n = nsink > 0 ? std::min<int64_t>(8, (tiles(queries) * rep + share - 1) / share) : 1;
  return {n > 1 ? (int)nsink : 0, (int)n};
}
// What the blocks of dk, dv share: block -> tile of keys, key head and sample, and its part of a shared tile. Shared tiles, the longest, first.
struct WinKeyTile {
  int tile, gb, split, splits;
  __device__ __forceinline__ WinKeyTile(int block, int tiles, int groups, const WinSinkPlan& plan) {
    const int shared = plan.tiles * plan.splits * groups;
    split = 0; splits = 1;
    if (block < shared) {
      gb = block % groups;
      split = block / groups % plan.splits; splits = plan.splits;
      tile = block / groups / plan.splits;
    } else {
      tile = plan.tiles + (block - shared) / groups; gb = (block - shared) % groups;
    }
  }
};
// dk, dv of the shared tiles from their blocks' sums [split][tile][group][rows of a tile][D + E]
int32_t win_sinks_join(const WinParams& p, const WinSinkPlan& plan, int tile, void* dk, void* dv, const float* sums, const void* dx, const float2* stats,
                       const float* delta, int32_t dtype, cudaStream_t st);

// ---- rows once more ---------------------------------------------------------------------------
// A tile's products multiply the weights that the mask made zero with whatever the array holds there: an infinity or NaN in a
// place that the row does not see would reach it. Rows whose results are not finite are therefore computed again by one warp over
// the visible keys (or queries) alone. Lane i holds features i, i + 32, ...
constexpr int kWinMaxDim = 256;
constexpr int kWinLaneDims = kWinMaxDim / 32;
template <typename T> __device__ __forceinline__ void win_load_lane(const T* row, int n, int lane, float (&v)[kWinLaneDims]) {
#pragma unroll
  for (int i = 0; i < kWinLaneDims; ++i) v[i] = lane + 32 * i < n ? to_f32(row[lane + 32 * i]) : 0.f;
}
template <typename T> __device__ __forceinline__ void win_store_lane(T* row, int n, int lane, const float (&v)[kWinLaneDims]) {
#pragma unroll
  for (int i = 0; i < kWinLaneDims; ++i)
    if (lane + 32 * i < n) row[lane + 32 * i] = from_f32<T>(v[i]);
}
// dot of n features; lanes past them hold zeros on both sides
__device__ __forceinline__ float win_dot_lane(const float (&a)[kWinLaneDims], const float (&b)[kWinLaneDims], int n) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kWinLaneDims; ++i)
    if (32 * i < n) s = fmaf(a[i], b[i], s);
  return warp_sum(s);
}
template <typename T> __device__ __forceinline__ const T* win_q_row(const WinParams& p, const void* base, int n, int l, int h, int b) {
  return static_cast<const T*>(base) + (((int64_t)b * p.L + l) * p.H + h) * n;
}
template <typename T> __device__ __forceinline__ const T* win_kv_row(const WinParams& p, const void* base, int n, int s, int g, int b) {
  return static_cast<const T*>(base) + (((int64_t)b * p.S + s) * p.Hkv + g) * n;
}

// stats of a row: the reference m2 that its logits were compared with (their maximum, or a little less) and log2(sum of 2^(z2 - m2)),
// apart: their sum would lose the second beside an m2 as large as the type's lowest value. A row that sees nothing has (0, inf).
// rest: x less its rounding, or null. ROUNDED: weights are summed as the
// tensor-core forward with a bias table sums them, rounded, and m2 grows by whole numbers.
template <typename T, bool ROUNDED = false> __device__ __noinline__ void win_row_fwd(const WinParams& p, T* x, T* rest, float2* stats, int l, int h, int b, int keys) {
  const int lane = threadIdx.x & 31, g = h / p.rep;
  float q[kWinLaneDims], t[kWinLaneDims], o[kWinLaneDims] = {};
  win_load_lane(win_q_row<T>(p, p.q, p.D, l, h, b), p.D, lane, q);
  float m = -INFINITY, sum = 0.f;
  int sinks, lo, hi;
  win_key_range(p, l, l + 1, keys, &sinks, &lo, &hi);
  for (int i0 = 0, n = sinks + max(0, hi - lo); i0 < n; ++i0) {
    const int s = i0 < sinks ? i0 : lo + (i0 - sinks);
    win_load_lane(win_kv_row<T>(p, p.k, p.D, s, g, b), p.D, lane, t);
    float z = win_dot_lane(q, t, p.D) * p.scale2;
    if (p.buckets.count > 0) z += win_bias<T>(p, h, s - l);
    const float mn = z > m ? (ROUNDED && z - m < 1024.f ? m + ceilf(z - m) : z) : m, ref = mn == -INFINITY ? 0.f : mn;
    const float keep = exp2f(m - ref);
    float w = exp2f(z - ref);
    if constexpr (ROUNDED) w = __bfloat162float(__float2bfloat16_rn(w));
    win_load_lane(win_kv_row<T>(p, p.v, p.E, s, g, b), p.E, lane, t);
#pragma unroll
    for (int i = 0; i < kWinLaneDims; ++i) o[i] = fmaf(w, t[i], o[i] * keep);
    sum = sum * keep + w;
    m = mn;
    if (isnan(sum)) break;                // so is the whole row
  }
#pragma unroll
  for (int i = 0; i < kWinLaneDims; ++i) o[i] /= sum;
  const int64_t at = (((int64_t)b * p.L + l) * p.H + h) * p.E;
  win_store_lane(x + at, p.E, lane, o);
  if (rest != nullptr) {
#pragma unroll
    for (int i = 0; i < kWinLaneDims; ++i) o[i] = win_rest(o[i], to_f32(from_f32<T>(o[i])));
    win_store_lane(rest + at, p.E, lane, o);
  }
  if (stats != nullptr && lane == 0) *stats = make_float2(m, log2f(sum));
}

// stats, delta: of query l, head h
template <typename T>
__device__ __noinline__ void win_row_dq(const WinParams& p, T* dq, const void* dx, float2 stats, float delta, int l, int h, int b, int keys) {
  const int lane = threadIdx.x & 31, g = h / p.rep;
  float q[kWinLaneDims], go[kWinLaneDims], t[kWinLaneDims], u[kWinLaneDims], o[kWinLaneDims] = {};
  win_load_lane(win_q_row<T>(p, p.q, p.D, l, h, b), p.D, lane, q);
  win_load_lane(win_q_row<T>(p, dx, p.E, l, h, b), p.E, lane, go);
  int sinks, lo, hi;
  win_key_range(p, l, l + 1, keys, &sinks, &lo, &hi);
  const bool single = win_single(p, l, keys);
  for (int i0 = 0, n = sinks + max(0, hi - lo); i0 < n; ++i0) {
    const int s = i0 < sinks ? i0 : lo + (i0 - sinks);
    win_load_lane(win_kv_row<T>(p, p.k, p.D, s, g, b), p.D, lane, t);
    win_load_lane(win_kv_row<T>(p, p.v, p.E, s, g, b), p.E, lane, u);
    float z = win_dot_lane(q, t, p.D) * p.scale2;
    if (p.buckets.count > 0) z += win_bias<T>(p, h, s - l);
    const float dp = win_dot_lane(go, u, p.E), ds = exp2f((z - stats.x) - stats.y) * (single ? dp - dp : dp - delta) * p.scale;
#pragma unroll
    for (int i = 0; i < kWinLaneDims; ++i) o[i] = fmaf(ds, t[i], o[i]);
  }
  win_store_lane(dq + (((int64_t)b * p.L + l) * p.H + h) * p.D, p.D, lane, o);
}

// stats, delta: [batch][head][query]
template <typename T>
__device__ __noinline__ void win_row_dkv(const WinParams& p, T* dk, T* dv, const void* dx, const float2* stats, const float* delta, int s, int g,
                                         int b, int queries, int keys) {
  const int lane = threadIdx.x & 31;
  float k[kWinLaneDims], v[kWinLaneDims], t[kWinLaneDims], u[kWinLaneDims], ok[kWinLaneDims] = {}, ov[kWinLaneDims] = {};
  win_load_lane(win_kv_row<T>(p, p.k, p.D, s, g, b), p.D, lane, k);
  win_load_lane(win_kv_row<T>(p, p.v, p.E, s, g, b), p.E, lane, v);
  int lo, hi;
  win_query_range(p, s, s + 1, queries, &lo, &hi);
  for (int j = 0; j < p.rep; ++j) {
    const int h = g * p.rep + j;
    for (int l = lo; l < hi; ++l) {
      win_load_lane(win_q_row<T>(p, p.q, p.D, l, h, b), p.D, lane, t);
      win_load_lane(win_q_row<T>(p, dx, p.E, l, h, b), p.E, lane, u);
      float z = win_dot_lane(t, k, p.D) * p.scale2;
      if (p.buckets.count > 0) z += win_bias<T>(p, h, s - l);
      const int64_t at = ((int64_t)b * p.H + h) * p.L + l;
      const float w = exp2f((z - stats[at].x) - stats[at].y), dp = win_dot_lane(u, v, p.E);
      const float ds = w * (win_single(p, l, keys) ? dp - dp : dp - delta[at]) * p.scale;
#pragma unroll
      for (int i = 0; i < kWinLaneDims; ++i) { ov[i] = fmaf(w, u[i], ov[i]); ok[i] = fmaf(ds, t[i], ok[i]); }
    }
  }
  win_store_lane(dk + (((int64_t)b * p.S + s) * p.Hkv + g) * p.D, p.D, lane, ok);
  win_store_lane(dv + (((int64_t)b * p.S + s) * p.Hkv + g) * p.E, p.E, lane, ov);
}

}  // namespace lb2
