// Windowed attention for one new token per sequence, over a ring cache of keys and values. The attention step itself is that of
// lib/LuxLib/src/impl/attention.jl:76-118; the reference keeps no cache.
//
// A cache of `capacity` slots holds position p in slot p while p < sinks, and later ones in
// sinks + (p - sinks) mod (capacity - sinks): the sinks stay, the rest is overwritten oldest first. With
// capacity >= sinks + window all that the new token sees is there.
#include <type_traits>

#include "common.cuh"
#include "window_tc.cuh"

namespace lb2 {

namespace {

__device__ __forceinline__ int64_t ring_slot(int64_t p, int sinks, int ring) { return p < sinks ? p : sinks + (p - sinks) % ring; }

struct StepParams {
  void *x, *kcache, *vcache;
  const void *q, *k, *v, *table;
  const int32_t* lengths;
  int D, E, H, Hkv, rep, C, window, sinks;
  float scale2;
  lb2_rel_buckets buckets;
};

// The keys that the new token at position n sees: n - lo + 1 of the window, `early` sinks before them. Key i lies in slot(i).
struct StepKeys {
  int count, early, first, capacity, ring;        // first: slot of the window's oldest key
  __device__ __forceinline__ StepKeys(const StepParams& p, int n) {
    const int lo = max(0, n - p.window + 1);
    capacity = p.C; ring = p.C - p.sinks;
    early = min(p.sinks, lo);
    count = early + (n - lo + 1);
    first = (int)ring_slot(lo, p.sinks, ring);
  }
  // lo < sinks: no slot has been taken twice among the visible ones, and key i is position and slot i
  __device__ __forceinline__ int64_t slot(int i) const {
    if (i < early) return i;
    const int s = first + (i - early);
    return s < capacity ? s : s - ring;
  }
  __device__ __forceinline__ int distance(int i, int n) const { return i < early ? n - i : count - 1 - i; }
};
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// ---- the kernels of long caches ----------------------------------------------------------------
// A cluster of blocks per (sequence, key head, up to R of its query heads) splits the visible keys; every key and value is read once
// for all R heads. Each warp (Float32: part of a warp) keeps its own running maximum, sum and accumulators; the block joins its
// warps', the cluster its blocks' through distributed shared memory, so there is no workspace and the order is fixed.
// Bounded by the cache's bytes: figures at the kernels.
constexpr int kStepThreads = 128, kStepWarps = 4;

template <int R, int DV, int PARTS> struct StepJoin {
  float o[PARTS][R][DV], m[PARTS][R], s[PARTS][R];
};
template <typename T, int R, int DV, int PARTS>
__device__ __forceinline__ void step_join(StepJoin<R, DV, PARTS>& j, const StepParams& p, T* x, int heads) {
  const int tid = threadIdx.x;
  __syncthreads();
  for (int i = tid; i < R * DV; i += kStepThreads) {
    const int r = i / DV, c = i % DV;
    float top = -INFINITY;
#pragma unroll
    for (int q = 0; q < PARTS; ++q) top = fmaxf(top, j.m[q][r]);
    const float ref = top == -INFINITY ? 0.f : top;
    float a = 0.f;
#pragma unroll
    for (int q = 0; q < PARTS; ++q) a = fmaf(j.o[q][r][c], exp2f(j.m[q][r] - ref), a);
    j.o[0][r][c] = a;                              // read and written by this thread alone
  }
  __syncthreads();
  if (tid < R) {
    float top = -INFINITY, t = 0.f;
    for (int q = 0; q < PARTS; ++q) top = fmaxf(top, j.m[q][tid]);
    const float ref = top == -INFINITY ? 0.f : top;
    for (int q = 0; q < PARTS; ++q) t = fmaf(j.s[q][tid], exp2f(j.m[q][tid] - ref), t);
    j.m[0][tid] = top; j.s[0][tid] = t;
  }
  uint32_t blocks;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
  __syncthreads();                                 // warps converge before the aligned barrier
  cluster_sync_all();
  const uint32_t rank = cluster_cta_rank(), mo = smem_u32(&j.m[0][0]), so = smem_u32(&j.s[0][0]), oo = smem_u32(&j.o[0][0][0]);
  for (int i = tid + (int)rank * kStepThreads; i < heads * DV; i += kStepThreads * (int)blocks) {
    const int r = i / DV, c = i % DV;
    float top = -INFINITY;
    for (uint32_t q = 0; q < blocks; ++q) top = fmaxf(top, ld_cluster_f32(map_to_cta(mo + 4 * r, q)));
    const float ref = top == -INFINITY ? 0.f : top;
    float a = 0.f, t = 0.f;
    for (uint32_t q = 0; q < blocks; ++q) {
      const float f = exp2f(ld_cluster_f32(map_to_cta(mo + 4 * r, q)) - ref);
      t = fmaf(ld_cluster_f32(map_to_cta(so + 4 * r, q)), f, t);
      a = fmaf(ld_cluster_f32(map_to_cta(oo + 4 * i, q)), f, a);
    }
    if (c < p.E) x[r * p.E + c] = from_f32<T>(a / t);
  }
  __syncthreads();
  cluster_sync_all();                              // nobody leaves while its shared memory is read
}

// What the kernels below have in common; `head0` is the first of up to R heads, `rank` of `blocks` the block's place in its cluster.
struct StepPlace {
  int b, g, head0, heads, n;
  uint32_t rank, blocks;
};
template <int R> __device__ __forceinline__ StepPlace step_place(const StepParams& p) {
  StepPlace w;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(w.blocks));
  w.rank = cluster_cta_rank();
  const int groups = (p.rep + R - 1) / R;
  int item = blockIdx.x / w.blocks;
  const int hg = item % groups;
  item /= groups;
  w.g = item % p.Hkv; w.b = item / p.Hkv;
  w.head0 = w.g * p.rep + hg * R;
  w.heads = min(R, p.rep - hg * R);
  w.n = p.lengths[w.b];
  return w;
}
// zeros where there is no sequence; the new row into the cache; the heads' bias per bucket
template <typename T, int R> __device__ __forceinline__ void step_edges(const StepParams& p, const StepPlace& w, float (*bias)[2 * kWinMaxBuckets]) {
  if (w.n < 0) {
    T* x = static_cast<T*>(p.x) + ((int64_t)w.b * p.H + w.head0) * p.E;
    if (w.rank == 0)
      for (int i = threadIdx.x; i < w.heads * p.E; i += kStepThreads) x[i] = from_f32<T>(0.f);
    return;
  }
  if (w.rank == 0 && w.head0 % p.rep == 0) {       // the slot holds nothing that is seen: no block reads it
    const int64_t row = ((int64_t)w.b * p.C + ring_slot(w.n, p.sinks, p.C - p.sinks)) * p.Hkv + w.g, in = (int64_t)w.b * p.Hkv + w.g;
    for (int i = threadIdx.x; i < p.D; i += kStepThreads) static_cast<T*>(p.kcache)[row * p.D + i] = static_cast<const T*>(p.k)[in * p.D + i];
    for (int i = threadIdx.x; i < p.E; i += kStepThreads) static_cast<T*>(p.vcache)[row * p.E + i] = static_cast<const T*>(p.v)[in * p.E + i];
  }
  const int columns = p.buckets.count * (p.buckets.bidirectional ? 2 : 1);
  for (int i = threadIdx.x; i < w.heads * columns; i += kStepThreads)
    bias[i % w.heads][i / w.heads] = win_bias2(to_f32(static_cast<const T*>(p.table)[w.head0 + i % w.heads + (int64_t)p.H * (i / w.heads)]));
}
// the share of `count` keys, in groups of `unit`, of a block
__device__ __forceinline__ void step_share(int count, int unit, const StepPlace& w, int* from, int* to) {
  const int groups = (count + unit - 1) / unit;
  *from = (int)((int64_t)groups * w.rank / w.blocks) * unit;
  *to = min(count, (int)((int64_t)groups * (w.rank + 1) / w.blocks) * unit);
}

// ---- BFloat16 -----------------------------------------------------------------------------------
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A warp takes 16 keys at a time. S[heads][keys] = Q K' and O[heads][features] += P V as m16n8k16 products (too small and too ragged for
// the TMEM path, and the cache's bytes bound them). The features of a contraction may come in any order, so a lane takes eight
// neighbouring ones of a key's row with one 16-byte load as its share of two steps; for V it joins two keys' rows by halves.
// Each warp has its own ring of kStepStages groups of keys in shared memory, filled by asynchronous copies: what is in flight does not
// depend on registers. 16-byte pieces are swizzled by row so that the fragments' loads meet no bank twice.
// Measured: 32 sequences of 1000 to 9000 tokens, 8 key heads of 128 features, 4 query heads each, window 4096: 455 MB in 91 us (5.0 TB/s, 0.77
// of the copy rate); 133 us with the loads in registers. One sequence, window 1024: 10 us, start, two groups of keys and the join.
constexpr int kStepStages = 3;
template <int DC, int R> struct StepRing {
  static constexpr int HALF = 16 * DC * 2, STAGE = 2 * HALF, WARP = kStepStages * STAGE;      // 16 keys, then their 16 values
  static constexpr int BYTES = kStepWarps * WARP > (int)sizeof(StepJoin<R, DC, kStepWarps>) ? kStepWarps * WARP : (int)sizeof(StepJoin<R, DC, kStepWarps>);
};
template <int DC, int R>
__global__ void __launch_bounds__(kStepThreads) win_step_bf16_kernel(const __grid_constant__ StepParams p) {
  using T = __nv_bfloat16;
  using Ring = StepRing<DC, R>;
  static_assert(R == 8 || R == 16, "rows of an m16 tile");
  extern __shared__ __align__(128) uint8_t raw[];
  __shared__ float head_bias[R][2 * kWinMaxBuckets];
  __shared__ int32_t first_of[kWinMaxBuckets];
  if (threadIdx.x < kWinMaxBuckets) first_of[threadIdx.x] = p.buckets.first[threadIdx.x];
  const StepPlace w = step_place<R>(p);
  step_edges<T, R>(p, w, head_bias);
  if (w.n < 0) return;                             // the whole cluster
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, u = lane >> 2, t = lane & 3;
  const StepKeys keys(p, w.n);
  const int64_t in = (int64_t)w.b * p.Hkv + w.g, row0 = (int64_t)w.b * p.C * p.Hkv + w.g;
  const T* kc = static_cast<const T*>(p.kcache) + row0 * p.D;
  const T* vc = static_cast<const T*>(p.vcache) + row0 * p.E;
  const T* kn = static_cast<const T*>(p.k) + in * p.D;
  const T* vn = static_cast<const T*>(p.v) + in * p.E;
  const int64_t ks = (int64_t)p.Hkv * p.D, vs = (int64_t)p.Hkv * p.E;
  constexpr int KC = DC / 32, VC = DC / 64, CPR = DC / 8;                  // CPR: 16-byte pieces of a row
  int from, to;
  step_share(keys.count, 16, w, &from, &to);
  const uint32_t ring = smem_u32(raw) + warp * Ring::WARP;
  const int piece = lane % CPR, first_row = lane / CPR;
  const bool kreal = piece * 8 < p.D, vreal = piece * 8 < p.E;
  // 16 keys from i0 on; past the end the last key once more, which does not count there
  auto fetch = [&](int i0, int stage) {
    if (i0 < to) {
#pragma unroll
      for (int r = 0; r < 16; r += 32 / CPR) {
        const int row = r + first_row, i = min(i0 + row, to - 1);
        const bool fresh = i == keys.count - 1;
        const int64_t slot = keys.slot(i);
        const uint32_t at = ring + stage * Ring::STAGE + row * (DC * 2);
        copy_async16(at + ((piece ^ ((row & 1) << 2)) * 16), (fresh ? kn : kc + slot * ks) + (kreal ? piece * 8 : 0), kreal);
        copy_async16(at + Ring::HALF + ((piece ^ (row & 6)) * 16), (fresh ? vn : vc + slot * vs) + (vreal ? piece * 8 : 0), vreal);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 q[R / 8][KC];
#pragma unroll
  for (int a = 0; a < R / 8; ++a)
#pragma unroll
    for (int c = 0; c < KC; ++c)
      q[a][c] = u + 8 * a < w.heads && c * 32 + t * 8 < p.D
                    ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + ((int64_t)w.b * p.H + w.head0 + u + 8 * a) * p.D + c * 32 + t * 8)
                    : zero;
  float o[VC][8][R / 4];
#pragma unroll
  for (int c = 0; c < VC; ++c)
#pragma unroll
    for (int f = 0; f < 8; ++f)
#pragma unroll
      for (int k = 0; k < R / 4; ++k) o[c][f][k] = 0.f;
  float m[R / 8], sum[R / 8];
#pragma unroll
  for (int a = 0; a < R / 8; ++a) { m[a] = -INFINITY; sum[a] = 0.f; }

  const int begin = from + warp * 16;
#pragma unroll
  for (int x = 0; x < kStepStages - 1; ++x) fetch(begin + x * kStepWarps * 16, x);
  int stage = 0;
  int i0 = begin;
  const auto group = [&](auto ends) {              // ends: some of the 16 keys are past the end
    constexpr bool ENDS = decltype(ends)::value;
    asm volatile("cp.async.wait_group %0;" ::"n"(kStepStages - 2) : "memory");
    __syncwarp();
    fetch(i0 + (kStepStages - 1) * kStepWarps * 16, stage == 0 ? kStepStages - 1 : stage - 1);      // over what was read last
    const uint8_t* at = raw + warp * Ring::WARP + stage * Ring::STAGE;
    stage = stage + 1 == kStepStages ? 0 : stage + 1;
    float s[2][4];
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      s[tile][0] = s[tile][1] = s[tile][2] = s[tile][3] = 0.f;
      const int row = tile * 8 + u;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint4 kv = *reinterpret_cast<const uint4*>(at + row * (DC * 2) + (((c * 4 + t) ^ ((row & 1) << 2)) * 16));
        const uint4 lo = q[0][c], hi = R == 16 ? q[R / 8 - 1][c] : zero;
        mma_bf16(s[tile], lo.x, hi.x, lo.y, hi.y, kv.x, kv.y);
        mma_bf16(s[tile], lo.z, hi.z, lo.w, hi.w, kv.z, kv.w);
      }
    }
    float z[R / 8][4], top[R / 8];                 // keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
    for (int a = 0; a < R / 8; ++a) top[a] = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + (k >> 1) * 8 + 2 * t + (k & 1);
      const int bk = p.buckets.count > 0 && (!ENDS || i < to) ? win_bucket(p.buckets, first_of, -keys.distance(i, w.n)) : 0;
#pragma unroll
      for (int a = 0; a < R / 8; ++a) {
        float v = s[k >> 1][2 * a + (k & 1)] * p.scale2;
        if (p.buckets.count > 0 && u + 8 * a < w.heads) v += head_bias[u + 8 * a][bk];
        z[a][k] = !ENDS || i < to ? v : -INFINITY;
        top[a] = fmaxf(top[a], z[a][k]);
      }
    }
    bool grow = false;
#pragma unroll
    for (int a = 0; a < R / 8; ++a) {
      top[a] = fmaxf(top[a], __shfl_xor_sync(0xffffffffu, top[a], 1));
      top[a] = fmaxf(top[a], __shfl_xor_sync(0xffffffffu, top[a], 2));
      grow = grow || top[a] > m[a] + 8.f;
    }
    if (__any_sync(0xffffffffu, grow)) {           // weights up to 2^8 are as exact in bf16
#pragma unroll
      for (int a = 0; a < R / 8; ++a) {
        const float to_m = top[a] > m[a] + 8.f ? top[a] : m[a], keep = to_m == m[a] ? 1.f : ex2(m[a] - to_m);
        m[a] = to_m;
        sum[a] *= keep;
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
          for (int f = 0; f < 8; ++f) { o[c][f][2 * a] *= keep; o[c][f][2 * a + 1] *= keep; }
      }
    }
    uint32_t pa[R / 8][2];
#pragma unroll
    for (int a = 0; a < R / 8; ++a) {
      const float ref = m[a] == -INFINITY ? 0.f : m[a];
      float e[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) e[k] = ex2(z[a][k] - ref);
      sum[a] += (e[0] + e[1]) + (e[2] + e[3]);
      pa[a][0] = pack_bf16(e[0], e[1]);
      pa[a][1] = pack_bf16(e[2], e[3]);
    }
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      uint4 vv[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = (r >> 1) * 8 + 2 * t + (r & 1);
        vv[r] = *reinterpret_cast<const uint4*>(at + Ring::HALF + row * (DC * 2) + (((c * 8 + u) ^ (row & 6)) * 16));
        if (ENDS && i0 + row >= to) vv[r] = zero;  // nothing times an infinite value is NaN
      }
      const uint32_t w0[4] = {vv[0].x, vv[0].y, vv[0].z, vv[0].w}, w1[4] = {vv[1].x, vv[1].y, vv[1].z, vv[1].w};
      const uint32_t w2[4] = {vv[2].x, vv[2].y, vv[2].z, vv[2].w}, w3[4] = {vv[3].x, vv[3].y, vv[3].z, vv[3].w};
#pragma unroll
      for (int f = 0; f < 8; ++f) {
        const uint32_t b0 = __byte_perm(w0[f >> 1], w1[f >> 1], f & 1 ? 0x7632 : 0x5410), b1 = __byte_perm(w2[f >> 1], w3[f >> 1], f & 1 ? 0x7632 : 0x5410);
        float d[4] = {o[c][f][0], o[c][f][1], R == 16 ? o[c][f][R / 4 - 2] : 0.f, R == 16 ? o[c][f][R / 4 - 1] : 0.f};
        mma_bf16(d, pa[0][0], R == 16 ? pa[R / 8 - 1][0] : 0u, pa[0][1], R == 16 ? pa[R / 8 - 1][1] : 0u, b0, b1);
#pragma unroll
        for (int k = 0; k < R / 4; ++k) o[c][f][k] = d[k];
      }
    }
    __syncwarp();                                  // all have read the stage before it is filled again
  };
  for (; i0 + 16 <= to; i0 += kStepWarps * 16) group(std::false_type{});
  if (i0 < to) group(std::true_type{});
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();                                 // the ring's memory becomes the join's
  auto& j = *reinterpret_cast<StepJoin<R, DC, kStepWarps>*>(raw);
#pragma unroll
  for (int a = 0; a < R / 8; ++a) {
    sum[a] += __shfl_xor_sync(0xffffffffu, sum[a], 1);
    sum[a] += __shfl_xor_sync(0xffffffffu, sum[a], 2);
    if (t == 0) { j.m[warp][u + 8 * a] = m[a]; j.s[warp][u + 8 * a] = sum[a]; }
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int f = 0; f < 8; ++f)
#pragma unroll
        for (int k = 0; k < 2; ++k) j.o[warp][u + 8 * a][c * 64 + (2 * t + k) * 8 + f] = o[c][f][2 * a + k];
  }
  step_join<T>(j, p, static_cast<T*>(p.x) + ((int64_t)w.b * p.H + w.head0) * p.E, w.heads);
}

// ---- Float32 ------------------------------------------------------------------------------------
// LPR lanes share a key's row, four features each; 32 / LPR keys per warp and load, four loads at a time. 5 sequences, 12 heads of 64
// features, window 500: 15 us, of which the kernel's own chain of loads is most.
template <int LPR, int R>
__global__ void __launch_bounds__(kStepThreads) win_step_f32_kernel(const __grid_constant__ StepParams p) {
  constexpr int DC = LPR * 4, PER = 32 / LPR, PARTS = kStepWarps * PER, U = 4;
  extern __shared__ __align__(16) uint8_t raw[];
  auto& j = *reinterpret_cast<StepJoin<R, DC, PARTS>*>(raw);
  __shared__ float head_bias[R][2 * kWinMaxBuckets];
  __shared__ int32_t first_of[kWinMaxBuckets];
  if (threadIdx.x < kWinMaxBuckets) first_of[threadIdx.x] = p.buckets.first[threadIdx.x];
  const StepPlace w = step_place<R>(p);
  step_edges<float, R>(p, w, head_bias);
  if (w.n < 0) return;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp * PER + lane / LPR, c = (lane % LPR) * 4;
  const StepKeys keys(p, w.n);
  const int64_t in = (int64_t)w.b * p.Hkv + w.g, row0 = (int64_t)w.b * p.C * p.Hkv + w.g;
  const float* kc = static_cast<const float*>(p.kcache) + row0 * p.D;
  const float* vc = static_cast<const float*>(p.vcache) + row0 * p.E;
  const float* kn = static_cast<const float*>(p.k) + in * p.D;
  const float* vn = static_cast<const float*>(p.v) + in * p.E;
  const int64_t ks = (int64_t)p.Hkv * p.D, vs = (int64_t)p.Hkv * p.E;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  float4 q[R], o[R];
  float m[R], sum[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    q[r] = r < w.heads && c < p.D ? *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + ((int64_t)w.b * p.H + w.head0 + r) * p.D + c) : zero;
    o[r] = zero; m[r] = -INFINITY; sum[r] = 0.f;
  }
  int from, to;
  step_share(keys.count, PARTS, w, &from, &to);
  for (int i0 = from; i0 < to; i0 += PARTS * U) {      // all lanes of a warp together
    float4 kv[U], vv[U];
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const int i = min(i0 + x * PARTS + part, to - 1);   // past the end the last key once more: it weighs nothing there
      const bool fresh = i == keys.count - 1;
      const int64_t slot = keys.slot(i);
      kv[x] = *reinterpret_cast<const float4*>((fresh ? kn : kc + slot * ks) + (c < p.D ? c : 0));
      vv[x] = *reinterpret_cast<const float4*>((fresh ? vn : vc + slot * vs) + (c < p.E ? c : 0));
    }
#pragma unroll
    for (int x = 0; x < U; ++x) {
      if (c >= p.D) kv[x] = zero;
      if (i0 + x * PARTS + part >= to) vv[x] = zero;      // it may be infinite
    }
    int bk[U];
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const int i = i0 + x * PARTS + part;
      bk[x] = p.buckets.count > 0 && i < to ? win_bucket(p.buckets, first_of, -keys.distance(i, w.n)) : 0;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= w.heads) break;
      float z[U], top = m[r];
#pragma unroll
      for (int x = 0; x < U; ++x) {
        float d = q[r].x * kv[x].x;
        d = fmaf(q[r].y, kv[x].y, d);
        d = fmaf(q[r].z, kv[x].z, d);
        d = fmaf(q[r].w, kv[x].w, d);
#pragma unroll
        for (int s = LPR / 2; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
        d *= p.scale2;
        if (p.buckets.count > 0) d += head_bias[r][bk[x]];
        z[x] = i0 + x * PARTS + part < to ? d : -INFINITY;
        top = fmaxf(top, z[x]);
      }
      const float ref = top == -INFINITY ? 0.f : top, keep = exp2f(m[r] - ref);
      m[r] = top;
      sum[r] *= keep;
      o[r].x *= keep; o[r].y *= keep; o[r].z *= keep; o[r].w *= keep;
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const float e = exp2f(z[x] - ref);
        sum[r] += e;
        o[r].x = fmaf(e, vv[x].x, o[r].x); o[r].y = fmaf(e, vv[x].y, o[r].y);
        o[r].z = fmaf(e, vv[x].z, o[r].z); o[r].w = fmaf(e, vv[x].w, o[r].w);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    *reinterpret_cast<float4*>(&j.o[part][r][c]) = o[r];
    if (lane % LPR == 0) { j.m[part][r] = m[r]; j.s[part][r] = sum[r]; }
  }
  step_join<float>(j, p, static_cast<float*>(p.x) + ((int64_t)w.b * p.H + w.head0) * p.E, w.heads);
}

// ---- any features: a block per (sequence, head); its warps take the keys in turn -----------------
template <typename T> __global__ void __launch_bounds__(256) win_step_kernel(const __grid_constant__ StepParams p) {
  __shared__ float so[8][kWinMaxDim], sm[8], ss[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H, g = h / p.rep;
  T* xr = static_cast<T*>(p.x) + ((int64_t)b * p.H + h) * p.E;
  const int n = p.lengths[b];
  if (n < 0) {                                  // no sequence in this place
    for (int e = threadIdx.x; e < p.E; e += 256) xr[e] = from_f32<T>(0.f);
    return;
  }
  const T* kn = static_cast<const T*>(p.k) + ((int64_t)b * p.Hkv + g) * p.D;
  const T* vn = static_cast<const T*>(p.v) + ((int64_t)b * p.Hkv + g) * p.E;
  T* kc = static_cast<T*>(p.kcache) + ((int64_t)b * p.C * p.Hkv + g) * p.D;
  T* vc = static_cast<T*>(p.vcache) + ((int64_t)b * p.C * p.Hkv + g) * p.E;
  const int ring = p.C - p.sinks;
  float q[kWinLaneDims], t[kWinLaneDims], o[kWinLaneDims] = {};
  win_load_lane(static_cast<const T*>(p.q) + ((int64_t)b * p.H + h) * p.D, p.D, lane, q);
  float m = -INFINITY, sum = 0.f;
  const int lo = max(0, n - p.window + 1), early = min(p.sinks, lo), count = early + (n - lo + 1);
  for (int i = warp; i < count; i += 8) {
    const int s = i < early ? i : lo + (i - early);
    const int64_t slot = ring_slot(s, p.sinks, ring);
    win_load_lane(s == n ? kn : kc + slot * p.Hkv * p.D, p.D, lane, t);
    float z = win_dot_lane(q, t, p.D) * p.scale2;
    if (p.buckets.count > 0) z += win_bias2(to_f32(static_cast<const T*>(p.table)[h + (int64_t)p.H * win_bucket(p.buckets, s - n)]));
    const float mn = fmaxf(m, z), ref = mn == -INFINITY ? 0.f : mn;
    const float keep = exp2f(m - ref), w = exp2f(z - ref);
    win_load_lane(s == n ? vn : vc + slot * p.Hkv * p.E, p.E, lane, t);
#pragma unroll
    for (int j = 0; j < kWinLaneDims; ++j) o[j] = fmaf(w, t[j], o[j] * keep);
    sum = sum * keep + w;
    m = mn;
  }
#pragma unroll
  for (int j = 0; j < kWinLaneDims; ++j) so[warp][lane + 32 * j] = o[j];
  if (lane == 0) { sm[warp] = m; ss[warp] = sum; }
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < 8; ++w) top = fmaxf(top, sm[w]);
  const float ref = top == -INFINITY ? 0.f : top;
  for (int w = 0; w < 8; ++w) total += ss[w] * exp2f(sm[w] - ref);
  for (int e = threadIdx.x; e < p.E; e += 256) {
    float a = 0.f;
    for (int w = 0; w < 8; ++w)
      if (w < count) a = fmaf(so[w][e], exp2f(sm[w] - ref), a);           // a warp without a key adds nothing
    xr[e] = from_f32<T>(a / total);
  }
  if (h % p.rep == 0) {
    const int64_t slot = ring_slot(n, p.sinks, ring);
    for (int d = threadIdx.x; d < p.D; d += 256) kc[slot * p.Hkv * p.D + d] = kn[d];
    for (int d = threadIdx.x; d < p.E; d += 256) vc[slot * p.Hkv * p.E + d] = vn[d];
  }
}

// the tokens of k and v that a cache holds after n of them: a warp per token and head
template <typename T>
__global__ void __launch_bounds__(256) win_fill_kernel(T* __restrict__ kc, T* __restrict__ vc, const T* __restrict__ k, const T* __restrict__ v,
                                                       const int32_t* __restrict__ lengths, int D, int E, int Hkv, int S, int C, int sinks, int64_t rows) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);     // (batch, slot, head)
  if (row >= rows) return;
  const int g = (int)(row % Hkv);
  const int64_t bs = row / Hkv, b = bs / C;
  const int slot = (int)(bs - b * C), ring = C - sinks;
  const int n = lengths == nullptr ? S : max(0, min(S, lengths[b]));
  int s = slot;                                                         // the newest position below n of this slot
  if (slot >= n) return;
  if (slot >= sinks) s = slot + (n - 1 - slot) / ring * ring;
  const int64_t src = (b * S + s) * Hkv + g;
  for (int d = lane; d < D; d += 32) kc[row * D + d] = k[src * D + d];
  for (int d = lane; d < E; d += 32) vc[row * E + d] = v[src * E + d];
}

int32_t step_check(const lb2_window_dims* d, const lb2_rel_buckets* t, const void* table, const int32_t* lengths, int32_t dtype) {
  LB2_REQUIRE(valid_dtype(dtype), LB2_UNSUPPORTED_DTYPE, "dtype %d not supported", (int)dtype);
  LB2_REQUIRE(d != nullptr, LB2_BAD_ARG, "window dims are null");
  LB2_REQUIRE(d->head_dim >= 0 && d->value_dim >= 0 && d->heads >= 0 && d->kv_heads >= 0 && d->queries >= 0 && d->keys >= 0 && d->batch >= 0,
              LB2_BAD_SHAPE, "negative extent");
  LB2_REQUIRE(d->head_dim <= kWinMaxDim && d->value_dim <= kWinMaxDim, LB2_BAD_SHAPE, "head_dim and value_dim may be %d at most", kWinMaxDim);
  const int64_t big = 1 << 29;
  LB2_REQUIRE(d->heads <= 65536 && d->kv_heads <= 65536 && d->keys <= big && d->queries <= big && d->batch <= big, LB2_BAD_SHAPE, "extent too large");
  LB2_REQUIRE(d->sinks >= 0, LB2_BAD_ARG, "negative number of sinks");
  LB2_REQUIRE(d->sinks < d->keys || d->batch == 0, LB2_BAD_ARG, "the cache must hold more than the sinks");
  LB2_REQUIRE(aligned_to(lengths, 4), LB2_BAD_ALIGN, "lengths must be 4-byte aligned");
  LB2_REQUIRE((t == nullptr) == (table == nullptr), LB2_BAD_ARG, "table and buckets must both be given or both be null");
  return t == nullptr ? LB2_OK : check_rel_buckets(t);
}

// Clusters: enough blocks for the device (six per SM even out sequences of different lengths) while each keeps 64 keys or more.
template <typename K> int32_t step_launch(K kernel, const StepParams& p, const lb2_window_dims* d, int heads_per_block, int smem, cudaStream_t st) {
  const int64_t items = d->batch * d->kv_heads * ((p.rep + heads_per_block - 1) / heads_per_block), seen = d->window + d->sinks;
  int blocks = 1;
  while (blocks < 8 && items * blocks < (int64_t)sm_count() * 6 && seen >= (int64_t)blocks * 2 * 64) blocks *= 2;
  LB2_REQUIRE(items * blocks <= 0x7FFFFFFF, LB2_BAD_SHAPE, "too many rows");
  if (smem > 0) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(LB2_LAUNCH_FAIL, "windowed attention step: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(items * blocks));
  cfg.blockDim = dim3(kStepThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)blocks; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) return fail(LB2_LAUNCH_FAIL, "windowed attention step: %s", cudaGetErrorString(e));
  return LB2_OK;
}

}  // namespace

}  // namespace lb2

using namespace lb2;

extern "C" {

int32_t lb2_window_attention_step(void* x, void* kcache, void* vcache, const void* q, const void* k, const void* v, const void* table,
                                  const lb2_rel_buckets* buckets, const int32_t* lengths, double scale, const lb2_window_dims* d, int32_t dtype,
                                  void* stream) {
  int32_t rc = step_check(d, buckets, table, lengths, dtype);
  if (rc != LB2_OK) return rc;
  LB2_REQUIRE(d->window >= 1, LB2_BAD_ARG, "the window must hold at least one token");
  LB2_REQUIRE(d->heads == 0 || (d->kv_heads > 0 && d->heads % d->kv_heads == 0), LB2_BAD_SHAPE, "heads must be a multiple of kv_heads");
  if (d->batch == 0 || d->kv_heads == 0) return LB2_OK;
  LB2_REQUIRE(d->heads > 0, LB2_BAD_SHAPE, "a step without query heads");       // it would leave the token out of the cache
  LB2_REQUIRE(d->window <= d->keys - d->sinks, LB2_BAD_ARG, "a cache of %lld slots does not hold %lld sinks and a window of %lld", (long long)d->keys,
              (long long)d->sinks, (long long)d->window);
  const size_t es = dtype_size(dtype);
  LB2_REQUIRE(lengths && ((x && vcache && v) || d->value_dim == 0) && ((q && kcache && k) || d->head_dim == 0), LB2_BAD_ARG, "null tensor pointer");
  LB2_REQUIRE(aligned_to(x, es) && aligned_to(kcache, es) && aligned_to(vcache, es) && aligned_to(q, es) && aligned_to(k, es) && aligned_to(v, es) &&
                  aligned_to(table, es),
              LB2_BAD_ALIGN, "pointer not aligned to the element size");
  LB2_REQUIRE(d->heads * d->batch <= 0x7FFFFFFF, LB2_BAD_SHAPE, "too many rows");
  StepParams p{};
  p.x = x; p.kcache = kcache; p.vcache = vcache; p.q = q; p.k = k; p.v = v; p.table = table; p.lengths = lengths;
  p.D = (int)d->head_dim; p.E = (int)d->value_dim; p.H = (int)d->heads; p.Hkv = (int)d->kv_heads; p.rep = (int)(d->heads / d->kv_heads);
  p.C = (int)d->keys; p.window = (int)d->window; p.sinks = (int)d->sinks;
  p.scale2 = (float)(scale * 1.4426950408889634);
  if (buckets != nullptr) p.buckets = *buckets;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t per16 = 16 / (int64_t)es;
  if (d->head_dim > 0 && d->value_dim > 0 && d->head_dim <= 128 && d->value_dim <= 128 && d->head_dim % per16 == 0 && d->value_dim % per16 == 0 &&
      aligned_to(kcache, 16) && aligned_to(vcache, 16) && aligned_to(q, 16) && aligned_to(k, 16) && aligned_to(v, 16)) {
    const int most = p.D > p.E ? p.D : p.E;
    if (dtype == LB2_BF16) {
      if (p.rep <= 8)
        return most <= 64 ? step_launch(win_step_bf16_kernel<64, 8>, p, d, 8, StepRing<64, 8>::BYTES, st)
                          : step_launch(win_step_bf16_kernel<128, 8>, p, d, 8, StepRing<128, 8>::BYTES, st);
      return most <= 64 ? step_launch(win_step_bf16_kernel<64, 16>, p, d, 16, StepRing<64, 16>::BYTES, st)
                        : step_launch(win_step_bf16_kernel<128, 16>, p, d, 16, StepRing<128, 16>::BYTES, st);
    }
    auto rows = [&](auto lpr) -> int32_t {
      constexpr int LPR = decltype(lpr)::value, PARTS = kStepWarps * 32 / LPR;
      if (p.rep == 1) return step_launch(win_step_f32_kernel<LPR, 1>, p, d, 1, (int)sizeof(StepJoin<1, LPR * 4, PARTS>), st);
      if (p.rep <= 4) return step_launch(win_step_f32_kernel<LPR, 4>, p, d, 4, (int)sizeof(StepJoin<4, LPR * 4, PARTS>), st);
      return step_launch(win_step_f32_kernel<LPR, 8>, p, d, 8, (int)sizeof(StepJoin<8, LPR * 4, PARTS>), st);
    };
    if (most <= 32) return rows(std::integral_constant<int, 8>{});
    return most <= 64 ? rows(std::integral_constant<int, 16>{}) : rows(std::integral_constant<int, 32>{});
  }
  LB2_DISPATCH_DTYPE(dtype, { win_step_kernel<T><<<(unsigned)(d->heads * d->batch), 256, 0, st>>>(p); });
  LB2_CHECK_LAUNCH("windowed attention step");
  return LB2_OK;
}

int32_t lb2_window_cache_fill(void* kcache, void* vcache, const void* k, const void* v, const int32_t* lengths, int64_t capacity,
                              const lb2_window_dims* d, int32_t dtype, void* stream) {
  LB2_REQUIRE(d != nullptr, LB2_BAD_ARG, "window dims are null");
  lb2_window_dims c = *d;
  c.keys = capacity; c.heads = 0; c.queries = d->keys;
  int32_t rc = step_check(&c, nullptr, nullptr, lengths, dtype);
  if (rc != LB2_OK) return rc;
  if (d->batch == 0 || d->kv_heads == 0 || d->keys == 0) return LB2_OK;
  const size_t es = dtype_size(dtype);
  LB2_REQUIRE(((vcache && v) || d->value_dim == 0) && ((kcache && k) || d->head_dim == 0), LB2_BAD_ARG, "null tensor pointer");
  LB2_REQUIRE(aligned_to(kcache, es) && aligned_to(vcache, es) && aligned_to(k, es) && aligned_to(v, es), LB2_BAD_ALIGN,
              "pointer not aligned to the element size");
  const int64_t rows = d->batch * capacity * d->kv_heads, blocks = (rows + 7) / 8;
  LB2_REQUIRE(blocks <= 0x7FFFFFFF, LB2_BAD_SHAPE, "too many rows");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LB2_DISPATCH_DTYPE(dtype, {
    win_fill_kernel<T><<<(unsigned)blocks, 256, 0, st>>>((T*)kcache, (T*)vcache, (const T*)k, (const T*)v, lengths, (int)d->head_dim, (int)d->value_dim,
                                                       (int)d->kv_heads, (int)d->keys, (int)capacity, (int)d->sinks, rows);
  });
  LB2_CHECK_LAUNCH("windowed cache fill");
  return LB2_OK;
}

}  // extern "C"
