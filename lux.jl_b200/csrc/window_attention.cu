// Attention with a sliding window and a few first tokens that stay visible (sinks), with its pullback: the softmax of
// scaled_dot_product_attention (lib/LuxLib/src/impl/attention.jl:76-131) over a band of keys, in one pass that keeps neither
// logits nor weights in memory, optionally with the learned bias table[h, bucket(s - l)] added to the logits.
//
// Forward, per tile of queries: running maximum m and sum of exp(z - m) over the tiles of visible keys, the accumulators scaled
// by exp(m_old - m_new); x = accumulator / sum. Pullback, from p = exp(z - m) / sum, dp = dx . v and
// delta = dx . x:  ds = p (dp - delta), dq = scale * ds k, dk = scale * ds' q, dv = p' dx, dtable = sums of ds by bucket.
// One kernel per tile of queries (dq, dtable) and one per tile of keys (dk, dv) form p anew; no result is added to by two
// blocks, so every sum has a fixed order.
//
// This file: the CUDA-core kernels, which serve Float32 and every feature count up to 256, and the entry points (window_tc.cu,
// window_tc_bwd.cu: the tensor-core kernels of BFloat16 with up to 128 features in whole 16-byte vectors). Measured, Float32, 4 x 8 heads of
// 64 features, 1024 tokens, window 256, 4 sinks, bias: forward 126 us, dq 206, dk dv 202 + 6; 17 TFLOP/s of the tiles' products, a quarter of
// the CUDA cores' rate. What bounds them: two blocks per SM (registers, shared memory) and 512 equal blocks, 1.7 rounds. BFloat16, the same tokens
// and heads: 36 features forward 104 us, pullback 304; 192 features 400 and 1473 (32 x 32 tiles).
#include "common.cuh"
#include "window_tc.cuh"

namespace lb2 {

namespace {

constexpr int kWinThreads = 256;      // 16 x 16, each TM x TN of a tile of logits

// rows [row0, row0 + ROWS) of n features, `stride` elements apart, as fp32 into rows of LD floats; zeros past `rows` and past n.
// Whole Float32 vectors are copied asynchronously: win_loaded() before the barrier that hands them on.
__device__ __forceinline__ void win_loaded() { asm volatile("cp.async.wait_all;" ::: "memory"); }
template <typename T, int ROWS, int LD>
__device__ __forceinline__ void win_load_tile(float* dst, const T* src, int64_t stride, int row0, int rows, int n, int n4, bool vec) {
  if (vec) {                          // rows are whole vectors of four
    const int quads = n4 >> 2;
    if constexpr (sizeof(T) == 4) {
      for (int i = threadIdx.x; i < ROWS * quads; i += kWinThreads) {
        const int r = i / quads, c = (i - r * quads) * 4;
        const bool in = row0 + r < rows;
        copy_async16(smem_u32(dst + r * LD + c), src + (int64_t)(in ? row0 + r : 0) * stride + c, in);
      }
    } else {
      for (int i = threadIdx.x; i < ROWS * quads; i += kWinThreads) {
        const int r = i / quads, c = (i - r * quads) * 4;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row0 + r < rows) {
          const uint2 u = *reinterpret_cast<const uint2*>(src + (int64_t)(row0 + r) * stride + c);
          f = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                          __uint_as_float(u.y & 0xFFFF0000u));
        }
        *reinterpret_cast<float4*>(dst + r * LD + c) = f;
      }
    }
  } else {
    for (int i = threadIdx.x; i < ROWS * n4; i += kWinThreads) {
      const int r = i / n4, c = i - r * n4;
      dst[r * LD + c] = row0 + r < rows && c < n ? to_f32(src[(int64_t)(row0 + r) * stride + c]) : 0.f;
    }
  }
}

// acc[i][j] = A[ty + 16 i] . B[tx + 16 j] over n4 features: even and odd ones side by side in one instruction, added at the end
template <int LD, int TM, int TN>
__device__ __forceinline__ void win_dots(float (&acc)[TM][TN], const float* A, const float* B, int n4, int ty, int tx) {
  uint64_t two[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) two[i][j] = 0;
#pragma unroll 2
  for (int d = 0; d < n4; d += 4) {
    ulonglong2 a[TM], b[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) a[i] = *reinterpret_cast<const ulonglong2*>(A + (ty + 16 * i) * LD + d);
#pragma unroll
    for (int j = 0; j < TN; ++j) b[j] = *reinterpret_cast<const ulonglong2*>(B + (tx + 16 * j) * LD + d);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) two[i][j] = fma2(a[i].y, b[j].y, fma2(a[i].x, b[j].x, two[i][j]));
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      float even, odd;
      unpack2(two[i][j], even, odd);
      acc[i][j] = even + odd;
    }
}
__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ void axpy4(float4& o, float w, const float4& v) {
  o.x = fmaf(w, v.x, o.x); o.y = fmaf(w, v.y, o.y); o.z = fmaf(w, v.z, o.z); o.w = fmaf(w, v.w, o.w);
}
// o[i][c] += sum over n of P[ty + 16 i][n] * V[n][4 tx + 64 c ..]
template <int LDP, int LD, int N, int TM, int NC>
__device__ __forceinline__ void win_rows(float4 (&o)[TM][NC], const float* P, const float* V, int ty, int tx) {
#pragma unroll 2
  for (int n = 0; n < N; n += 4) {
    float w[TM][4];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const float4 f = ld4(P + (ty + 16 * i) * LDP + n);
      w[i][0] = f.x; w[i][1] = f.y; w[i][2] = f.z; w[i][3] = f.w;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float4 f = ld4(V + (n + u) * LD + 4 * tx + 64 * c);
#pragma unroll
        for (int i = 0; i < TM; ++i) axpy4(o[i][c], w[i][u], f);
      }
  }
}
// o[i][c] += sum over m of P[m][TN ty + i] * G[m][4 tx + 64 c ..]
template <int LDP, int LD, int M, int TN, int NC>
__device__ __forceinline__ void win_cols(float4 (&o)[TN][NC], const float* P, const float* G, int ty, int tx) {
#pragma unroll 4
  for (int m = 0; m < M; ++m) {
    float w[TN];
    if constexpr (TN == 4) {
      const float4 f = ld4(P + m * LDP + 4 * ty);
      w[0] = f.x; w[1] = f.y; w[2] = f.z; w[3] = f.w;
    } else {
#pragma unroll
      for (int i = 0; i < TN; ++i) w[i] = P[m * LDP + TN * ty + i];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float4 f = ld4(G + m * LD + 4 * tx + 64 * c);
#pragma unroll
      for (int i = 0; i < TN; ++i) axpy4(o[i][c], w[i], f);
    }
  }
}
__device__ __forceinline__ bool finite4(const float4& v) { return isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w); }
template <typename T> __device__ __forceinline__ void win_put4(T* row, int c, int n, const float4& v, float f, T* rest = nullptr) {
  const float a[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < n) {
      row[c + i] = from_f32<T>(a[i]);
      if (rest != nullptr) rest[c + i] = from_f32<T>(win_rest(a[i], to_f32(from_f32<T>(a[i]))));
    }
}
// the maximum / sum over the 16 threads that share rows
__device__ __forceinline__ float half_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float half_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int DP> struct WinTile {
  static constexpr int BM = DP <= 128 ? 64 : 32, TM = BM / 16;        // 64 x 64 logits; 256 features leave room for 32 x 32
  static constexpr int LD = DP + 4, LDP = BM + 4, NC = DP / 64;
  static constexpr int TILE = BM * LD, PTILE = BM * LDP, DIAG = 2 * BM;
  static constexpr int FWD_BYTES = (3 * TILE + PTILE + DIAG) * 4;
  static constexpr int DQ_BYTES = (4 * TILE + PTILE + 3 * DIAG + BM) * 4;
  static constexpr int DKV_BYTES = (4 * TILE + 2 * PTILE + DIAG) * 4;
};

// a thread's bias of the tile's diagonals: index (l - s) + BM - 1, l - s from l0 - s0 - (BM - 1) on
template <typename T, int BM> __device__ __forceinline__ void win_fill_diag(float* diag, int* bucket, const WinParams& p, int h, int l0, int s0) {
  for (int i = threadIdx.x; i < 2 * BM - 1; i += kWinThreads) {
    const int rel = -(l0 - s0 + i - (BM - 1)), b = win_bucket(p.buckets, rel);
    diag[i] = win_bias2(to_f32(static_cast<const T*>(p.table)[h + (int64_t)p.H * b]));
    if (bucket != nullptr) bucket[i] = b;
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kWinThreads) win_fwd_kernel(T* __restrict__ x, T* __restrict__ rest, float2* __restrict__ stats, const __grid_constant__ WinParams p,
                                                              int tiles, int vecq, int vecv) {
  using C = WinTile<DP>;
  constexpr int BM = C::BM, TM = C::TM, LD = C::LD, LDP = C::LDP, NC = C::NC;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sK = sQ + C::TILE, *sV = sK + C::TILE, *sP = sV + C::TILE, *sD = sP + C::PTILE;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int tile = blockIdx.x % tiles, hb = blockIdx.x / tiles, h = hb % p.H, b = hb / p.H, g = h / p.rep;
  const int l0 = tile * BM, queries = win_tokens(p, b, p.L), keys = win_tokens(p, b, p.S);
  const int D4 = (p.D + 3) & ~3, E4 = (p.E + 3) & ~3;
  const T* kb = win_kv_row<T>(p, p.k, p.D, 0, g, b);
  const T* vb = win_kv_row<T>(p, p.v, p.E, 0, g, b);
  win_load_tile<T, BM, LD>(sQ, win_q_row<T>(p, p.q, p.D, 0, h, b), (int64_t)p.H * p.D, l0, queries, p.D, D4, vecq);
  for (int i = threadIdx.x; i < BM * (LD - E4); i += kWinThreads) sV[(i / (LD - E4)) * LD + E4 + i % (LD - E4)] = 0.f;

  float4 o[TM][NC];
  float m[TM], sum[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    m[i] = -INFINITY; sum[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  int sinks, lo, hi;
  win_key_range(p, l0, min(l0 + BM, queries), keys, &sinks, &lo, &hi);
  if (l0 >= queries) sinks = hi = 0;
  const int nsink = (sinks + BM - 1) / BM, first = max(nsink, lo / BM), last = (hi + BM - 1) / BM;
  for (int t = nsink > 0 ? 0 : first; t < max(last, nsink); t = (t + 1 == nsink ? first : t + 1)) {
    const int s0 = t * BM;
    __syncthreads();
    win_load_tile<T, BM, LD>(sK, kb, (int64_t)p.Hkv * p.D, s0, keys, p.D, D4, vecq);
    win_load_tile<T, BM, LD>(sV, vb, (int64_t)p.Hkv * p.E, s0, keys, p.E, E4, vecv);
    if (p.buckets.count > 0) win_fill_diag<T, BM>(sD, nullptr, p, h, l0, s0);
    win_loaded();
    __syncthreads();
    float z[TM][TM];
    win_dots<LD>(z, sQ, sK, D4, ty, tx);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int r = ty + 16 * i, l = l0 + r;
      float mx = m[i];
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int c = tx + 16 * j, s = s0 + c;
        float u = z[i][j] * p.scale2;
        if (p.buckets.count > 0) u += sD[r - c + BM - 1];
        z[i][j] = s < keys && win_sees(p, l, s) ? u : -INFINITY;
        mx = fmaxf(mx, z[i][j]);
      }
      mx = half_max(mx);
      const float ref = mx == -INFINITY ? 0.f : mx, keep = exp2f(m[i] - ref);
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const float w = exp2f(z[i][j] - ref);
        part += w;
        sP[r * LDP + tx + 16 * j] = w;
      }
      m[i] = mx;
      sum[i] = sum[i] * keep + half_sum(part);
#pragma unroll
      for (int c = 0; c < NC; ++c) { o[i][c].x *= keep; o[i][c].y *= keep; o[i][c].z *= keep; o[i][c].w *= keep; }
    }
    __syncwarp();                       // the rows of P that a warp reads are its own
    win_rows<LDP, LD, BM>(o, sP, sV, ty, tx);
  }
  T* xb = x + ((int64_t)b * p.L * p.H + h) * p.E;
  float2* lb = stats != nullptr ? stats + ((int64_t)b * p.H + h) * p.L : nullptr;
  __syncthreads();
  int* bad = reinterpret_cast<int*>(sD);
  for (int i = threadIdx.x; i < BM; i += kWinThreads) bad[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int l = l0 + ty + 16 * i;
    if (l >= p.L) continue;
    const bool any = l < queries && win_any(p, l, keys);
    const float inv = any ? 1.f / sum[i] : 0.f;
    bool ok = isfinite(inv);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      ok = ok && finite4(o[i][c]);
      win_put4(xb + (int64_t)l * p.H * p.E, 4 * tx + 64 * c, p.E, any ? o[i][c] : make_float4(0.f, 0.f, 0.f, 0.f), inv,
               rest != nullptr ? rest + (xb - x) + (int64_t)l * p.H * p.E : nullptr);
    }
    if (lb != nullptr && tx == 0) lb[l] = any ? make_float2(m[i], log2f(sum[i])) : make_float2(0.f, INFINITY);
    if (any && !ok) bad[ty + 16 * i] = 1;
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < BM; r += kWinThreads / 32)
    if (bad[r]) win_row_fwd<T>(p, x, rest, lb != nullptr ? lb + l0 + r : nullptr, l0 + r, h, b, keys);
}

// delta[batch][head][query] = dx . x; LR lanes share a row and take a 16-byte vector each, or (LR = 0) a warp walks it
template <typename T, int LR>
__global__ void __launch_bounds__(256) win_delta_kernel(float* __restrict__ delta, const T* __restrict__ dx, const T* __restrict__ x,
                                                        const T* __restrict__ rest, int E, int H, int L, int64_t rows) {
  constexpr int LANES = LR == 0 ? 32 : LR, V = Vec16<T>::N;
  const int lane = threadIdx.x % LANES;
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;      // (batch, query, head)
  float s = 0.f;
  if (row < rows) {
    const T *a = dx + row * E, *c = x + row * E;
    if constexpr (LR == 0) {
      for (int e = lane; e < E; e += 32) s = fmaf(to_f32(a[e]), to_f32(c[e]) + (rest != nullptr ? to_f32(rest[row * E + e]) : 0.f), s);
    } else if (lane * V < E) {
      const Vec16<T> u = load16(a + lane * V), v = load16(c + lane * V);
      Vec16<T> r;
      r.raw = make_uint4(0, 0, 0, 0);
      if (rest != nullptr) r = load16(rest + row * E + lane * V);
#pragma unroll
      for (int i = 0; i < V; ++i) s = fmaf(u.get(i), v.get(i) + r.get(i), s);
    }
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0 && row < rows) {
    const int64_t h = row % H, bl = row / H, b = bl / L, l = bl - b * L;
    delta[(b * H + h) * L + l] = s;
  }
}

// dq, and partial[tile][batch][head][bucket] of dtable. `rounded`: the forward pass with a table ran on the tensor cores, over the sum of
// weights rounded to bf16; the gradients of a row add up to nothing with those alone.
template <typename T, int DP>
__global__ void __launch_bounds__(kWinThreads, DP == 64 ? 2 : 1) win_dq_kernel(T* __restrict__ dq, float* __restrict__ partial, const T* __restrict__ dx,
                                                             const float2* __restrict__ stats, const float* __restrict__ delta,
                                                             const __grid_constant__ WinParams p, int tiles, int vecq, int vecv, int rounded) {
  using C = WinTile<DP>;
  constexpr int BM = C::BM, TM = C::TM, LD = C::LD, LDP = C::LDP, NC = C::NC;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sG = sQ + C::TILE, *sK = sG + C::TILE, *sV = sK + C::TILE, *sP = sV + C::TILE, *sD = sP + C::PTILE, *sSum = sD + C::DIAG;
  int* sB = reinterpret_cast<int*>(sSum + C::DIAG);
  int* bad = sB + C::DIAG;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int tile = blockIdx.x % tiles, hb = blockIdx.x / tiles, h = hb % p.H, b = hb / p.H, g = h / p.rep;
  const int l0 = tile * BM, queries = win_tokens(p, b, p.L), keys = win_tokens(p, b, p.S);
  const int D4 = (p.D + 3) & ~3, E4 = (p.E + 3) & ~3, columns = p.buckets.count * (p.buckets.bidirectional ? 2 : 1);
  const T* kb = win_kv_row<T>(p, p.k, p.D, 0, g, b);
  const T* vb = win_kv_row<T>(p, p.v, p.E, 0, g, b);
  win_load_tile<T, BM, LD>(sQ, win_q_row<T>(p, p.q, p.D, 0, h, b), (int64_t)p.H * p.D, l0, queries, p.D, D4, vecq);
  win_load_tile<T, BM, LD>(sG, win_q_row<T>(p, dx, p.E, 0, h, b), (int64_t)p.H * p.E, l0, queries, p.E, E4, vecv);
  for (int i = threadIdx.x; i < BM * (LD - D4); i += kWinThreads) sK[(i / (LD - D4)) * LD + D4 + i % (LD - D4)] = 0.f;
  const float2* lb = stats + ((int64_t)b * p.H + h) * p.L;
  const float* db = delta + ((int64_t)b * p.H + h) * p.L;
  float4 o[TM][NC];
  float2 ls[TM];
  float de[TM], of_bucket = 0.f;
  bool single[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int l = l0 + ty + 16 * i;
    ls[i] = l < queries ? lb[l] : make_float2(0.f, INFINITY);
    de[i] = l < queries ? db[l] : 0.f;
    single[i] = win_single(p, l, keys);
#pragma unroll
    for (int c = 0; c < NC; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  int sinks, lo, hi;
  win_key_range(p, l0, min(l0 + BM, queries), keys, &sinks, &lo, &hi);
  if (l0 >= queries) sinks = hi = 0;
  const int nsink = (sinks + BM - 1) / BM, first = max(nsink, lo / BM), last = (hi + BM - 1) / BM;
  for (int t = nsink > 0 ? 0 : first; t < max(last, nsink); t = (t + 1 == nsink ? first : t + 1)) {
    const int s0 = t * BM;
    __syncthreads();
    win_load_tile<T, BM, LD>(sK, kb, (int64_t)p.Hkv * p.D, s0, keys, p.D, D4, vecq);
    win_load_tile<T, BM, LD>(sV, vb, (int64_t)p.Hkv * p.E, s0, keys, p.E, E4, vecv);
    if (p.buckets.count > 0) win_fill_diag<T, BM>(sD, sB, p, h, l0, s0);
    win_loaded();
    __syncthreads();
    float z[TM][TM], dp[TM][TM];
    win_dots<LD>(z, sQ, sK, D4, ty, tx);
    win_dots<LD>(dp, sG, sV, E4, ty, tx);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int r = ty + 16 * i, c = tx + 16 * j, l = l0 + r, s = s0 + c;
        float u = z[i][j] * p.scale2;
        if (p.buckets.count > 0) u += sD[r - c + BM - 1];
        const auto weight = [&] {
          if constexpr (sizeof(T) == 2)
            if (rounded) return __bfloat162float(__float2bfloat16_rn(exp2f(u - ls[i].x))) * exp2f(-ls[i].y);
          return exp2f((u - ls[i].x) - ls[i].y);
        };
        sP[r * LDP + c] = l < queries && s < keys && win_sees(p, l, s) ? weight() * (dp[i][j] - (single[i] ? dp[i][j] : de[i])) : 0.f;
      }
    if (p.buckets.count > 0) {          // sums along the diagonals, then those of a bucket, each in order
      __syncthreads();
      if (threadIdx.x < 2 * BM - 1) {
        const int d = (int)threadIdx.x - (BM - 1);
        float t = 0.f;
        for (int r = max(0, d); r < min(BM, BM + d); ++r) t += sP[r * LDP + r - d];
        sSum[threadIdx.x] = t;
      }
      __syncthreads();
      if (threadIdx.x < columns)
        for (int i = 0; i < 2 * BM - 1; ++i)
          if (sB[i] == (int)threadIdx.x) of_bucket += sSum[i];
    } else {
      __syncwarp();
    }
    win_rows<LDP, LD, BM>(o, sP, sK, ty, tx);
  }
  if (p.buckets.count > 0 && threadIdx.x < columns)
    partial[((int64_t)tile * p.B * p.H + (int64_t)b * p.H + h) * columns + threadIdx.x] = of_bucket;
  T* out = dq + ((int64_t)b * p.L * p.H + h) * p.D;
  for (int i = threadIdx.x; i < BM; i += kWinThreads) bad[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int l = l0 + ty + 16 * i;
    if (l >= p.L) continue;
    bool ok = true;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      ok = ok && finite4(o[i][c]);
      win_put4(out + (int64_t)l * p.H * p.D, 4 * tx + 64 * c, p.D, l < queries ? o[i][c] : make_float4(0.f, 0.f, 0.f, 0.f), p.scale);
    }
    if (l < queries && !ok) bad[ty + 16 * i] = 1;
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < BM; r += kWinThreads / 32)
    if (bad[r]) win_row_dq<T>(p, dq, dx, lb[l0 + r], db[l0 + r], l0 + r, h, b, keys);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kWinThreads, DP == 64 ? 2 : 1) win_dkv_kernel(T* __restrict__ dk, T* __restrict__ dv, const T* __restrict__ dx,
                                                              const float2* __restrict__ stats, const float* __restrict__ delta,
                                                              float* __restrict__ sums, const __grid_constant__ WinParams p, WinSinkPlan plan,
                                                              int tiles, int vecq, int vecv) {
  using C = WinTile<DP>;
  constexpr int BM = C::BM, TM = C::TM, LD = C::LD, LDP = C::LDP, NC = C::NC;
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sG = sQ + C::TILE, *sK = sG + C::TILE, *sV = sK + C::TILE, *sP = sV + C::TILE, *sS = sP + C::PTILE, *sD = sS + C::PTILE;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int groups = p.Hkv * p.B;
  const WinKeyTile mine(blockIdx.x, tiles, groups, plan);
  const int tile = mine.tile, gb = mine.gb, g = gb % p.Hkv, b = gb / p.Hkv;
  const int s0 = tile * BM, queries = win_tokens(p, b, p.L), keys = win_tokens(p, b, p.S);
  const int D4 = (p.D + 3) & ~3, E4 = (p.E + 3) & ~3;
  win_load_tile<T, BM, LD>(sK, win_kv_row<T>(p, p.k, p.D, 0, g, b), (int64_t)p.Hkv * p.D, s0, keys, p.D, D4, vecq);
  win_load_tile<T, BM, LD>(sV, win_kv_row<T>(p, p.v, p.E, 0, g, b), (int64_t)p.Hkv * p.E, s0, keys, p.E, E4, vecv);
  for (int i = threadIdx.x; i < BM * (LD - D4); i += kWinThreads) sQ[(i / (LD - D4)) * LD + D4 + i % (LD - D4)] = 0.f;
  for (int i = threadIdx.x; i < BM * (LD - E4); i += kWinThreads) sG[(i / (LD - E4)) * LD + E4 + i % (LD - E4)] = 0.f;
  float4 ok4[TM][NC], ov4[TM][NC];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int c = 0; c < NC; ++c) ok4[i][c] = ov4[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
  int lo, hi;
  win_query_range(p, s0, min(s0 + BM, keys), queries, &lo, &hi);
  if (s0 >= keys) hi = 0;
  const int per_head = lo < hi ? (hi + BM - 1) / BM - lo / BM : 0, count = per_head * p.rep;
  for (int it = (int)((int64_t)count * mine.split / mine.splits), end = (int)((int64_t)count * (mine.split + 1) / mine.splits); it < end; ++it) {
    const int h = g * p.rep + it / per_head, l0 = (lo / BM + it % per_head) * BM;
    const float2* lb = stats + ((int64_t)b * p.H + h) * p.L;
    const float* db = delta + ((int64_t)b * p.H + h) * p.L;
    __syncthreads();
    win_load_tile<T, BM, LD>(sQ, win_q_row<T>(p, p.q, p.D, 0, h, b), (int64_t)p.H * p.D, l0, queries, p.D, D4, vecq);
    win_load_tile<T, BM, LD>(sG, win_q_row<T>(p, dx, p.E, 0, h, b), (int64_t)p.H * p.E, l0, queries, p.E, E4, vecv);
    if (p.buckets.count > 0) win_fill_diag<T, BM>(sD, nullptr, p, h, l0, s0);
    win_loaded();
    __syncthreads();
    float z[TM][TM], dp[TM][TM];
    win_dots<LD>(z, sQ, sK, D4, ty, tx);
    win_dots<LD>(dp, sG, sV, E4, ty, tx);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int r = ty + 16 * i, l = l0 + r;
      const float2 ls = l < queries ? lb[l] : make_float2(0.f, INFINITY);
      const float de = l < queries ? db[l] : 0.f;
      const bool single = win_single(p, l, keys);
#pragma unroll
      for (int jj = 0; jj < TM; ++jj) {
        const int c = tx + 16 * jj, s = s0 + c;
        float u = z[i][jj] * p.scale2;
        if (p.buckets.count > 0) u += sD[r - c + BM - 1];
        const bool in = l < queries && s < keys && win_sees(p, l, s);
        const float w = in ? exp2f((u - ls.x) - ls.y) : 0.f;
        sP[r * LDP + c] = w;
        sS[r * LDP + c] = in ? w * (dp[i][jj] - (single ? dp[i][jj] : de)) : 0.f;
      }
    }
    __syncthreads();
    win_cols<LDP, LD, BM>(ov4, sP, sG, ty, tx);
    win_cols<LDP, LD, BM>(ok4, sS, sQ, ty, tx);
  }
  if (mine.splits > 1) {
    float* out = sums + (((int64_t)mine.split * plan.tiles + tile) * groups + gb) * BM * (p.D + p.E);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        win_put4(out + (TM * ty + i) * (p.D + p.E), 4 * tx + 64 * c, p.D, ok4[i][c], p.scale);
        win_put4(out + (TM * ty + i) * (p.D + p.E) + p.D, 4 * tx + 64 * c, p.E, ov4[i][c], 1.f);
      }
    return;
  }
  T* dkb = dk + ((int64_t)b * p.S * p.Hkv + g) * p.D;
  T* dvb = dv + ((int64_t)b * p.S * p.Hkv + g) * p.E;
  __syncthreads();
  int* bad = reinterpret_cast<int*>(sD);
  for (int i = threadIdx.x; i < BM; i += kWinThreads) bad[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int s = s0 + TM * ty + i;
    if (s >= p.S) continue;
    bool ok = true;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      ok = ok && finite4(ok4[i][c]) && finite4(ov4[i][c]);
      win_put4(dkb + (int64_t)s * p.Hkv * p.D, 4 * tx + 64 * c, p.D, ok4[i][c], p.scale);
      win_put4(dvb + (int64_t)s * p.Hkv * p.E, 4 * tx + 64 * c, p.E, ov4[i][c], 1.f);
    }
    if (s < keys && !ok) bad[TM * ty + i] = 1;
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < BM; r += kWinThreads / 32)
    if (bad[r]) win_row_dkv<T>(p, dk, dv, dx, stats, delta, s0 + r, g, b, queries, keys);
}

// the sums of a shared tile's blocks in order, a warp per key and head
template <typename T>
__global__ void __launch_bounds__(256) win_sinks_kernel(T* __restrict__ dk, T* __restrict__ dv, const float* __restrict__ sums, const T* __restrict__ dx,
                                                        const float2* __restrict__ stats, const float* __restrict__ delta,
                                                        const __grid_constant__ WinParams p, WinSinkPlan plan, int tile) {
  const int lane = threadIdx.x & 31, groups = p.Hkv * p.B, width = p.D + p.E;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), all = (int64_t)plan.tiles * groups * tile;
  if (row >= all) return;
  const int r = (int)(row % tile), gb = (int)(row / tile % groups), g = gb % p.Hkv, b = gb / p.Hkv, s = (int)(row / tile / groups) * tile + r;
  if (s >= p.S) return;
  const int keys = win_tokens(p, b, p.S);
  T* dkr = dk + (((int64_t)b * p.S + s) * p.Hkv + g) * p.D;
  T* dvr = dv + (((int64_t)b * p.S + s) * p.Hkv + g) * p.E;
  bool fine = true;
  for (int c = lane; c < width; c += 32) {
    float t = 0.f;
    for (int i = 0; i < plan.splits; ++i) t += sums[(i * all + row) * width + c];
    fine = fine && isfinite(t);
    (c < p.D ? dkr[c] : dvr[c - p.D]) = from_f32<T>(s < keys ? t : 0.f);
  }
  if (s < keys && !__all_sync(0xffffffffu, fine)) win_row_dkv<T>(p, dk, dv, dx, stats, delta, s, g, b, win_tokens(p, b, p.L), keys);
}

// ----------------------------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------------------------
int32_t win_check(const lb2_window_dims* d, const lb2_rel_buckets* t, const void* table, const int32_t* lengths, int32_t dtype) {
  LB2_REQUIRE(valid_dtype(dtype), LB2_UNSUPPORTED_DTYPE, "dtype %d not supported", (int)dtype);
  LB2_REQUIRE(d != nullptr, LB2_BAD_ARG, "window dims are null");
  LB2_REQUIRE(d->head_dim >= 0 && d->value_dim >= 0 && d->heads >= 0 && d->kv_heads >= 0 && d->queries >= 0 && d->keys >= 0 && d->batch >= 0,
              LB2_BAD_SHAPE, "negative extent");
  LB2_REQUIRE(d->window >= 1, LB2_BAD_ARG, "the window must hold at least one token");
  LB2_REQUIRE(d->sinks >= 0, LB2_BAD_ARG, "negative number of sinks");
  LB2_REQUIRE(d->head_dim <= kWinMaxDim && d->value_dim <= kWinMaxDim, LB2_BAD_SHAPE, "head_dim and value_dim may be %d at most", kWinMaxDim);
  LB2_REQUIRE(d->heads == 0 || (d->kv_heads > 0 && d->heads % d->kv_heads == 0), LB2_BAD_SHAPE, "heads must be a multiple of kv_heads");
  const int64_t big = 1 << 29;
  LB2_REQUIRE(d->heads <= 65536 && d->queries <= big && d->keys <= big && d->batch <= big, LB2_BAD_SHAPE, "extent too large");
  LB2_REQUIRE((t == nullptr) == (table == nullptr), LB2_BAD_ARG, "table and buckets must both be given or both be null");
  LB2_REQUIRE(aligned_to(lengths, 4), LB2_BAD_ALIGN, "lengths must be 4-byte aligned");
  return t == nullptr ? LB2_OK : check_rel_buckets(t);
}
bool win_empty(const lb2_window_dims* d) { return d->batch == 0 || d->heads == 0; }

WinParams win_params(const lb2_window_dims* d, const void* q, const void* k, const void* v, const void* table, const lb2_rel_buckets* t,
                     const int32_t* lengths, double scale) {
  WinParams p{};
  p.q = q; p.k = k; p.v = v; p.table = table; p.lengths = lengths;
  p.D = (int)d->head_dim; p.E = (int)d->value_dim; p.H = (int)d->heads; p.Hkv = (int)d->kv_heads; p.rep = (int)(d->heads / d->kv_heads);
  p.L = (int)d->queries; p.S = (int)d->keys; p.B = (int)d->batch;
  const int64_t most = d->queries + d->keys + 1;            // a wider window sees no more
  p.window = (int)(d->window < most ? d->window : most);
  p.sinks = (int)(d->sinks < d->keys ? d->sinks : d->keys);
  p.causal = d->causal != 0;
  p.scale = (float)scale; p.scale2 = (float)(scale * 1.4426950408889634);
  if (t != nullptr) p.buckets = *t;
  return p;
}
int win_columns(const lb2_rel_buckets* t) { return t == nullptr ? 0 : t->count * (t->bidirectional ? 2 : 1); }
int win_simt_tile(const lb2_window_dims* d) { return d->head_dim <= 128 && d->value_dim <= 128 ? 64 : 32; }
int64_t win_tiles(int64_t n, int tile) { return (n + tile - 1) / tile; }
size_t win_partial_bytes(const lb2_window_dims* d, const lb2_rel_buckets* t) {
  return align_up((size_t)(win_tiles(d->queries, win_simt_tile(d)) * d->batch * d->heads * win_columns(t)) * sizeof(float), 256);
}
// four features at a time: rows and bases of whole vectors
bool win_vec(int64_t n, const void* a, const void* b, size_t es) { return n % 4 == 0 && aligned_to(a, 4 * es) && aligned_to(b, 4 * es); }

#define LB2_WIN_DISPATCH(d, ...)                                                                   \
  do {                                                                                             \
    const int64_t most_ = (d)->head_dim > (d)->value_dim ? (d)->head_dim : (d)->value_dim;         \
    if (most_ <= 64) { constexpr int DP = 64; __VA_ARGS__; }                                       \
    else if (most_ <= 128) { constexpr int DP = 128; __VA_ARGS__; }                                \
    else { constexpr int DP = 256; __VA_ARGS__; }                                                  \
  } while (0)

template <typename K> int32_t win_smem(K kernel, int bytes) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(LB2_LAUNCH_FAIL, "windowed attention: cannot reserve %d bytes of shared memory: %s", bytes, cudaGetErrorString(e));
  return LB2_OK;
}

template <typename T> int32_t win_delta(float* delta, const T* dx, const T* x, const T* rest, const WinParams& p, int64_t rows, cudaStream_t st) {
  const int lanes = p.E / Vec16<T>::N;
  const bool vec = p.E > 0 && p.E % Vec16<T>::N == 0 && lanes <= 32 && aligned_to(dx, 16) && aligned_to(x, 16) && aligned_to(rest, 16);
  auto launch = [&](auto kernel, int per_row) {
    kernel<<<(unsigned)((rows * per_row + 255) / 256), 256, 0, st>>>(delta, dx, x, rest, p.E, p.H, p.L, rows);
  };
  if (!vec) launch(win_delta_kernel<T, 0>, 32);
  else if (lanes <= 8) launch(win_delta_kernel<T, 8>, 8);
  else if (lanes <= 16) launch(win_delta_kernel<T, 16>, 16);
  else launch(win_delta_kernel<T, 32>, 32);
  LB2_CHECK_LAUNCH("windowed attention delta");
  return LB2_OK;
}

WinSinkPlan win_plan(const lb2_window_dims* d, int tile) {
  return win_sink_plan(tile, d->queries, d->keys, std::min(d->window, d->queries + d->keys + 1), d->sinks, d->heads / d->kv_heads, d->kv_heads * d->batch);
}
// scratch of the tiles whose keys all later queries see
size_t win_sink_bytes(const lb2_window_dims* d, int32_t dtype) {
  auto bytes = [&](int tile) {
    const WinSinkPlan n = win_plan(d, tile);
    return (size_t)n.tiles * n.splits * (size_t)(d->batch * d->kv_heads * tile * (d->head_dim + d->value_dim)) * sizeof(float);
  };
  return align_up(std::max(bytes(win_simt_tile(d)), win_tc_serves(d, dtype) ? bytes(kWtTile) : 0), 256);
}

}  // namespace

int32_t win_sinks_join(const WinParams& p, const WinSinkPlan& plan, int tile, void* dk, void* dv, const float* sums, const void* dx, const float2* stats,
                       const float* delta, int32_t dtype, cudaStream_t st) {
  const int64_t rows = (int64_t)plan.tiles * p.Hkv * p.B * tile;
  LB2_DISPATCH_DTYPE(dtype, {
    win_sinks_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>((T*)dk, (T*)dv, sums, (const T*)dx, stats, delta, p, plan, tile);
  });
  LB2_CHECK_LAUNCH("windowed attention dk, dv of the sinks");
  return LB2_OK;
}

}  // namespace lb2

using namespace lb2;

extern "C" {

int32_t lb2_window_attention_fwd(void* x, void* x_rest, float* stats, const void* q, const void* k, const void* v, const void* table,
                                 const lb2_rel_buckets* buckets, const int32_t* lengths, double scale, const lb2_window_dims* d,
                                 int32_t dtype, void* stream) {
  int32_t rc = win_check(d, buckets, table, lengths, dtype);
  if (rc != LB2_OK) return rc;
  if (win_empty(d) || d->queries == 0) return LB2_OK;
  const size_t es = dtype_size(dtype);
  LB2_REQUIRE((x || d->value_dim == 0) && (q || d->head_dim == 0) && (d->keys == 0 || ((k || d->head_dim == 0) && (v || d->value_dim == 0))), LB2_BAD_ARG,
              "null tensor pointer");
  LB2_REQUIRE(aligned_to(x, es) && aligned_to(x_rest, es) && aligned_to(q, es) && aligned_to(k, es) && aligned_to(v, es) && aligned_to(table, es) &&
                  aligned_to(stats, 8),
              LB2_BAD_ALIGN, "pointer not aligned to the element size");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const WinParams p = win_params(d, q, k, v, table, buckets, lengths, scale);
  if (win_tc_serves(d, dtype) && aligned_to(x, 16) && aligned_to(x_rest, 16) && aligned_to(q, 16) && aligned_to(k, 16) && aligned_to(v, 16))
    return win_tc_fwd(p, x, x_rest, reinterpret_cast<float2*>(stats), st);
  const int tile = win_simt_tile(d);
  const int64_t tiles = win_tiles(d->queries, tile), blocks = tiles * d->heads * d->batch;
  LB2_REQUIRE(blocks <= 0x7FFFFFFF, LB2_BAD_SHAPE, "too many rows");
  LB2_DISPATCH_DTYPE(dtype, LB2_WIN_DISPATCH(d, {
    auto kernel = win_fwd_kernel<T, DP>;
    if ((rc = win_smem(kernel, WinTile<DP>::FWD_BYTES)) != LB2_OK) return rc;
    kernel<<<(unsigned)blocks, kWinThreads, WinTile<DP>::FWD_BYTES, st>>>((T*)x, (T*)x_rest, (float2*)stats, p, (int)tiles, win_vec(d->head_dim, q, k, es),
                                                                          win_vec(d->value_dim, v, nullptr, es));
  }));
  LB2_CHECK_LAUNCH("windowed attention");
  return LB2_OK;
}

size_t lb2_window_attention_bwd_workspace_bytes(const lb2_window_dims* d, const lb2_rel_buckets* buckets, int32_t dtype) {
  if (d == nullptr || !valid_dtype(dtype) || d->queries <= 0 || d->heads <= 0 || d->batch <= 0) return 0;
  if (d->kv_heads <= 0 || d->heads % d->kv_heads != 0) return 0;
  const size_t rows = (size_t)(d->queries * d->heads * d->batch);
  return align_up(rows * sizeof(float), 256) + win_partial_bytes(d, buckets) + win_sink_bytes(d, dtype) + (win_tc_serves(d, dtype) ? win_tc_row_bytes(d) : 0);
}

int32_t lb2_window_attention_bwd(void* dq, void* dk, void* dv, void* dtable, const void* dx, const void* x, const void* x_rest, const float* stats, const void* q,
                                 const void* k, const void* v, const void* table, const lb2_rel_buckets* buckets, const int32_t* lengths,
                                 double scale, const lb2_window_dims* d, int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int32_t rc = win_check(d, buckets, table, lengths, dtype);
  if (rc != LB2_OK) return rc;
  const size_t es = dtype_size(dtype);
  if (win_empty(d)) {                   // no samples or no query heads: the gradients are sums over nothing
    const int64_t keys = d->kv_heads * d->keys * d->batch;
    void* at[3] = {dk, dv, dtable};
    const int64_t count[3] = {keys * d->head_dim, keys * d->value_dim, dtable == nullptr ? 0 : d->heads * win_columns(buckets)};
    for (int i = 0; i < 3; ++i) {
      if (count[i] == 0) continue;
      LB2_REQUIRE(at[i] != nullptr, LB2_BAD_ARG, "null tensor pointer");
      const cudaError_t e = cudaMemsetAsync(at[i], 0, (size_t)count[i] * es, static_cast<cudaStream_t>(stream));
      if (e != cudaSuccess) return fail(LB2_LAUNCH_FAIL, "windowed attention: gradients of nothing: %s", cudaGetErrorString(e));
    }
    return LB2_OK;
  }
  const bool nq = d->queries > 0, nk = d->keys > 0, nd = d->head_dim > 0, ne = d->value_dim > 0;
  LB2_REQUIRE((dq || !nq || !nd) && (dk || !nk || !nd) && (dv || !nk || !ne) && (dx || !nq || !ne) && (x || !nq || !ne) && (stats || !nq) &&
                  (q || !nq || !nd) && (k || !nk || !nd) && (v || !nk || !ne) && (dtable || buckets == nullptr),
              LB2_BAD_ARG, "null tensor pointer");
  LB2_REQUIRE(aligned_to(dq, es) && aligned_to(dk, es) && aligned_to(dv, es) && aligned_to(dtable, es) && aligned_to(dx, es) && aligned_to(x, es) && aligned_to(x_rest, es) &&
                  aligned_to(stats, 8) && aligned_to(q, es) && aligned_to(k, es) && aligned_to(v, es) && aligned_to(table, es),
              LB2_BAD_ALIGN, "pointer not aligned to the element size");
  const size_t need = lb2_window_attention_bwd_workspace_bytes(d, buckets, dtype);
  LB2_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), LB2_WORKSPACE_TOO_SMALL, "workspace of %zu bytes needed", need);
  LB2_REQUIRE(aligned_to(workspace, 256), LB2_BAD_ALIGN, "workspace must be 256-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const WinParams p = win_params(d, q, k, v, table, buckets, lengths, scale);
  const int tile = win_simt_tile(d), columns = win_columns(buckets);
  const int64_t rows = d->queries * d->heads * d->batch;
  float* delta = static_cast<float*>(workspace);
  float* partial = delta + align_up((size_t)rows * sizeof(float), 256) / sizeof(float);
  float* sink_sums = partial + win_partial_bytes(d, buckets) / sizeof(float);
  const int vecq = win_vec(d->head_dim, q, k, es), vecv = win_vec(d->value_dim, v, dx, es);
  const int64_t qt = win_tiles(d->queries, tile), kt = win_tiles(d->keys, tile);
  LB2_REQUIRE(qt * d->heads * d->batch <= 0x7FFFFFFF && kt * d->kv_heads * d->batch <= 0x7FFFFFFF && (rows + 7) / 8 <= 0x7FFFFFFF, LB2_BAD_SHAPE,
              "too many rows");
  const bool tc = win_tc_serves(d, dtype) && aligned_to(x, 16) && aligned_to(x_rest, 16) && aligned_to(q, 16) && aligned_to(k, 16) && aligned_to(v, 16);
  const int rounded = tc && columns > 0;                                         // as the forward pass decided
  if (tc && aligned_to(dq, 16) && aligned_to(dk, 16) && aligned_to(dv, 16) && aligned_to(dx, 16)) {
    float* constants = sink_sums + win_sink_bytes(d, dtype) / sizeof(float);
    rc = win_tc_bwd(p, dq, dk, dv, partial, sink_sums, constants, dx, x, x_rest, reinterpret_cast<const float2*>(stats), delta, st);
    if (rc != LB2_OK || columns == 0) return rc;
    win_dtable_kernel<<<(unsigned)((p.H * columns + 7) / 8), 256, 0, st>>>((__nv_bfloat16*)dtable, partial, p.H, columns, win_tc_partials(d) * d->batch);
    LB2_CHECK_LAUNCH("windowed attention dtable");
    return LB2_OK;
  }
  LB2_DISPATCH_DTYPE(dtype, LB2_WIN_DISPATCH(d, {
    using C = WinTile<DP>;
    if (nq) {
      if ((rc = win_delta(delta, (const T*)dx, (const T*)x, (const T*)x_rest, p, rows, st)) != LB2_OK) return rc;
      if ((rc = win_smem(win_dq_kernel<T, DP>, C::DQ_BYTES)) != LB2_OK) return rc;
      win_dq_kernel<T, DP><<<(unsigned)(qt * d->heads * d->batch), kWinThreads, C::DQ_BYTES, st>>>((T*)dq, partial, (const T*)dx, (const float2*)stats, delta, p, (int)qt,
                                                                                                   vecq, vecv, rounded);
      LB2_CHECK_LAUNCH("windowed attention dq");
    }
    if (columns > 0) {
      win_dtable_kernel<T><<<(unsigned)((p.H * columns + 7) / 8), 256, 0, st>>>((T*)dtable, partial, p.H, columns, nq ? qt * d->batch : 0);
      LB2_CHECK_LAUNCH("windowed attention dtable");
    }
    if (nk) {
      if ((rc = win_smem(win_dkv_kernel<T, DP>, C::DKV_BYTES)) != LB2_OK) return rc;
      const WinSinkPlan plan = win_plan(d, tile);
      const int64_t blocks = (kt - plan.tiles + (int64_t)plan.tiles * plan.splits) * d->kv_heads * d->batch;
      LB2_REQUIRE(blocks <= 0x7FFFFFFF, LB2_BAD_SHAPE, "too many rows");
      win_dkv_kernel<T, DP><<<(unsigned)blocks, kWinThreads, C::DKV_BYTES, st>>>((T*)dk, (T*)dv, (const T*)dx, (const float2*)stats, delta, sink_sums, p, plan,
                                                                                (int)kt, vecq, vecv);
      LB2_CHECK_LAUNCH("windowed attention dk, dv");
      if (plan.tiles > 0 && (rc = win_sinks_join(p, plan, tile, dk, dv, sink_sums, dx, (const float2*)stats, delta, dtype, st)) != LB2_OK) return rc;
    }
  }));
  return LB2_OK;
}

}  // extern "C"
