// Learned relative position bias by buckets: bias[s, l, h] = table[h, bucket(s - l - offset)], the bias that
// scaled_dot_product_attention (lib/LuxLib/src/api/attention.jl, impl/attention.jl:76-118) adds to its logits, and its gradient
// dtable[h, j] = sum of dbias over the pairs (and samples) of bucket j.
#include "common.cuh"
#include "window_tc.cuh"

namespace lb2 {

int32_t check_rel_buckets(const lb2_rel_buckets* t) {
  LB2_REQUIRE(t != nullptr, LB2_BAD_ARG, "buckets are null");
  LB2_REQUIRE(t->count >= 1 && t->count <= kWinMaxBuckets, LB2_BAD_ARG, "1 to %d buckets per side", kWinMaxBuckets);
  LB2_REQUIRE(t->first[0] == 0, LB2_BAD_ARG, "the first bucket starts at distance 0");
  for (int i = 1; i < t->count; ++i) LB2_REQUIRE(t->first[i] >= t->first[i - 1], LB2_BAD_ARG, "the buckets' first distances must not fall");
  return LB2_OK;
}

namespace {

constexpr int kRelRows = 64;      // queries per block

// Forward: a block writes kRelRows x kRelKeys values of a head, all from the kRelRows + kRelKeys - 1 diagonals that it works out once.
// Shared memory holds the diagonals once per alignment (copy r starts at diagonal r), so that a 16-byte store of neighbouring keys is
// one aligned 16-byte load whatever the row. Bounded by the stores: 16 heads of 1024 x 1024 bf16, 33.5 MB in 9.6 us (3.5 TB/s).
constexpr int kRelKeys = 1024;
template <typename T>
__global__ void __launch_bounds__(256) relpos_fwd_kernel(T* __restrict__ bias, const T* __restrict__ table, const __grid_constant__ lb2_rel_buckets t,
                                                         int S, int L, int H, int offset) {
  constexpr int V = 16 / sizeof(T), N = kRelRows + kRelKeys;
  __shared__ __align__(16) T lut[V][N];
  const int h = blockIdx.z, s0 = blockIdx.x * kRelKeys, l0 = blockIdx.y * kRelRows, keys = min(kRelKeys, S - s0), rows = min(kRelRows, L - l0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ int32_t first_of[kWinMaxBuckets];
  if (threadIdx.x < kWinMaxBuckets) first_of[threadIdx.x] = t.first[threadIdx.x];
  __syncthreads();
  // diagonal i: s - l = s0 - l0 - (kRelRows - 1) + i
  for (int i = threadIdx.x; i < keys + kRelRows - 1; i += 256) {
    const T v = table[h + (int64_t)H * win_bucket(t, first_of, s0 - l0 - (kRelRows - 1) + i - offset)];
#pragma unroll
    for (int r = 0; r < V; ++r)
      if (i >= r) lut[r][i - r] = v;
  }
  __syncthreads();
  for (int row = warp; row < rows; row += 8) {
    T* out = bias + ((int64_t)h * L + l0 + row) * S + s0;
    const int first = kRelRows - 1 - row;                                 // diagonal of the row's first key
    const int head = min(keys, (int)((16 - reinterpret_cast<uintptr_t>(out) % 16) % 16 / sizeof(T))), end = head + (keys - head) / V * V;
    if (lane < head) out[lane] = lut[0][first + lane];
    if (end + lane < keys) out[end + lane] = lut[0][first + end + lane];
    const int r = (first + head) % V;
    for (int s = head + lane * V; s < end; s += 32 * V) store16_stream(out + s, load16(&lut[r][first + s - r]));
  }
}

// Backward: a warp takes 32 V neighbouring keys (V per lane, one load) of V queries at a time. A lane's V x V values lie on 2 V - 1
// diagonals; V of them, complete for this lane, are the next lane's upper ones in the next V queries: they move there with
// a shuffle, and out of lane 31 to the warp's sums in shared memory. The block joins its warps, then diagonals by bucket;
// all in a fixed order. Measured: 16 heads of 1024 x 1024, 4 samples, bf16: 134 MB in 33.6 us (4.0 TB/s, 0.61 of the copy rate); the conversions
// and sums of a value are five instructions. A diagonal's 32 rows (and all samples of a warp) are summed in fp32, the blocks' sums in
// 64 bits: 197 x 197 Float32 values are off by 9e-8 where 64 bits throughout leave 2.4e-8, the result's own rounding.
constexpr int kRelWarps = 4, kRelBwdRows = 32;    // 32 rows: blocks enough to even out over the SMs
template <typename T, int V>
__global__ void __launch_bounds__(32 * kRelWarps) relpos_bwd_kernel(float* __restrict__ partial, const T* __restrict__ dbias,
                                                                    const __grid_constant__ lb2_rel_buckets t, int S, int L, int H, int B, int offset,
                                                                    int columns) {
  constexpr int KEYS = 32 * V, N = KEYS + kRelBwdRows;                       // diagonal i: s - l = s0 - l0 - (kRelBwdRows - 1) + i
  __shared__ __align__(16) float sums[kRelWarps][N];
  __shared__ uint4 ring[kRelWarps][2][V == 1 ? 1 : V][32];                // each lane's next loads, two blocks of rows ahead
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.z, s0 = blockIdx.x * KEYS, l0 = blockIdx.y * kRelBwdRows;
  for (int i = threadIdx.x; i < N; i += 32 * kRelWarps) {
#pragma unroll
    for (int w = 0; w < kRelWarps; ++w) sums[w][i] = 0.f;
  }
  __syncthreads();
  // the warps share the samples, or the rows where samples are few
  const bool by_sample = B >= kRelWarps;
  const int lo = by_sample ? 0 : warp * (kRelBwdRows / kRelWarps), hi = min(L - l0, by_sample ? kRelBwdRows : lo + kRelBwdRows / kRelWarps);
  const int s = s0 + lane * V;
  float* my = sums[warp];
  for (int b = by_sample ? warp : 0; b < B; b += by_sample ? kRelWarps : 1) {
    const T* in = dbias + (((int64_t)b * H + h) * L + l0) * S + min(s, S - V);
    float a[2 * V - 1];                                                   // diagonal s - row + x - (V - 1) of the block of V rows
#pragma unroll
    for (int x = 0; x < 2 * V - 1; ++x) a[x] = 0.f;
    auto fetch = [&](int r0, int stage) {
      if constexpr (V > 1) {
        if (r0 < hi) {
#pragma unroll
          for (int k = 0; k < V; ++k) copy_async16(smem_u32(&ring[warp][stage][k][lane]), in + (int64_t)min(r0 + k, hi - 1) * S);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
    };
    float next[8];                                                        // V = 1: eight rows at a time
    auto load8 = [&](int r0) {
      if constexpr (V == 1) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float v = to_f32(in[(int64_t)min(r0 + k, max(hi - 1, 0)) * S]);
          next[k] = r0 + k < hi && s < S ? v : 0.f;
        }
      }
    };
    if (lo < hi) load8(lo);
    fetch(lo, 0);
    fetch(lo + V, 1);
    int row = lo, stage = 0;
    for (; row < hi; row += V) {
      if (row > lo) {
#pragma unroll
        for (int x = 0; x < V; ++x) {
          const float up = __shfl_up_sync(0xffffffffu, a[V - 1 + x], 1);
          if (lane == 31) my[31 * V + x + kRelBwdRows - 1 - (row - V)] += a[V - 1 + x];
          a[V - 1 + x] = (lane == 0 ? 0.f : up) + (x > 0 ? a[x - 1] : 0.f);
        }
#pragma unroll
        for (int x = 0; x < V - 1; ++x) a[x] = 0.f;
      }
      if constexpr (V == 1) {
        a[0] += next[(row - lo) & 7];
        if (((row - lo) & 7) == 7) load8(row + 1);
      } else {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
#pragma unroll
        for (int k = 0; k < V; ++k) {
          Vec16<T> v;
          v.raw = ring[warp][stage][k][lane];
          if (row + k >= hi || s >= S) v.raw = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < V; ++e) a[e - k + V - 1] += v.get(e);
        }
        fetch(row + 2 * V, stage);
        stage ^= 1;
      }
    }
    row -= V;                                                             // the last block's first row; empty where lo >= hi
    __syncwarp();
    if (lo < hi) {
      // neighbouring lanes share diagonals: the upper ones first, then the lower ones
#pragma unroll
      for (int x = 0; x < V; ++x) my[lane * V + x + kRelBwdRows - 1 - row] += a[V - 1 + x];
      __syncwarp();
#pragma unroll
      for (int x = 0; x < V - 1; ++x) {
        const int i = lane * V + x - (V - 1) + kRelBwdRows - 1 - row;
        if (i >= 0) my[i] += a[x];                                        // rows past the last held zeros
      }
      __syncwarp();
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < N; i += 32 * kRelWarps) {
    float v = sums[0][i];
#pragma unroll
    for (int w = 1; w < kRelWarps; ++w) v += sums[w][i];
    sums[0][i] = v;
  }
  __syncthreads();
  // a bucket's diagonals lie side by side: a warp per bucket
  const int base = s0 - l0 - (kRelBwdRows - 1) - offset;
  for (int j = warp; j < columns; j += kRelWarps) {
    const int k = j < t.count ? j : j - t.count, near = t.first[k], past = k + 1 < t.count ? t.first[k + 1] : 0x7FFFFFFF;
    int lo, hi;                                                           // relative positions of the bucket
    if (j < t.count) {
      lo = -(past - 1);
      hi = t.bidirectional || near > 0 ? -near : 0x7FFFFFFF;
      if (!t.bidirectional && near == 0 && past == 0) hi = lo - 1;
    } else {
      lo = max(near, 1); hi = past - 1;
    }
    float v = 0.f;
    const int64_t end = min((int64_t)hi - base, (int64_t)N - 1);
    for (int64_t i = max((int64_t)lo - base, (int64_t)0) + lane; i <= end; i += 32) v += sums[0][i];
    v = warp_sum(v);
    if (lane == 0) partial[(((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * H + h) * columns + j] = v;
  }
}
int rel_columns(const lb2_rel_buckets* t) { return t->count * (t->bidirectional ? 2 : 1); }
int64_t rel_blocks(int64_t n, int64_t per) { return (n + per - 1) / per; }

int32_t relpos_check(const lb2_rel_buckets* t, int64_t S, int64_t L, int64_t H, int64_t offset, int32_t dtype) {
  LB2_REQUIRE(valid_dtype(dtype), LB2_UNSUPPORTED_DTYPE, "dtype %d not supported", (int)dtype);
  LB2_REQUIRE(S >= 0 && L >= 0 && H >= 0, LB2_BAD_SHAPE, "negative extent");
  const int64_t big = 65535 * kRelBwdRows;                 // blocks along a grid's second axis
  LB2_REQUIRE(S <= big && L <= big && H <= 65535, LB2_BAD_SHAPE, "extent too large");
  LB2_REQUIRE(offset >= -(1 << 29) && offset <= (1 << 29), LB2_BAD_ARG, "offset too large");
  return check_rel_buckets(t);
}
}  // namespace

}  // namespace lb2

using namespace lb2;

extern "C" {

int32_t lb2_relpos_bias_fwd(void* bias, const void* table, const lb2_rel_buckets* buckets, int64_t S, int64_t L, int64_t H, int64_t offset,
                            int32_t dtype, void* stream) {
  int32_t rc = relpos_check(buckets, S, L, H, offset, dtype);
  if (rc != LB2_OK) return rc;
  if (S == 0 || L == 0 || H == 0) return LB2_OK;
  LB2_REQUIRE(bias && table, LB2_BAD_ARG, "null tensor pointer");
  const size_t es = dtype_size(dtype);
  LB2_REQUIRE(aligned_to(bias, es) && aligned_to(table, es), LB2_BAD_ALIGN, "pointer not aligned to the element size");
  const dim3 grid((unsigned)rel_blocks(S, kRelKeys), (unsigned)rel_blocks(L, kRelRows), (unsigned)H);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LB2_DISPATCH_DTYPE(dtype, {
    relpos_fwd_kernel<T><<<grid, 256, 0, st>>>((T*)bias, (const T*)table, *buckets, (int)S, (int)L, (int)H, (int)offset);
  });
  LB2_CHECK_LAUNCH("relative position bias");
  return LB2_OK;
}

size_t lb2_relpos_bias_bwd_workspace_bytes(const lb2_rel_buckets* buckets, int64_t S, int64_t L, int64_t H, int64_t B) {
  if (buckets == nullptr || S <= 0 || L <= 0 || H <= 0 || B <= 0) return 0;
  return align_up((size_t)(rel_blocks(S, 32) * rel_blocks(L, kRelBwdRows) * H * rel_columns(buckets)) * sizeof(float), 256);
}

int32_t lb2_relpos_bias_bwd(void* dtable, const void* dbias, const lb2_rel_buckets* buckets, int64_t S, int64_t L, int64_t H, int64_t B,
                            int64_t offset, int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int32_t rc = relpos_check(buckets, S, L, H, offset, dtype);
  if (rc != LB2_OK) return rc;
  LB2_REQUIRE(B >= 0 && B <= (1 << 29), LB2_BAD_SHAPE, "batch out of range");
  if (H == 0) return LB2_OK;
  LB2_REQUIRE(dtable != nullptr, LB2_BAD_ARG, "null tensor pointer");
  const size_t es = dtype_size(dtype);
  LB2_REQUIRE(aligned_to(dtable, es) && aligned_to(dbias, es), LB2_BAD_ALIGN, "pointer not aligned to the element size");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool none = S == 0 || L == 0 || B == 0;           // a sum over nothing
  LB2_REQUIRE(none || dbias != nullptr, LB2_BAD_ARG, "null tensor pointer");
  const size_t need = lb2_relpos_bias_bwd_workspace_bytes(buckets, S, L, H, B);
  LB2_REQUIRE(none || (workspace != nullptr && workspace_bytes >= need), LB2_WORKSPACE_TOO_SMALL, "workspace of %zu bytes needed", need);
  LB2_REQUIRE(aligned_to(workspace, 256), LB2_BAD_ALIGN, "workspace must be 256-byte aligned");
  float* partial = static_cast<float*>(workspace);
  const int columns = rel_columns(buckets);
  int64_t blocks = 0;
  LB2_DISPATCH_DTYPE(dtype, {
    if (!none) {
      constexpr int V = Vec16<T>::N;
      auto launch = [&](auto kernel, int keys) {       // whole vectors only where every row starts on one
        const dim3 grid((unsigned)rel_blocks(S, keys), (unsigned)rel_blocks(L, kRelBwdRows), (unsigned)H);
        blocks = (int64_t)grid.x * grid.y;
        kernel<<<grid, 32 * kRelWarps, 0, st>>>(partial, (const T*)dbias, *buckets, (int)S, (int)L, (int)H, (int)B, (int)offset, columns);
      };
      if (S % V == 0 && aligned_to(dbias, 16)) launch(relpos_bwd_kernel<T, V>, 32 * V);
      else launch(relpos_bwd_kernel<T, 1>, 32);
      LB2_CHECK_LAUNCH("relative position bias gradient");
    }
    win_dtable_kernel<T><<<(unsigned)rel_blocks(H * columns, 8), 256, 0, st>>>((T*)dtable, partial, (int)H, columns, blocks);
  });
  LB2_CHECK_LAUNCH("relative position bias gradient's sums");
  return LB2_OK;
}

}  // extern "C"
