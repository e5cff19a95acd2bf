// Learned relative position bias by buckets: bias[s, l, h] = table[h, bucket(s - l - offset)], the bias that
// scaled_dot_product_attention (lib/LuxLib/src/api/attention.jl, impl/attention.jl:76-118) adds to its logits, and its gradient
// dtable[h, j] = sum of dbias over the pairs (and samples) of bucket j.
#include "common.cuh"
#include "window.cuh"

namespace lb2 {

int32_t check_rel_buckets(const lb2_rel_buckets* t) {
  LB2_REQUIRE(t != nullptr, LB2_BAD_ARG, "buckets are null");
  LB2_REQUIRE(t->count >= 1 && t->count <= kWinMaxBuckets, LB2_BAD_ARG, "1 to %d buckets per side", kWinMaxBuckets);
  LB2_REQUIRE(t->first[0] == 0, LB2_BAD_ARG, "the first bucket starts at distance 0");
  for (int i = 1; i < t->count; ++i) LB2_REQUIRE(t->first[i] >= t->first[i - 1], LB2_BAD_ARG, "the buckets' first distances must not fall");
  return LB2_OK;
}

namespace {

constexpr int kRelRows = 64;      // queries per partial sum

template <typename T>
__global__ void __launch_bounds__(256) relpos_fwd_kernel(T* __restrict__ bias, const T* __restrict__ table, const __grid_constant__ lb2_rel_buckets t,
                                                         int S, int L, int H, int offset, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / S;
    const int s = (int)(i - row * S), h = (int)(row / L), l = (int)(row - (int64_t)h * L);
    bias[i] = table[h + (int64_t)H * win_bucket(t, s - l - offset)];
  }
}

// partial[chunk][h][diagonal]: diagonal i holds s - l = i - (L - 1)
template <typename T>
__global__ void __launch_bounds__(256) relpos_diag_kernel(float* __restrict__ partial, const T* __restrict__ dbias, int S, int L, int H, int B) {
  const int i = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y, chunk = blockIdx.z, d = i - (L - 1);
  if (i >= S + L - 1) return;
  const int lo = max(chunk * kRelRows, -d), hi = min(min((chunk + 1) * kRelRows, L), S - d);
  float sum = 0.f;
  for (int b = 0; b < B; ++b)
    for (int l = lo; l < hi; ++l) sum += to_f32(dbias[(((int64_t)b * H + h) * L + l) * S + l + d]);
  partial[((int64_t)chunk * H + h) * (S + L - 1) + i] = sum;
}
// a block per (head, bucket): its diagonals of all chunks, 64 bits
template <typename T>
__global__ void __launch_bounds__(256) relpos_bucket_kernel(T* __restrict__ dtable, const float* __restrict__ partial,
                                                            const __grid_constant__ lb2_rel_buckets t, int S, int L, int H, int offset, int chunks) {
  __shared__ double red[8];
  const int h = blockIdx.x, j = blockIdx.y, n = S + L - 1;
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += 256)
    if (win_bucket(t, i - (L - 1) - offset) == j)
      for (int c = 0; c < chunks; ++c) sum += partial[((int64_t)c * H + h) * n + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) sum += red[w];
    dtable[h + (int64_t)H * j] = from_f32<T>((float)sum);
  }
}

int32_t relpos_check(const lb2_rel_buckets* t, int64_t S, int64_t L, int64_t H, int64_t offset, int32_t dtype) {
  LB2_REQUIRE(valid_dtype(dtype), LB2_UNSUPPORTED_DTYPE, "dtype %d not supported", (int)dtype);
  LB2_REQUIRE(S >= 0 && L >= 0 && H >= 0, LB2_BAD_SHAPE, "negative extent");
  const int64_t big = 1 << 22;
  LB2_REQUIRE(S <= big && L <= big && H <= 65535, LB2_BAD_SHAPE, "extent too large");
  LB2_REQUIRE(offset >= -(1 << 29) && offset <= (1 << 29), LB2_BAD_ARG, "offset too large");
  return check_rel_buckets(t);
}
int rel_columns(const lb2_rel_buckets* t) { return t->count * (t->bidirectional ? 2 : 1); }

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
  const int64_t n = S * L * H, blocks = (n + 255) / 256, cap = (int64_t)sm_count() * 8;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LB2_DISPATCH_DTYPE(dtype, {
    relpos_fwd_kernel<T><<<(unsigned)(blocks < cap ? blocks : cap), 256, 0, st>>>((T*)bias, (const T*)table, *buckets, (int)S, (int)L, (int)H, (int)offset, n);
  });
  LB2_CHECK_LAUNCH("relative position bias");
  return LB2_OK;
}

size_t lb2_relpos_bias_bwd_workspace_bytes(const lb2_rel_buckets* buckets, int64_t S, int64_t L, int64_t H, int64_t B) {
  (void)buckets;
  if (S <= 0 || L <= 0 || H <= 0 || B <= 0) return 0;
  return align_up((size_t)((L + kRelRows - 1) / kRelRows * H * (S + L - 1)) * sizeof(float), 256);
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
  const int chunks = none ? 0 : (int)((L + kRelRows - 1) / kRelRows);
  LB2_REQUIRE(chunks <= 65535, LB2_BAD_SHAPE, "too many queries");
  float* partial = static_cast<float*>(workspace);
  LB2_DISPATCH_DTYPE(dtype, {
    if (!none) {
      relpos_diag_kernel<T><<<dim3((unsigned)((S + L - 1 + 255) / 256), (unsigned)H, (unsigned)chunks), 256, 0, st>>>(partial, (const T*)dbias, (int)S, (int)L,
                                                                                                                   (int)H, (int)B);
      LB2_CHECK_LAUNCH("relative position bias diagonals");
    }
    relpos_bucket_kernel<T><<<dim3((unsigned)H, (unsigned)rel_columns(buckets)), 256, 0, st>>>((T*)dtable, partial, *buckets, (int)S, (int)L, (int)H,
                                                                                            (int)offset, chunks);
  });
  LB2_CHECK_LAUNCH("relative position bias buckets");
  return LB2_OK;
}

}  // extern "C"
