// Windowed attention for one new token per sequence, over a ring cache of keys and values. The attention step itself is that of
// lib/LuxLib/src/impl/attention.jl:76-118; the reference keeps no cache.
//
// A cache of `capacity` slots holds position p in slot p while p < sinks, and later ones in
// sinks + (p - sinks) mod (capacity - sinks): the sinks stay, the rest is overwritten oldest first. With
// capacity >= sinks + window all that the new token sees is there.
#include "common.cuh"
#include "window.cuh"

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

// a block per (sequence, head); its warps take the keys in turn
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
  const int lo = max(0, n - p.window + 1), early = min(p.sinks, lo), count = early + (n + 1 - lo);
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
  if (d->batch == 0 || d->heads == 0) return LB2_OK;
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
