// Windowed attention on the tensor cores (BFloat16, up to 128 features): declarations shared by its forward and backward kernels.
#pragma once
#include "tc_ptx.cuh"
#include "window.cuh"

namespace lb2 {

constexpr int kWtTile = 128;                 // queries and keys of a tile
constexpr int kWtBox = kWtTile * 128;        // bytes of a TMA box: 128 tokens x 64 features
// what the tensor-core kernels serve: rows of whole 16-byte vectors for TMA, at most two boxes of features
bool win_tc_serves(const lb2_window_dims* d, int32_t dtype);
int64_t win_tc_partials(const lb2_window_dims* d);      // blocks that leave a partial sum of dtable per head and sample
size_t win_tc_row_bytes(const lb2_window_dims* d);     // scratch for the rows' constants
int32_t win_tc_bwd(const WinParams& p, void* dq, void* dk, void* dv, float* partial, float* sink_sums, float* rows, const void* dx, const void* x,
                   const void* rest, const float2* stats, float* delta, cudaStream_t st);
int32_t win_tc_fwd(const WinParams& p, void* x, void* rest, float2* stats, cudaStream_t st);

// token arrays (features, heads, tokens, batch) in boxes of 64 features x 128 tokens of one head
inline bool wt_encode(CUtensorMap* map, const void* ptr, int64_t features, int64_t heads, int64_t tokens, int64_t batch) {
  TensorMapEncodeFn enc = tensor_map_encoder();
  if (!enc) return false;
  cuuint64_t dims[4] = {(cuuint64_t)features, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)batch};
  cuuint64_t strides[3] = {(cuuint64_t)(features * 2), (cuuint64_t)(features * heads * 2), (cuuint64_t)(features * heads * tokens * 2)};
  cuuint32_t box[4] = {64, 1, kWtTile, 1}, estr[4] = {1, 1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Blocks for `items`: one per SM that takes its items in turn, or one per item, which the device hands out as SMs come free. Taking them
// in turn saves some 3 us an item (start, first loads, last stores); the other way saves about half an item where they do not come out
// even. `steps`: tiles of one window, though queries that look both ways see two: what does not come out even is that the first
// tokens see fewer, and with two sides they see half as many, not one. Measured at 16 heads on 4, 8192 tokens, 128 features, in turn and
// as they come, us, an asterisk at the side that the rule takes:
//   window            512         1024        2048        4096      both ways  512         1024        2048        4096
//   forward           76* 87      107* 116    167* 162    265 229*             107* 118    168* 172    266* 270    433 420*
//   dq                78* 93      116* 127    187* 191    297* 286             114* 129    186* 198    299* 322    492* 511
//   dk dv             100 104*    158 164*    276 282*    467 434*             157 161*    274 275*    464 464*    709 711*
// With 2048 sinks and window 512, whose tiles `steps` leaves out: forward 195* 181, dq 219* 219, dk dv 305 281*; with 512 sinks 105* 114,
// 115* 127, 164 170*. 16 heads of 64 features, 4096 tokens, both ways, window 1024: 71* 74, 82* 86, 108* 115; 2048: 105 111*, 125* 128, 165* 172.
inline unsigned wt_blocks(int items, int sms, int64_t steps) { return (unsigned)(items <= sms || (int64_t)items * 7 > steps * sms ? std::min(items, sms) : items); }

// Shared-memory descriptors of a tile of 128 tokens in boxes: features as the contraction (K-major: 32 bytes per step of 16, the
// next box after four) or tokens as the contraction (MN-major: 16 rows of 128 bytes per step, boxes side by side along N).
constexpr uint32_t kWtDescHi = ((1024u >> 4) & 0x3FFFu) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint64_t wt_desc_k(uint32_t addr) { return ((uint64_t)kWtDescHi << 32) | ((addr >> 4) & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ uint64_t wt_desc_mn(uint32_t addr) {
  return ((uint64_t)kWtDescHi << 32) | ((addr >> 4) & 0x3FFFu) | ((uint32_t)(kWtBox >> 4) << 16);
}
__host__ __device__ constexpr uint32_t wt_idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kWtTile >> 4) << 24);
}
// D[128][128] = A . B' over NB boxes of features, both K-major in shared memory
template <int NB> __device__ __forceinline__ void wt_mma_features(uint32_t d, uint32_t a, uint32_t b) {
  const uint64_t ad = wt_desc_k(a), bd = wt_desc_k(b);
#pragma unroll
  for (int ks = 0; ks < 4 * NB; ++ks) {
    const uint32_t at = (ks >> 2) * (kWtBox >> 4) + (ks & 3) * 2;
    umma<false>(d, ad + at, bd + at, wt_idesc(kWtTile, false), ks != 0 ? 1u : 0u);
  }
}
// A operand in TMEM: 128 lanes x 128 values, two bf16 per column
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[128][64 NB] (+)= P . V: P from TMEM, V a tile of 128 tokens
template <int NB> __device__ __forceinline__ void wt_mma_tokens(uint32_t d, uint32_t p, uint32_t v, bool accumulate) {
  const uint64_t vd = wt_desc_mn(v);
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) umma_ts(d, p + ks * 8, vd + ks * ((16 * 128) >> 4), wt_idesc(64 * NB, true), (accumulate || ks != 0) ? 1u : 0u);
}
// with P in two halves 64 columns apart, each over the columns that its own threads have read
template <int NB> __device__ __forceinline__ void wt_mma_tokens_halves(uint32_t d, uint32_t p, uint32_t v, bool accumulate) {
  const uint64_t vd = wt_desc_mn(v);
#pragma unroll
  for (int ks = 0; ks < 8; ++ks)
    umma_ts(d, p + (ks >> 2) * 64 + (ks & 3) * 8, vd + ks * ((16 * 128) >> 4), wt_idesc(64 * NB, true), (accumulate || ks != 0) ? 1u : 0u);
}
// `N` columns of a row and the wait for them in one statement, so that nothing reads the registers in between
template <int O, int M> __device__ __forceinline__ void tmem_row32(uint32_t taddr, float (&z)[M]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(z[O + 0]), "=f"(z[O + 1]), "=f"(z[O + 2]), "=f"(z[O + 3]), "=f"(z[O + 4]), "=f"(z[O + 5]), "=f"(z[O + 6]), "=f"(z[O + 7]),
        "=f"(z[O + 8]), "=f"(z[O + 9]), "=f"(z[O + 10]), "=f"(z[O + 11]), "=f"(z[O + 12]), "=f"(z[O + 13]), "=f"(z[O + 14]), "=f"(z[O + 15]),
        "=f"(z[O + 16]), "=f"(z[O + 17]), "=f"(z[O + 18]), "=f"(z[O + 19]), "=f"(z[O + 20]), "=f"(z[O + 21]), "=f"(z[O + 22]), "=f"(z[O + 23]),
        "=f"(z[O + 24]), "=f"(z[O + 25]), "=f"(z[O + 26]), "=f"(z[O + 27]), "=f"(z[O + 28]), "=f"(z[O + 29]), "=f"(z[O + 30]), "=f"(z[O + 31])
      : "r"(taddr)
      : "memory");
}
template <int O, int M> __device__ __forceinline__ void tmem_row64(uint32_t taddr, float (&z)[M]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(z[O + 0]), "=f"(z[O + 1]), "=f"(z[O + 2]), "=f"(z[O + 3]), "=f"(z[O + 4]), "=f"(z[O + 5]), "=f"(z[O + 6]), "=f"(z[O + 7]),
        "=f"(z[O + 8]), "=f"(z[O + 9]), "=f"(z[O + 10]), "=f"(z[O + 11]), "=f"(z[O + 12]), "=f"(z[O + 13]), "=f"(z[O + 14]), "=f"(z[O + 15]),
        "=f"(z[O + 16]), "=f"(z[O + 17]), "=f"(z[O + 18]), "=f"(z[O + 19]), "=f"(z[O + 20]), "=f"(z[O + 21]), "=f"(z[O + 22]), "=f"(z[O + 23]),
        "=f"(z[O + 24]), "=f"(z[O + 25]), "=f"(z[O + 26]), "=f"(z[O + 27]), "=f"(z[O + 28]), "=f"(z[O + 29]), "=f"(z[O + 30]), "=f"(z[O + 31]),
        "=f"(z[O + 32]), "=f"(z[O + 33]), "=f"(z[O + 34]), "=f"(z[O + 35]), "=f"(z[O + 36]), "=f"(z[O + 37]), "=f"(z[O + 38]), "=f"(z[O + 39]),
        "=f"(z[O + 40]), "=f"(z[O + 41]), "=f"(z[O + 42]), "=f"(z[O + 43]), "=f"(z[O + 44]), "=f"(z[O + 45]), "=f"(z[O + 46]), "=f"(z[O + 47]),
        "=f"(z[O + 48]), "=f"(z[O + 49]), "=f"(z[O + 50]), "=f"(z[O + 51]), "=f"(z[O + 52]), "=f"(z[O + 53]), "=f"(z[O + 54]), "=f"(z[O + 55]),
        "=f"(z[O + 56]), "=f"(z[O + 57]), "=f"(z[O + 58]), "=f"(z[O + 59]), "=f"(z[O + 60]), "=f"(z[O + 61]), "=f"(z[O + 62]), "=f"(z[O + 63])
      : "r"(taddr)
      : "memory");
}
template <int O, int M> __device__ __forceinline__ void tmem_row128(uint32_t taddr, float (&z)[M]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63, "
      "%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, "
      "%80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95, "
      "%96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, "
      "%112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127}, [%128];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(z[O + 0]), "=f"(z[O + 1]), "=f"(z[O + 2]), "=f"(z[O + 3]), "=f"(z[O + 4]), "=f"(z[O + 5]), "=f"(z[O + 6]), "=f"(z[O + 7]),
        "=f"(z[O + 8]), "=f"(z[O + 9]), "=f"(z[O + 10]), "=f"(z[O + 11]), "=f"(z[O + 12]), "=f"(z[O + 13]), "=f"(z[O + 14]), "=f"(z[O + 15]),
        "=f"(z[O + 16]), "=f"(z[O + 17]), "=f"(z[O + 18]), "=f"(z[O + 19]), "=f"(z[O + 20]), "=f"(z[O + 21]), "=f"(z[O + 22]), "=f"(z[O + 23]),
        "=f"(z[O + 24]), "=f"(z[O + 25]), "=f"(z[O + 26]), "=f"(z[O + 27]), "=f"(z[O + 28]), "=f"(z[O + 29]), "=f"(z[O + 30]), "=f"(z[O + 31]),
        "=f"(z[O + 32]), "=f"(z[O + 33]), "=f"(z[O + 34]), "=f"(z[O + 35]), "=f"(z[O + 36]), "=f"(z[O + 37]), "=f"(z[O + 38]), "=f"(z[O + 39]),
        "=f"(z[O + 40]), "=f"(z[O + 41]), "=f"(z[O + 42]), "=f"(z[O + 43]), "=f"(z[O + 44]), "=f"(z[O + 45]), "=f"(z[O + 46]), "=f"(z[O + 47]),
        "=f"(z[O + 48]), "=f"(z[O + 49]), "=f"(z[O + 50]), "=f"(z[O + 51]), "=f"(z[O + 52]), "=f"(z[O + 53]), "=f"(z[O + 54]), "=f"(z[O + 55]),
        "=f"(z[O + 56]), "=f"(z[O + 57]), "=f"(z[O + 58]), "=f"(z[O + 59]), "=f"(z[O + 60]), "=f"(z[O + 61]), "=f"(z[O + 62]), "=f"(z[O + 63]),
        "=f"(z[O + 64]), "=f"(z[O + 65]), "=f"(z[O + 66]), "=f"(z[O + 67]), "=f"(z[O + 68]), "=f"(z[O + 69]), "=f"(z[O + 70]), "=f"(z[O + 71]),
        "=f"(z[O + 72]), "=f"(z[O + 73]), "=f"(z[O + 74]), "=f"(z[O + 75]), "=f"(z[O + 76]), "=f"(z[O + 77]), "=f"(z[O + 78]), "=f"(z[O + 79]),
        "=f"(z[O + 80]), "=f"(z[O + 81]), "=f"(z[O + 82]), "=f"(z[O + 83]), "=f"(z[O + 84]), "=f"(z[O + 85]), "=f"(z[O + 86]), "=f"(z[O + 87]),
        "=f"(z[O + 88]), "=f"(z[O + 89]), "=f"(z[O + 90]), "=f"(z[O + 91]), "=f"(z[O + 92]), "=f"(z[O + 93]), "=f"(z[O + 94]), "=f"(z[O + 95]),
        "=f"(z[O + 96]), "=f"(z[O + 97]), "=f"(z[O + 98]), "=f"(z[O + 99]), "=f"(z[O + 100]), "=f"(z[O + 101]), "=f"(z[O + 102]), "=f"(z[O + 103]),
        "=f"(z[O + 104]), "=f"(z[O + 105]), "=f"(z[O + 106]), "=f"(z[O + 107]), "=f"(z[O + 108]), "=f"(z[O + 109]), "=f"(z[O + 110]), "=f"(z[O + 111]),
        "=f"(z[O + 112]), "=f"(z[O + 113]), "=f"(z[O + 114]), "=f"(z[O + 115]), "=f"(z[O + 116]), "=f"(z[O + 117]), "=f"(z[O + 118]), "=f"(z[O + 119]),
        "=f"(z[O + 120]), "=f"(z[O + 121]), "=f"(z[O + 122]), "=f"(z[O + 123]), "=f"(z[O + 124]), "=f"(z[O + 125]), "=f"(z[O + 126]), "=f"(z[O + 127])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A tile's one bias may join the reference instead of every logit while it does not swallow them.
__device__ __forceinline__ bool wt_apart(float c2, float flat) { return c2 > 0.f && fabsf(flat) < 65536.f; }
// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <int N> __device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t u;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
  return u;
}
// lo and hi plus the halves of a pair of bf16, in one mixed-precision instruction each
__device__ __forceinline__ void add_bf16(float& lo, float& hi, uint32_t pair) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\nadd.rn.f32.bf16 %0, a, %0;\nadd.rn.f32.bf16 %1, b, %1;\n}\n" : "+f"(lo), "+f"(hi) : "r"(pair));
}
__device__ __forceinline__ void bar_group(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// The tiles of 128 keys that a tile of queries visits: [0, nsink) and [first, last).
struct WtTiles {
  int nsink, first, last;
  __device__ __forceinline__ int count() const { return nsink + max(0, last - first); }
  __device__ __forceinline__ int at(int i) const { return i < nsink ? i : first + (i - nsink); }
};
__device__ __forceinline__ WtTiles wt_key_tiles(const WinParams& p, int l0, int queries, int keys) {
  WtTiles r{0, 0, 0};
  if (l0 >= queries) return r;
  int sinks, lo, hi;
  win_key_range(p, l0, min(l0 + kWtTile, queries), keys, &sinks, &lo, &hi);
  r.nsink = (sinks + kWtTile - 1) / kWtTile;
  if (lo < hi) { r.first = max(r.nsink, lo / kWtTile); r.last = (hi + kWtTile - 1) / kWtTile; }
  return r;
}
// the tiles of both
__device__ __forceinline__ WtTiles wt_union(const WtTiles& a, const WtTiles& b) {
  if (a.count() == 0) return b;
  if (b.count() == 0) return a;
  WtTiles r;
  r.nsink = max(a.nsink, b.nsink);
  const bool ea = a.first >= a.last, eb = b.first >= b.last;
  r.first = ea ? b.first : (eb ? a.first : min(a.first, b.first));
  r.last = ea ? b.last : (eb ? a.last : max(a.last, b.last));
  r.first = max(r.first, r.nsink);
  return r;
}
__device__ __forceinline__ int warp_uniform(int v) { return __reduce_max_sync(0xffffffffu, v); }   // the same in all lanes, and known to be
// A warp's wait that is mostly over before it begins: one look by all lanes, and lane 0 alone only where that was too early.
__device__ __forceinline__ bool wt_wait(uint64_t* bar, uint32_t parity, unsigned int* status, unsigned int code) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || mbar_wait_warp(bar, parity, status, code);
}
// Where a tile of 128 queries from l0 on stands to `N` keys from s0 on: some row sees some of them; every row sees all of them.
template <int N> struct WtView {
  int sinks, lo, hi, whole_sinks, whole_lo, whole_hi, whole_end;
  __device__ __forceinline__ WtView(const WinParams& p, int l0, int queries, int keys) {
    sinks = lo = hi = whole_sinks = whole_lo = 0;
    whole_hi = whole_end = -1;
    if (l0 >= queries) return;
    win_key_range(p, l0, min(l0 + kWtTile, queries), keys, &sinks, &lo, &hi);
    if (lo >= hi) lo = hi = 0;
    if (l0 + kWtTile > queries) return;
    whole_sinks = p.sinks - N;
    whole_lo = l0 + kWtTile - p.window;
    whole_end = min(keys, p.causal ? l0 + 1 : keys) - N;
    whole_hi = min(whole_end, l0 + p.window - N);
  }
  __device__ __forceinline__ bool some(int s0) const { return s0 < sinks || (s0 < hi && s0 + N > lo); }
  __device__ __forceinline__ bool whole(int s0) const { return s0 <= whole_end && (s0 <= whole_sinks || (s0 >= whole_lo && s0 <= whole_hi)); }
};
// The bias of N keys from s0 on for a tile of queries from l0 on: one value where all pairs lie in a side's last bucket.
struct WtFlat {
  float left, right;
  int last, left_bucket, right_bucket;    // where a side's last bucket starts; the table's columns
  template <typename T> __device__ __forceinline__ WtFlat(const WinParams& p, const T* table, int h) {
    left = right = 0.f; last = left_bucket = right_bucket = 0;
    if (p.buckets.count == 0) return;
    last = p.buckets.first[p.buckets.count - 1];
    left_bucket = p.buckets.count - 1;
    right_bucket = p.buckets.bidirectional ? 2 * p.buckets.count - 1 : win_bucket(p.buckets, 1);     // one-sided: distance 0 for all of them
    left = win_bias2(to_f32(table[h + (int64_t)p.H * left_bucket]));
    right = win_bias2(to_f32(table[h + (int64_t)p.H * right_bucket]));
  }
  // low, high: of key - query over the pairs
  __device__ __forceinline__ bool is_left(int high) const { return high <= 0 && -high >= last; }
  __device__ __forceinline__ bool is_right(const WinParams& p, int low) const { return low > 0 && (!p.buckets.bidirectional || low >= last); }
};
__device__ __forceinline__ uint32_t wt_below(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u); }
// Which keys of a tile a row of queries sees, 32 columns at a time: s = s0 + j with j < end and (j < sink or from <= j < past).
struct WtSeen {
  int from, past, sink, end;
  __device__ __forceinline__ WtSeen(const WinParams& p, int l, int queries, int s0, int keys) {
    from = l - p.window + 1 - s0;
    past = l + p.window - s0;
    sink = p.sinks - s0;
    end = l >= queries ? 0 : (p.causal ? min(l + 1, keys) : keys) - s0;
  }
  __device__ __forceinline__ uint32_t bits(int j) const {
    return wt_below(end - j) & (wt_below(sink - j) | (wt_below(past - j) & ~wt_below(from - j)));
  }
};
// every one of 128 queries from l0 on sees every one of `n` keys from s0 on
__device__ __forceinline__ bool wt_all_seen(const WinParams& p, int l0, int queries, int s0, int keys, int n = kWtTile) {
  if (l0 + kWtTile > queries || s0 + n > keys) return false;
  if (p.causal && s0 + n - 1 > l0) return false;
  const bool sinks = s0 + n <= p.sinks;
  return sinks || (l0 + kWtTile - 1 - s0 < p.window && s0 + n - 1 - l0 < p.window);
}
// 16 columns of a row as bf16, 32 bytes in one store where rows allow it
__device__ __forceinline__ void wt_store16(__nv_bfloat16* to, const uint32_t (&v)[8], int columns, bool wide) {
  if (wide && columns >= 16) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    if (columns >= 8) *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
    if (columns >= 16) *reinterpret_cast<uint4*>(to + 8) = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

}  // namespace lb2
