// Windowed attention on the tensor cores, pullback: BFloat16, up to 128 features.
//
// Two kernels form the weights anew from the stats of the forward pass, so that no result is summed by more than one block:
//   dq: a tile of 128 queries walks its tiles of keys;        S = Q K', dP = dX V', dS = p (dP - delta), dQ += dS K
//   dk, dv: a tile of 128 keys walks its tiles of queries;    S' = K Q', dP' = V dX', dV += p' dX, dK += dS' Q
// Rows are the block's own tokens, a thread holds half a row; p and dS go back to TMEM as bf16, over the columns of S and dP that
// the same threads have read, and are the A operand of the next product, whose B operand is the tile that is in shared memory
// already (tokens as the contraction). Two warpgroups share the exponentials of a tile.
//
// The weights of the logits' gradient are rounded to bf16 for dq and dk, as the weights are for dv: with the result's own rounding that leaves
// 0.0024 of the result, where a result rounded once has 0.0017. The table's gradient sums them in fp32, from weights rounded as the forward pass rounded
// them: over a row those add up to nothing, so that a bucket that holds nearly all of a row's weight gets minus the sum of the few others
// and not what rounding leaves (2 samples of 1100 tokens, window 246, four buckets: error 0.0087 -> 0.0028 of the gradient; all in one
// bucket: 40 times what dx . x rounds to -> a fifth of it). dq takes 8 % longer for it.
//
// Measured: 32 heads on 8, 128 features, 8192 tokens, window 1024, 4 sinks, bias: rows' constants 43 us (201 MB), dq 313 us, dk dv 331 us.
// What bounds them: in dq a tile's chain through the softmax warps (weights 1140 cycles, their gradients 650, the signals and waits between
// 700) and at 128 features the values, whose one place in shared memory is free only after the product before; in dk dv, whose four
// accumulators leave TMEM no second S, weights and products take turns, and the products and loads take 2300 cycles a tile of
// shared memory at 128 bytes per cycle.
//
// The bias table's gradient: sums of dS (fp32) by bucket. A tile of one bucket is summed in registers; in the others each warp adds
// along its diagonals with shuffles, then joins neighbouring diagonals of a bucket; per-warp sums, fixed order.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "window_tc.cuh"

namespace lb2 {

namespace {

// warp 0: TMA, warp 1: MMA, warps 4-11: softmax; registers 88 + 2 x 208 = 3 x 168 per thread at launch
constexpr int kWtBwdThreads = 384, kWtBwdFew = 88, kWtBwdMany = 208, kWtSoft = 256;
constexpr uint32_t kWtRowBytes = 3 * kWtTile * 4;

struct WtBwdParams {
  WinParams w;
  void *dq, *dk, *dv;
  const void* dx;
  const float2* stats;
  const float* delta;
  float* rows;                               // [batch][head][tile][-m2 | -log2 sum | -delta][128]
  float* partial;
  float* sink_sums;                          // [split][tile][batch][kv head][128][D + E], fp32
  int tiles, query_tiles, items, columns, boxes_d, boxes_e, wide_d, wide_kv;
  WinSinkPlan sinks;
  unsigned int* status;
};

template <int NB> struct WtBwd {
  static constexpr int TILE = NB * kWtBox;
  static constexpr int STAGES = NB == 1 ? 6 : 4;
  // dq: the ring's tiles of keys and how far their loads run ahead of the values'. Keys are held until the product that ends a tile,
  // values only for the one that begins it: 3 + 1 tiles of 128 features, one ahead, 361 us at window 4096 where 2 + 2 took 384 (before the product order below); 3 + 3 of
  // 64 features, in turn, 264 us, one ahead 301
  static constexpr int KS = 3, AHEAD = NB == 1 ? 0 : 1;
  // dq: bias and bucket of the diagonals (two tiles), diagonal sums of 8 warps, bucket sums of 8 warps; dk, dv: bias, columns' stats
  static constexpr int EXTRA = 2 * 256 * 4 + 2 * 256 + 8 * 4 * 48 * 4 + 8 * 2 * kWinMaxBuckets * 4 + 128 * 4 + kWinMaxBuckets * 4;
  static constexpr int SMEM = (2 + STAGES) * TILE + EXTRA + 256 + 1024;
};

// a tile of queries and the tiles of keys that it visits; the longest (last) tiles first
struct WtQueries {
  int l0, h, b, queries, keys;
  WtTiles own;
  __device__ __forceinline__ WtQueries(const WtBwdParams& p, int item) {
    const int rest = item / p.tiles;
    l0 = (p.tiles - 1 - item % p.tiles) * kWtTile;
    h = rest % p.w.H; b = rest / p.w.H;
    queries = warp_uniform(win_tokens(p.w, b, p.w.L)); keys = warp_uniform(win_tokens(p.w, b, p.w.S));
    own = wt_key_tiles(p.w, l0, queries, keys);
  }
};
// a tile of keys, or its part of the queries: tiles of queries first .. first + per_head of each head, n of them from `begin` on
struct WtKeys {
  WinKeyTile mine;
  int s0, g, b, queries, keys, first, per_head, begin, n;
  __device__ __forceinline__ WtKeys(const WtBwdParams& p, int item) : mine(item, p.tiles, p.w.Hkv * p.w.B, p.sinks) {
    const WinParams& w = p.w;
    g = mine.gb % w.Hkv; b = mine.gb / w.Hkv; s0 = mine.tile * kWtTile;
    queries = warp_uniform(win_tokens(w, b, w.L)); keys = warp_uniform(win_tokens(w, b, w.S));
    int lo, hi;
    win_query_range(w, s0, min(s0 + kWtTile, keys), queries, &lo, &hi);
    first = lo / kWtTile;
    per_head = s0 < keys && lo < hi ? (hi + kWtTile - 1) / kWtTile - first : 0;
    const int64_t all = (int64_t)per_head * w.rep;
    begin = (int)(all * mine.split / mine.splits);
    n = (int)(all * (mine.split + 1) / mine.splits) - begin;
  }
  __device__ __forceinline__ int head(const WinParams& w) const { return g * w.rep + (per_head > 0 ? begin / per_head : 0); }
  __device__ __forceinline__ int query_tile() const { return first + (per_head > 0 ? begin % per_head : 0); }
};
// 32 NB columns of a row from column c0 on, times f: whether all are finite. `in`: the row exists; `real`: it counts, else zeros
template <int NB>
__device__ __forceinline__ bool wt_store_row(__nv_bfloat16* to, const float (&v)[32 * NB], float f, int c0, int width, bool in, bool real, bool wide) {
  bool fine = true;
#pragma unroll
  for (int q = 0; q < 2 * NB; ++q) {
    uint32_t o[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const float a = v[q * 16 + 2 * x] * f, c = v[q * 16 + 2 * x + 1] * f;
      if (c0 + q * 16 + 2 * x < width) fine = fine && isfinite(a) && isfinite(c);
      o[x] = real ? pack_bf16(a, c) : 0u;
    }
    if (in) wt_store16(to + c0 + q * 16, o, width - c0 - q * 16, wide);
  }
  return fine;
}
// Adds 32 rows x 64 columns of d to the warp's sums by bucket. 16 columns at a time a lane hands the sum of its diagonal r - j on to the
// next lane's column; lane 31's is complete. Then neighbouring diagonals of one bucket join.
__device__ __forceinline__ void wt_diagonals(const float (&d)[64], float* my_diag, float* my_bsum, const uint8_t* bucket, int half, int quarter, int lane) {
  float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      a[c] += d[16 * c + j];
      if (j < 15) {
        if (lane == 31) my_diag[c * 48 + 46 - j] = a[c];                // diagonal d at d + 15
        const float up = __shfl_up_sync(0xffffffffu, a[c], 1);
        a[c] = lane == 0 ? 0.f : up;
      }
    }
#pragma unroll
  for (int c = 0; c < 4; ++c) my_diag[c * 48 + lane] = a[c];            // r - 15
  __syncwarp();
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    const int D = part * 32 + lane;                                     // r - j + 63 over the 64 columns, 95 of them
    float t = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int k = D - 63 + 16 * c + 15;
      if (k >= 0 && k < 47 && D < 95) t += my_diag[c * 48 + k];
    }
    // key - query, from the tile's lowest: j_tile - r_tile + 127
    const int bk = bucket[min(254, max(0, (63 - D) + half * 64 - quarter * 32 + 127))];
    const int mine = D < 95 ? bk : -1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float up = __shfl_up_sync(0xffffffffu, t, o);
      const int other = __shfl_up_sync(0xffffffffu, mine, o);
      if (lane >= o && other == mine) t += up;
    }
    const int following = __shfl_down_sync(0xffffffffu, mine, 1);
    if (mine >= 0 && (lane == 31 || following != mine)) my_bsum[mine] += t;
    __syncwarp();
  }
}
__device__ __forceinline__ float4 lds4(const float* p) { return *reinterpret_cast<const float4*>(p); }

template <int NB, bool BIASED>
__global__ void __launch_bounds__(kWtBwdThreads, 1)
win_tc_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ WtBwdParams p) {
  using C = WtBwd<NB>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  float* lut = reinterpret_cast<float*>(gen + (2 + C::STAGES) * C::TILE);          // [parity][256]
  float* diag = lut + 2 * 256;                                                     // [warp][4][48]
  float* bsum = diag + 8 * 4 * 48;                                                 // [warp][buckets]
  int* bad = reinterpret_cast<int*>(bsum + 8 * 2 * kWinMaxBuckets);
  uint8_t* of = reinterpret_cast<uint8_t*>(bad + 128);                             // [parity][256]
  int32_t* first_of = reinterpret_cast<int32_t*>(of + 2 * 256);                    // where the buckets start
  uint64_t* bars = reinterpret_cast<uint64_t*>(first_of + kWinMaxBuckets);
  uint64_t *q_full = bars, *q_empty = bars + 1, *full = bars + 2, *empty = full + C::STAGES, *s_full = empty + C::STAGES, *dp_full = s_full + 2,
           *ds_ready = dp_full + 1, *o_full = ds_ready + 1, *o_empty = o_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_empty + 1);
  const uint32_t sQ = base, sG = base + C::TILE, sKV = base + 2 * C::TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WinParams& w = p.w;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmG); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
    mbar_init(q_full, 1); mbar_init(q_empty, 1);
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(&s_full[0], 1); mbar_init(&s_full[1], 1); mbar_init(dp_full, 1); mbar_init(ds_ready, 8); mbar_init(o_full, 1); mbar_init(o_empty, 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x >= 64 && threadIdx.x < 64 + kWinMaxBuckets) first_of[threadIdx.x - 64] = w.buckets.first[threadIdx.x - 64];
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) *bad = 0;
  for (int i = threadIdx.x; i < 8 * 2 * kWinMaxBuckets; i += kWtBwdThreads) bsum[i] = 0.f;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tDP = tmem + 256, tDQ = tmem + 384;            // S of even and odd tiles at 0 and 128

  if (warp < 4) {
    regs_less<kWtBwdFew>();
    if (warp == 0) {
      uint32_t kst = 0, vst = 0, ph_k = 0, ph_v = 0, turn = 0;
      bool ok = true;
      for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
        const WtQueries t(p, item);
        const int n = t.own.count();
        if (n == 0) continue;
        if (!mbar_wait_uniform(q_empty, (turn & 1u) ^ 1u, p.status, 0x80u)) break;
        ++turn;
        if (elect_one()) {
          mbar_expect_tx(q_full, (uint32_t)((p.boxes_d + p.boxes_e) * kWtBox));
          for (int x = 0; x < p.boxes_d; ++x) tma_load_4d(sQ + x * kWtBox, &tmQ, x * 64, t.h, t.l0, t.b, q_full);
          for (int x = 0; x < p.boxes_e; ++x) tma_load_4d(sG + x * kWtBox, &tmG, x * 64, t.h, t.l0, t.b, q_full);
        }
        __syncwarp();
        for (int i = 0; i < n + C::AHEAD && ok; ++i) {
          for (int which = 0; which < 2; ++which) {
            const bool is_k = which == 0;
            const int tile = is_k ? i : i - C::AHEAD;
            if (tile < 0 || tile >= n) continue;
            const uint32_t slot = is_k ? kst : C::KS + vst;
            if (!mbar_wait_uniform(&empty[slot], (is_k ? ph_k : ph_v) ^ 1u, p.status, 0x100u)) { ok = false; break; }
            if (elect_one()) {
              const int boxes = is_k ? p.boxes_d : p.boxes_e, s0 = t.own.at(tile) * kWtTile;
              mbar_expect_tx(&full[slot], (uint32_t)(boxes * kWtBox));
              for (int x = 0; x < boxes; ++x) tma_load_4d(sKV + slot * C::TILE + x * kWtBox, is_k ? &tmK : &tmV, x * 64, t.h / w.rep, s0, t.b, &full[slot]);
            }
            __syncwarp();
            if (is_k) { if (++kst == C::KS) { kst = 0; ph_k ^= 1u; } }
            else if (++vst == C::STAGES - C::KS) { vst = 0; ph_v ^= 1u; }
          }
        }
      }
    } else if (warp == 1) {
      uint32_t turn = 0, kst = 0, vst = 0, ph_k = 0, ph_v = 0, done = 0;   // items; the ring's next tiles; tiles so far
      bool ok = true;
      for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
        const WtQueries t(p, item);
        const int n = t.own.count();
        if (n == 0) continue;
        if (!mbar_wait_uniform(q_full, turn & 1u, p.status, 0x200u)) break;
        uint32_t kprev = 0;                                                // where tile i's keys are
        for (int i = -1; i < n; ++i) {
          const bool next = i + 1 < n;
          const uint32_t cur = (done + (uint32_t)i) & 1u, nxt = cur ^ 1u, k = sKV + kst * C::TILE, v = sKV + (C::KS + vst) * C::TILE;
          if (next) {
            if (!mbar_wait_uniform(&full[kst], ph_k, p.status, 0x400u)) { ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
              if (NB == 2 && p.boxes_d == 2) wt_mma_features<NB>(tmem + nxt * 128, sQ, k);
              else wt_mma_features<1>(tmem + nxt * 128, sQ, k);
              umma_commit(&s_full[nxt]);
            }
            __syncwarp();
          }
          if (i >= 0) {
            if (!mbar_wait_uniform(ds_ready, cur, p.status, 0x800u)) { ok = false; break; }
            if (i == 0 && !mbar_wait_uniform(o_empty, (turn & 1u) ^ 1u, p.status, 0x40u)) { ok = false; break; }
            tc_fence_after();
          }
          // 128 features wait for their one tile of values here: the product with the finished tile first (361 -> 303 us at window 4096; 297 as the kernel is now)
          const auto product_dq = [&] {
            if (i < 0) return;
            if (elect_one()) {
              const uint32_t kc = sKV + kprev * C::TILE;
              if (NB == 2 && p.boxes_d == 2) wt_mma_tokens_halves<NB>(tDQ, tmem + cur * 128, kc, i > 0);
              else wt_mma_tokens_halves<1>(tDQ, tmem + cur * 128, kc, i > 0);
              umma_commit(&empty[kprev]);
              if (!next) umma_commit(o_full);
            }
            __syncwarp();
          };
          if (NB == 2) product_dq();
          if (next) {
            if (!mbar_wait_uniform(&full[C::KS + vst], ph_v, p.status, 0x400u)) { ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
              if (NB == 2 && p.boxes_e == 2) wt_mma_features<NB>(tDP, sG, v);
              else wt_mma_features<1>(tDP, sG, v);
              umma_commit(dp_full);
              umma_commit(&empty[C::KS + vst]);
              if (i + 2 == n) umma_commit(q_empty);
            }
            __syncwarp();
          }
          if (NB == 1) product_dq();
          kprev = kst;
          if (next) {
            if (++kst == C::KS) { kst = 0; ph_k ^= 1u; }
            if (++vst == C::STAGES - C::KS) { vst = 0; ph_v ^= 1u; }
          }
        }
        ++turn;
        done += (uint32_t)n;
      }
    }
  } else {
    regs_more<kWtBwdMany>();
    const int sw = warp - 4, half = sw >> 2, quarter = warp & 3, row = quarter * 32 + lane, st = threadIdx.x - 128;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const float c2 = w.scale2;
    float* my_bsum = bsum + sw * 2 * kWinMaxBuckets;
    float* my_diag = diag + sw * 4 * 48;
    bool ok = true;                     // after a wait that ran out: no more waits, but the same way through, whose barriers all warps share
    uint32_t done = 0, turn = 0;        // tiles and items so far
    int table = 0;                      // of the tiles with more than one bucket: each has a barrier, two tables are enough
    for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
      const WtQueries t(p, item);
      const int l0 = t.l0, l = l0 + row, n = t.own.count(), h = t.h;
      const WtView<kWtTile> view(w, l0, t.queries, t.keys);
      const WtFlat tail(w, static_cast<const __nv_bfloat16*>(w.table), h);
      const float* of_row = p.rows + (((int64_t)t.b * w.H + h) * p.query_tiles + l0 / kWtTile) * 3 * kWtTile + row;
      const float neg_m = of_row[0], neg_l = of_row[kWtTile], neg_d = of_row[2 * kWtTile];
      // ds = p / sum (dp - delta); a row that sees one key alone: dp times nothing, which is nothing unless dp is not finite
      const bool single = win_single(w, l, t.keys);
      const float inv = single ? 0.f : ex2(neg_l), off_d = single ? 0.f : neg_d * inv;
      const uint64_t nm = pack2(neg_m, neg_m), inv2 = pack2(inv, inv), off_d2 = pack2(off_d, off_d);
      float left_sum = 0.f, right_sum = 0.f;
      for (int i = 0; i < n; ++i) {
        const int s0 = t.own.at(i) * kWtTile, low = s0 - l0 - (kWtTile - 1);
        const uint32_t cur = (done + (uint32_t)i) & 1u;
        float flat = 0.f;
        const float* bias = nullptr;
        const uint8_t* bucket = nullptr;
        const bool whole = view.whole(s0), in_left = BIASED && tail.is_left(low + 2 * (kWtTile - 1));
        if constexpr (BIASED) {
          if (in_left) {
            flat = tail.left;
          } else if (tail.is_right(w, low)) {
            flat = tail.right;
          } else {
            float* to = lut + table * 256;
            if (st < 255) {
              const int bk = win_bucket(w.buckets, first_of, low + st);
              to[st] = win_bias2(to_f32(static_cast<const __nv_bfloat16*>(w.table)[h + (int64_t)w.H * bk]));
              of[table * 256 + st] = (uint8_t)bk;
            }
            bar_group(1, kWtSoft);
            bias = to + (kWtTile - 1 - row) + half * 64;
            bucket = of + table * 256;
            table ^= 1;
          }
        }
        ok = ok && wt_wait(&s_full[cur], ((done + (uint32_t)i) >> 1) & 1u, p.status, 0x1000u);
        tc_fence_after();
        const uint32_t tS = tmem + lanes + cur * 128 + half * 64;
        float d[64];
        tmem_row64<0>(tS, d);
        const uint64_t mul2_ = pack2(c2, c2);
        if (bias == nullptr && wt_apart(c2, flat)) {
          const float off = flat + neg_m;
          const uint64_t off2_ = pack2(off, off);
#pragma unroll
          for (int j = 0; j < 64; j += 2) {
            float e0, e1;
            unpack2(fma2(pack2(d[j], d[j + 1]), mul2_, off2_), e0, e1);
            d[j] = ex2(e0); d[j + 1] = ex2(e1);
          }
        } else {
          const uint64_t flat2_ = pack2(flat, flat);
#pragma unroll
          for (int j = 0; j < 64; j += 2) {
            const uint64_t add = bias != nullptr ? pack2(bias[j], bias[j + 1]) : flat2_;
            float e0, e1;
            unpack2(add2(fma2(pack2(d[j], d[j + 1]), mul2_, add), nm), e0, e1);
            d[j] = ex2(e0); d[j + 1] = ex2(e1);
          }
        }
        ok = ok && wt_wait(dp_full, cur, p.status, 0x2000u);
        tc_fence_after();
        float e[64];
        tmem_row64<0>(tDP + lanes + half * 64, e);
        uint32_t bits[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
        if (!whole) {
          const WtSeen seen(w, l, t.queries, s0, t.keys);
          bits[0] = seen.bits(half * 64);
          bits[1] = seen.bits(half * 64 + 32);
        }
        {
          uint32_t v[32];
          const auto gradients = [&](auto masked) {                       // e: what the weights are multiplied with
#pragma unroll
            for (int j = 0; j < 64; j += 2) {
              const uint64_t f = fma2(pack2(e[j], e[j + 1]), inv2, off_d2);
              float y0, y1;
              unpack2(mul2(f, pack2(d[j], d[j + 1])), y0, y1);
              unpack2(f, e[j], e[j + 1]);
              if constexpr (decltype(masked)::value) {
                y0 = bits[j >> 5] >> (j & 31) & 1u ? y0 : 0.f;
                y1 = bits[j >> 5] >> ((j + 1) & 31) & 1u ? y1 : 0.f;
              }
              v[j >> 1] = pack_bf16(y0, y1);
            }
          };
          if (whole) gradients(std::false_type{});
          else gradients(std::true_type{});
          tmem_st32(tS, v);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
        if constexpr (BIASED) {                    // the table's share, of the weights that the forward pass used
#pragma unroll
          for (int j = 0; j < 64; j += 2) {
            const uint32_t both = pack_bf16(d[j], d[j + 1]);
            unpack2(mul2(pack2(e[j], e[j + 1]), pack2(__uint_as_float(both << 16), __uint_as_float(both & 0xFFFF0000u))), d[j], d[j + 1]);
          }
          if (!whole) {
#pragma unroll
            for (int j = 0; j < 64; ++j) d[j] = bits[j >> 5] >> (j & 31) & 1u ? d[j] : 0.f;
          }
          if (bucket == nullptr) {
            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 64; ++j) part[j & 3] += d[j];
            (in_left ? left_sum : right_sum) += (part[0] + part[1]) + (part[2] + part[3]);
          } else {
            wt_diagonals(d, my_diag, my_bsum, bucket, half, quarter, lane);
          }
        }
      }
      done += (uint32_t)n;
      if constexpr (BIASED) {
        const float a = warp_sum(left_sum), c = warp_sum(right_sum);
        if (lane == 0) {
          my_bsum[tail.left_bucket] += a;
          my_bsum[tail.right_bucket] += c;
        }
        bar_group(1, kWtSoft);
        if (st < p.columns) {
          float sum = 0.f;
          for (int x = 0; x < 8; ++x) {
            sum += bsum[x * 2 * kWinMaxBuckets + st];
            bsum[x * 2 * kWinMaxBuckets + st] = 0.f;
          }
          p.partial[((int64_t)(l0 / kWtTile) * w.B * w.H + (int64_t)t.b * w.H + h) * p.columns + st] = sum;
        }
        bar_group(1, kWtSoft);
      }
      float o[32 * NB];
      if (n > 0) {
        ok = ok && wt_wait(o_full, turn & 1u, p.status, 0x4000u);
        ++turn;
        tc_fence_after();
        if constexpr (NB == 2) tmem_row64<0>(tDQ + lanes + half * 64, o);
        else tmem_row32<0>(tDQ + lanes + half * 32, o);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_empty);
      } else {
#pragma unroll
        for (int j = 0; j < 32 * NB; ++j) o[j] = 0.f;
      }
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.dq) + (((int64_t)t.b * w.L + l) * w.H + h) * w.D;
      const bool fine = wt_store_row<NB>(out, o, w.scale, half * NB * 32, w.D, l < w.L, l < t.queries, p.wide_d != 0);
      if (l < t.queries && !fine) *bad = 1;
    }
    // rows that an infinity or NaN reached, once the pipeline no longer waits for these warps
    bar_group(1, kWtSoft);
    if (*bad != 0 && ok) {
      for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
        const WtQueries t(p, item);
        for (int r = sw; r < kWtTile && t.l0 + r < t.queries; r += 8) {
          const int64_t at = ((int64_t)t.b * w.H + t.h) * w.L + t.l0 + r;
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.dq) + (((int64_t)t.b * w.L + t.l0 + r) * w.H + t.h) * w.D;
          bool fine = true;
          for (int e = lane; e < w.D; e += 32) fine = fine && isfinite(__bfloat162float(out[e]));
          if (!__all_sync(0xffffffffu, fine))
            win_row_dq<__nv_bfloat16>(w, static_cast<__nv_bfloat16*>(p.dq), p.dx, p.stats[at], p.delta[at], t.l0 + r, t.h, t.b, t.keys);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (*reinterpret_cast<volatile unsigned int*>(p.status) != 0) drain_after_abort();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int NB>
__global__ void __launch_bounds__(kWtBwdThreads, 1)
win_tc_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ WtBwdParams p) {
  using C = WtBwd<NB>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  float* lut = reinterpret_cast<float*>(gen + (2 + C::STAGES) * C::TILE);          // [parity][256]
  float* cols = lut + 2 * 256;                                                     // per query tile of the ring: -m2 | -log2 sum | -delta
  int* bad = reinterpret_cast<int*>(cols + C::STAGES / 2 * 3 * 128);
  int32_t* first_of = reinterpret_cast<int32_t*>(bad + 128);                       // where the buckets start
  uint64_t* bars = reinterpret_cast<uint64_t*>(first_of + kWinMaxBuckets);
  uint64_t *k_full = bars, *k_empty = bars + 1, *full = bars + 2, *empty = full + C::STAGES, *s_full = empty + C::STAGES, *dp_full = s_full + 1,
           *p_ready = dp_full + 1, *ds_ready = p_ready + 1, *o_full = ds_ready + 1, *o_empty = o_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_empty + 1);
  const uint32_t sK = base, sV = base + C::TILE, sQG = base + 2 * C::TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WinParams& w = p.w;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmG); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
    mbar_init(k_full, 1); mbar_init(k_empty, 1);
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(s_full, 1); mbar_init(dp_full, 1); mbar_init(p_ready, 8); mbar_init(ds_ready, 8); mbar_init(o_full, 1); mbar_init(o_empty, 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x >= 64 && threadIdx.x < 64 + kWinMaxBuckets) first_of[threadIdx.x - 64] = w.buckets.first[threadIdx.x - 64];
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) *bad = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tDP = tmem + 128, tDV = tmem + 256, tDK = tmem + 384;

  if (warp < 4) {
    regs_less<kWtBwdFew>();
    if (warp == 0) {
      uint32_t stage = 0, phase = 0, turn = 0;
      bool ok = true;
      for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
        const WtKeys t(p, item);
        if (t.n == 0) continue;
        if (!mbar_wait_uniform(k_empty, (turn & 1u) ^ 1u, p.status, 0x80u)) break;
        ++turn;
        if (elect_one()) {
          mbar_expect_tx(k_full, (uint32_t)((p.boxes_d + p.boxes_e) * kWtBox));
          for (int x = 0; x < p.boxes_d; ++x) tma_load_4d(sK + x * kWtBox, &tmK, x * 64, t.g, t.s0, t.b, k_full);
          for (int x = 0; x < p.boxes_e; ++x) tma_load_4d(sV + x * kWtBox, &tmV, x * 64, t.g, t.s0, t.b, k_full);
        }
        __syncwarp();
        int h = t.head(w), qt = t.query_tile();
        for (int i = 0; i < 2 * t.n; ++i) {
          if (!mbar_wait_uniform(&empty[stage], phase ^ 1u, p.status, 0x100u)) { ok = false; break; }
          if (elect_one()) {
            const bool is_q = (i & 1) == 0;
            const int boxes = is_q ? p.boxes_d : p.boxes_e;
            mbar_expect_tx(&full[stage], (uint32_t)(boxes * kWtBox + (is_q ? kWtRowBytes : 0)));
            for (int x = 0; x < boxes; ++x) tma_load_4d(sQG + stage * C::TILE + x * kWtBox, is_q ? &tmQ : &tmG, x * 64, h, qt * kWtTile, t.b, &full[stage]);
            if (is_q)
              bulk_load_1d(smem_u32(cols) + (stage >> 1) * kWtRowBytes, p.rows + (((int64_t)t.b * w.H + h) * p.query_tiles + qt) * 3 * kWtTile, kWtRowBytes,
                           &full[stage]);
          }
          __syncwarp();
          if ((i & 1) == 1 && ++qt == t.first + t.per_head) { qt = t.first; ++h; }
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    } else if (warp == 1) {
      uint32_t turn = 0, done = 0, qst = 0, gst = 0, ph_q = 0, ph_g = 0;   // items, tiles of queries so far; the ring's next tiles
      bool ok = true;
      for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
        const WtKeys t(p, item);
        const int n = t.n;
        if (n == 0) continue;
        if (!mbar_wait_uniform(k_full, turn & 1u, p.status, 0x200u)) break;
        uint32_t qprev = 0, gprev = 0;
        for (int i = -1; i < n; ++i) {
          const bool next = i + 1 < n;
          const uint32_t par = (done + (uint32_t)i) & 1u;
          const uint32_t qn = sQG + 2 * qst * C::TILE, gn = sQG + (2 * gst + 1) * C::TILE, qc = sQG + 2 * qprev * C::TILE, gc = sQG + (2 * gprev + 1) * C::TILE;
          if (i >= 0 && !mbar_wait_uniform(p_ready, par, p.status, 0x800u)) { ok = false; break; }
          if (i == 0 && !mbar_wait_uniform(o_empty, (turn & 1u) ^ 1u, p.status, 0x40u)) { ok = false; break; }
          tc_fence_after();
          if (i >= 0 && elect_one()) {
            if (NB == 2 && p.boxes_e == 2) wt_mma_tokens_halves<NB>(tDV, tmem, gc, i > 0);
            else wt_mma_tokens_halves<1>(tDV, tmem, gc, i > 0);
            umma_commit(&empty[2 * gprev + 1]);
          }
          __syncwarp();
          if (next && !mbar_wait_uniform(&full[2 * qst], ph_q, p.status, 0x400u)) { ok = false; break; }
          tc_fence_after();
          if (next && elect_one()) {
            if (NB == 2 && p.boxes_d == 2) wt_mma_features<NB>(tmem, sK, qn);
            else wt_mma_features<1>(tmem, sK, qn);
            umma_commit(s_full);
          }
          __syncwarp();
          if (i >= 0 && !mbar_wait_uniform(ds_ready, par, p.status, 0x8000u)) { ok = false; break; }
          tc_fence_after();
          if (i >= 0 && elect_one()) {
            if (NB == 2 && p.boxes_d == 2) wt_mma_tokens_halves<NB>(tDK, tDP, qc, i > 0);
            else wt_mma_tokens_halves<1>(tDK, tDP, qc, i > 0);
            umma_commit(&empty[2 * qprev]);
            if (!next) umma_commit(o_full);
          }
          __syncwarp();
          if (next && !mbar_wait_uniform(&full[2 * gst + 1], ph_g, p.status, 0x400u)) { ok = false; break; }
          tc_fence_after();
          if (next && elect_one()) {
            if (NB == 2 && p.boxes_e == 2) wt_mma_features<NB>(tDP, sV, gn);
            else wt_mma_features<1>(tDP, sV, gn);
            umma_commit(dp_full);
            if (i + 2 == n) umma_commit(k_empty);
          }
          __syncwarp();
          qprev = qst; gprev = gst;
          if (next) {
            if (++qst == C::STAGES / 2) { qst = 0; ph_q ^= 1u; }
            if (++gst == C::STAGES / 2) { gst = 0; ph_g ^= 1u; }
          }
        }
        ++turn;
        done += (uint32_t)n;
      }
    }
  } else {
    regs_more<kWtBwdMany>();
    const int sw = warp - 4, half = sw >> 2, quarter = warp & 3, row = quarter * 32 + lane, st = threadIdx.x - 128;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, tS = tmem + lanes + half * 64, tD = tDP + lanes + half * 64;
    const float c2 = w.scale2;
    const bool biased = w.buckets.count > 0;
    bool ok = true;                     // after a wait that ran out: no more waits, but the same way through, whose barriers all warps share
    int table = 0;
    uint32_t qst = 0, ph_q = 0, done = 0, turn = 0;
    for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
      const WtKeys t(p, item);
      const int n = t.n, s0 = t.s0, s = s0 + row, b = t.b, g = t.g, queries = t.queries, keys = t.keys;
      int h = t.head(w), qt = t.query_tile();
      WtFlat tail(w, static_cast<const __nv_bfloat16*>(w.table), h);
      for (int i = 0; i < n; ++i) {
        const int l0 = qt * kWtTile;
        const uint32_t par = (done + (uint32_t)i) & 1u;
        const float* col = cols + qst * 3 * kWtTile;
        float flat = 0.f;
        const float* bias = nullptr;
        if (biased) {
          const int low = s0 - l0 - (kWtTile - 1);
          if (tail.is_left(low + 2 * (kWtTile - 1))) {
            flat = tail.left;
          } else if (tail.is_right(w, low)) {
            flat = tail.right;
          } else {                                   // index (column - row) + 127: rel = low + 254 - index
            float* to = lut + table * 256;
            table ^= 1;                              // each use has a barrier: two tables are enough
            if (st < 255) to[st] = win_bias<__nv_bfloat16>(w, first_of, h, low + 254 - st);
            bar_group(1, kWtSoft);
            bias = to + (kWtTile - 1 - row) + half * 64;
          }
        }
        // the queries that see key s: columns from..to
        int from = w.causal ? s - l0 : (s < w.sinks ? 0 : s - w.window + 1 - l0);
        int to = (s < w.sinks ? queries - 1 : min(queries - 1, s + w.window - 1)) - l0;
        if (s >= keys) to = -1;
        const bool whole = wt_all_seen(w, l0, queries, s0, keys, kWtTile);
        ok = ok && wt_wait(&full[2 * qst], ph_q, p.status, 0x8u);       // the columns' stats
        ok = ok && wt_wait(s_full, par, p.status, 0x1000u);
        tc_fence_after();
        float d[64];
        const bool apart = bias == nullptr && wt_apart(c2, flat);
        const uint64_t mul2_ = pack2(c2, c2), flat2_ = pack2(flat, flat);
        tmem_row64<0>(tS, d);
        if (apart) {
#pragma unroll
          for (int j = 0; j < 64; j += 4) {
            const float4 m = lds4(col + half * 64 + j), e = lds4(col + 128 + half * 64 + j);
            float y[4];
            unpack2(add2(fma2(pack2(d[j], d[j + 1]), mul2_, add2(flat2_, pack2(m.x, m.y))), pack2(e.x, e.y)), y[0], y[1]);
            unpack2(add2(fma2(pack2(d[j + 2], d[j + 3]), mul2_, add2(flat2_, pack2(m.z, m.w))), pack2(e.z, e.w)), y[2], y[3]);
#pragma unroll
            for (int k = 0; k < 4; ++k) d[j + k] = ex2(y[k]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 64; j += 4) {
            const float4 m = lds4(col + half * 64 + j), e = lds4(col + 128 + half * 64 + j);
            const uint64_t add0 = bias != nullptr ? pack2(bias[j], bias[j + 1]) : flat2_, add1 = bias != nullptr ? pack2(bias[j + 2], bias[j + 3]) : flat2_;
            float y[4];
            unpack2(add2(add2(fma2(pack2(d[j], d[j + 1]), mul2_, add0), pack2(m.x, m.y)), pack2(e.x, e.y)), y[0], y[1]);
            unpack2(add2(add2(fma2(pack2(d[j + 2], d[j + 3]), mul2_, add1), pack2(m.z, m.w)), pack2(e.z, e.w)), y[2], y[3]);
#pragma unroll
            for (int k = 0; k < 4; ++k) d[j + k] = ex2(y[k]);
          }
        }
        if (!whole) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const uint32_t bits = wt_below(to + 1 - half * 64 - q * 32) & ~wt_below(from - half * 64 - q * 32);
#pragma unroll
            for (int j = 0; j < 32; ++j) d[q * 32 + j] = bits >> j & 1u ? d[q * 32 + j] : 0.f;
          }
        }
        {
          uint32_t v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = pack_bf16(d[2 * j], d[2 * j + 1]);
          tmem_st32(tS, v);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
        ok = ok && wt_wait(dp_full, par, p.status, 0x2000u);
        tc_fence_after();
        uint32_t o[32];
        {
          float e[64];
          tmem_row64<0>(tD, e);
          if (!whole) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const uint32_t single = __ballot_sync(0xffffffffu, win_single(w, l0 + half * 64 + q * 32 + lane, keys));
              if (single != 0) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  e[q * 32 + j] = single >> j & 1u ? (e[q * 32 + j] - e[q * 32 + j]) - col[256 + half * 64 + q * 32 + j] : e[q * 32 + j];
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 64; j += 4) {
            const float4 nd = lds4(col + 256 + half * 64 + j);
            unpack2(mul2(add2(pack2(e[j], e[j + 1]), pack2(nd.x, nd.y)), pack2(d[j], d[j + 1])), d[j], d[j + 1]);
            unpack2(mul2(add2(pack2(e[j + 2], e[j + 3]), pack2(nd.z, nd.w)), pack2(d[j + 2], d[j + 3])), d[j + 2], d[j + 3]);
          }
        }
        if (!whole) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const uint32_t bits = wt_below(to + 1 - half * 64 - q * 32) & ~wt_below(from - half * 64 - q * 32);
#pragma unroll
            for (int j = 0; j < 32; ++j) d[q * 32 + j] = bits >> j & 1u ? d[q * 32 + j] : 0.f;
          }
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = pack_bf16(d[2 * j], d[2 * j + 1]);
        tmem_st32(tD, o);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
        if (++qst == C::STAGES / 2) { qst = 0; ph_q ^= 1u; }
        if (++qt == t.first + t.per_head) {
          qt = t.first; ++h;
          if (biased && i + 1 < n) tail = WtFlat(w, static_cast<const __nv_bfloat16*>(w.table), h);
        }
      }
      done += (uint32_t)n;
      float ak[32 * NB], av[32 * NB];
      if (n > 0) {
        ok = ok && wt_wait(o_full, turn & 1u, p.status, 0x4000u);
        ++turn;
        tc_fence_after();
        if constexpr (NB == 2) {
          tmem_row64<0>(tDK + lanes + half * 64, ak);
          tmem_row64<0>(tDV + lanes + half * 64, av);
        } else {
          tmem_row32<0>(tDK + lanes + half * 32, ak);
          tmem_row32<0>(tDV + lanes + half * 32, av);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_empty);
      } else {
#pragma unroll
        for (int x = 0; x < 32 * NB; ++x) ak[x] = av[x] = 0.f;
      }
      const int c0 = half * NB * 32;
      if (t.mine.splits > 1) {
        float* out = p.sink_sums + ((((int64_t)t.mine.split * p.sinks.tiles + t.mine.tile) * (w.Hkv * w.B) + t.mine.gb) * kWtTile + row) * (w.D + w.E);
#pragma unroll
        for (int x = 0; x < 32 * NB; x += 4) {
          if (c0 + x < w.D) *reinterpret_cast<float4*>(out + c0 + x) = make_float4(ak[x] * w.scale, ak[x + 1] * w.scale, ak[x + 2] * w.scale, ak[x + 3] * w.scale);
          if (c0 + x < w.E) *reinterpret_cast<float4*>(out + w.D + c0 + x) = make_float4(av[x], av[x + 1], av[x + 2], av[x + 3]);
        }
      } else {
        bool fine = wt_store_row<NB>(static_cast<__nv_bfloat16*>(p.dk) + (((int64_t)b * w.S + s) * w.Hkv + g) * w.D, ak, w.scale, c0, w.D, s < w.S, s < keys,
                                     p.wide_kv != 0);
        fine = wt_store_row<NB>(static_cast<__nv_bfloat16*>(p.dv) + (((int64_t)b * w.S + s) * w.Hkv + g) * w.E, av, 1.f, c0, w.E, s < w.S, s < keys,
                                p.wide_kv != 0) && fine;
        if (s < keys && !fine) *bad = 1;
      }
    }
    // rows that an infinity or NaN reached, once the pipeline no longer waits for these warps
    bar_group(1, kWtSoft);
    if (*bad != 0) {
      for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
        const WtKeys t(p, item);
        if (t.mine.splits > 1) continue;
        for (int r = sw; r < kWtTile && t.s0 + r < t.keys; r += 8) {
          const int64_t at = ((int64_t)t.b * w.S + t.s0 + r) * w.Hkv + t.g;
          bool fine = true;
          for (int e = lane; e < w.D; e += 32) fine = fine && isfinite(__bfloat162float(static_cast<const __nv_bfloat16*>(p.dk)[at * w.D + e]));
          for (int e = lane; e < w.E; e += 32) fine = fine && isfinite(__bfloat162float(static_cast<const __nv_bfloat16*>(p.dv)[at * w.E + e]));
          if (!__all_sync(0xffffffffu, fine))
            win_row_dkv<__nv_bfloat16>(w, static_cast<__nv_bfloat16*>(p.dk), static_cast<__nv_bfloat16*>(p.dv), p.dx, p.stats, p.delta, t.s0 + r, t.g, t.b,
                                       t.queries, t.keys);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (*reinterpret_cast<volatile unsigned int*>(p.status) != 0) drain_after_abort();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// delta[batch][head][query] = dx . x and the rows' constants, LR lanes of a row taking eight features each
template <int LR>
__global__ void __launch_bounds__(256) win_tc_rows_kernel(const __grid_constant__ WtBwdParams p, float* __restrict__ delta, const __nv_bfloat16* __restrict__ x,
                                                          const __nv_bfloat16* __restrict__ rest) {
  const WinParams& w = p.w;
  const int lane = threadIdx.x % LR, padded = p.query_tiles * kWtTile;
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LR;         // (batch, query up to whole tiles, head)
  const int h = (int)(row % w.H);
  const int64_t bl = row / w.H;
  const int b = (int)(bl / padded), l = (int)(bl - (int64_t)b * padded);
  const bool in = b < w.B && l < w.L;
  float s = 0.f;
  if (in && lane * 8 < w.E) {
    const int64_t at = (((int64_t)b * w.L + l) * w.H + h) * w.E + lane * 8;
    const Vec16<__nv_bfloat16> u = load16(static_cast<const __nv_bfloat16*>(p.dx) + at), v = load16(x + at);
    Vec16<__nv_bfloat16> r;
    r.raw = make_uint4(0, 0, 0, 0);
    if (rest != nullptr) r = load16(rest + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(u.get(i), v.get(i) + r.get(i), s);
  }
#pragma unroll
  for (int o = LR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane != 0 || b >= w.B) return;
  const int64_t hb = (int64_t)b * w.H + h;
  const bool counts = l < win_tokens(w, b, w.L);
  const float2 stat = counts ? p.stats[hb * w.L + l] : make_float2(0.f, INFINITY);
  float* to = p.rows + (hb * p.query_tiles + l / kWtTile) * 3 * kWtTile + l % kWtTile;
  to[0] = -stat.x; to[kWtTile] = -stat.y; to[2 * kWtTile] = counts ? -s : 0.f;
  if (in) delta[hb * w.L + l] = s;
}

}  // namespace

size_t win_tc_row_bytes(const lb2_window_dims* d) {
  return (size_t)((d->queries + kWtTile - 1) / kWtTile * d->heads * d->batch) * kWtRowBytes;
}

int64_t win_tc_partials(const lb2_window_dims* d) { return (d->queries + kWtTile - 1) / kWtTile; }

int32_t win_tc_bwd(const WinParams& w, void* dq, void* dk, void* dv, float* partial, float* sink_sums, float* rows, const void* dx, const void* x,
                   const void* rest, const float2* stats, float* delta, cudaStream_t st) {
  WtBwdParams p{};
  p.w = w; p.dq = dq; p.dk = dk; p.dv = dv; p.dx = dx; p.stats = stats; p.delta = delta; p.partial = partial; p.sink_sums = sink_sums; p.rows = rows;
  p.sinks = win_sink_plan(kWtTile, w.L, w.S, w.window, w.sinks, w.rep, (int64_t)w.Hkv * w.B);
  p.columns = w.buckets.count * (w.buckets.bidirectional ? 2 : 1);
  p.boxes_d = (w.D + 63) / 64; p.boxes_e = (w.E + 63) / 64;
  p.status = device_status_word();
  LB2_REQUIRE(p.status != nullptr, LB2_LAUNCH_FAIL, "windowed attention: device status word unavailable");
  CUtensorMap mq, mg, mk, mv;
  if (!wt_encode(&mq, w.q, w.D, w.H, w.L, w.B) || !wt_encode(&mg, dx, w.E, w.H, w.L, w.B) || !wt_encode(&mk, w.k, w.D, w.Hkv, w.S, w.B) ||
      !wt_encode(&mv, w.v, w.E, w.Hkv, w.S, w.B))
    return fail(LB2_LAUNCH_FAIL, "windowed attention: cuTensorMapEncodeTiled failed");
  const int64_t qt = (w.L + kWtTile - 1) / kWtTile, kt = (w.S + kWtTile - 1) / kWtTile;
  LB2_REQUIRE(qt * w.H * w.B <= 0x7FFFFFFF && kt * w.Hkv * w.B <= 0x7FFFFFFF, LB2_BAD_SHAPE, "too many rows");
  p.query_tiles = (int)qt;
  const int lanes = w.E <= 64 ? 8 : 16;
  const int64_t row_blocks = (qt * kWtTile * w.H * w.B * lanes + 255) / 256;
  LB2_REQUIRE(row_blocks <= 0x7FFFFFFF, LB2_BAD_SHAPE, "too many rows");
  if (lanes == 8) win_tc_rows_kernel<8><<<(unsigned)row_blocks, 256, 0, st>>>(p, delta, static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(rest));
  else win_tc_rows_kernel<16><<<(unsigned)row_blocks, 256, 0, st>>>(p, delta, static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(rest));
  LB2_CHECK_LAUNCH("windowed attention rows");
  auto launch = [&](auto kernel, int smem, int64_t tiles, int64_t blocks) -> int32_t {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(LB2_LAUNCH_FAIL, "windowed attention: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(e));
    p.tiles = (int)tiles;
    kernel<<<(unsigned)blocks, kWtBwdThreads, smem, st>>>(mq, mg, mk, mv, p);
    LB2_CHECK_LAUNCH("windowed attention pullback");
    return LB2_OK;
  };
  const bool one = p.boxes_d == 1 && p.boxes_e == 1;
  LB2_REQUIRE(qt * w.H * w.B <= 0x7FFF0000, LB2_BAD_SHAPE, "too many rows");           // and a grid more
  p.items = (int)(qt * w.H * w.B);
  p.wide_d = aligned_to(dq, 32) && w.D % 16 == 0;
  const int64_t steps = std::min<int64_t>(w.S, (int64_t)w.window + kWtTile) / kWtTile + 1, resident = wt_blocks(p.items, sm_count(), steps);
  int32_t rc = w.buckets.count > 0 ? (one ? launch(win_tc_dq_kernel<1, true>, WtBwd<1>::SMEM, qt, resident) : launch(win_tc_dq_kernel<2, true>, WtBwd<2>::SMEM, qt, resident))
                                    : (one ? launch(win_tc_dq_kernel<1, false>, WtBwd<1>::SMEM, qt, resident) : launch(win_tc_dq_kernel<2, false>, WtBwd<2>::SMEM, qt, resident));
  if (rc != LB2_OK) return rc;
  const int64_t blocks = (kt - p.sinks.tiles + (int64_t)p.sinks.tiles * p.sinks.splits) * w.Hkv * w.B;
  LB2_REQUIRE(blocks <= 0x7FFF0000, LB2_BAD_SHAPE, "too many rows");
  p.items = (int)blocks;
  p.wide_kv = aligned_to(dk, 32) && aligned_to(dv, 32) && w.D % 16 == 0 && w.E % 16 == 0;
  const int64_t resident_kv = wt_blocks(p.items, sm_count(), (std::min<int64_t>(w.L, (int64_t)w.window + kWtTile) / kWtTile + 1) * w.rep);
  rc = one ? launch(win_tc_dkv_kernel<1>, WtBwd<1>::SMEM, kt, resident_kv) : launch(win_tc_dkv_kernel<2>, WtBwd<2>::SMEM, kt, resident_kv);
  if (rc != LB2_OK || p.sinks.tiles == 0) return rc;
  return win_sinks_join(w, p.sinks, kWtTile, dk, dv, sink_sums, dx, stats, delta, LB2_BF16, st);
}

}  // namespace lb2
