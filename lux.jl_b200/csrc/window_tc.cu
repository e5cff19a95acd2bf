// Windowed attention on the tensor cores, forward: BFloat16, up to 128 features.
//
// A block owns two tiles of 128 queries that read the same keys: the tiles of two heads that share a key head, or two
// neighbouring tiles of one head; each has its softmax group of four warps, a thread per row.
// Per tile of 128 keys: S = Q K' into TMEM, the group turns S into weights 2^(z2 - m2), which go back to TMEM as bf16 over S,
// O += P V with P taken from TMEM. While one group is in its softmax the tensor cores work for the other. O is rescaled only when
// a row's maximum has grown by more than 2^8 (the reference m2 may lag behind the maximum by that: weights up to 256 are as exact in
// bf16 as weights up to 1). With a bias table the sum is that of the rounded weights, and m2 grows by whole numbers, so
// that rescaling changes no rounding: x is the average over weights that the pullback can form again bit by bit, so that the gradients of
// a row's logits, summed by bucket, add up to zero as they must.
//
// Blocks stay on their SM and take pairs of tiles in turn: the next pair's Q and keys are loaded, and its first logits formed, while
// the groups finish and store this one's.
//
// Measured: 32 heads on 8, 128 features, 16384 tokens, window 4096: 0.93 ms by itself, 1031 TFLOP/s of the visible pairs (0.63 of the GEMM
// rate), 1.05 ms where calls follow one another under the power limit; 8192 tokens, window 1024, bias: 217 us. What bounds it: a group's chain per tile, 3780 cycles by the SM's clock: from its signal to
// the next logits 1600 (1024 of MMA time at full rate; S from shared memory takes all of its 128 bytes per cycle), reading S 140,
// maximum 560, exponentials 1370 (the 16 per cycle and SM), storing 130; the other group's fills the same time.
// A third of the chain would go if the next S were formed during the softmax, but 512 TMEM columns hold two S and two O and no more;
// 64 keys at a time with two S each were slower (303 against 262 us at 8192 tokens, 16 heads, window 4096; the kernel as it is takes 229): S at N = 64 is bound by its shared-memory reads.
//
// TMEM columns: S0 | S1 | O0 | O1, 128 each. Shared memory: both tiles of Q, a ring of key and value tiles in turn.
#include "common.cuh"
#include "window_tc.cuh"

namespace lb2 {

namespace {

// warp 0: TMA, warp 1: MMA, warps 4-7 and 8-11: one softmax group each; registers 104 + 2 x 200 = 3 x 168 per thread at launch
constexpr int kWtFwdThreads = 384, kWtFwdFew = 104, kWtFwdMany = 200;

template <int NB> struct WtFwd {
  static constexpr int TILE = NB * kWtBox;
  static constexpr int STAGES = NB == 1 ? 6 : 4;
  static constexpr int SMEM = 2 * TILE + STAGES * TILE + 2 * 2 * 256 * 4 + kWinMaxBuckets * 4 + 256 + 1024;
};

struct WtFwdParams {
  WinParams w;
  void *x, *rest;                            // rest: x less its rounding, or null
  float2* stats;
  int items, pairs, by_head;                        // by_head: a pair is two heads of a group, else two neighbouring tiles
  int boxes_d, boxes_e, wide;
  unsigned int* status;
};

// a pair of tiles of queries and the tiles of keys that either visits
struct WtPair {
  int head[2], l0[2], b, g, queries, keys;
  WtTiles all;
  __device__ __forceinline__ WtPair(const WtFwdParams& p, int item) {
    const WinParams& w = p.w;
    const int pr = p.pairs - 1 - item % p.pairs, rest = item / p.pairs;   // the longest (last) tiles first
    if (p.by_head) {
      const int heads2 = w.H / 2;
      head[0] = (rest % heads2) * 2; head[1] = head[0] + 1; b = rest / heads2;
      l0[0] = l0[1] = pr * kWtTile;
    } else {
      head[0] = head[1] = rest % w.H; b = rest / w.H;
      l0[0] = pr * 2 * kWtTile; l0[1] = l0[0] + kWtTile;
    }
    g = head[0] / w.rep;
    queries = warp_uniform(win_tokens(w, b, w.L)); keys = warp_uniform(win_tokens(w, b, w.S));
    all = wt_union(wt_key_tiles(w, l0[0], queries, keys), wt_key_tiles(w, l0[1], queries, keys));
  }
};

template <int NB, bool BIASED>
__global__ void __launch_bounds__(kWtFwdThreads, 1)
win_tc_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ WtFwdParams p) {
  using C = WtFwd<NB>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  float* lut = reinterpret_cast<float*>(gen + (2 + C::STAGES) * C::TILE);      // [group][parity][256]
  int32_t* first = reinterpret_cast<int32_t*>(lut + 2 * 2 * 256);              // where the buckets start
  uint64_t* bars = reinterpret_cast<uint64_t*>(first + kWinMaxBuckets);
  // [group]: S is there, P is there, its product is in O, O has been read
  uint64_t *q_full = bars, *q_empty = bars + 1, *full = bars + 2, *empty = full + C::STAGES, *s_full = empty + C::STAGES, *p_ready = s_full + 2,
           *pv_done = p_ready + 2, *o_empty = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_empty + 2);
  const uint32_t sQ = base, sKV = base + 2 * C::TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WinParams& w = p.w;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
    mbar_init(q_full, 1); mbar_init(q_empty, 1);
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_ready[i], 4); mbar_init(&pv_done[i], 1); mbar_init(&o_empty[i], 4); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x >= 64 && threadIdx.x < 64 + kWinMaxBuckets) first[threadIdx.x - 64] = w.buckets.first[threadIdx.x - 64];
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    regs_less<kWtFwdFew>();
    if (warp == 0) {
      uint32_t stage = 0, phase = 0, turn = 0;
      bool ok = true;
      for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
        const WtPair t(p, item);
        const int n = t.all.count();
        if (n == 0) continue;
        if (!mbar_wait_uniform(q_empty, (turn & 1u) ^ 1u, p.status, 0x80u)) break;
        ++turn;
        if (elect_one()) {
          mbar_expect_tx(q_full, (uint32_t)(2 * p.boxes_d * kWtBox));
          for (int i = 0; i < 2; ++i)
            for (int x = 0; x < p.boxes_d; ++x) tma_load_4d(sQ + i * C::TILE + x * kWtBox, &tmQ, x * 64, t.head[i], min(t.l0[i], w.L - 1), t.b, q_full);
        }
        __syncwarp();
        for (int i = 0; i < 2 * n; ++i) {
          if (!mbar_wait_uniform(&empty[stage], phase ^ 1u, p.status, 0x100u)) { ok = false; break; }
          if (elect_one()) {
            const bool is_k = (i & 1) == 0;
            const int boxes = is_k ? p.boxes_d : p.boxes_e, s0 = t.all.at(i >> 1) * kWtTile;
            mbar_expect_tx(&full[stage], (uint32_t)(boxes * kWtBox));
            for (int x = 0; x < boxes; ++x) tma_load_4d(sKV + stage * C::TILE + x * kWtBox, is_k ? &tmK : &tmV, x * 64, t.g, s0, t.b, &full[stage]);
          }
          __syncwarp();
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    } else if (warp == 1) {
      // one warp for both groups keeps them half a tile apart: their products do not run into one another
      uint32_t turn = 0, kst = 0, kph = 0, vst = 0, vph = 0;               // pairs; the ring's next key and value tile
      uint32_t used[2] = {0, 0}, outs[2] = {0, 0};                         // P consumed, O begun
      bool ok = true;
      for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
        const WtPair t(p, item);
        const int n = t.all.count();
        if (n == 0) continue;
        const WtView<128> view[2] = {WtView<128>(w, t.l0[0], t.queries, t.keys), WtView<128>(w, t.l0[1], t.queries, t.keys)};
        if (!mbar_wait_uniform(q_full, turn & 1u, p.status, 0x200u)) break;
        ++turn;
        bool begun[2] = {false, false};
        // the next tile's logits after this one's product, whose weights they overwrite
        for (int j = -1; j < n && ok; ++j) {
          const bool next = j + 1 < n;
          const int s0 = j >= 0 ? t.all.at(j) * kWtTile : 0, s1 = next ? t.all.at(j + 1) * kWtTile : 0;
          if (next && !mbar_wait_uniform(&full[2 * kst], kph, p.status, 0x400u)) { ok = false; break; }
          if (j >= 0 && !mbar_wait_uniform(&full[2 * vst + 1], vph, p.status, 0x400u)) { ok = false; break; }
          const uint32_t k = sKV + 2 * kst * C::TILE, v = sKV + (2 * vst + 1) * C::TILE;
#pragma unroll
          for (int grp = 0; grp < 2; ++grp) {
            const bool use = j >= 0 && view[grp].some(s0), make = next && view[grp].some(s1);
            if (use) {
              if (!begun[grp] && !mbar_wait_uniform(&o_empty[grp], (outs[grp] & 1u) ^ 1u, p.status, 0x4000u)) ok = false;
              if (!mbar_wait_uniform(&p_ready[grp], used[grp] & 1u, p.status, 0x800u)) ok = false;
              if (!ok) break;
            }
            tc_fence_after();
            if (elect_one()) {
              const uint32_t tS = tmem + grp * 128, tO = tmem + 256 + grp * 128;
              if (use) {
                if (NB == 2 && p.boxes_e == 2) wt_mma_tokens<NB>(tO, tS, v, begun[grp]);
                else wt_mma_tokens<1>(tO, tS, v, begun[grp]);
                umma_commit(&pv_done[grp]);
              }
              if (make) {
                if (NB == 2 && p.boxes_d == 2) wt_mma_features<NB>(tS, sQ + grp * C::TILE, k);
                else wt_mma_features<1>(tS, sQ + grp * C::TILE, k);
                umma_commit(&s_full[grp]);
              }
            }
            __syncwarp();
            if (use) {
              if (!begun[grp]) ++outs[grp];
              ++used[grp];
              begun[grp] = true;
            }
          }
          if (!ok) break;
          if (elect_one()) {
            if (j >= 0) umma_commit(&empty[2 * vst + 1]);
            if (next) umma_commit(&empty[2 * kst]);
            if (j + 1 == n - 1) umma_commit(q_empty);
          }
          __syncwarp();
          if (j >= 0 && ++vst == C::STAGES / 2) { vst = 0; vph ^= 1u; }
          if (next && ++kst == C::STAGES / 2) { kst = 0; kph ^= 1u; }
        }
      }
    }
  } else {
    regs_more<kWtFwdMany>();
    const int grp = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane, gt = threadIdx.x - 128 - grp * 128;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, tS = tmem + lanes + grp * 128, tO = tmem + lanes + 256 + grp * 128;
    const float c2 = w.scale2;
    __nv_bfloat16* rest = static_cast<__nv_bfloat16*>(p.rest);
    bool ok = true, redo = false;                // after a wait that ran out: no more waits, but the same way through, whose barriers all warps share
    uint32_t made = 0;                           // steps so far
    int turn = 0;                                // of the bias tables: each use has a barrier of the group, two are enough
    for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
      const WtPair t(p, item);
      const int h = t.head[grp], l0 = t.l0[grp], l = l0 + row, n = t.all.count();
      const WtView<128> view(w, l0, t.queries, t.keys);
      const WtFlat tail(w, static_cast<const __nv_bfloat16*>(w.table), h);
      float m2 = -INFINITY, sum = 0.f;
      bool begun = false;
      for (int j = 0; j < n; ++j) {
        const int s0 = t.all.at(j) * kWtTile;
        if (!view.some(s0)) continue;
        float flat = 0.f;
        const float* bias = nullptr;
        if constexpr (BIASED) {
          const int low = s0 - l0 - (kWtTile - 1);
          if (tail.is_left(low + 2 * (kWtTile - 1))) {
            flat = tail.left;
          } else if (tail.is_right(w, low)) {
            flat = tail.right;
          } else {                               // index j - row + 127: rel = low + index
            float* at = lut + (grp * 2 + turn) * 256;
            turn ^= 1;
            for (int x = gt; x < 2 * kWtTile - 1; x += 128) at[x] = win_bias<__nv_bfloat16>(w, first, h, low + x);
            bar_group(1 + grp, 128);
            bias = at + (kWtTile - 1 - row);
          }
        }
        ok = ok && wt_wait(&s_full[grp], made & 1u, p.status, 0x1000u);
        tc_fence_after();
        // logits = mul * z + add, mul > 0; what a row does not see is -inf
        const bool apart = bias == nullptr && wt_apart(c2, flat);
        const float mul = apart ? c2 : 1.f, add = apart ? flat : 0.f;
        float z[128];
        tmem_row128<0>(tS, z);
        if (!apart) {
          if (bias != nullptr) {
#pragma unroll
            for (int x = 0; x < 128; ++x) z[x] = fmaf(z[x], c2, bias[x]);
          } else {
#pragma unroll
            for (int x = 0; x < 128; ++x) z[x] = fmaf(z[x], c2, flat);
          }
        }
        if (!view.whole(s0)) {
          const WtSeen seen(w, l, t.queries, s0, t.keys);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t bits = seen.bits(q * 32);
#pragma unroll
            for (int x = 0; x < 32; ++x) z[q * 32 + x] = bits >> x & 1u ? z[q * 32 + x] : -INFINITY;
          }
        }
        float top[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
        for (int x = 4; x < 128; ++x) top[x & 3] = fmaxf(top[x & 3], z[x]);
        const float mx = fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), mul, add);
        const bool grow = mx > m2 + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
          const float to = BIASED && mx - m2 < 1024.f ? m2 + ceilf(mx - m2) : mx, keep = grow ? ex2(m2 - to) : 1.f;     // beyond, nothing of the old weights is left
          if (grow) { m2 = to; sum *= keep; }
          if (begun) {                           // the logits came after the last product: O is still
#pragma unroll 1
            for (int q = 0; q < 4 * NB; ++q) {
              uint32_t v[16];
              tmem_ld16(tO + q * 16, v);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < 16; ++x) v[x] = __float_as_uint(__uint_as_float(v[x]) * keep);
              tmem_st16(tO + q * 16, v);
            }
          }
        }
        const float ref = m2 == -INFINITY ? 0.f : m2;
        const uint64_t mul_2 = pack2(mul, mul), off_2 = pack2(add - ref, add - ref);
        uint64_t part[2] = {0, 0};
        float each[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t v[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            float a, c;
            unpack2(fma2(pack2(z[q * 64 + 2 * x], z[q * 64 + 2 * x + 1]), mul_2, off_2), a, c);
            a = ex2(a); c = ex2(c);
            if constexpr (!BIASED) part[x & 1] = add2(part[x & 1], pack2(a, c));
            v[x] = pack_bf16(a, c);
            if constexpr (BIASED) add_bf16(each[2 * x & 3], each[(2 * x + 1) & 3], v[x]);
          }
          tmem_st32(tS + q * 32, v);
        }
        if constexpr (BIASED) {
          sum += (each[0] + each[1]) + (each[2] + each[3]);
        } else {
          float a, c;
          unpack2(add2(part[0], part[1]), a, c);
          sum += a + c;
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[grp]);
        ++made;
        begun = true;
      }
      if (l0 >= w.L) continue;
      const bool any = l < t.queries && win_any(w, l, t.keys), in = l < w.L;
      const float inv = 1.f / sum;
      bool fine = isfinite(inv);
      __nv_bfloat16* xr = static_cast<__nv_bfloat16*>(p.x) + (((int64_t)t.b * w.L + l) * w.H + h) * w.E;
      float o[64 * NB];
      if (begun) {
        ok = ok && wt_wait(&pv_done[grp], (made - 1) & 1u, p.status, 0x2000u);
        tc_fence_after();
        tmem_row64<0>(tO, o);
        if constexpr (NB == 2) tmem_row64<64>(tO + 64, o);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[grp]);
      } else {
#pragma unroll
        for (int x = 0; x < 64 * NB; ++x) o[x] = 0.f;
      }
#pragma unroll
      for (int q = 0; q < 4 * NB; ++q) {
        uint32_t v[8], r[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float a = o[q * 16 + 2 * x] * inv, c = o[q * 16 + 2 * x + 1] * inv;
          if (q * 16 + 2 * x < w.E) fine = fine && isfinite(a) && isfinite(c);
          v[x] = any ? pack_bf16(a, c) : 0u;
          r[x] = any ? pack_bf16(win_rest(a, __uint_as_float(v[x] << 16)), win_rest(c, __uint_as_float(v[x] & 0xFFFF0000u))) : 0u;
        }
        if (in) {
          wt_store16(xr + q * 16, v, w.E - q * 16, p.wide != 0);
          if (rest != nullptr) wt_store16(rest + (xr - static_cast<__nv_bfloat16*>(p.x)) + q * 16, r, w.E - q * 16, p.wide != 0);
        }
      }
      float2* st = p.stats != nullptr ? p.stats + ((int64_t)t.b * w.H + h) * w.L : nullptr;
      if (st != nullptr && in) st[l] = any ? make_float2(m2, log2f(sum)) : make_float2(0.f, INFINITY);
      redo = redo || (any && !fine);
      __syncwarp();
    }
    // rows that an infinity or NaN reached, once the pipeline no longer waits for this group
    if (__any_sync(0xffffffffu, redo)) {
      for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
        const WtPair t(p, item);
        const int h = t.head[grp], l = t.l0[grp] + row;
        const __nv_bfloat16* xr = static_cast<const __nv_bfloat16*>(p.x) + (((int64_t)t.b * w.L + l) * w.H + h) * w.E;
        bool bad = false;
        if (l < t.queries && win_any(w, l, t.keys))
          for (int e = 0; e < w.E; ++e) bad = bad || !isfinite(__bfloat162float(xr[e]));
        for (uint32_t again = __ballot_sync(0xffffffffu, bad); again != 0; again &= again - 1) {
          const int r = l - lane + __ffs(again) - 1;
          win_row_fwd<__nv_bfloat16, BIASED>(w, static_cast<__nv_bfloat16*>(p.x), rest, p.stats != nullptr ? p.stats + ((int64_t)t.b * w.H + h) * w.L + r : nullptr, r, h,
                                     t.b, t.keys);
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

}  // namespace

bool win_tc_serves(const lb2_window_dims* d, int32_t dtype) {
  return dtype == LB2_BF16 && d->head_dim >= 8 && d->value_dim >= 8 && d->head_dim <= 128 && d->value_dim <= 128 && d->head_dim % 8 == 0 &&
         d->value_dim % 8 == 0 && d->keys > 0 && d->queries > 0 && tensor_map_encoder() != nullptr;
}

int32_t win_tc_fwd(const WinParams& w, void* x, void* rest, float2* stats, cudaStream_t st) {
  WtFwdParams p{};
  p.w = w; p.x = x; p.rest = rest; p.stats = stats;
  const int tiles = (w.L + kWtTile - 1) / kWtTile;
  p.by_head = w.rep % 2 == 0;
  p.pairs = p.by_head ? tiles : (tiles + 1) / 2;
  p.boxes_d = (w.D + 63) / 64; p.boxes_e = (w.E + 63) / 64;
  p.wide = aligned_to(x, 32) && aligned_to(rest, 32) && w.E % 16 == 0;
  p.status = device_status_word();
  LB2_REQUIRE(p.status != nullptr, LB2_LAUNCH_FAIL, "windowed attention: device status word unavailable");
  CUtensorMap mq, mk, mv;
  if (!wt_encode(&mq, w.q, w.D, w.H, w.L, w.B) || !wt_encode(&mk, w.k, w.D, w.Hkv, w.S, w.B) || !wt_encode(&mv, w.v, w.E, w.Hkv, w.S, w.B))
    return fail(LB2_LAUNCH_FAIL, "windowed attention: cuTensorMapEncodeTiled failed");
  const int64_t items = (int64_t)p.pairs * (p.by_head ? w.H / 2 : w.H) * w.B;
  LB2_REQUIRE(items <= 0x7FFF0000, LB2_BAD_SHAPE, "too many rows");        // and a grid more
  p.items = (int)items;
  const int sms = sm_count();
  const int64_t steps = std::min<int64_t>(w.S, (int64_t)w.window + kWtTile) / kWtTile + 1;
  auto launch = [&](auto kernel, int smem) -> int32_t {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(LB2_LAUNCH_FAIL, "windowed attention: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(e));
    kernel<<<wt_blocks(p.items, sms, steps), kWtFwdThreads, smem, st>>>(mq, mk, mv, p);
    LB2_CHECK_LAUNCH("windowed attention");
    return LB2_OK;
  };
  if (w.buckets.count > 0)
    return p.boxes_d == 1 && p.boxes_e == 1 ? launch(win_tc_fwd_kernel<1, true>, WtFwd<1>::SMEM) : launch(win_tc_fwd_kernel<2, true>, WtFwd<2>::SMEM);
  return p.boxes_d == 1 && p.boxes_e == 1 ? launch(win_tc_fwd_kernel<1, false>, WtFwd<1>::SMEM) : launch(win_tc_fwd_kernel<2, false>, WtFwd<2>::SMEM);
}

}  // namespace lb2
