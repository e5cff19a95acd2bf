// Windowed attention on the tensor cores, forward: BFloat16, up to 128 features.
//
// A block owns two tiles of 128 queries that read the same keys: the tiles of two heads that share a key head, or two
// neighbouring tiles of one head. Per tile of 128 keys and tile of queries: S = Q K' into TMEM, one thread per row turns S into
// weights 2^(z2 - m2), which go back to TMEM as bf16 over S, O += P V with P taken from TMEM. While one tile of queries is in its
// softmax the tensor cores work for the other. O is rescaled only when a row's maximum has grown by more than 2^8 (the
// reference m2 may lag behind the maximum by that: weights up to 256 are as exact in bf16 as weights up to 1).
//
// TMEM columns: S0 | S1 | O0 | O1, 128 each. Shared memory: both tiles of Q, a ring of key and value tiles in turn.
#include "common.cuh"
#include "window_tc.cuh"

namespace lb2 {

namespace {

// warp 0: TMA, warp 1: MMA, warps 4-7 and 8-11: one softmax group each. The softmax keeps a row of S in registers: the first four
// warps give up theirs (56 + 2 x 224 = 3 x 168 per thread at launch).
constexpr int kWtFwdThreads = 384, kWtFwdFew = 56, kWtFwdMany = 224;

template <int NB> struct WtFwd {
  static constexpr int TILE = NB * kWtBox;
  static constexpr int STAGES = NB == 1 ? 6 : 4;
  static constexpr int SMEM = 2 * TILE + STAGES * TILE + 2 * 2 * 256 * 4 + 256 + 1024;
};

struct WtFwdParams {
  WinParams w;
  void* x;
  float2* stats;
  int tiles, pairs, by_head;                 // by_head: a pair is two heads of a group, else two neighbouring tiles
  int boxes_d, boxes_e;
  unsigned int* status;
};

template <int NB>
__global__ void __launch_bounds__(kWtFwdThreads, 1)
win_tc_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ WtFwdParams p) {
  using C = WtFwd<NB>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  float* lut = reinterpret_cast<float*>(gen + (2 + C::STAGES) * C::TILE);      // [group][parity][256]
  uint64_t* bars = reinterpret_cast<uint64_t*>(lut + 2 * 2 * 256);
  uint64_t *q_full = bars, *full = bars + 1, *empty = full + C::STAGES, *s_full = empty + C::STAGES, *p_ready = s_full + 2, *o_full = p_ready + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  const uint32_t sQ = base, sKV = base + 2 * C::TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WinParams& w = p.w;

  // the pair's two tiles of queries
  int item = blockIdx.x;
  const int pr = item % p.pairs;
  item /= p.pairs;
  int head[2], l0[2], b;
  if (p.by_head) {
    const int heads2 = w.H / 2;
    head[0] = (item % heads2) * 2; head[1] = head[0] + 1; b = item / heads2;
    l0[0] = l0[1] = pr * kWtTile;
  } else {
    head[0] = head[1] = item % w.H; b = item / w.H;
    l0[0] = pr * 2 * kWtTile; l0[1] = l0[0] + kWtTile;
  }
  const int g = head[0] / w.rep;
  const int queries = win_tokens(w, b, w.L), keys = win_tokens(w, b, w.S);
  const WtTiles own[2] = {wt_key_tiles(w, l0[0], queries, keys), wt_key_tiles(w, l0[1], queries, keys)};
  const WtTiles all = wt_union(own[0], own[1]);
  const int n = all.count();

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_ready[i], 4); mbar_init(&o_full[i], 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
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
      if (n > 0) {
        if (elect_one()) {
          mbar_expect_tx(q_full, (uint32_t)(2 * p.boxes_d * kWtBox));
          for (int i = 0; i < 2; ++i)
            for (int x = 0; x < p.boxes_d; ++x) tma_load_4d(sQ + i * C::TILE + x * kWtBox, &tmQ, x * 64, head[i], min(l0[i], w.L - 1), b, q_full);
        }
        __syncwarp();
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        for (int i = 0; i < 2 * n && ok; ++i) {
          if (!mbar_wait_uniform(&empty[stage], phase ^ 1u, p.status, 0x100u)) { ok = false; break; }
          if (elect_one()) {
            const bool is_k = (i & 1) == 0;
            const int boxes = is_k ? p.boxes_d : p.boxes_e, s0 = all.at(i >> 1) * kWtTile;
            mbar_expect_tx(&full[stage], (uint32_t)(boxes * kWtBox));
            for (int x = 0; x < boxes; ++x) tma_load_4d(sKV + stage * C::TILE + x * kWtBox, is_k ? &tmK : &tmV, x * 64, g, s0, b, &full[stage]);
          }
          __syncwarp();
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    } else if (warp == 1) {
      // in order: S0 S1 of the first tile; then per tile, O of it and S of the next for each group in turn
      bool ok = n == 0 || mbar_wait_uniform(q_full, 0, p.status, 0x200u);
      uint32_t ready[2] = {0, 0};              // phases of p_ready
      bool begun[2] = {false, false};
      auto wait_stage = [&](int i) { return mbar_wait_uniform(&full[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1u, p.status, 0x400u); };
      auto scores = [&](int i, int grp) {
        if (elect_one()) {
          const uint32_t k = sKV + (2 * i % C::STAGES) * C::TILE, q = sQ + grp * C::TILE, d = tmem + grp * 128;
          if (NB == 2 && p.boxes_d == 2) wt_mma_features<NB>(d, q, k);
          else wt_mma_features<1>(d, q, k);
          umma_commit(&s_full[grp]);
        }
        __syncwarp();
      };
      auto release = [&](int i) {
        if (elect_one()) umma_commit(&empty[i % C::STAGES]);
        __syncwarp();
      };
      for (int i = -1; i < n && ok; ++i) {
        const bool next = i + 1 < n;
        if (next && !wait_stage(2 * (i + 1))) { ok = false; break; }
        if (i >= 0 && !wait_stage(2 * i + 1)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int grp = 0; grp < 2; ++grp) {
          if (!ok) break;
          if (i >= 0 && own[grp].has(all.at(i))) {
            if (!mbar_wait_uniform(&p_ready[grp], ready[grp], p.status, 0x800u)) { ok = false; break; }
            ready[grp] ^= 1u;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t v = sKV + ((2 * i + 1) % C::STAGES) * C::TILE, d = tmem + 256 + grp * 128, a = tmem + grp * 128;
              if (NB == 2 && p.boxes_e == 2) wt_mma_tokens<NB>(d, a, v, begun[grp]);
              else wt_mma_tokens<1>(d, a, v, begun[grp]);
            }
            __syncwarp();
            begun[grp] = true;
          }
          if (next && own[grp].has(all.at(i + 1))) scores(i + 1, grp);
        }
        if (!ok) break;
        if (i >= 0) release(2 * i + 1);
        if (next) release(2 * (i + 1));
      }
      if (ok && elect_one()) { umma_commit(&o_full[0]); umma_commit(&o_full[1]); }
      __syncwarp();
    }
  } else {
    regs_more<kWtFwdMany>();
    const int grp = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane, l = l0[grp] + row, h = head[grp];
    const int gt = threadIdx.x - 128 - grp * 128;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, tS = tmem + lanes + grp * 128, tO = tmem + lanes + 256 + grp * 128;
    const float c2 = w.scale2;
    const bool biased = w.buckets.count > 0;
    float m2 = -INFINITY, sum = 0.f;
    bool ok = true, begun = false;
    uint32_t phase = 0;
    int turn = 0;
    for (int i = 0; i < n; ++i) {
      const int t = all.at(i), s0 = t * kWtTile;
      if (!own[grp].has(t)) continue;
      float flat = 0.f;
      const float* bias = nullptr;
      if (biased) {
        const int low = s0 - l0[grp] - (kWtTile - 1), high = s0 - l0[grp] + (kWtTile - 1);
        const int bl = win_bucket(w.buckets, low);
        if (bl == win_bucket(w.buckets, high)) {
          flat = win_bias2(to_f32(static_cast<const __nv_bfloat16*>(w.table)[h + (int64_t)w.H * bl]));
        } else {                               // index j - row + 127: rel = low + index
          float* at = lut + (grp * 2 + turn) * 256;
          for (int x = gt; x < 255; x += 128) at[x] = win_bias<__nv_bfloat16>(w, h, low + x);
          bar_group(1 + grp, 128);
          bias = at + (kWtTile - 1 - row);
        }
      }
      turn ^= 1;                               // whoever is past the next s_full knows that all have read this tile's
      if (!mbar_wait_warp(&s_full[grp], phase, p.status, 0x1000u)) { ok = false; break; }
      phase ^= 1u;
      tc_fence_after();
      // logits = mul * z + add, mul > 0; what a row does not see is -inf
      const bool apart = bias == nullptr && wt_apart(c2, flat);
      const float mul = apart ? c2 : 1.f, add = apart ? flat : 0.f;
      float z[128];
      tmem_row128<0>(tS, z);
      if (!apart) {
        if (bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 128; ++j) z[j] = fmaf(z[j], c2, bias[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 128; ++j) z[j] = fmaf(z[j], c2, flat);
        }
      }
      if (!wt_all_seen(w, l0[grp], queries, s0, keys)) {
        const WtSeen seen(w, l, queries, s0, keys);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t bits = seen.bits(q * 32);
#pragma unroll
          for (int j = 0; j < 32; ++j) z[q * 32 + j] = bits >> j & 1u ? z[q * 32 + j] : -INFINITY;
        }
      }
      float top[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
      for (int j = 4; j < 128; ++j) top[j & 3] = fmaxf(top[j & 3], z[j]);
      const float mx = fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), mul, add);
      const bool grow = mx > m2 + 8.f;
      if (__any_sync(0xffffffffu, grow)) {
        const float keep = grow ? ex2(m2 - mx) : 1.f;
        if (grow) { m2 = mx; sum *= keep; }
        if (begun) {
#pragma unroll 1
          for (int q = 0; q < 4 * NB; ++q) {
            uint32_t v[16];
            tmem_ld16(tO + q * 16, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * keep);
            tmem_st16(tO + q * 16, v);
          }
        }
      }
      const float ref = m2 == -INFINITY ? 0.f : m2;
      const uint64_t mul_2 = pack2(mul, mul), off_2 = pack2(add - ref, add - ref);
      uint64_t part[2] = {0, 0};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float a, c;
          unpack2(fma2(pack2(z[q * 32 + 2 * j], z[q * 32 + 2 * j + 1]), mul_2, off_2), a, c);
          a = ex2(a); c = ex2(c);
          part[j & 1] = add2(part[j & 1], pack2(a, c));
          v[j] = pack_bf16(a, c);
        }
        tmem_st16(tS + q * 16, v);
      }
      {
        float a, c;
        unpack2(add2(part[0], part[1]), a, c);
        sum += a + c;
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[grp]);
      begun = true;
    }
    if (ok) ok = mbar_wait_warp(&o_full[grp], 0, p.status, 0x2000u);
    if (ok && l0[grp] < w.L) {
      tc_fence_after();
      const bool any = l < queries && win_any(w, l, keys), in = l < w.L;
      const float inv = 1.f / sum;
      bool fine = isfinite(inv);
      __nv_bfloat16* xr = static_cast<__nv_bfloat16*>(p.x) + (((int64_t)b * w.L + l) * w.H + h) * w.E;
#pragma unroll
      for (int q = 0; q < 2 * NB; ++q) {
        if (q * 32 >= w.E) break;
        uint32_t v[32];
        if (begun) {
          tmem_ld32(tO + q * 32, v);
          tmem_ld_wait();
        }
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float a = __uint_as_float(v[j + 2 * k]) * inv, c = __uint_as_float(v[j + 2 * k + 1]) * inv;
            if (q * 32 + j < w.E) fine = fine && isfinite(a) && isfinite(c);
            o[k] = any ? pack_bf16(a, c) : 0u;
          }
          if (in && q * 32 + j < w.E) *reinterpret_cast<uint4*>(xr + q * 32 + j) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
      float2* st = p.stats != nullptr ? p.stats + ((int64_t)b * w.H + h) * w.L : nullptr;
      if (st != nullptr && in) st[l] = any ? make_float2(m2, log2f(sum)) : make_float2(0.f, INFINITY);
      __syncwarp();
      for (uint32_t again = __ballot_sync(0xffffffffu, any && !fine); again != 0; again &= again - 1) {
        const int r = l - lane + __ffs(again) - 1;
        win_row_fwd<__nv_bfloat16>(w, static_cast<__nv_bfloat16*>(p.x), st != nullptr ? st + r : nullptr, r, h, b, keys);
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

int32_t win_tc_fwd(const WinParams& w, void* x, float2* stats, cudaStream_t st) {
  WtFwdParams p{};
  p.w = w; p.x = x; p.stats = stats;
  p.tiles = (w.L + kWtTile - 1) / kWtTile;
  p.by_head = w.rep % 2 == 0;
  p.pairs = p.by_head ? p.tiles : (p.tiles + 1) / 2;
  p.boxes_d = (w.D + 63) / 64; p.boxes_e = (w.E + 63) / 64;
  p.status = device_status_word();
  LB2_REQUIRE(p.status != nullptr, LB2_LAUNCH_FAIL, "windowed attention: device status word unavailable");
  CUtensorMap mq, mk, mv;
  if (!wt_encode(&mq, w.q, w.D, w.H, w.L, w.B) || !wt_encode(&mk, w.k, w.D, w.Hkv, w.S, w.B) || !wt_encode(&mv, w.v, w.E, w.Hkv, w.S, w.B))
    return fail(LB2_LAUNCH_FAIL, "windowed attention: cuTensorMapEncodeTiled failed");
  const int64_t items = (int64_t)p.pairs * (p.by_head ? w.H / 2 : w.H) * w.B;
  LB2_REQUIRE(items <= 0x7FFFFFFF, LB2_BAD_SHAPE, "too many rows");
  auto launch = [&](auto kernel, int smem) -> int32_t {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(LB2_LAUNCH_FAIL, "windowed attention: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(e));
    kernel<<<(unsigned)items, kWtFwdThreads, smem, st>>>(mq, mk, mv, p);
    LB2_CHECK_LAUNCH("windowed attention");
    return LB2_OK;
  };
  return p.boxes_d == 1 && p.boxes_e == 1 ? launch(win_tc_fwd_kernel<1>, WtFwd<1>::SMEM) : launch(win_tc_fwd_kernel<2>, WtFwd<2>::SMEM);
}

}  // namespace lb2
