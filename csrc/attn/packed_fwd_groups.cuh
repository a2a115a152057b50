// Attention forward over packed sequences (packed.cuh) for heads of 64 in groups: four chains a CTA instead of two.
//
// At d = 64 a tile of scores costs twice the time in exponentials (16 a clock and SM) that it costs in products, and with two chains the
// exponentials stand still for nearly half of the time: after its own a chain waits for P V and the next scores while the other chain has the unit
// to itself (2 x 4096 tokens, 32 / 8 heads: 3700 clocks for two tiles of 128 x 128 where the exponentials need 2048).  Here four
// chains of 128 rows share the unit, with key tiles of 64 so that scores and output of all of them fit tensor memory (4 x (64 + 64) columns).
// The chains are heads of one group at the same rows (four, or two at two tiles of rows), so they read the same K and V tiles, begin and end
// together, and a CTA has 128 rows of every sequence it meets, not 256.  4096 x 2 tokens, 32 / 8 heads: 227 -> 192 us; 8192 tokens in
// documents of some 700, 32 / 4 heads: 154 -> 113 us.
//
// Per chain and key tile j:  S = Q K_j^T (SS, fp32 in TMEM);  P = exp2(S c - m c), 128 softmax threads, a row each, over the first 32
// columns of S as bf16;  O += P V_j (TS).  One warp issues, in the order PV_0(j) QK_0(j+1) PV_1(j) QK_1(j+1) ..., and waits for data
// alone.  O is rescaled in TMEM only when a row's maximum grew by more than 2^8.
//
// Warps 0-15: softmax, chain warp / 4; 16: MMA issuer + TMEM owner; 17: TMA producer; 18, 19: idle.
#pragma once
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "packed.cuh"

namespace zb {

struct GroupsParams {
  float* lse;
  const int2* bounds;
  const PackedPair* pairs;
  const PackedTile* tiles;
  int T, Hq, rep, causal, window;
  float scale_log2;
  int* status;
};

struct GroupsCfg {
  static constexpr int CHAINS = 4, BM = 128, BN = 64, D = 64, NSLOT = 12;
  static constexpr int Q_BYTES = BM * D * 2, KV_BYTES = BN * D * 2;
  static constexpr int SMEM_BYTES = CHAINS * Q_BYTES + NSLOT * KV_BYTES + 1024 + 512;
  static constexpr int THREADS = 640;
  // registers of the softmax warps and of the rest: together what the CTA was launched with (640 x 96)
  static constexpr int SOFTMAX_REGS = 104, OTHER_REGS = 64;
  static_assert(512 * SOFTMAX_REGS + 128 * OTHER_REGS == THREADS * 96, "register budget");
};

// HEADS: chains at the same rows, 4 or 2.
template <int HEADS>
__global__ void __launch_bounds__(GroupsCfg::THREADS, 1)
packed_fwd_groups_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                         const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_o, const GroupsParams p) {
  using Cfg = GroupsCfg;
  constexpr int BM = Cfg::BM, BN = Cfg::BN, D = Cfg::D, NSLOT = Cfg::NSLOT, CHAINS = Cfg::CHAINS, TILES = CHAINS / HEADS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sR = sQ + CHAINS * Cfg::Q_BYTES;       // ring: K_j, V_j, K_j+1, ...
  uint64_t* bars = reinterpret_cast<uint64_t*>(sR + NSLOT * Cfg::KV_BYTES);
  uint64_t* q_full = bars;                  // [CHAINS]
  uint64_t* s_full = q_full + CHAINS;       // [CHAINS]
  uint64_t* p_full = s_full + CHAINS;       // [CHAINS], one arrival a warp
  uint64_t* o_done = p_full + CHAINS;       // [CHAINS]
  uint64_t* r_full = o_done + CHAINS;       // [NSLOT]
  uint64_t* r_empty = r_full + NSLOT;       // [NSLOT]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(r_empty + NSLOT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head0 = int(blockIdx.x) * HEADS, kv_head = head0 / p.rep;
  WaitCtx wctx{abort_flag, p.status};

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int c = 0; c < CHAINS; ++c) {
      mbar_init(&q_full[c], 1);
      mbar_init(&s_full[c], 1);
      mbar_init(&p_full[c], 4);
      mbar_init(&o_done[c], 1);
    }
    for (int i = 0; i < NSLOT; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], 1);
    }
    mbar_fence_init();
  }
  if (warp == 16) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_trigger();
  chain_wait();

  // tiles of rows of this CTA, and the key tiles that each of them meets
  int row_tile, total;
  int2 first[TILES], last[TILES];
  if constexpr (TILES == 1) {
    const PackedTile mine = load_packed(p.tiles + blockIdx.y);
    row_tile = mine.tile;
    total = mine.total;
    first[0] = mine.first;
    last[0] = mine.last;
  } else {
    const PackedPair mine = load_packed(p.pairs + blockIdx.y);
    row_tile = 2 * mine.pair;
    total = mine.total;
#pragma unroll
    for (int i = 0; i < TILES; ++i) { first[i] = mine.first[i]; last[i] = mine.last[i]; }
  }
  int lo[TILES], hi[TILES], j_lo = 1 << 30, j_hi = 0;
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    const KeyRange r = key_range(first[i], last[i], (row_tile + i) * BM, p.causal, p.window);
    lo[i] = r.lo / BN;
    hi[i] = r.hi > r.lo ? (r.hi + BN - 1) / BN : lo[i];
    if (hi[i] > lo[i]) { j_lo = min(j_lo, lo[i]); j_hi = max(j_hi, hi[i]); }
  }
  const int n_tiles = max(j_hi - j_lo, 0);
  auto tile_of = [&](int c) { return TILES == 1 ? 0 : c / HEADS; };
  auto lo_of = [&](int c) { return TILES == 1 || c < HEADS ? lo[0] : lo[TILES - 1]; };
  auto hi_of = [&](int c) { return TILES == 1 || c < HEADS ? hi[0] : hi[TILES - 1]; };

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::OTHER_REGS));
    if (warp == 17) {
      // ------------------------------ TMA producer ------------------------------
      if (lane == 0) {
        tma_prefetch_desc(&tmap_q);
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
#pragma unroll 1
        for (int c = 0; c < CHAINS; ++c) {
          if (hi_of(c) <= lo_of(c)) continue;
          mbar_expect_tx(&q_full[c], Cfg::Q_BYTES);
          tma_load_4d(sQ + c * Cfg::Q_BYTES, &tmap_q, &q_full[c], 0, head0 + c % HEADS, (row_tile + tile_of(c)) * BM, 0);
        }
        for (int t = 0; t < 2 * n_tiles; ++t) {
          const int slot = t % NSLOT, kv0 = (j_lo + (t >> 1)) * BN;
          if (!zb_in_bounds(kv0 >= 0 && kv0 < p.T, p.status, 8)) break;
          if (!mbar_wait(&r_empty[slot], (uint32_t(t / NSLOT) & 1) ^ 1, wctx, ST_TIMEOUT_EMPTY)) break;
          mbar_expect_tx(&r_full[slot], Cfg::KV_BYTES);
          tma_load_4d(sR + slot * Cfg::KV_BYTES, (t & 1) ? &tmap_v : &tmap_k, &r_full[slot], 0, kv_head, kv0, 0);
        }
      }
    } else if (warp == 16) {
      // ------------------------------ MMA issuer (all chains) ------------------------------
      // Chains and products are unrolled and places in the ring counted along: with a loop over chains (operands formed product by product) or chains
      // taken as their weights come in, the issuing itself bounds the kernel (2 x 4096 tokens: 192 us unrolled, 220 and 422).
      const bool elected = elect_one();
      constexpr uint32_t idesc_s = umma_idesc_bf16(BM, BN, false, false);
      constexpr uint32_t idesc_o = umma_idesc_bf16(BM, D, false, true);
      constexpr uint64_t KV_STEP = Cfg::KV_BYTES >> 4;      // of a descriptor, to the next entry of the ring
      const uint64_t q_desc = umma_desc_kmajor(smem_u32(sQ)), k_desc = umma_desc_kmajor(smem_u32(sR)), v_desc = umma_desc_mnmajor(smem_u32(sR), BN * 128);
      bool ok = true;
      auto has = [&](int c, int j) { return TILES == 1 || (j >= lo_of(c) && j < hi_of(c)); };
      auto issue_qk = [&](int c, uint64_t k_at) {
        if (elected) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_f16_ss(tmem_base + uint32_t(c * 64), q_desc + uint64_t(c * (Cfg::Q_BYTES >> 4) + kk * 2), k_at + uint64_t(kk * 2), idesc_s, kk != 0 ? 1u : 0u);
          umma_commit(&s_full[c]);
        }
        __syncwarp();
      };
      int slot = 0;                 // the ring's entry that comes next
      uint32_t phase = 0;
      auto next_entry = [&] {
        if (++slot == NSLOT) { slot = 0; phase ^= 1; }
      };
      if (n_tiles > 0) {
        ok = mbar_wait_warp(&r_full[0], 0, wctx, ST_TIMEOUT_FULL);
#pragma unroll
        for (int c = 0; c < CHAINS; ++c)
          if (ok && has(c, j_lo)) {
            ok = mbar_wait_warp(&q_full[c], 0, wctx, ST_TIMEOUT_FULL);
            tc_fence_after();
            if (ok) issue_qk(c, k_desc);
          }
        if (ok && elected) umma_commit(&r_empty[0]);
        __syncwarp();
        next_entry();
      }
      for (int j = j_lo; j < j_hi && ok; ++j) {
        const bool more = j + 1 < j_hi;
        const int vslot = slot;
        if (!mbar_wait_warp(&r_full[vslot], phase, wctx, ST_TIMEOUT_FULL)) { ok = false; break; }
        next_entry();
        const int kslot = slot;
        if (more && !mbar_wait_warp(&r_full[kslot], phase, wctx, ST_TIMEOUT_FULL)) { ok = false; break; }
        next_entry();
        tc_fence_after();
        clear_tail_rows<D, BN>(smem_u32(sR + vslot * Cfg::KV_BYTES), total - j * BN, lane);   // their weights are 0, but 0 times a NaN is one
        const uint64_t v_at = v_desc + uint64_t(vslot) * KV_STEP, k_at = k_desc + uint64_t(kslot) * KV_STEP;
#pragma unroll
        for (int c = 0; c < CHAINS; ++c) {
          if (ok && has(c, j)) {
            ok = mbar_wait_warp(&p_full[c], uint32_t(j - lo_of(c)) & 1, wctx, ST_TIMEOUT_MISC);
            tc_fence_after();
            if (ok && elected) {
#pragma unroll
              for (int kk = 0; kk < BN / 16; ++kk)
                umma_f16_ts(tmem_base + uint32_t(256 + c * 64), tmem_base + uint32_t(c * 64 + kk * 8), v_at + uint64_t(kk * 128), idesc_o,
                            j != lo_of(c) || kk != 0 ? 1u : 0u);
              if (j == hi_of(c) - 1) umma_commit(&o_done[c]);
            }
            __syncwarp();
          }
          if (ok && more && has(c, j + 1)) {
            if (TILES > 1 && j + 1 == lo_of(c)) {
              ok = mbar_wait_warp(&q_full[c], 0, wctx, ST_TIMEOUT_FULL);
              tc_fence_after();
            }
            if (ok) issue_qk(c, k_at);
          }
        }
        if (ok && elected) {
          umma_commit(&r_empty[vslot]);
          if (more) umma_commit(&r_empty[kslot]);
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------ softmax warps of chain c ------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::SOFTMAX_REGS));
    const int c = warp >> 2, t = threadIdx.x & 127, head = head0 + c % HEADS;
    const int q0 = (row_tile + tile_of(c)) * BM, row = q0 + t;
    const uint32_t lane_addr = tmem_base + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t s_col = lane_addr + uint32_t(c * 64), o_col = lane_addr + uint32_t(256 + c * 64);
    const int my_lo = lo_of(c), my_tiles = max(hi_of(c) - my_lo, 0);
    const int2 b = p.bounds[row];
    const int key_lo = p.window > 0 ? max(b.x, row - p.window + 1) : b.x, key_hi = p.causal ? min(row + 1, b.y) : b.y;
    // keys that every row of the tile sees
    const int last_begin = TILES == 1 || c < HEADS ? last[0].x : last[TILES - 1].x, first_end = TILES == 1 || c < HEADS ? first[0].y : first[TILES - 1].y;
    const int all_lo = p.window > 0 ? max(last_begin, q0 + BM - p.window) : last_begin, all_hi = p.causal ? min(first_end, q0 + 1) : first_end;
    const float scale = p.scale_log2;
    float m_run = -INFINITY, l_run = total < 0 ? PACKED_NAN : 0.f;
    bool ok = true;
    for (int i = 0; i < my_tiles; ++i) {
      const int kv0 = (my_lo + i) * BN;
      if (!__all_sync(0xffffffffu, mbar_wait(&s_full[c], uint32_t(i) & 1, wctx, ST_TIMEOUT_TMEM_FULL))) { ok = false; break; }
      tc_fence_after();
      uint32_t s0[32], s1[32];
      tmem_ld32(s_col, s0);
      tmem_ld32(s_col + 32u, s1);
      tmem_wait_ld();
      if (kv0 < all_lo || kv0 + BN > all_hi) {
        const int vis_lo = max(key_lo - kv0, 0);
        const uint32_t vis_n = uint32_t(max(key_hi - kv0 - vis_lo, 0));
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          s0[k] = uint32_t(k - vis_lo) < vis_n ? s0[k] : 0xff800000u;        // -inf
          s1[k] = uint32_t(32 + k - vis_lo) < vis_n ? s1[k] : 0xff800000u;
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int k = 0; k < 32; k += 4) {
        mx[0] = fmax3(mx[0], __uint_as_float(s0[k]), __uint_as_float(s0[k + 1]));
        mx[1] = fmax3(mx[1], __uint_as_float(s0[k + 2]), __uint_as_float(s0[k + 3]));
        mx[2] = fmax3(mx[2], __uint_as_float(s1[k]), __uint_as_float(s1[k + 1]));
        mx[3] = fmax3(mx[3], __uint_as_float(s1[k + 2]), __uint_as_float(s1[k + 3]));
      }
      const float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      if (i == 0) {
        m_run = tmax;
      } else {
        const bool need = (tmax - m_run) * scale > 8.f;
        if (__any_sync(0xffffffffu, need)) {
          float alpha = 1.f;
          if (need) {
            alpha = (m_run == -INFINITY) ? 0.f : exp2f((m_run - tmax) * scale);
            m_run = tmax;
            l_run *= alpha;
          }
          // these scores are complete, so every product issued before them is, P V of the tile before among them
#pragma unroll 1
          for (int ch = 0; ch < 4; ++ch) {
            uint32_t r[16];
            tmem_ld16(o_col + uint32_t(ch * 16), r);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
            tmem_st16(o_col + uint32_t(ch * 16), r);
          }
          tmem_wait_st();
        }
      }
      const float m_eff = (m_run == -INFINITY) ? 0.f : m_run, neg_mc = -m_eff * scale;
      float ls[4] = {0.f, 0.f, 0.f, 0.f};
      auto exp_store = [&](uint32_t (&r)[32], uint32_t col) {
        uint32_t pk[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          float x0, x1;
          ffma2(x0, x1, __uint_as_float(r[k]), __uint_as_float(r[k + 1]), scale, scale, neg_mc, neg_mc);
          const float e0 = exp2f(x0), e1 = exp2f(x1);
          const int a = ((k >> 1) & 1) * 2;
          fadd2(ls[a], ls[a + 1], ls[a], ls[a + 1], e0, e1);
          pk[k >> 1] = pack_bf16x2(e0, e1);
        }
        tmem_st16(s_col + col, pk);
      };
      exp_store(s0, 0u);
      exp_store(s1, 16u);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[c]);
      l_run += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    }
    // ------------------------------ epilogue ------------------------------
    if (ok && my_tiles > 0) ok = mbar_wait(&o_done[c], 0, wctx, ST_TIMEOUT_MISC);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    const float inv_l = l_run != 0.f ? 1.f / l_run : 0.f;      // (NaN stays NaN)
    // O leaves through the chain's Q tile, whose last reader is done, and TMA, which drops the rows behind the batch
    const uint32_t orow = smem_u32(sQ) + uint32_t(c * Cfg::Q_BYTES) + uint32_t(t) * 128;
#pragma unroll 1
    for (int ch = 0; ch < 2; ++ch) {
      uint32_t r[32];
      if (my_tiles > 0) {
        tmem_ld32(o_col + uint32_t(ch * 32), r);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) r[k] = 0u;
      }
#pragma unroll
      for (int v4 = 0; v4 < 4; ++v4)
        st_shared_v4(orow + ((uint32_t(ch * 4 + v4) ^ uint32_t(t & 7)) << 4),
                     pack_bf16x2(__uint_as_float(r[v4 * 8 + 0]) * inv_l, __uint_as_float(r[v4 * 8 + 1]) * inv_l),
                     pack_bf16x2(__uint_as_float(r[v4 * 8 + 2]) * inv_l, __uint_as_float(r[v4 * 8 + 3]) * inv_l),
                     pack_bf16x2(__uint_as_float(r[v4 * 8 + 4]) * inv_l, __uint_as_float(r[v4 * 8 + 5]) * inv_l),
                     pack_bf16x2(__uint_as_float(r[v4 * 8 + 6]) * inv_l, __uint_as_float(r[v4 * 8 + 7]) * inv_l));
    }
    fence_proxy_async_smem();
    asm volatile("bar.sync %0, 128;" ::"r"(1 + c) : "memory");   // the chain's four warps (all of them come here)
    if ((warp & 3) == 0 && lane == 0 && ok && *abort_flag == 0 && q0 < p.T) {
      tma_store_4d(&tmap_o, sQ + c * Cfg::Q_BYTES, 0, head, q0, 0);
      bulk_commit();
    }
    if (ok && row < p.T)
      p.lse[size_t(head) * p.T + row] =
          l_run != 0.f ? ((m_run == -INFINITY ? 0.f : m_run) * scale + log2f(l_run)) * 0.6931471805599453f : -INFINITY;
    if ((warp & 3) == 0 && lane == 0) bulk_wait_read<0>();
  }

  __syncwarp();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

inline int groups_map(CUtensorMap* out, const __nv_bfloat16* base, int T, int heads, int width, uint32_t rows) {
  const uint64_t dims[4] = {64, uint64_t(heads), uint64_t(T), 1};
  const uint64_t strides[3] = {128, uint64_t(width) * 2, uint64_t(width) * 2 * uint64_t(T)};
  const uint32_t box[4] = {64, 1, rows, 1};
  return make_tmap_nd_bf16(out, base, 4, dims, strides, box);
}

template <int HEADS>
inline int launch_groups(const __nv_bfloat16* qkv, __nv_bfloat16* out, int Hkv, const GroupsParams& p, cudaStream_t stream) {
  using Cfg = GroupsCfg;
  const int width = (p.Hq + 2 * Hkv) * Cfg::D;
  CUtensorMap tq, tk, tv, to;
  int rc = groups_map(&tq, qkv, p.T, p.Hq, width, Cfg::BM);
  if (!rc) rc = groups_map(&tk, qkv + size_t(p.Hq) * Cfg::D, p.T, Hkv, width, Cfg::BN);
  if (!rc) rc = groups_map(&tv, qkv + size_t(p.Hq + Hkv) * Cfg::D, p.T, Hkv, width, Cfg::BN);
  if (!rc) rc = groups_map(&to, out, p.T, p.Hq, p.Hq * Cfg::D, Cfg::BM);
  if (rc) return rc;
  const auto kern = packed_fwd_groups_kernel<HEADS>;
  static SharedLimit limit;
  ZB_CUDA_OK(limit.raise(kern, Cfg::SMEM_BYTES));
  const dim3 grid(p.Hq / HEADS, HEADS == 4 ? (p.T + 127) / 128 : (p.T + 255) / 256);
  ZB_CUDA_OK(launch_chained(kern, grid, Cfg::THREADS, Cfg::SMEM_BYTES, stream, 0, tq, tk, tv, to, p));
  return 0;
}

// Whether the four chains are the faster form (heads of 64 in even groups); `pairs`: CTAs that the kernel of two chains (flash_fwd4.cu) would have.  Of a
// CTA by itself the two chains are done 1.3 to 2 times sooner, which decides where all CTAs run at once or one long sequence goes on
// behind the rest; with several rounds of CTAs the exponential unit decides.  The lengths are not known here, so by `pairs` alone.  us of four
// chains / two:  groups of 4 and 8, `pairs` of up to 128 12.3 / 10.3 to 30.7 / 20.5; 256 14.6 / 24.6 and 20.5 / 28.7 for documents of 90 and
// 300 tokens, 30.8 / 36.9 of 700, 65 / 43 and 102 / 60 for one of 2047 and 4096; 512 and more 32.8 / 49.2, 203 / 278, one of 8192 196 / 204 and
// 366 / 400.  Groups of 2, 6 and 10 (two heads a CTA, so two tiles of rows): `pairs` of 128 36 / 21; 320 and 384 32.8 / 36.9 and 43 / 49, one of 4096
// 125 / 80 and 125 / 93; 512 37 / 49, one of 4096 124 / 117; 1024 and 2048 86 / 107 and 241 / 278, one of 8192 444 / 400.
inline bool groups_pay(int T, int Hq, int Hkv) {
  const long pairs = long(Hq) * ((T + 255) / 256);
  return pairs > (Hq / Hkv % 4 == 0 ? 1l : 3l) * num_sms();
}

// Hq / Hkv even; heads of 64.
inline int packed_fwd_groups(const __nv_bfloat16* qkv, __nv_bfloat16* out, float* lse, const int2* bounds, const PackedPair* pairs,
                      const PackedTile* tiles, int T, int Hq, int Hkv, int causal, int window, float scale_log2, int* status,
                      cudaStream_t stream) {
  const GroupsParams p = {lse, bounds, pairs, tiles, T, Hq, Hq / Hkv, causal, window, scale_log2, status};
  return Hq / Hkv % 4 == 0 ? launch_groups<4>(qkv, out, Hkv, p, stream) : launch_groups<2>(qkv, out, Hkv, p, stream);
}

}  // namespace zb
