// The products of the Newton-Schulz iterations (newton_schulz.cu): fp16 operands, fp32 sums, all matrices of up to NS_GROUPS shapes in one
// launch.  Two forms, by shape:
//     symmetric   out = alpha P P^T + beta R + diag I
//     plain       out = alpha P X + beta R + gamma (R + its remainder)      P symmetric, X [n, m]
// Of a symmetric result only the tiles on and above the diagonal are formed; the others are stored as well, turned over.  A tile on the
// diagonal has the same rows on both sides, which are loaded once (8 blocks of 1024: X X^T 99.7 -> 98.2 us, A A 56.4 -> 55.0; 24 blocks, at the
// power limit, 7680 -> 7390).
//
// Persistent CTA pairs on tiles of 256 x 256, the form of the framework's bf16 product (csrc/gemm/gemm2_bf16.cu): one warp loads, one
// issues, eight take the accumulators out while the next tile is under way, in boxes of 32 rows and 64 columns through shared memory.  A warp has
// at most two boxes of a tile, so what is added to them (R) is asked for before the accumulators are complete.  With four warps,
// boxes loaded two at a time and the turned tiles stored from registers a tile took 14 us (26 thousand clocks) to leave, more than the
// 8 thousand of a reduction of 1024.
//
// Bound by the tensor pipe, and under load by the power limit: 4 x 4096 x 4096 and 3 x 4096 x 11008 take 601 us for X X^T (1380 TFLOP/s of the half
// that is needed), 351 for A A (1370) and 1085 for B X (1530; 1126 with remainders), launch by launch under a profiler; 8 blocks of 1024 keep the pipe
// busy for 86 and 69 %, and in B X for 81 % without remainders (137 us) and 69 % with them (160 us: the epilogue has twice as many instructions).
#pragma once
#include "../common/host.h"
#include "../common/pair.cuh"
#include "../common/ptx.cuh"
#include <cuda_fp16.h>
#include <algorithm>
#include <type_traits>

namespace zb {

constexpr int NS_GROUPS = 8;         // shapes of a launch

struct NsCfg {
  static constexpr int BM = 256, BN = 256, BK = 64, HALF_N = 128;
  static constexpr int A_BYTES = 128 * BK * 2, B_BYTES = HALF_N * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  // Shared memory is split at launch: a second box for each epilogue warp, or a sixth stage for long reductions, under which the
  // epilogue has time.  us with five stages / six, always:  12 matrices of 128 and 512 98.3 / 100.3, 16 of 512 157.7 / 161.6, 16 of 256 x 4096
  // (reductions of 256 mostly) 331 / 341, 8 of 1024 292 / 289, 4 of 2048 687 / 658, 2 of 4096 2500 / 2420.
  static constexpr int EP_WARPS = 8, BOX_BYTES = 32 * 128, MAX_STAGES = 6;
  static constexpr int RING_BYTES = MAX_STAGES * STAGE_BYTES + EP_WARPS * BOX_BYTES;
  static constexpr int LONG_K = 2048;
  static_assert(STAGE_BYTES == EP_WARPS * BOX_BYTES, "a stage makes room for a box a warp");
  static constexpr int SMEM_BYTES = RING_BYTES + 1024 + 512;
  static constexpr int THREADS = 64 + 32 * EP_WARPS;
};

// Matrices of one shape.
struct alignas(64) NsGroup {
  CUtensorMap a, b;       // operands: boxes of 128 rows (plain: b's of 64 rows of the reduction)
  CUtensorMap x, c, t;    // R, the result, and the result in boxes of 64 rows and 32 columns for turned tiles
  int M, N, K, tiles_m, tiles;
  int symmetric;
  int first;              // its first item
  float alpha, beta, diag;
  float gamma;            // plain, with R's remainder
  int remainders;         // 1: of R are read, 2: of the result are written (over those of R, by the thread that read them)
  int rem_rows, rem_cols; // boxes of the remainders of one matrix
  uint8_t* rem;
};
struct NsParams {
  NsGroup g[NS_GROUPS];
  int groups, items;
  int stages;             // 6 with one box a warp, 5 with two
  int* status;
};

__host__ __device__ constexpr uint32_t umma_idesc_f16(int M, int N, bool a_mn_major, bool b_mn_major) {
  return umma_idesc_bf16(M, N, a_mn_major, b_mn_major) & ~((7u << 7) | (7u << 10));   // operand types 0: fp16
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// Remainders: eight more bits of a value behind its fp16 form, as the difference of the two as whole numbers.  fp16 keeps 10 of fp32's 23 bits of a
// mantissa, so rounding moves the number by at most 2^12, and a byte holds that in steps of 2^5.  (Values below fp16's normal numbers are
// further off and keep what a byte can: they are small against the rest.)  A box of 32 rows and 64 columns lies together, 16 columns
// of a row in one piece and the rows behind one another: the products read and write it 512 bytes a warp, without shared memory.
constexpr int NS_REM_BOX = 32 * 64;
__device__ __forceinline__ size_t ns_rem_at(size_t box, int row, int col) { return box * NS_REM_BOX + (col & 48) * 32 + (row & 31) * 16 + (col & 15); }
__device__ __forceinline__ uint32_t ns_remainders(float2 x01, float2 x23, uint32_t h01, uint32_t h23) {
  const float2 a = unpack_half2(h01), b = unpack_half2(h23);
  auto q = [](float x, float h) { return (__float_as_int(x) - __float_as_int(h) + 16) >> 5; };
  uint32_t hi, all;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(q(x23.y, b.y)), "r"(q(x23.x, b.x)));
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(all) : "r"(q(x01.y, a.y)), "r"(q(x01.x, a.x)), "r"(hi));
  return all;
}
template <int K>      // byte K of the word belongs to h
__device__ __forceinline__ float ns_with_remainder(float h, uint32_t word) {
  int q;      // the byte with its sign in the other three
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(q) : "r"(word), "n"(K | (K | 8) << 4 | (K | 8) << 8 | (K | 8) << 12));
  return __int_as_float(__float_as_int(h) + q * 32);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NsCfg::THREADS, 1) newton_schulz_kernel(const __grid_constant__ NsParams p) {
  using Cfg = NsCfg;
  constexpr int BK = Cfg::BK, BN = Cfg::BN, EP_WARPS = Cfg::EP_WARPS;
  const int STAGES = p.stages, BOXES = Cfg::MAX_STAGES + 1 - STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* boxes = smem + STAGES * Cfg::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::RING_BYTES);   // the leader's are in use
  uint64_t* empty = full + Cfg::MAX_STAGES;   // each CTA waits on its own
  uint64_t* tmem_full = empty + Cfg::MAX_STAGES;   // [2], each CTA waits on its own
  uint64_t* tmem_empty = tmem_full + 2;       // [2], the leader's, one arrival per epilogue warp of both CTAs
  uint64_t* x_full = tmem_empty + 2;          // [EP_WARPS][2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(x_full + EP_WARPS * 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();
  const bool leader = cta == 0;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  WaitCtx wctx{abort_flag, p.status};

  // Item -> shape, matrix, tile.  Symmetric: the tiles tn >= tm, row by row; else column by column, so that pairs at work
  // together read few columns of the wide operand.
  struct Item { int g, matrix, tm, tn; };
  auto item_at = [&](int item) {
    Item it;
    it.g = 0;
    while (it.g + 1 < p.groups && item >= p.g[it.g + 1].first) ++it.g;
    const NsGroup& g = p.g[it.g];
    int r = item - g.first;
    it.matrix = r / g.tiles;
    r -= it.matrix * g.tiles;
    if (g.symmetric) {
      it.tm = 0;
      for (int n = g.tiles_m; r >= n; --n) { r -= n; ++it.tm; }
      it.tn = it.tm + r;
    } else {
      it.tn = r / g.tiles_m;
      it.tm = r - it.tn * g.tiles_m;
    }
    return it;
  };

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tmem_full[i], 1);
      mbar_init(&tmem_empty[i], 2 * EP_WARPS);
    }
    for (int i = 0; i < EP_WARPS * 2; ++i) mbar_init(&x_full[i], 1);
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_wait();
  chain_trigger();

  if (warp == 0) {
    // ------------------------------ TMA producer (both CTAs) ------------------------------
    const bool elected = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int item = pair; item < p.items && ok; item += num_pairs) {
      const Item it = item_at(item);
      const NsGroup& g = p.g[it.g];
      const bool sym = g.symmetric != 0, diagonal = sym && it.tm == it.tn;
      const int m0 = it.tm * Cfg::BM + int(cta) * 128, n0 = it.tn * BN + int(cta) * Cfg::HALF_N;
      if (!zb_in_bounds(it.tm * Cfg::BM < g.M && it.tn * BN < g.N, p.status, 1)) break;
      const int num_kb = (g.K + BK - 1) / BK;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, wctx, ST_TIMEOUT_EMPTY)) { ok = false; break; }
        uint8_t* sa = smem + stage * Cfg::STAGE_BYTES;
        uint8_t* sb = sa + Cfg::A_BYTES;
        if (elected) {
          if (leader) mbar_expect_tx(&full[stage], diagonal ? 2 * Cfg::A_BYTES : 2 * Cfg::STAGE_BYTES);
          tma_load_3d_pair(sa, &g.a, &full[stage], kb * BK, m0, it.matrix);
          if (diagonal) {
            // one operand's rows are the other's
          } else if (sym) {
            tma_load_3d_pair(sb, &g.b, &full[stage], kb * BK, n0, it.matrix);
          } else {
            tma_load_3d_pair(sb, &g.b, &full[stage], n0, kb * BK, it.matrix);
            tma_load_3d_pair(sb + BK * 128, &g.b, &full[stage], n0 + 64, kb * BK, it.matrix);
          }
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
    // the leader's commits arrive on the barriers of both CTAs: none may be on its way to a CTA that has left
    for (int i = 0; i < STAGES && ok; ++i) {
      ok = mbar_wait_warp(&empty[stage], phase ^ 1, wctx, ST_TIMEOUT_EMPTY);
      if (++stage == STAGES) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer (leader CTA only) ------------------------------
    if (leader) {
      const bool elected = elect_one();
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int item = pair; item < p.items && ok; item += num_pairs, ++local) {
        const Item it = item_at(item);
        const NsGroup& g = p.g[it.g];
        const int num_kb = (g.K + BK - 1) / BK;
        // b: rows of the tile with the reduction inside a row, or rows of the reduction (16 of them a product, 128 bytes apart, and
        // 64-column blocks behind one another)
        const bool sym = g.symmetric != 0;
        const uint32_t b_at = sym && it.tm == it.tn ? 0u : uint32_t(Cfg::A_BYTES);
        const uint32_t idesc = sym ? umma_idesc_f16(256, BN, false, false) : umma_idesc_f16(256, BN, false, true);
        const uint32_t b_step = sym ? 32u : 16u * 128u, b_lbo = sym ? 16u : uint32_t(BK * 128);
        const int buf = local & 1;
        ok = mbar_wait_warp(&tmem_empty[buf], (uint32_t(local >> 1) & 1) ^ 1, wctx, ST_TIMEOUT_TMEM_EMPTY);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + uint32_t(buf * BN);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait_warp(&full[stage], phase, wctx, ST_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * Cfg::STAGE_BYTES), sb = sa + b_at;
          const uint64_t a_desc = umma_desc_kmajor(sa), b_desc = umma_desc_sw128(sb, b_lbo, 1024);
          if (elected) {
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk)
              umma_f16_ss_pair(d_tmem, umma_desc_add(a_desc, kk * 32), umma_desc_add(b_desc, kk * b_step), idesc,
                               kb != 0 || kk != 0 ? 1u : 0u);
            umma_commit_pair(&empty[stage]);
          }
          __syncwarp();
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (ok && elected) umma_commit_pair(&tmem_full[buf]);
        __syncwarp();
      }
      // arrivals of the second CTA's epilogue warps: those of two more tiles have landed before this CTA leaves
      for (int i = 0; i < 2 && ok; ++i, ++local)
        ok = mbar_wait_warp(&tmem_empty[local & 1], (uint32_t(local >> 1) & 1) ^ 1, wctx, ST_TIMEOUT_TMEM_EMPTY);
    }
  } else {
    // ------------------------------ epilogue (own 128 rows) ------------------------------
    const int q = warp & 3, h = (warp - 2) >> 2;     // which 32 rows; boxes h and h + 2 of a tile
    uint8_t* my_boxes = boxes + (warp - 2) * BOXES * Cfg::BOX_BYTES;
    uint64_t* my_full = x_full + (warp - 2) * 2;
    uint32_t phases = 0;     // bit u: phase of my_full[u]
    int local = 0;
    for (int item = pair; item < p.items; item += num_pairs, ++local) {
      const Item it = item_at(item);
      const NsGroup& g = p.g[it.g];
      const int row0 = it.tm * Cfg::BM + int(cta) * 128 + q * 32, n0 = it.tn * BN;
      const int n_boxes = row0 < g.M ? min(BN / 64, (g.N - n0 + 63) / 64) : 0;
      const int mine = (n_boxes - h + 1) >> 1;
      const int buf = local & 1;
      const float alpha = g.alpha, beta = g.beta, diag = g.diag, gamma = g.gamma;
      const bool rem_in = (g.remainders & 1) != 0, rem_out = (g.remainders & 2) != 0;
      auto rem_box = [&](int u) {   // of this thread's row in box u
        const size_t at = (size_t(it.matrix) * g.rem_rows + (row0 >> 5)) * g.rem_cols + (n0 >> 6) + h + 2 * u;
        return reinterpret_cast<uint4*>(g.rem + ns_rem_at(at, lane, 0));
      };
      uint32_t rem[16];          // of this thread's 64 columns of a box, four a word
      auto load_rem = [&](int u) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint4 v = ld_v4(rem_box(u) + 32 * k);
          rem[4 * k] = v.x; rem[4 * k + 1] = v.y; rem[4 * k + 2] = v.z; rem[4 * k + 3] = v.w;
        }
      };
      if (rem_in && mine > 0) load_rem(0);
      const bool add = beta != 0.f, turned = g.symmetric && it.tm != it.tn;
      auto load_box = [&](int u) {   // lane 0; every store from its place has left
        mbar_expect_tx(&my_full[u], Cfg::BOX_BYTES);
        tma_load_3d(my_boxes + (u & (BOXES - 1)) * Cfg::BOX_BYTES, &g.x, &my_full[u], n0 + (h + 2 * u) * 64, row0, it.matrix);
      };
      if (lane == 0) {
        bulk_wait_read<0>();      // (of boxes stored a main loop ago)
        if (add)
          for (int u = 0; u < min(mine, BOXES); ++u) load_box(u);
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[buf], uint32_t(local >> 1) & 1, wctx, ST_TIMEOUT_TMEM_FULL))) break;
      tc_fence_after();
      auto release_tmem = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(&tmem_empty[buf], 0);
      };
      bool ok = true;
      if (mine <= 0) release_tmem();
      // (two forms: with the remainders' branches inside the loop each of fifteen small products took 2.4 us longer, not only those with some)
      auto boxes_out = [&](auto with_remainders) {
        constexpr bool REM = decltype(with_remainders)::value;
#pragma unroll 1
        for (int u = 0; u < mine; ++u) {
          const int col0 = n0 + (h + 2 * u) * 64;
          const uint32_t t_addr = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(buf * BN + (h + 2 * u) * 64);
          uint32_t r[32], s[32];
          tmem_ld32(t_addr, r);
          tmem_ld32(t_addr + 32u, s);
          if (BOXES == 1 && u == 1 && lane == 0) {
            bulk_wait_read<0>();
            if (add) load_box(1);
          }
          tmem_wait_ld();
          if (u == mine - 1) release_tmem();
          else __syncwarp();
          uint8_t* box = my_boxes + (u & (BOXES - 1)) * Cfg::BOX_BYTES;
          const uint32_t row_at = smem_u32(box) + uint32_t(lane) * 128;
          if (add) {
            ok = __all_sync(0xffffffffu, mbar_wait(&my_full[u], (phases >> u) & 1, wctx, ST_TIMEOUT_FULL));
            if (!ok) break;
            phases ^= 1u << u;
          }
          // the one column of this box that lies on the diagonal in this thread's row
          const int diag_at = it.tm == it.tn && (row0 & ~63) == col0 ? (row0 & 32) + lane : -1;
          uint32_t o[32];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t at = row_at + uint32_t((j ^ (lane & 7)) << 4);
            uint32_t x[4] = {0u, 0u, 0u, 0u};
            if (add) {
              const uint4 v = ld_shared_v4(at);
              x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
            }
            float2 v[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int e = (j & 3) * 8 + 2 * w;
              float lo = __uint_as_float(j < 4 ? r[e] : s[e]) * alpha, hi = __uint_as_float(j < 4 ? r[e + 1] : s[e + 1]) * alpha;
              const float2 more = unpack_half2(x[w]);
              lo = fmaf(beta, more.x, lo);
              hi = fmaf(beta, more.y, hi);
              if (REM) {
                const uint32_t word = rem[j * 2 + (w >> 1)];
                lo = fmaf(gamma, (w & 1) ? ns_with_remainder<2>(more.x, word) : ns_with_remainder<0>(more.x, word), lo);
                hi = fmaf(gamma, (w & 1) ? ns_with_remainder<3>(more.y, word) : ns_with_remainder<1>(more.y, word), hi);
              }
              if (diag_at >= 0) {
                lo += diag_at == j * 8 + 2 * w ? diag : 0.f;
                hi += diag_at == j * 8 + 2 * w + 1 ? diag : 0.f;
              }
              o[j * 4 + w] = pack_half2(lo, hi);
              v[w] = make_float2(lo, hi);
            }
            if (REM && rem_out) {
              rem[j * 2] = ns_remainders(v[0], v[1], o[j * 4], o[j * 4 + 1]);
              rem[j * 2 + 1] = ns_remainders(v[2], v[3], o[j * 4 + 2], o[j * 4 + 3]);
            }
            st_shared_v4(at, o[j * 4], o[j * 4 + 1], o[j * 4 + 2], o[j * 4 + 3]);
          }
          if (REM && rem_out) {
#pragma unroll
            for (int k = 0; k < 4; ++k) rem_box(u)[32 * k] = make_uint4(rem[4 * k], rem[4 * k + 1], rem[4 * k + 2], rem[4 * k + 3]);
          }
          if (REM && u + 1 < mine) load_rem(u + 1);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (zb_in_bounds(row0 < g.M && col0 < g.N, p.status, 2)) tma_store_3d(&g.c, box, col0, row0, it.matrix);
            bulk_commit();
            // turned boxes leave from the first place: what it holds (this box, or the turned one before it) has been read by then
            if (turned) {
              if (u == 0 || BOXES == 1) bulk_wait_read<0>();
              else bulk_wait_read<1>();
            }
          }
          if (turned) {
            // Two lanes trade halves, so that each has two rows of one column: 64 rows of 32 of the turned box, 128 bytes a store.
            __syncwarp();
            const uint32_t to = smem_u32(my_boxes) + uint32_t(lane & 1) * 64 + uint32_t(lane >> 1) * 4;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const uint32_t other = __shfl_xor_sync(0xffffffffu, o[j], 1);
              const uint32_t v = lane & 1 ? __byte_perm(other, o[j], 0x7632) : __byte_perm(o[j], other, 0x5410);
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + uint32_t(j * 128)), "r"(v) : "memory");
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (zb_in_bounds(row0 < g.M && col0 < g.N, p.status, 2)) tma_store_3d(&g.t, my_boxes, row0, col0, it.matrix);
              bulk_commit();
            }
          }
        }
      };
      if (rem_in) boxes_out(std::true_type());
      else boxes_out(std::false_type());
      if (!ok) break;
    }
  }

  __syncwarp();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // (what was sent to the other CTA's barriers has been waited for)
  if (warp >= 2 && lane == 0) bulk_wait_read<0>();
  __syncwarp();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

inline int ns_launch(const NsParams& p, cudaStream_t stream) {
  static SharedLimit limit;
  ZB_CUDA_OK(limit.raise(newton_schulz_kernel, NsCfg::SMEM_BYTES));
  const int pairs = std::min(num_sms() / 2, p.items);
  ZB_CUDA_OK(launch_chained(newton_schulz_kernel, dim3(2 * pairs), NsCfg::THREADS, NsCfg::SMEM_BYTES, stream, 0, p));
  return 0;
}

}  // namespace zb
