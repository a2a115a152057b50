// RMS norm of every query and key head with the rotate-half rotation in the same pass, forward and backward, on the packed
// projection [T, (Hq + 2 Hkv) d] (query heads, key heads, value heads).  With x one head of one token, w the weights of its kind
// (wq or wk, [d], shared by the heads) and R the rotation by the angles of position t mod S:
//   forward   rstd = 1 / sqrt(mean(x^2) + eps),  y = R(x rstd w)
//   backward  g = R^T dy,  xh = x rstd,  dx = rstd (w g - xh mean(w g xh)),  dw += sum over tokens and heads of g xh
// Sums and products are in fp32 and a value is rounded to bf16 once, at the end: as two passes the normalised heads would be
// rounded in between.
// Both directions are bound by memory: 16384 tokens of 32 + 8 + 8 heads of 128 forward into a new tensor 64 to 66 us, 6.2 TB/s or
// 96 % of a copy's rate; 8192 tokens of 32 + 32 heads of 128 backward 71 us, 5.7 TB/s or 89 %, of which about 3 are the sum over
// the CTAs in a launch of its own.  Small ones are bound by their launches: 256 tokens of 8 + 2 x 8 heads of 64 2.2 us forward in a
// graph and 4.9 backward, 5.3 and 6.7 called from Python.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "norm_common.cuh"

namespace zb {

struct QkNormArgs {
  const __nv_bfloat16* x;   // the projection, row stride ldx
  __nv_bfloat16* y;         // forward: where heads go; backward: the packed gradient, in place
  const __nv_bfloat16 *wq, *wk;
  const float* cs;          // [S, d] cosines | sines; null: no rotation
  float* rstd;              // [T, nq + nk]; forward: null if not kept
  float* partial;           // backward: [CTAs, d]
  long ldx, ldy;
  int T, S, nq, nk, nv, d;  // nv: value heads to copy (forward into another tensor), else 0
  int span;                 // forward: units of a warp's item
  int ctas_q;               // backward: CTAs of the query heads
  float eps, inv_d;
};

// Sixteen values of a head per lane: eight from either half, so that a lane has both members of its pairs.
struct HeadChunk {
  uint4 lo, hi;
};
__device__ __forceinline__ HeadChunk load_head(const __nv_bfloat16* p, int half) { return {ld_v4(p), ld_v4(p + half)}; }
__device__ __forceinline__ void store_head(__nv_bfloat16* p, int half, const HeadChunk& h) {
  *reinterpret_cast<uint4*>(p) = h.lo;
  *reinterpret_cast<uint4*>(p + half) = h.hi;
}
template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void load_angles(const float* row, int half, float (&co)[8], float (&si)[8]) {
#pragma unroll
  for (int k = 0; k < 8; k += 4) {
    *reinterpret_cast<float4*>(co + k) = *reinterpret_cast<const float4*>(row + k);
    *reinterpret_cast<float4*>(si + k) = *reinterpret_cast<const float4*>(row + half + k);
  }
}

// Bytes on the way bound these passes: with a unit's operands in registers, and a hundred of those a thread, an SM has too few
// requests out.  So every thread copies its own chunks some units ahead into a ring of its own in shared memory (the two large
// cases above 81 -> 66 us, with packed arithmetic and the angles kept for a token's heads, and 141 -> 74).
constexpr int QK_RING = 3;
// Two values an instruction (fma.rn.f32x2 and the like): a head's arithmetic is most of what an SM issues here.
struct Pair {
  float a, b;
};
__device__ __forceinline__ Pair operator*(Pair x, Pair y) {
  Pair r;
  fmul2(r.a, r.b, x.a, x.b, y.a, y.b);
  return r;
}
__device__ __forceinline__ Pair fma2(Pair x, Pair y, Pair z) {
  Pair r;
  ffma2(r.a, r.b, x.a, x.b, y.a, y.b, z.a, z.b);
  return r;
}
__device__ __forceinline__ Pair both(float v) { return {v, v}; }
__device__ __forceinline__ Pair pair_of(uint32_t u) {
  const float2 f = unpack_bf16x2(u);
  return {f.x, f.y};
}
// A head chunk as pairs: 0 .. 3 of the low half, 4 .. 7 of the high one
__device__ __forceinline__ void unpack_pairs(const HeadChunk& h, Pair (&p)[8]) {
  p[0] = pair_of(h.lo.x); p[1] = pair_of(h.lo.y); p[2] = pair_of(h.lo.z); p[3] = pair_of(h.lo.w);
  p[4] = pair_of(h.hi.x); p[5] = pair_of(h.hi.y); p[6] = pair_of(h.hi.z); p[7] = pair_of(h.hi.w);
}
__device__ __forceinline__ HeadChunk pack_pairs(const Pair (&p)[8]) {
  HeadChunk h;
  h.lo = make_uint4(pack_bf16x2(p[0].a, p[0].b), pack_bf16x2(p[1].a, p[1].b), pack_bf16x2(p[2].a, p[2].b), pack_bf16x2(p[3].a, p[3].b));
  h.hi = make_uint4(pack_bf16x2(p[4].a, p[4].b), pack_bf16x2(p[5].a, p[5].b), pack_bf16x2(p[6].a, p[6].b), pack_bf16x2(p[7].a, p[7].b));
  return h;
}
__device__ __forceinline__ float sum_of_squares(const Pair (&x)[8]) {
  Pair s = x[0] * x[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) s = fma2(x[j], x[j], s);
  return s.a + s.b;
}

// LANES lanes share a head (a power of two, at least d / 16: for d = 96 two of eight idle); a warp takes 32 / LANES neighbouring
// heads at a time, a unit.  A warp's item is `span` units of one token in a row.  The weights of a lane's kind of head and the
// token's angles are multiplied once for all its heads: lo = x_lo a - x_hi b, hi = x_hi c + x_lo d, times rstd.
template <int LANES, bool ROPE>
__global__ void __launch_bounds__(128, 6) qk_norm_rope_fwd_kernel(const QkNormArgs a) {
  chain_trigger();
  chain_wait();
  constexpr int HEADS = 32 / LANES;
  __shared__ uint4 ring[QK_RING][2][128];
  const int half = a.d >> 1, lane = threadIdx.x & 31, c = (lane % LANES) * 8;
  const int nqk = a.nq + a.nk, units = (nqk + a.nv + HEADS - 1) / HEADS;
  const unsigned parts = (units + a.span - 1) / a.span, i = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (i >= unsigned(a.T) * parts) return;
  const int t = int(i / parts), first = int(i - t * parts) * a.span;
  int h = first * HEADS + lane / LANES;                       // this lane's head, HEADS further on with every unit
  const int end = c < half ? min(nqk + a.nv, (first + a.span) * HEADS) : 0;
  const __nv_bfloat16* src = a.x + t * a.ldx + h * a.d + c;
  __nv_bfloat16* dst = a.y + t * a.ldy + h * a.d + c;
  const int step = HEADS * a.d;
  int ahead = h;
  auto request = [&](int slot) {
    if (ahead < end) {
      ring_load16(&ring[slot][0][threadIdx.x], src);
      ring_load16(&ring[slot][1][threadIdx.x], src + half);
      ahead += HEADS;
      src += step;
    }
    ring_commit();
  };
#pragma unroll
  for (int k = 0; k < QK_RING - 1; ++k) request(k);
  const float* angles = ROPE ? a.cs + size_t(t % a.S) * a.d + c : nullptr;
  Pair lo_lo[4], lo_hi[4], hi_hi[4], hi_lo[4];
  int kind = -1, slot = 0;
  const int last = min(first + a.span, units);
  for (int u = first; u < last; ++u) {
    const int now = h < a.nq ? 0 : 1;
    if (now != kind && h < nqk && c < half) {
      kind = now;
      Pair w[8];
      unpack_pairs(load_head((now ? a.wk : a.wq) + c, half), w);
      float co[8], si[8];
      if (ROPE) load_angles(angles, half, co, si);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo_lo[j] = w[j];
        hi_hi[j] = w[4 + j];
        if (ROPE) {
          const Pair cc = {co[2 * j], co[2 * j + 1]}, ss = {si[2 * j], si[2 * j + 1]};
          lo_lo[j] = w[j] * cc;
          hi_hi[j] = w[4 + j] * cc;
          lo_hi[j] = w[4 + j] * Pair{-ss.a, -ss.b};
          hi_lo[j] = w[j] * ss;
        }
      }
    }
    request((slot + QK_RING - 1) % QK_RING);
    ring_wait<QK_RING - 1>();
    HeadChunk out = {};
    if (h < end) out = {ring[slot][0][threadIdx.x], ring[slot][1][threadIdx.x]};
    slot = (slot + 1) % QK_RING;
    Pair x[8];
    unpack_pairs(out, x);
    const float rstd = rsqrtf(head_sum<LANES>(sum_of_squares(x)) * a.inv_d + a.eps);
    if (h < end) {
      if (h < nqk) {
        Pair y[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const Pair lo = x[j] * both(rstd), hi = x[4 + j] * both(rstd);
          y[j] = ROPE ? fma2(hi, lo_hi[j], lo * lo_lo[j]) : lo * lo_lo[j];
          y[4 + j] = ROPE ? fma2(lo, hi_lo[j], hi * hi_hi[j]) : hi * hi_hi[j];
        }
        out = pack_pairs(y);
        if (a.rstd != nullptr && c == 0) a.rstd[long(t) * nqk + h] = rstd;
      }
      store_head(dst, half, out);
    }
    h += HEADS;
    dst += step;
  }
}

// Tokens beside one another in a unit of the backward pass (9068 tokens of 4 + 1 heads of 64 12.1 -> 8.0 us, 8192 of 4 + 1 of 128 12.4 -> 10.6)
__host__ __device__ constexpr int qk_norm_side(int n, int heads) { return n > 0 && n < heads && heads % n == 0 ? heads / n : 1; }

struct QkRing {
  uint4 chunk[QK_RING][4][256];    // x low, x high, gradient low, gradient high
  float rstd[QK_RING][256];
};
// The first `ctas_q` CTAs have the query heads, the others the key heads: one set of weights and of weight-gradient sums a thread.
// A warp takes an equal stretch of its kind's units of all tokens; the ring runs on over its tokens.  Where a token has fewer heads of a
// kind than a unit, `side` tokens lie side by side in one.
template <int LANES, bool ROPE>
__global__ void __launch_bounds__(256, 2) qk_norm_rope_bwd_kernel(const QkNormArgs a) {
  chain_trigger();
  chain_wait();
  constexpr int HEADS = 32 / LANES;
  extern __shared__ __align__(16) unsigned char raw[];
  QkRing& ring = *reinterpret_cast<QkRing*>(raw);
  __shared__ float part[8][LANES * 16];
  const int tid = threadIdx.x, half = a.d >> 1, lane = tid & 31, warp = tid >> 5, c = (lane % LANES) * 8, sub = lane / LANES;
  const bool used = c < half;
  const int step = HEADS * a.d, nqk = a.nq + a.nk, kind = int(blockIdx.x) >= a.ctas_q;
  const int n = kind ? a.nk : a.nq, h0 = kind ? a.nq : 0, units = (n + HEADS - 1) / HEADS, side = qk_norm_side(n, HEADS);
  const int beside = side > 1 ? sub / n : 0, sub_head = sub - beside * n;      // this lane's token of those, and head
  Pair w[8], dw[8];
  HeadChunk wu = {};
  if (used) wu = load_head((kind ? a.wk : a.wq) + c, half);
  unpack_pairs(wu, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) dw[j] = both(0.f);
  const long all = long((a.T + side - 1) / side) * units, me = (blockIdx.x - (kind ? a.ctas_q : 0)) * 8 + warp;
  const long warps = (kind ? gridDim.x - a.ctas_q : a.ctas_q) * 8;
  const long first = all * me / warps;
  int left = int(all * (me + 1) / warps - first), to_ask = left;
  int t = int(first / units);
  int u = int(first - long(t) * units);
  t = t * side + beside;
  // the next unit to ask for: its number in the token, this lane's token, its head among the kind's, and where that lies
  int ask_u = u, ask_t = t, ask_k = u * HEADS + sub_head;
  size_t col = size_t(h0 + ask_k) * a.d + c;
  const __nv_bfloat16 *ask_x = a.x + t * a.ldx + col, *ask_g = a.y + t * a.ldy + col;
  __nv_bfloat16* dst = a.y + t * a.ldy + col;
  const float* ask_r = a.rstd + size_t(t) * nqk + h0 + ask_k;
  const long next_x = side * a.ldx - long(units) * step, next_g = side * a.ldy - long(units) * step;   // from behind a token's units to the next one's
  auto request = [&](int slot) {
    if (to_ask > 0) {
      if (used && ask_k < n && ask_t < a.T) {
        ring_load16(&ring.chunk[slot][0][tid], ask_x);
        ring_load16(&ring.chunk[slot][1][tid], ask_x + half);
        ring_load16(&ring.chunk[slot][2][tid], ask_g);
        ring_load16(&ring.chunk[slot][3][tid], ask_g + half);
        ring_load4(&ring.rstd[slot][tid], ask_r);
      }
      --to_ask;
      ask_x += step;
      ask_g += step;
      ask_r += HEADS;
      ask_k += HEADS;
      if (++ask_u == units) {
        ask_u = 0;
        ask_t += side;
        ask_k = sub_head;
        ask_x += next_x;
        ask_g += next_g;
        ask_r += side * nqk - units * HEADS;
      }
    }
    ring_commit();
  };
#pragma unroll
  for (int k = 0; k < QK_RING - 1; ++k) request(k);
  int slot = 0, pos = t % a.S;
  while (left > 0) {
    const bool there = used && t < a.T;
    float co[8] = {}, si[8] = {};
    if (ROPE && there) load_angles(a.cs + size_t(pos) * a.d + c, half, co, si);
    const int here = min(left, units - u);
    left -= here;
    int k = u * HEADS + sub_head;
    for (int i = 0; i < here; ++i) {
      request((slot + QK_RING - 1) % QK_RING);
      ring_wait<QK_RING - 1>();
      const bool live = there && k < n;
      HeadChunk xu = {}, gu = {};
      float rstd = 0.f;
      if (live) {
        xu = {ring.chunk[slot][0][tid], ring.chunk[slot][1][tid]};
        gu = {ring.chunk[slot][2][tid], ring.chunk[slot][3][tid]};
        rstd = ring.rstd[slot][tid];
      }
      slot = (slot + 1) % QK_RING;
      // with g = rstd R^T dy:  dw += g x,  dx = w g - x rstd^2 mean(w g x)
      Pair x[8], g[8], along = both(0.f);
      unpack_pairs(xu, x);
      unpack_pairs(gu, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Pair lo = g[j] * both(rstd), hi = g[4 + j] * both(rstd);
        const Pair cc = {co[2 * j], co[2 * j + 1]}, ss = {si[2 * j], si[2 * j + 1]}, back = {-ss.a, -ss.b};
        g[j] = ROPE ? fma2(hi, ss, lo * cc) : lo;
        g[4 + j] = ROPE ? fma2(lo, back, hi * cc) : hi;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dw[j] = fma2(g[j], x[j], dw[j]);
        g[j] = g[j] * w[j];
        along = fma2(g[j], x[j], along);
      }
      const float m = -head_sum<LANES>(along.a + along.b) * a.inv_d * (rstd * rstd);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = fma2(x[j], both(m), g[j]);
      if (live) store_head(dst, half, pack_pairs(g));
      k += HEADS;
      dst += step;
    }
    u = 0;
    t += side;
    dst += next_g;
    pos += side;
    if (pos >= a.S) pos %= a.S;
  }
  ring_wait<0>();
  // over the heads of a warp, then over its CTA's warps
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = 16; o >= LANES; o >>= 1) {
      dw[j].a += __shfl_xor_sync(0xffffffffu, dw[j].a, o);
      dw[j].b += __shfl_xor_sync(0xffffffffu, dw[j].b, o);
    }
    if (lane < LANES && used) {
      const int at = (j < 4 ? 0 : half) + c + 2 * (j & 3);
      part[warp][at] = dw[j].a;
      part[warp][at + 1] = dw[j].b;
    }
  }
  __syncthreads();
  for (int j = tid; j < a.d; j += 256) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < 8; ++v) s += part[v][j];
    a.partial[size_t(blockIdx.x) * a.d + j] = s;
  }
}

// slot[j] += sum of partial[row][j] over a kind's rows, in a fixed order: 32 columns per CTA, its warps over the rows.
template <typename GT>
__global__ void __launch_bounds__(1024) qk_norm_weight_grad_kernel(const float* partial, GT* gwq, GT* gwk, int ctas_q, int ctas, int d) {
  chain_trigger();
  chain_wait();
  __shared__ float part[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = (d + 31) / 32, kind = int(blockIdx.x) >= per;
  const int col = (blockIdx.x - kind * per) * 32 + lane, end = kind ? ctas : ctas_q;
  GT* slot = (kind ? gwk : gwq) + col;
  float s = 0.f, old = 0.f;
  if (col < d) {
    if (warp == 0) old = float(*slot);
    for (int r = (kind ? ctas_q : 0) + warp; r < end; r += 8 * 32) {
      float v[8];                        // (all asked for before the first is added)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = r + 32 * i < end ? partial[size_t(r + 32 * i) * d + col] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || col >= d) return;
#pragma unroll
  for (int v = 1; v < 32; ++v) s += part[v][lane];
  *slot = GT(old + s);
}

static int qk_norm_lanes(int d) {
  int n = 1;
  while (n * 16 < d) n *= 2;
  return n;
}
// Units to a warp's item: as many of a token's as leave `warps` warps with work, so that its angles are loaded and multiplied
// out for many heads, but not for so many that the last items run alone.
static int qk_norm_span(long T, int units, long warps, int most) {
  const long s = T * units / warps;
  return int(s < 1 ? 1 : s > most ? most : s);
}
// CTAs of the backward pass for either kind of head: a unit for every warp, but no more than are on the GPU at once.  Those are dealt
// out by the work on a token: its units, and its angles and place, which take as long as one more.  (One kind behind the other on all
// CTAs: 256 tokens of 8 + 8 heads of 64 6.0 us instead of 4.6, 8192 of 32 + 8 heads of 128 46.7 instead of 46.1.)
static void qk_norm_bwd_ctas(int T, int nq, int nk, int d, int* of_q, int* of_all) {
  const int per = 32 / qk_norm_lanes(d), side_q = qk_norm_side(nq, per), side_k = qk_norm_side(nk, per);
  const long uq = (nq + per - 1) / per, uk = (nk + per - 1) / per, cap = long(num_sms()) * 2;
  long q = ((T + side_q - 1) / side_q * uq + 7) / 8, k = ((T + side_k - 1) / side_k * uk + 7) / 8;
  if (q + k > cap) {
    const long of_token_q = (uq + 1) * side_k, of_token_k = (uk + 1) * side_q;
    q = q == 0 ? 0 : k == 0 ? cap : cap * of_token_q / (of_token_q + of_token_k);
    q = uq > 0 && q < 1 ? 1 : uk > 0 && q > cap - 1 ? cap - 1 : q;
    k = cap - q;
  }
  *of_q = int(q);
  *of_all = int(q + k);
}

// What has to hold before anything is counted in heads: the lanes and units of other widths mean nothing.
static int qk_norm_heads_check(int nq, int nk, int d) {
  if (d % 16 != 0 || d < 16 || d > 512) ZB_FAIL(-1, "qk_norm_rope: head width %d is not a multiple of 16 up to 512", d);
  if (nq < 0 || nk < 0) ZB_FAIL(-1, "qk_norm_rope: %d + %d heads", nq, nk);
  return 0;
}
static int qk_norm_check(const QkNormArgs& a) {
  if (int rc = qk_norm_heads_check(a.nq, a.nk, a.d)) return rc;
  if (a.S < 1) ZB_FAIL(-1, "qk_norm_rope: sequences of %d", a.S);
  // a token's elements, and the heads that a warp's last item counts up to behind them (six units of 32 at most), in 32 bits
  const long heads = long(a.nq) + a.nk + a.nv;
  if ((heads + 192) * a.d >= 1L << 31) ZB_FAIL(-1, "qk_norm_rope: rows of %ld heads of %d", heads, a.d);
  // units of all tokens, and what a warp of the last CTA counts up to behind them, in 32 bits
  if (a.T * (heads + 3) >= (1L << 31) - (1L << 20)) ZB_FAIL(-1, "qk_norm_rope: %d tokens of %d heads", a.T, a.nq + a.nk);
  if (a.T > 1 && a.ldy < heads * a.d) ZB_FAIL(-1, "qk_norm_rope: rows to write lie over one another (stride %ld)", a.ldy);
  if (a.ldx % 8 != 0 || a.ldy % 8 != 0) ZB_FAIL(-1, "qk_norm_rope: row strides %ld, %ld not a multiple of 8", a.ldx, a.ldy);
  if ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.wq) |
       reinterpret_cast<uintptr_t>(a.wk) | reinterpret_cast<uintptr_t>(a.cs)) & 15)
    ZB_FAIL(-1, "qk_norm_rope: operands must be 16-byte aligned");
  return 0;
}

template <int LANES>
static int qk_norm_fwd_launch(const QkNormArgs& a, int grid, cudaStream_t stream) {
  auto kern = qk_norm_rope_fwd_kernel<LANES, true>;
  if (a.cs == nullptr) kern = qk_norm_rope_fwd_kernel<LANES, false>;
  ZB_CUDA_OK(launch_pass(kern, grid, 128, 0, stream, a));
  return 0;
}
template <int LANES>
static int qk_norm_bwd_launch(const QkNormArgs& a, int grid, cudaStream_t stream) {
  auto kern = qk_norm_rope_bwd_kernel<LANES, true>;
  if (a.cs == nullptr) kern = qk_norm_rope_bwd_kernel<LANES, false>;
  static SharedLimit limit[2];
  ZB_CUDA_OK(limit[a.cs == nullptr].raise(kern, sizeof(QkRing)));
  ZB_CUDA_OK(launch_pass(kern, grid, 256, sizeof(QkRing), stream, a));
  return 0;
}

}  // namespace zb

extern "C" {

int zb_qk_norm_rope_fwd(const void* x, void* y, const void* wq, const void* wk, const float* cs, float* rstd, int T, int S, int nq,
                        int nk, int nv, int d, long ldx, long ldy, float eps, cudaStream_t stream) {
  using namespace zb;
  QkNormArgs a = {};
  a.x = static_cast<const __nv_bfloat16*>(x); a.y = static_cast<__nv_bfloat16*>(y);
  a.wq = static_cast<const __nv_bfloat16*>(wq); a.wk = static_cast<const __nv_bfloat16*>(wk);
  a.cs = cs; a.rstd = rstd; a.ldx = ldx; a.ldy = ldy;
  a.T = T; a.S = S; a.nq = nq; a.nk = nk; a.nv = nv; a.d = d; a.eps = eps; a.inv_d = 1.f / d;
  if (int rc = qk_norm_check(a)) return rc;
  const int per = 32 / qk_norm_lanes(d), units = (nq + nk + nv + per - 1) / per;
  if (T <= 0 || units == 0) return 0;
  // (the warps that are on the GPU at once; for twice as many, 4094 tokens of 40 heads of 64 in place took 9.4 us instead of 8.3)
  a.span = qk_norm_span(T, units, long(num_sms()) * 24, 6);
  const int grid = int((long(T) * ((units + a.span - 1) / a.span) + 3) / 4);
  switch (qk_norm_lanes(d)) {
    case 1: return qk_norm_fwd_launch<1>(a, grid, stream);
    case 2: return qk_norm_fwd_launch<2>(a, grid, stream);
    case 4: return qk_norm_fwd_launch<4>(a, grid, stream);
    case 8: return qk_norm_fwd_launch<8>(a, grid, stream);
    case 16: return qk_norm_fwd_launch<16>(a, grid, stream);
    default: return qk_norm_fwd_launch<32>(a, grid, stream);
  }
}

// *floats: what zb_qk_norm_rope_bwd wants as workspace
int zb_qk_norm_rope_workspace(int T, int nq, int nk, int d, long* floats) {
  using namespace zb;
  int of_q = 0, ctas = 0;
  if (int rc = qk_norm_heads_check(nq, nk, d)) return rc;
  if (T > 0) qk_norm_bwd_ctas(T, nq, nk, d, &of_q, &ctas);
  *floats = long(ctas) * d;
  return 0;
}

int zb_qk_norm_rope_bwd(void* dy, const void* x, const void* wq, const void* wk, float* rstd, const float* cs, float* partial,
                        void* gwq, void* gwk, int T, int S, int nq, int nk, int d, long ldx, long ldy, int grad_f32,
                        cudaStream_t stream) {
  using namespace zb;
  QkNormArgs a = {};
  a.x = static_cast<const __nv_bfloat16*>(x); a.y = static_cast<__nv_bfloat16*>(dy);
  a.wq = static_cast<const __nv_bfloat16*>(wq); a.wk = static_cast<const __nv_bfloat16*>(wk);
  a.cs = cs; a.rstd = rstd; a.partial = partial; a.ldx = ldx; a.ldy = ldy;
  a.T = T; a.S = S; a.nq = nq; a.nk = nk; a.d = d; a.inv_d = 1.f / d;
  if (int rc = qk_norm_check(a)) return rc;
  if (T <= 0 || nq + nk == 0) return 0;
  int grid = 0;
  qk_norm_bwd_ctas(T, nq, nk, d, &a.ctas_q, &grid);
  int rc;
  switch (qk_norm_lanes(d)) {
    case 1: rc = qk_norm_bwd_launch<1>(a, grid, stream); break;
    case 2: rc = qk_norm_bwd_launch<2>(a, grid, stream); break;
    case 4: rc = qk_norm_bwd_launch<4>(a, grid, stream); break;
    case 8: rc = qk_norm_bwd_launch<8>(a, grid, stream); break;
    case 16: rc = qk_norm_bwd_launch<16>(a, grid, stream); break;
    default: rc = qk_norm_bwd_launch<32>(a, grid, stream); break;
  }
  if (rc) return rc;
  const int columns = 2 * ((d + 31) / 32);
  if (grad_f32)
    ZB_CUDA_OK(launch_pass(qk_norm_weight_grad_kernel<float>, columns, 1024, 0, stream, partial, static_cast<float*>(gwq),
                           static_cast<float*>(gwk), a.ctas_q, grid, d));
  else
    ZB_CUDA_OK(launch_pass(qk_norm_weight_grad_kernel<__nv_bfloat16>, columns, 1024, 0, stream, partial,
                           static_cast<__nv_bfloat16*>(gwq), static_cast<__nv_bfloat16*>(gwk), a.ctas_q, grid, d));
  return 0;
}

}  // extern "C"
