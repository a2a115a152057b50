// RMS norm of every query and key head with the rotate-half rotation in the same pass, forward and backward, on the packed
// projection [T, (Hq + 2 Hkv) d] (query heads, key heads, value heads).  With x one head of one token, w the weights of its kind
// (wq or wk, [d], shared by the heads) and R the rotation by the angles of position t mod S:
//   forward   rstd = 1 / sqrt(mean(x^2) + eps),  y = R(x rstd w)
//   backward  g = R^T dy,  xh = x rstd,  dx = rstd (w g - xh mean(w g xh)),  dw += sum over tokens and heads of g xh
// Sums and products are in fp32 and a value is rounded to bf16 once, at the end: as two passes the normalised heads would be
// rounded in between.
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
  float* partial;           // backward: [CTAs, 2, d]
  long ldx, ldy;
  int T, S, nq, nk, nv, d;  // nv: value heads to copy (forward into another tensor), else 0
  float eps;
};

// Sixteen values of a head per lane: eight from either half, so that a lane has both members of its pairs.
struct HeadChunk {
  uint4 lo, hi;
};
__device__ __forceinline__ void unpack16(const HeadChunk& h, float (&f)[16]) {
  unpack8(h.lo, f);
  unpack8(h.hi, f + 8);
}
__device__ __forceinline__ HeadChunk pack16(const float (&f)[16]) { return {pack8(f), pack8(f + 8)}; }
__device__ __forceinline__ HeadChunk load_head(const __nv_bfloat16* p, int half) { return {ld_v4(p), ld_v4(p + half)}; }
__device__ __forceinline__ void store_head(__nv_bfloat16* p, int half, const HeadChunk& h) {
  *reinterpret_cast<uint4*>(p) = h.lo;
  *reinterpret_cast<uint4*>(p + half) = h.hi;
}
// f becomes R f (sign 1) or R^T f (sign -1); row: the cosines of the position
__device__ __forceinline__ void rotate16(float (&f)[16], const float* row, int c, int half, float sign) {
#pragma unroll
  for (int k = 0; k < 8; k += 4) {
    const float4 co = *reinterpret_cast<const float4*>(row + c + k), si = *reinterpret_cast<const float4*>(row + half + c + k);
    const float cc[4] = {co.x, co.y, co.z, co.w}, ss[4] = {si.x, si.y, si.z, si.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = f[k + j], b = f[8 + k + j], s = ss[j] * sign;
      f[k + j] = a * cc[j] - b * s;
      f[8 + k + j] = b * cc[j] + a * s;
    }
  }
}
template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// LANES lanes share a head (a power of two, at least d / 16: for d = 96 two of eight idle); a warp takes 32 / LANES heads of a token.
template <int LANES>
__global__ void __launch_bounds__(256) qk_norm_rope_fwd_kernel(const QkNormArgs a) {
  chain_trigger();
  chain_wait();
  constexpr int HEADS = 32 / LANES;
  const int half = a.d >> 1, lane = threadIdx.x & 31, c = (lane % LANES) * 8;
  const bool used = c < half;
  const int nqk = a.nq + a.nk, heads = nqk + a.nv, groups = (heads + HEADS - 1) / HEADS;
  const long items = long(a.T) * groups;
  for (long i = blockIdx.x * 8L + (threadIdx.x >> 5); i < items; i += gridDim.x * 8L) {
    const int t = int(i / groups), h = int(i - long(t) * groups) * HEADS + lane / LANES;
    const bool live = used && h < heads;
    const size_t col = size_t(h) * a.d + c;
    HeadChunk u = {};
    if (live) u = load_head(a.x + t * a.ldx + col, half);
    float f[16], ss = 0.f;
    unpack16(u, f);
#pragma unroll
    for (int j = 0; j < 16; ++j) ss += f[j] * f[j];
    const float rstd = rsqrtf(head_sum<LANES>(ss) / a.d + a.eps);
    if (!live) continue;
    if (h < nqk) {
      const HeadChunk wu = load_head((h < a.nq ? a.wq : a.wk) + c, half);
      float w[16];
      unpack16(wu, w);
#pragma unroll
      for (int j = 0; j < 16; ++j) f[j] *= rstd * w[j];
      if (a.cs != nullptr) rotate16(f, a.cs + size_t(t % a.S) * a.d, c, half, 1.f);
      u = pack16(f);
      if (a.rstd != nullptr && c == 0) a.rstd[long(t) * nqk + h] = rstd;
    }
    store_head(a.y + t * a.ldy + col, half, u);
  }
}

template <int LANES>
__global__ void __launch_bounds__(256) qk_norm_rope_bwd_kernel(const QkNormArgs a) {
  chain_trigger();
  chain_wait();
  constexpr int HEADS = 32 / LANES;
  __shared__ float part[8][LANES * 16];
  const int half = a.d >> 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = (lane % LANES) * 8;
  const bool used = c < half;
  for (int kind = 0; kind < 2; ++kind) {          // query heads, then key heads: one set of weight-gradient sums at a time
    const int n = kind ? a.nk : a.nq, h0 = kind ? a.nq : 0, groups = (n + HEADS - 1) / HEADS;
    float w[16], dw[16];
    HeadChunk wu = {};
    if (used) wu = load_head((kind ? a.wk : a.wq) + c, half);
    unpack16(wu, w);
#pragma unroll
    for (int j = 0; j < 16; ++j) dw[j] = 0.f;
    const long items = long(a.T) * groups;
    for (long i = blockIdx.x * 8L + warp; i < items; i += gridDim.x * 8L) {
      const int t = int(i / groups), k = int(i - long(t) * groups) * HEADS + lane / LANES, h = h0 + k;
      const bool live = used && k < n;
      const size_t col = size_t(h) * a.d + c;
      HeadChunk xu = {}, gu = {};
      float rstd = 0.f;
      if (live) {
        xu = load_head(a.x + t * a.ldx + col, half);
        gu = load_head(a.y + t * a.ldy + col, half);
        rstd = a.rstd[long(t) * (a.nq + a.nk) + h];
      }
      float x[16], g[16], along = 0.f;
      unpack16(xu, x);
      unpack16(gu, g);
      if (a.cs != nullptr && live) rotate16(g, a.cs + size_t(t % a.S) * a.d, c, half, -1.f);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        x[j] *= rstd;
        dw[j] += g[j] * x[j];
        g[j] *= w[j];
        along += g[j] * x[j];
      }
      along = head_sum<LANES>(along) / a.d;
#pragma unroll
      for (int j = 0; j < 16; ++j) g[j] = rstd * (g[j] - x[j] * along);
      if (live) store_head(a.y + t * a.ldy + col, half, pack16(g));
    }
    // over the heads of a warp, then over its CTA's warps
#pragma unroll
    for (int j = 0; j < 16; ++j) {
#pragma unroll
      for (int o = 16; o >= LANES; o >>= 1) dw[j] += __shfl_xor_sync(0xffffffffu, dw[j], o);
    }
    __syncthreads();
    if (lane < LANES && used) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        part[warp][c + j] = dw[j];
        part[warp][half + c + j] = dw[8 + j];
      }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < a.d; j += 256) {
      float s = 0.f;
#pragma unroll
      for (int v = 0; v < 8; ++v) s += part[v][j];
      a.partial[(size_t(blockIdx.x) * 2 + kind) * a.d + j] = s;
    }
  }
}

// slot[j] += sum over `rows` of partial[row][j], in a fixed order: 32 columns per CTA, eight warps over the rows.
template <typename GT>
__global__ void __launch_bounds__(256) qk_norm_weight_grad_kernel(const float* partial, GT* gwq, GT* gwk, int rows, int d) {
  chain_trigger();
  chain_wait();
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < 2 * d)
    for (int r = warp; r < rows; r += 8) s += partial[size_t(r) * 2 * d + col];
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || col >= 2 * d) return;
#pragma unroll
  for (int v = 1; v < 8; ++v) s += part[v][lane];
  GT* slot = col < d ? gwq + col : gwk + (col - d);
  *slot = GT(float(*slot) + s);
}

static int qk_norm_lanes(int d) {
  int n = 1;
  while (n * 16 < d) n *= 2;
  return n;
}
static int qk_norm_bwd_ctas(int T, int nq, int nk, int d) {
  const int per = 32 / qk_norm_lanes(d), most = nq > nk ? nq : nk;
  const long want = (long(T) * ((most + per - 1) / per) + 7) / 8, cap = long(num_sms()) * 3;
  return int(want < cap ? want : cap);
}

static int qk_norm_check(const QkNormArgs& a) {
  if (a.d % 16 != 0 || a.d < 16 || a.d > 512) ZB_FAIL(-1, "qk_norm_rope: head width %d is not a multiple of 16 up to 512", a.d);
  if (a.nq < 0 || a.nk < 0 || a.nv < 0 || a.S < 1) ZB_FAIL(-1, "qk_norm_rope: %d + %d heads, sequences of %d", a.nq, a.nk, a.S);
  if (a.ldx % 8 != 0 || a.ldy % 8 != 0) ZB_FAIL(-1, "qk_norm_rope: row strides %ld, %ld not a multiple of 8", a.ldx, a.ldy);
  if ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.wq) |
       reinterpret_cast<uintptr_t>(a.wk) | reinterpret_cast<uintptr_t>(a.cs)) & 15)
    ZB_FAIL(-1, "qk_norm_rope: operands must be 16-byte aligned");
  return 0;
}

#define QK_NORM_LAUNCH(KERNEL, GRID)                                                                        \
  switch (qk_norm_lanes(a.d)) {                                                                             \
    case 1: ZB_CUDA_OK(launch_pass(KERNEL<1>, GRID, 256, 0, stream, a)); break;                             \
    case 2: ZB_CUDA_OK(launch_pass(KERNEL<2>, GRID, 256, 0, stream, a)); break;                             \
    case 4: ZB_CUDA_OK(launch_pass(KERNEL<4>, GRID, 256, 0, stream, a)); break;                             \
    case 8: ZB_CUDA_OK(launch_pass(KERNEL<8>, GRID, 256, 0, stream, a)); break;                             \
    case 16: ZB_CUDA_OK(launch_pass(KERNEL<16>, GRID, 256, 0, stream, a)); break;                           \
    default: ZB_CUDA_OK(launch_pass(KERNEL<32>, GRID, 256, 0, stream, a)); break;                           \
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
  a.T = T; a.S = S; a.nq = nq; a.nk = nk; a.nv = nv; a.d = d; a.eps = eps;
  if (int rc = qk_norm_check(a)) return rc;
  const int per = 32 / qk_norm_lanes(d);
  const long items = long(T) * ((nq + nk + nv + per - 1) / per);
  if (items <= 0) return 0;
  const long ctas = (items + 7) / 8, cap = long(num_sms()) * 16;
  const int grid = int(ctas < cap ? ctas : cap);
  QK_NORM_LAUNCH(qk_norm_rope_fwd_kernel, grid)
  return 0;
}

// *floats: what zb_qk_norm_rope_bwd wants as workspace
int zb_qk_norm_rope_workspace(int T, int nq, int nk, int d, long* floats) {
  using namespace zb;
  *floats = d > 0 && T > 0 ? 2L * d * qk_norm_bwd_ctas(T, nq, nk, d) : 0;
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
  a.T = T; a.S = S; a.nq = nq; a.nk = nk; a.d = d;
  if (int rc = qk_norm_check(a)) return rc;
  if (T <= 0 || nq + nk == 0) return 0;
  const int grid = qk_norm_bwd_ctas(T, nq, nk, d);
  QK_NORM_LAUNCH(qk_norm_rope_bwd_kernel, grid)
  const int columns = (2 * d + 31) / 32;
  if (grad_f32)
    ZB_CUDA_OK(launch_pass(qk_norm_weight_grad_kernel<float>, columns, 256, 0, stream, partial, static_cast<float*>(gwq),
                           static_cast<float*>(gwk), grid, d));
  else
    ZB_CUDA_OK(launch_pass(qk_norm_weight_grad_kernel<__nv_bfloat16>, columns, 256, 0, stream, partial,
                           static_cast<__nv_bfloat16*>(gwq), static_cast<__nv_bfloat16*>(gwk), grid, d));
  return 0;
}

}  // extern "C"
