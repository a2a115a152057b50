// Updates orthogonalised by Newton-Schulz products, over a list of matrices.
//
// U (n x m, n <= m; a matrix with more rows than columns is taken transposed) becomes X = U / ||U||_F and then, five times,
//     A = X X^T,   B = b A + c A A,   X <- a X + B X
// an odd polynomial of the singular values that drives them all towards 1 without an SVD.  Three products an iteration; A and A A
// are symmetric, so only their tiles on and above the diagonal are formed and every other one is stored a second time, turned
// over: down to 3 n^2 m + n^3 floating-point operations instead of 4 n^2 m + 2 n^3.  (Tiles on the diagonal are formed whole: of t x t tiles, t = n / 256
// rounded up, t (t + 1) / 2 are formed, all of them for n of up to 256.)
//
// Every matrix of the list takes part in each launch: those of one shape lie one behind the other in the workspace under one tensor
// map, and the tiles of up to GROUPS shapes are dealt to persistent CTA pairs.  A model's matrices of 512 to 1024 columns have 3 to 10
// tiles each, one by one a launch would leave most of the GPU idle.
//
// Operands are fp16, sums fp32 in tensor memory.  All values are bounded (singular values stay below 1.21), so the range of bf16 is
// not needed and its eight bits would cost: relative error of X after five iterations 1.0e-2 with bf16 and 1.0e-3 with fp16 (noise of 512 x
// 512 to 1024 x 1024).  What rounding leaves where a matrix has nothing is a singular value like others and grows by a = 3.4 an iteration, 485 times in
// five, so X itself has to be held more exactly than the products read it: eight more bits of it go from product to product beside it
// (ns_remainders) in all iterations but the last two, into a X alone, since B takes nothing from where X has nothing.  Relative errors (1024 x 1024)
// without them and with them: rank 1 0.15 and 3.0e-3, 16 0.045 and 2.7e-3, 64 0.024 and 2.6e-3, 256 8.6e-3 and 2.3e-3; singular values as
// 1 / k 3.7e-3 and 7e-4, 1 / k^2 0.021 and 1.4e-3; noise 1.0e-3 either way (of a handful of entries, 2 x 2 to 3 x 5, 2e-3 on average and up to 1e-2).  They cost 3 to 8 % (24 blocks of 1024 6600 -> 6830 us, 16 matrices
// of 512 199 -> 214); more bits of the last two iterations' X would take 1e-3 off ranks below 64.  X is held times 2^round(log2(sqrt m)), so its entries are near 1 at the end,
// A and B times 64, so that what the first iteration's small values round to stays far below what they add.
//
// Around the products: one pass over gradient and momentum with the sum of squares, one that scales, turns and rounds into the
// workspace, and one that applies the result (momentum and scale come from fp32, sums of squares are held in 64 bits: no normal number of fp32 is too
// small or too large for them; below those, 1.2e-38, values count as zeros).
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "newton_schulz.cuh"
#include <algorithm>
#include <cmath>
#include <exception>
#include <vector>

namespace zb {

constexpr float NS_A_SCALE = 64.f;   // what is n x n is held times this

// --------------------------------------------------------------------------------------------- passes before and behind
constexpr int NS_MATRICES = 64;      // of a launch of a pass
constexpr int NS_PARTS = 256;        // sums of squares of one matrix, at most

// What a caller hands over for each matrix.
struct NsMatrix {
  float* p;               // muon: fp32, rows x cols; else null
  float* m;               // muon: momentum
  const void* g;          // gradient (muon), or the matrix
  __nv_bfloat16* out;     // muon: p's copy in bf16, or null; else the result
  long rows, cols;
  int g_f32, unused;
};

struct NsPassMatrix {
  float* p;
  float* m;
  const void* g;
  __nv_bfloat16* out;
  __half* x;              // first the scaled matrix, at the end the result: [n, ld]
  uint8_t* rem;           // remainders of the scaled matrix, or null
  double* sums;           // [parts]
  long ld;
  int rem_cols;
  int rows, cols, parts, tiles_c, first;   // first: of the blocks of a launch
  int g_f32, wide;        // wide: rows start on 16 bytes in every type
  float scale, step;      // X is held times scale; muon: what the result is multiplied with
};
struct NsPass {
  NsPassMatrix t[NS_MATRICES];
  int count;
  float momentum, grad_scale, keep;
  int nesterov, muon;
  int span;               // tiles of a block that scales
};

__device__ __forceinline__ int ns_find(const NsPass& a, int block) {
  int lo = 0, hi = a.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.t[mid].first <= block) lo = mid; else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ float4 ns_load4(const void* base, bool f32, size_t at) {
  if (f32) {
    const uint4 v = ld_v4(static_cast<const float*>(base) + at);
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
  }
  const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + at);
  const float2 a = unpack_bf16x2(v.x), b = unpack_bf16x2(v.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float ns_load1(const void* base, bool f32, size_t at) {
  return f32 ? static_cast<const float*>(base)[at] : __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at]);
}
// The update from the scaled gradient and the new momentum.
__device__ __forceinline__ float ns_update(const NsPass& a, float g, float m) { return a.nesterov ? fmaf(a.momentum, m, g) : m; }

// Momentum (written back) and the sum of squares of the update; a block has an equal part of its matrix's elements.
__global__ void __launch_bounds__(256) ns_sums_kernel(const __grid_constant__ NsPass a) {
  chain_trigger();
  chain_wait();
  const NsPassMatrix& t = a.t[ns_find(a, blockIdx.x)];
  const int part = int(blockIdx.x) - t.first;
  const size_t n = size_t(t.rows) * t.cols, each = ((n + t.parts - 1) / t.parts + 3) / 4 * 4;
  const size_t lo = each * part, hi = lo + each < n ? lo + each : n;
  double sum = 0.0;
  auto one = [&](size_t i) {
    float u = ns_load1(t.g, t.g_f32, i);
    if (a.muon) {
      const float g = u * a.grad_scale, m = fmaf(a.momentum, t.m[i], g);
      t.m[i] = m;
      u = ns_update(a, g, m);
    }
    sum += double(u) * double(u);
  };
  if (t.wide) {
    constexpr int U = 4;     // loads in flight
    const size_t whole = lo < hi ? lo + (hi - lo) / 4 * 4 : lo;
    for (size_t i = lo + threadIdx.x * 4; i < whole; i += 256 * 4 * U) {
      float4 g[U], m[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (i + k * 1024 < whole) {
          g[k] = ns_load4(t.g, t.g_f32, i + k * 1024);
          if (a.muon) m[k] = ns_load4(t.m, true, i + k * 1024);
        }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (i + k * 1024 < whole) {
          float u[4] = {g[k].x, g[k].y, g[k].z, g[k].w};
          if (a.muon) {
            float w[4] = {m[k].x, m[k].y, m[k].z, m[k].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float x = u[j] * a.grad_scale;
              w[j] = fmaf(a.momentum, w[j], x);
              u[j] = ns_update(a, x, w[j]);
            }
            *reinterpret_cast<float4*>(t.m + i + k * 1024) = make_float4(w[0], w[1], w[2], w[3]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) sum += double(u[j]) * double(u[j]);
        }
    }
    if (whole + threadIdx.x < hi) one(whole + threadIdx.x);
  } else {
    for (size_t i = lo + threadIdx.x; i < hi; i += 256) one(i);
  }
  __shared__ double part_sums[8];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if ((threadIdx.x & 31) == 0) part_sums[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += part_sums[i];
    t.sums[part] = s;
  }
}

// Tiles of 64 x 64, `span` a block: the update times scale / norm in fp16, turned over where the matrix has more rows than columns.  All of a
// tile's loads are asked for before the first is used, and a block finds its matrix and factor once for up to four tiles: 101 million
// elements of 48 matrices (bf16 gradients, 8 bytes an element in all) 227 -> 175 us (198 with one tile a block).  With the remainders, 9 bytes an
// element, 203 (207 with five blocks an SM instead of six, which spares the 130 bytes that spill, and 228 with four).
__global__ void __launch_bounds__(256, 6) ns_scale_kernel(const __grid_constant__ NsPass a) {
  chain_trigger();
  chain_wait();
  const NsPassMatrix& t = a.t[ns_find(a, blockIdx.x)];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  __shared__ float tile_s[64][65];
  const bool turned = t.rows > t.cols;
  double s = 0.0;      // every warp adds the parts up for itself
#pragma unroll
  for (int i = 0; i < NS_PARTS; i += 32)
    if (i + int(threadIdx.x & 31) < t.parts) s += t.sums[i + (threadIdx.x & 31)];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  // scale / norm as a power of two and the rest, either of which fp32 holds for any norm; NaN and infinite norms give NaN
  int e = 0;
  const double by = s == 0.0 ? 0.0 : double(t.scale) / sqrt(s);
  const float low = float(frexp(by, &e) * 2.0);
  const float half = exp2f(float((e - 1) / 2)), rest = exp2f(float(e - 1 - (e - 1) / 2)) * low;
  auto put = [&](int r, int c, float2 x01, float2 x23) {     // of X
    const uint2 h = make_uint2(pack_half2(x01.x, x01.y), pack_half2(x23.x, x23.y));
    *reinterpret_cast<uint2*>(t.x + size_t(r) * t.ld + c) = h;
    if (t.rem != nullptr)
      *reinterpret_cast<uint32_t*>(t.rem + ns_rem_at(size_t(r >> 5) * t.rem_cols + (c >> 6), r, c)) = ns_remainders(x01, x23, h.x, h.y);
  };
  const int tiles = (t.rows + 63) / 64 * t.tiles_c, first = (int(blockIdx.x) - t.first) * a.span;
#pragma unroll 1
  for (int tile = first; tile < min(first + a.span, tiles); ++tile) {
    const int r0 = tile / t.tiles_c * 64, c0 = tile % t.tiles_c * 64, c = c0 + tx * 4;
    float u[4][4], m[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = r0 + ty + 16 * k;
      const size_t at = size_t(r) * t.cols + c;
#pragma unroll
      for (int j = 0; j < 4; ++j) u[k][j] = m[k][j] = 0.f;
      if (t.wide) {
        if (r < t.rows && c < t.cols) {
          const float4 g = ns_load4(t.g, t.g_f32, at);
          u[k][0] = g.x; u[k][1] = g.y; u[k][2] = g.z; u[k][3] = g.w;
          if (a.muon) *reinterpret_cast<float4*>(m[k]) = ns_load4(t.m, true, at);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r < t.rows && c + j < t.cols) {
            u[k][j] = ns_load1(t.g, t.g_f32, at + j);
            if (a.muon) m[k][j] = t.m[at + j];
          }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = r0 + ty + 16 * k;
#pragma unroll
      for (int j = 0; j < 4; ++j) u[k][j] = (a.muon ? ns_update(a, u[k][j] * a.grad_scale, m[k][j]) : u[k][j]) * half * rest;
      if (turned) {
#pragma unroll
        for (int j = 0; j < 4; ++j) tile_s[ty + 16 * k][tx * 4 + j] = u[k][j];
      } else if (r < t.rows && c < t.cols) {      // (rows of the workspace are padded to 64)
        put(r, c, make_float2(u[k][0], u[k][1]), make_float2(u[k][2], u[k][3]));
      }
    }
    if (!turned) continue;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int cc = c0 + ty + 16 * k, r = r0 + tx * 4;
      if (cc < t.cols && r < t.rows)
        put(cc, r, make_float2(tile_s[tx * 4][ty + 16 * k], tile_s[tx * 4 + 1][ty + 16 * k]),
            make_float2(tile_s[tx * 4 + 2][ty + 16 * k], tile_s[tx * 4 + 3][ty + 16 * k]));
    }
    __syncthreads();
  }
}

// Tiles of 64 x 64: the result in bf16, or the step of the parameters.
__global__ void __launch_bounds__(256) ns_apply_kernel(const __grid_constant__ NsPass a) {
  chain_trigger();
  chain_wait();
  const NsPassMatrix& t = a.t[ns_find(a, blockIdx.x)];
  const int tile = int(blockIdx.x) - t.first, r0 = tile / t.tiles_c * 64, c0 = tile % t.tiles_c * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, c = c0 + tx * 4;
  const bool turned = t.rows > t.cols;
  __shared__ float tile_s[64][65];
  float4 old[4];
  uint2 x[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + ty + 16 * k, xr = turned ? c0 + ty + 16 * k : r, xc = turned ? r0 + tx * 4 : c;
    x[k] = make_uint2(0u, 0u);
    if (xr < (turned ? t.cols : t.rows) && xc < (turned ? t.rows : t.cols)) x[k] = *reinterpret_cast<const uint2*>(t.x + size_t(xr) * t.ld + xc);
    if (a.muon && t.wide && r < t.rows && c < t.cols) old[k] = ns_load4(t.p, true, size_t(r) * t.cols + c);
  }
  if (turned) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 lo = unpack_half2(x[k].x), hi = unpack_half2(x[k].y);
      float* to = &tile_s[ty + 16 * k][tx * 4];
      to[0] = lo.x; to[1] = lo.y; to[2] = hi.x; to[3] = hi.y;
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + ty + 16 * k;
    float v[4];
    if (turned) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = tile_s[tx * 4 + j][ty + 16 * k];
    } else {
      const float2 lo = unpack_half2(x[k].x), hi = unpack_half2(x[k].y);
      v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
    }
    if (r >= t.rows) continue;
    const size_t at = size_t(r) * t.cols + c;
    const float w[4] = {old[k].x, old[k].y, old[k].z, old[k].w};
    const bool four = t.wide && c < t.cols;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] *= t.step;
      if (a.muon && c + j < t.cols) v[j] = fmaf(four ? w[j] : t.p[at + j], a.keep, -v[j]);
    }
    if (four) {
      if (a.muon) *reinterpret_cast<float4*>(t.p + at) = make_float4(v[0], v[1], v[2], v[3]);
      if (t.out != nullptr) *reinterpret_cast<uint2*>(t.out + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < t.cols) {
          if (a.muon) t.p[at + j] = v[j];
          if (t.out != nullptr) t.out[at + j] = __float2bfloat16(v[j]);
        }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ the list
enum : int { NS_X0 = 0, NS_X1 = 1, NS_A = 2, NS_B = 3, NS_BUFFERS = 4 };   // X in turns, and what is n x n

struct NsShape {
  long n, m;                       // short and long side
  std::vector<int> members;        // of the list
  size_t at[NS_BUFFERS], rem;      // places in the workspace
  // Rows start on 128-byte lines, so that a row of a box is one line and not parts of two: lists of 3 x 1000 x 333 and 4097 x 641 and the
  // like 310 -> 265 us.
  long ld(int buffer) const { return ((buffer < NS_A ? m : n) + 63) / 64 * 64; }
  long cols(int buffer) const { return buffer < NS_A ? m : n; }
  long rem_rows() const { return (n + 31) / 32; }      // boxes of remainders of one matrix
  long rem_cols() const { return (m + 63) / 64; }
  size_t rem_bytes() const { return size_t(rem_rows()) * rem_cols() * NS_REM_BOX; }
};
struct NsPlan {
  std::vector<NsShape> shapes;     // long sides first
  std::vector<size_t> sums;        // of each matrix
  std::vector<int> parts;
  size_t bytes = 0;
};

static NsPlan ns_plan(const NsMatrix* t, int count) {
  NsPlan plan;
  auto take = [&](size_t n) {
    const size_t at = plan.bytes;
    plan.bytes += (n + 1023) / 1024 * 1024;
    return at;
  };
  for (int i = 0; i < count; ++i) {
    const long n = std::min(t[i].rows, t[i].cols), m = std::max(t[i].rows, t[i].cols);
    auto s = std::find_if(plan.shapes.begin(), plan.shapes.end(), [&](const NsShape& x) { return x.n == n && x.m == m; });
    if (s == plan.shapes.end()) s = plan.shapes.insert(s, NsShape{n, m, {}, {}, 0});
    s->members.push_back(i);
  }
  std::stable_sort(plan.shapes.begin(), plan.shapes.end(), [](const NsShape& a, const NsShape& b) { return a.m > b.m; });
  for (NsShape& s : plan.shapes) {
    for (int i = 0; i < NS_BUFFERS; ++i) s.at[i] = take(s.members.size() * s.n * s.ld(i) * 2);
    s.rem = take(s.members.size() * s.rem_bytes());
  }
  for (int i = 0; i < count; ++i) {
    const long parts = (t[i].rows * t[i].cols + 4095) / 4096;
    plan.parts.push_back(int(std::min<long>(parts, NS_PARTS)));
    plan.sums.push_back(take(size_t(plan.parts.back()) * 8));
  }
  return plan;
}

static float ns_scale(long m) { return exp2f(float(std::min(13l, std::lround(0.5 * std::log2(double(m)))))); }

// out = alpha P P^T + beta R + diag I (symmetric), or alpha P X + beta R + gamma (R + its remainder); numbers of buffers, add < 0: no R.
struct NsStep {
  bool symmetric;
  int p, q, add, out;
  float alpha, beta, diag, gamma;
  int remainders;         // 1: R's are read, 2: the result's are kept
};
// X of all iterations but the last two keeps what its rounding to fp16 leaves over (ns_remainders).
constexpr bool ns_keeps_remainder(int iteration, int iterations) { return iteration + 2 < iterations; }
// Launch by launch.  B goes with 2 I added and X with a - 2: once singular values are near 1, B is nearly -2.7 I, most of which a takes
// away again, rounding errors excepted.  (1.43e-3 -> 0.95e-3 for 512 x 1376 noise, 1.64e-3 -> 0.69e-3 for 8 x 600, never more.)  (Two iterations of long matrices taken as one, X2 = q(A1) q(A) X0 with A1 = q(A) A q(A), save 3 n^2 m - 3 n^3 operations,
// but q(A1) q(A) is 11.9 I less as much along a direction that holds most of a matrix: 1.4e-2 of a matrix of ones instead of 1e-4.)
static std::vector<NsStep> ns_program(int iterations, float a, float b, float c) {
  std::vector<NsStep> steps;
  for (int i = 0, x = NS_X0; i < iterations; ++i, x = 1 - x) {
    const bool more = ns_keeps_remainder(i, iterations);
    steps.push_back({true, x, x, -1, NS_A, 1.f, 0.f, 0.f, 0.f, 0});
    steps.push_back({true, NS_A, NS_A, NS_A, NS_B, c, b, 2.f, 0.f, 0});
    steps.push_back({false, NS_B, x, x, 1 - x, 1.f, more ? -2.f : a - 2.f, 0.f, more ? a : 0.f, more + 2 * ns_keeps_remainder(i + 1, iterations)});
  }
  return steps;
}

// The maps of a shape's buffers, made when first asked for: boxes of `rows` rows of 64 columns, or (rows 0) of 64 rows of 32.
struct NsMaps {
  CUtensorMap map[NS_BUFFERS][4];
  bool made[NS_BUFFERS][4] = {};
  int get(CUtensorMap* out, const NsShape& s, char* ws, int buffer, uint32_t rows) {
    const int i = rows == 128 ? 0 : rows == 64 ? 1 : rows == 32 ? 2 : 3;
    if (!made[buffer][i]) {
      const uint64_t dims[3] = {uint64_t(s.cols(buffer)), uint64_t(s.n), s.members.size()};
      const uint64_t strides[2] = {uint64_t(s.ld(buffer)) * 2, uint64_t(s.n * s.ld(buffer)) * 2};
      const uint32_t box[3] = {rows ? 64u : 32u, rows ? rows : 64u, 1};
      if (int rc = make_tmap_nd_bf16(&map[buffer][i], ws + s.at[buffer], 3, dims, strides, box,
                                     rows ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE))
        return rc;
      made[buffer][i] = true;
    }
    *out = map[buffer][i];
    return 0;
  }
};

static int ns_products(const NsPlan& plan, char* ws, const std::vector<NsStep>& program, int* status, cudaStream_t stream, int* launches) {
  std::vector<NsMaps> maps(plan.shapes.size());
  std::vector<size_t> order(plan.shapes.size());
  for (const NsStep& e : program) {
    for (size_t i = 0; i < order.size(); ++i) order[i] = i;
    // the longest reductions first: the last wave of a launch is then of short ones
    std::stable_sort(order.begin(), order.end(), [&](size_t i, size_t j) { return plan.shapes[i].cols(e.p) > plan.shapes[j].cols(e.p); });
    for (size_t first = 0; first < order.size(); first += NS_GROUPS) {
      NsParams p;
      p.status = status;
      p.groups = p.items = 0;
      for (size_t k = first; k < std::min(first + NS_GROUPS, order.size()); ++k) {
        const NsShape& s = plan.shapes[order[k]];
        NsMaps& m = maps[order[k]];
        NsGroup& g = p.g[p.groups++];
        int rc = m.get(&g.a, s, ws, e.p, 128);
        if (!rc) rc = m.get(&g.b, s, ws, e.q, e.symmetric ? 128 : 64);
        if (!rc) rc = m.get(&g.c, s, ws, e.out, 32);
        if (!rc) rc = m.get(&g.x, s, ws, e.add >= 0 ? e.add : e.out, 32);
        if (!rc && e.symmetric) rc = m.get(&g.t, s, ws, e.out, 0);
        if (rc) return rc;
        const float scale = ns_scale(s.m);
        g.symmetric = e.symmetric;
        g.M = int(s.n);
        g.N = int(s.cols(e.out));
        g.K = int(s.cols(e.p));
        g.alpha = e.alpha * (e.p < NS_A ? NS_A_SCALE / (scale * scale) : 1.f / NS_A_SCALE);
        g.beta = e.beta;
        g.diag = e.diag * NS_A_SCALE;
        g.gamma = e.gamma;
        g.remainders = e.remainders;
        g.rem = reinterpret_cast<uint8_t*>(ws + s.rem);
        g.rem_rows = int(s.rem_rows());
        g.rem_cols = int(s.rem_cols());
        g.tiles_m = (g.M + NsCfg::BM - 1) / NsCfg::BM;
        const long columns = (g.N + NsCfg::BN - 1) / NsCfg::BN, count = long(s.members.size());
        const long tiles = e.symmetric ? long(g.tiles_m) * (g.tiles_m + 1) / 2 : g.tiles_m * columns;
        if (p.items + tiles * count > 0x7fffffffL) ZB_FAIL(-1, "newton_schulz: %ld matrices of %ld x %ld", count, s.n, s.m);
        g.tiles = int(tiles);
        g.first = p.items;
        p.items += int(tiles * count);
      }
      p.stages = p.g[0].K >= NsCfg::LONG_K ? 6 : 5;
      if (int rc = ns_launch(p, stream)) return rc;
      ++*launches;
    }
  }
  return 0;
}

// One of the passes over all matrices; PASS 0: sums, 1: scale, 2: apply.
template <int PASS>
static int ns_pass(const NsPlan& plan, const NsMatrix* t, const NsPass& common, float step, char* ws, int x, bool remainders, cudaStream_t stream, int* launches) {
  NsPass a = common;
  a.count = 0;
  long all = 0;
  for (const NsShape& s : plan.shapes) all += long(s.members.size()) * ((s.n + 63) / 64) * ((s.m + 63) / 64);
  a.span = int(std::min(4l, std::max(1l, all / (2 * num_sms() * 6))));      // two rounds of blocks on all SMs at the least
  long blocks = 0;
  auto flush = [&]() -> int {
    if (a.count == 0) return 0;
    if (blocks > 0x7fffffffL) ZB_FAIL(-1, "newton_schulz: %ld blocks", blocks);
    const dim3 grid{unsigned(blocks)};
    if (PASS == 0) ZB_CUDA_OK(launch_pass(ns_sums_kernel, grid, 256, 0, stream, a));
    else if (PASS == 1) ZB_CUDA_OK(launch_pass(ns_scale_kernel, grid, 256, 0, stream, a));
    else ZB_CUDA_OK(launch_pass(ns_apply_kernel, grid, 256, 0, stream, a));
    ++*launches;
    a.count = 0;
    blocks = 0;
    return 0;
  };
  for (const NsShape& s : plan.shapes) {
    const float scale = ns_scale(s.m);
    for (size_t k = 0; k < s.members.size(); ++k) {
      const int i = s.members[k];
      NsPassMatrix& e = a.t[a.count++];
      e.p = t[i].p;
      e.m = t[i].m;
      e.g = t[i].g;
      e.out = t[i].out;
      e.x = reinterpret_cast<__half*>(ws + s.at[x]) + k * s.n * s.ld(NS_X0);
      e.rem = remainders ? reinterpret_cast<uint8_t*>(ws + s.rem) + k * s.rem_bytes() : nullptr;
      e.rem_cols = int(s.rem_cols());
      e.sums = reinterpret_cast<double*>(ws + plan.sums[i]);
      e.ld = s.ld(NS_X0);
      e.rows = int(t[i].rows);
      e.cols = int(t[i].cols);
      e.parts = plan.parts[i];
      e.tiles_c = (e.cols + 63) / 64;
      e.first = int(blocks);
      e.g_f32 = t[i].g_f32;
      const uintptr_t f32 = reinterpret_cast<uintptr_t>(e.p) | reinterpret_cast<uintptr_t>(e.m) | (e.g_f32 ? reinterpret_cast<uintptr_t>(e.g) : 0);
      const uintptr_t b16 = reinterpret_cast<uintptr_t>(e.out) | (e.g_f32 ? 0 : reinterpret_cast<uintptr_t>(e.g));
      e.wide = e.cols % 4 == 0 && (f32 & 15) == 0 && (b16 & 7) == 0;
      e.scale = scale;
      e.step = (common.muon ? step * sqrtf(float(s.m)) : 1.f) / scale;
      const long tiles = long((e.rows + 63) / 64) * e.tiles_c;
      blocks += PASS == 0 ? e.parts : PASS == 1 ? (tiles + a.span - 1) / a.span : tiles;
      if (a.count == NS_MATRICES)
        if (int rc = flush()) return rc;
    }
  }
  return flush();
}

static int ns_check(const NsMatrix* t, int count) {
  for (int i = 0; i < count; ++i)
    if (t[i].rows < 1 || t[i].cols < 1 || t[i].rows > 0x7fffffffL || t[i].cols > 0x7fffffffL)
      ZB_FAIL(-1, "newton_schulz: matrix %d is %ld x %ld", i, t[i].rows, t[i].cols);
  return 0;
}

// How many of the list's first matrices are taken together.
static int ns_together(const NsMatrix* t, int count, long limit) {
  double room = double(limit);
  for (int i = 0; i < count; ++i) {
    const double n = double(std::min(t[i].rows, t[i].cols)), m = double(std::max(t[i].rows, t[i].cols));
    room -= 4 * n * (m + 64) + 4 * n * (n + 64) + (n + 32) * (m + 64) + 8192;
    if (room < 0) return std::max(i, 1);
  }
  return count;
}

}  // namespace zb

extern "C" {

// Bytes of workspace for a list (of zb_newton_schulz's table only rows and cols are looked at).  Its matrices are taken together as far as their
// workspace stays below `limit`, or one by one.
int zb_newton_schulz_workspace(const void* table, int count, long limit, long* bytes) {
  using namespace zb;
  try {
    const NsMatrix* t = static_cast<const NsMatrix*>(table);
    if (int rc = ns_check(t, count)) return rc;
    *bytes = 0;
    for (int i = 0, n; i < count; i += n) {
      n = ns_together(t + i, count - i, limit);
      *bytes = std::max(*bytes, long(ns_plan(t + i, n).bytes));
    }
    return 0;
  } catch (const std::exception& e) {      // (the host's memory for the plan)
    ZB_FAIL(-4, "newton_schulz: %s", e.what());
  }
}

// table: `count` NsMatrix, none of them empty.  muon: p and m are stepped with lr times `size` sqrt(long side), momentum (nesterov: the gradient looks ahead by it), the
// gradient times grad_scale, and keep = 1 - lr weight_decay; else the orthogonalised matrices go to `out`.  a, b, c: coefficients.
int zb_newton_schulz(const void* table, int count, int muon, float lr, float momentum, int nesterov, float keep, float grad_scale, int iterations,
                     float a, float b, float c, float size, long limit, void* workspace, long bytes, int* launches, int* status, cudaStream_t stream) {
  using namespace zb;
  try {
    const NsMatrix* t = static_cast<const NsMatrix*>(table);
    *launches = 0;
    if (count <= 0) return 0;
    if (int rc = ns_check(t, count)) return rc;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) ZB_FAIL(-4, "newton_schulz: the workspace is not on a 16-byte boundary");
    NsPass pass = {};
    pass.momentum = momentum;
    pass.grad_scale = grad_scale;
    pass.keep = keep;
    pass.nesterov = nesterov;
    pass.muon = muon;
    char* ws = static_cast<char*>(workspace);
    const std::vector<NsStep> program = ns_program(iterations, a, b, c);
    for (int i = 0, n; i < count; i += n) {
      n = ns_together(t + i, count - i, limit);
      const NsPlan plan = ns_plan(t + i, n);
      if (bytes < long(plan.bytes)) ZB_FAIL(-4, "newton_schulz: %ld bytes of workspace, %zu are needed", bytes, plan.bytes);
      int rc = ns_pass<0>(plan, t + i, pass, lr * size, ws, NS_X0, false, stream, launches);
      if (!rc) rc = ns_pass<1>(plan, t + i, pass, lr * size, ws, NS_X0, ns_keeps_remainder(0, iterations), stream, launches);
      if (!rc) rc = ns_products(plan, ws, program, status, stream, launches);
      if (!rc) rc = ns_pass<2>(plan, t + i, pass, lr * size, ws, iterations & 1 ? NS_X1 : NS_X0, false, stream, launches);
      if (rc) return rc;
    }
    return 0;
  } catch (const std::exception& e) {
    ZB_FAIL(-4, "newton_schulz: %s", e.what());
  }
}

}  // extern "C"
