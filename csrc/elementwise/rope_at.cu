// Rotation of heads by given positions, of one or several axes, in place.
//
// Pair i of a head (columns i and i + d / 2) turns by the angle of pair i in row positions[axis(i)][t] of the table, whose rows
// hold the cosines of all pairs, then the sines; the first sections[0] pairs belong to axis 0, the next sections[1] to
// axis 1, and so on.  One axis with the places within packed sequences is the plain rotation restarted in each of
// them; three axes are time, height and width of what an image or a video has given tokens for.
//
// Bound by memory: 4 bytes an element, 8 flops a pair.  A thread has 8 pairs of a token (two 16-byte pieces a head), keeps
// their cosines and sines in registers and walks over HEADS heads with all their loads in flight; neighbouring threads have
// neighbouring pieces, so a head's halves are read in whole lines.  Rows of the table come through L2.  16384 tokens of 40 heads of
// 128 by three axes: 57 us, 92 % of a copy's rate.
#include "../common/host.h"
#include "../common/ptx.cuh"

namespace zb {

constexpr int ROPE_AXES = 4;
struct RopeAt {
  __nv_bfloat16* buf;
  const float* cs;
  const int* positions;
  long ld;
  int T, P, heads, d, groups;
  int ends[ROPE_AXES];      // pairs [ends[a - 1], ends[a]) are axis a's
};

__device__ __forceinline__ int rope_axis(const RopeAt& p, int i) {
  int a = 0;
#pragma unroll
  for (int k = 0; k + 1 < ROPE_AXES; ++k) a += i >= p.ends[k];
  return a;
}
__device__ __forceinline__ const float* rope_row(const RopeAt& p, int axis, int t) {
  const int at = min(max(p.positions[size_t(axis) * p.T + t], 0), p.P - 1);   // a position outside the table takes its nearest row
  return p.cs + size_t(at) * p.d;
}

template <int HEADS>
__global__ void __launch_bounds__(256)
rope_at_kernel(const RopeAt p, const float sign) {
  chain_trigger();
  chain_wait();
  const int h = p.d >> 1, pieces = h >> 3;
  const long n = long(p.T) * p.groups * pieces;
  const long at = long(blockIdx.x) * 256 + threadIdx.x;
  if (at >= n) return;
  const int piece = int(at % pieces);
  const long rest = at / pieces;
  const int group = int(rest % p.groups), t = int(rest / p.groups);
  const int i0 = piece * 8;
  float co[8], si[8];
  const int a0 = rope_axis(p, i0);
  if (a0 == rope_axis(p, i0 + 7)) {
    const float* row = rope_row(p, a0, t) + i0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint4 c = ld_v4(row + 4 * j), s = ld_v4(row + h + 4 * j);
      co[4 * j] = __uint_as_float(c.x); co[4 * j + 1] = __uint_as_float(c.y);
      co[4 * j + 2] = __uint_as_float(c.z); co[4 * j + 3] = __uint_as_float(c.w);
      si[4 * j] = __uint_as_float(s.x); si[4 * j + 1] = __uint_as_float(s.y);
      si[4 * j + 2] = __uint_as_float(s.z); si[4 * j + 3] = __uint_as_float(s.w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float* row = rope_row(p, rope_axis(p, i0 + j), t) + i0 + j;
      co[j] = row[0];
      si[j] = row[h];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) si[j] *= sign;
  __nv_bfloat16* x = p.buf + size_t(t) * p.ld + size_t(group) * HEADS * p.d + i0;
  const int m = min(HEADS, p.heads - group * HEADS);
  uint4 u[HEADS], v[HEADS];
#pragma unroll
  for (int k = 0; k < HEADS; ++k)
    if (k < m) {
      u[k] = ld_v4(x + size_t(k) * p.d);
      v[k] = ld_v4(x + size_t(k) * p.d + h);
    }
#pragma unroll
  for (int k = 0; k < HEADS; ++k)
    if (k < m) {
      uint32_t us[4] = {u[k].x, u[k].y, u[k].z, u[k].w}, vs[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = unpack_bf16x2(us[j]), b = unpack_bf16x2(vs[j]);
        us[j] = pack_bf16x2(a.x * co[2 * j] - b.x * si[2 * j], a.y * co[2 * j + 1] - b.y * si[2 * j + 1]);
        vs[j] = pack_bf16x2(b.x * co[2 * j] + a.x * si[2 * j], b.y * co[2 * j + 1] + a.y * si[2 * j + 1]);
      }
      *reinterpret_cast<uint4*>(x + size_t(k) * p.d) = make_uint4(us[0], us[1], us[2], us[3]);
      *reinterpret_cast<uint4*>(x + size_t(k) * p.d + h) = make_uint4(vs[0], vs[1], vs[2], vs[3]);
    }
}

// A pair at a time: widths that are no multiple of 16, rows that do not start on 16 bytes.
__global__ void __launch_bounds__(256)
rope_at_pairs_kernel(const RopeAt p, const float sign) {
  chain_trigger();
  chain_wait();
  const int h = p.d >> 1;
  const long n = long(p.T) * p.heads * h;
  for (long at = long(blockIdx.x) * 256 + threadIdx.x; at < n; at += long(gridDim.x) * 256) {
    const int i = int(at % h), head = int(at / h % p.heads), t = int(at / h / p.heads);
    const float* row = rope_row(p, rope_axis(p, i), t) + i;
    const float c = row[0], s = row[h] * sign;
    __nv_bfloat16* x = p.buf + size_t(t) * p.ld + size_t(head) * p.d + i;
    const float a = __bfloat162float(x[0]), b = __bfloat162float(x[h]);
    x[0] = __float2bfloat16(a * c - b * s);
    x[h] = __float2bfloat16(b * c + a * s);
  }
}

}  // namespace zb

// buf: bf16, rows ld elements apart, heads [0, heads) of d columns at their start; cs [P, d]; positions [axes, T]; sections [axes] (host).
extern "C" int zb_rope_at(void* buf, const float* cs, const int* positions, const int* sections, int axes, int T, int P, int heads, int d,
                          long ld, int backward, cudaStream_t stream) {
  using namespace zb;
  if (T <= 0 || heads <= 0) return 0;
  if (P <= 0) ZB_FAIL(-1, "rope_at: an empty table");
  if (d <= 0 || d % 2 != 0) ZB_FAIL(-1, "rope_at: heads of %d columns", d);
  if (axes < 1 || axes > ROPE_AXES) ZB_FAIL(-1, "rope_at: %d axes, 1 to %d", axes, ROPE_AXES);
  RopeAt p = {};
  p.buf = static_cast<__nv_bfloat16*>(buf);
  p.cs = cs;
  p.positions = positions;
  p.ld = ld;
  p.T = T; p.P = P; p.heads = heads; p.d = d;
  long end = 0;
  for (int a = 0; a < ROPE_AXES; ++a) {
    if (a < axes) {
      if (sections[a] < 0) ZB_FAIL(-1, "rope_at: a section of %d", sections[a]);
      end += sections[a];
    }
    p.ends[a] = a < axes - 1 ? int(end) : d;   // (behind the last axis: never reached)
  }
  if (end != d / 2) ZB_FAIL(-1, "rope_at: sections of %ld pairs, heads have %d", end, d / 2);
  const float sign = backward ? -1.f : 1.f;
  const bool wide = d % 16 == 0 && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(buf) & 15) == 0 && (reinterpret_cast<uintptr_t>(cs) & 15) == 0;
  if (wide) {
    constexpr int HEADS = 4;
    p.groups = (heads + HEADS - 1) / HEADS;
    const long blocks = (long(T) * p.groups * (d / 16) + 255) / 256;
    if (blocks > 0x7fffffffL) ZB_FAIL(-1, "rope_at: %d tokens of %d heads", T, heads);
    ZB_CUDA_OK(launch_pass(rope_at_kernel<HEADS>, dim3(unsigned(blocks)), 256, 0, stream, p, sign));
  } else {
    const long blocks = (long(T) * heads * (d / 2) + 255) / 256, most = 64l * num_sms();
    ZB_CUDA_OK(launch_pass(rope_at_pairs_kernel, dim3(unsigned(blocks < most ? blocks : most)), 256, 0, stream, p, sign));
  }
  return 0;
}
