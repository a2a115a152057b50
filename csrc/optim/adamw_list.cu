// AdamW (decoupled weight decay) over a list of tensors in one launch, with its two moments in fp32 or in 8 bits:
//   g' = g s,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g' g'
//   p = p (1 - lr wd) - lr / (1 - b1^k) m / (sqrt(v) / sqrt(1 - b2^k) + eps),  p16 = bf16(p)
//
// Moments in 8 bits.  A value is held as the leading bits of its fp32 pattern: exponent and three bits of mantissa,
// u = bits >> 20, counted from the base of its block of 256 values, which is an int16 beside it: m as its sign and u - base in
// 0 .. 127 (16 binades below the block's largest), v as u - base in 0 .. 255 (32 binades).  Code 0 is zero; a v that is not
// zero keeps at least code 1, so that no step is divided by eps alone.  The base follows from the largest value of the
// block.  Before the 20 low bits are cut off, a dither of 16 bits is added to them, so that the expectation of what is held
// is the value: rounded to nearest, v would never move (b2 = 0.999 changes it by a thousandth a step, neighbouring codes
// differ by an eighth) and m would come to rest at less than two thirds of a constant gradient.  The dither is half of a
// hash of the tensor's seed and the number of the pair of elements, the same half for m and v: a Weyl sequence (odd multiple
// near 2^32 / golden ratio) through two rounds of shift-xor and multiplication by the fraction bits of sqrt 2 and sqrt 3.
// m and v are computed by multiplications and additions that round one by one, so that the codes are a function of the
// inputs and not of the compiler's contractions; encoding and decoding are integer operations.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include <type_traits>

namespace zb {

constexpr int ADAMW_BLOCK = 256;                     // values with one base; a warp's work at a time
constexpr int ADAMW_TILE = 8 * ADAMW_BLOCK;          // a CTA's

struct AdamwTensor {                                 // as the caller packs it
  float* p;
  void *m, *v;                                       // fp32, or codes
  short *mb, *vb;                                    // bases of codes
  const void* g;
  __nv_bfloat16* p16;                                // may be null
  long n;
  float step, inv_bc2;                               // lr / (1 - b1^k), 1 / sqrt(1 - b2^k)
  unsigned seed, grad_f32;
};
struct AdamwHyper {
  float beta1, c1, beta2, c2, eps, keep, grad_scale; // c = 1 - beta, keep = 1 - lr wd
};
template <int N>
struct AdamwList {
  AdamwTensor t[N];
  long end[N];                                       // tiles up to and with this tensor
  int count;
  AdamwHyper h;
};

// one operation, rounded to nearest, subnormals kept
__device__ __forceinline__ float mul1(float a, float b) {
  float d;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float add1(float a, float b) {
  float d;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ unsigned adamw_hash(unsigned pair, unsigned seed) {
  unsigned x = pair * 0x9E3779B1u + seed;
  x = (x ^ (x >> 15)) * 0x6A09E667u;
  x = (x ^ (x >> 13)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}
__device__ __forceinline__ unsigned decode_bits(unsigned code, unsigned base) { return code ? (code + base) << 20 : 0u; }
__device__ __forceinline__ float decode_m(unsigned byte, unsigned base) {
  return __uint_as_float(decode_bits(byte & 0x7fu, base) | (byte & 0x80u) << 24);
}
// The base of a block whose largest pattern is `top`: the highest code that a dither can give still fits
__device__ __forceinline__ int code_base(unsigned top, int most) {
  const int b = int((top + 0xfffffu) >> 20) - most;
  return b > 0 ? b : 0;
}
constexpr unsigned ADAMW_TOP = 0x7fe00000u;          // NaNs are held as this one, and keep clear of the sign bit

__device__ __forceinline__ void adamw_moments(float g, float& m, float& v, const AdamwHyper& h) {
  g = mul1(g, h.grad_scale);
  m = add1(mul1(m, h.beta1), mul1(g, h.c1));
  v = add1(mul1(v, h.beta2), mul1(mul1(g, h.c2), g));
}
__device__ __forceinline__ float adamw_param(float p, float m, float v, const AdamwTensor& t, const AdamwHyper& h) {
  return p * h.keep - t.step * (m / (sqrtf(v) * t.inv_bc2 + h.eps));
}

// Four consecutive elements of a tensor, n of them there (4 but at its end)
template <typename T>
__device__ __forceinline__ void load4(const T* src, int n, float (&f)[4]) {
  if (n == 4) {
    if constexpr (sizeof(T) == 4) {
      const uint4 u = ld_v4(src);
      f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(src);
      const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
      f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = j < n ? float(src[j]) : 0.f;
  }
}
__device__ __forceinline__ void store4(float* dst, int n, const float (&f)[4]) {
  if (n == 4) {
    *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) dst[j] = f[j];
  }
}
__device__ __forceinline__ void store4(__nv_bfloat16* dst, int n, const float (&f)[4]) {
  if (n == 4) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) dst[j] = __float2bfloat16(f[j]);
  }
}
__device__ __forceinline__ unsigned load_codes(const unsigned char* src, int n) {
  if (n == 4) return *reinterpret_cast<const unsigned*>(src);
  unsigned u = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) u |= unsigned(src[j]) << (8 * j);
  return u;
}
__device__ __forceinline__ void store_codes(unsigned char* dst, int n, unsigned u) {
  if (n == 4) {
    *reinterpret_cast<unsigned*>(dst) = u;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) dst[j] = static_cast<unsigned char>(u >> (8 * j));
  }
}

// One warp, one block of 256: lane l has elements 4 l .. 4 l + 3 and 128 + 4 l ..
template <int BITS, typename GT>
__device__ __forceinline__ void adamw_block(const AdamwTensor& t, const AdamwHyper& h, long block, int lane) {
  const long e0 = block * ADAMW_BLOCK + lane * 4;
  int n[2];
  float p[2][4], g[2][4], m[2][4], v[2][4];
  unsigned mu[2], vu[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long e = e0 + k * 128, left = t.n - e;
    n[k] = left >= 4 ? 4 : left > 0 ? int(left) : 0;
    load4(t.p + e, n[k], p[k]);
    load4(static_cast<const GT*>(t.g) + e, n[k], g[k]);
    if constexpr (BITS == 32) {
      load4(static_cast<const float*>(t.m) + e, n[k], m[k]);
      load4(static_cast<const float*>(t.v) + e, n[k], v[k]);
    } else {
      mu[k] = load_codes(static_cast<const unsigned char*>(t.m) + e, n[k]);
      vu[k] = load_codes(static_cast<const unsigned char*>(t.v) + e, n[k]);
    }
  }
  if constexpr (BITS == 8) {
    const unsigned mb = unsigned(t.mb[block]), vb = unsigned(t.vb[block]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[k][j] = decode_m(mu[k] >> (8 * j) & 0xffu, mb);
        v[k][j] = __uint_as_float(decode_bits(vu[k] >> (8 * j) & 0xffu, vb));
      }
    }
  }
  unsigned mtop = 0, vtop = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      adamw_moments(g[k][j], m[k][j], v[k][j], h);
      p[k][j] = adamw_param(p[k][j], m[k][j], v[k][j], t, h);
      if constexpr (BITS == 8) {
        mtop = max(mtop, __float_as_uint(m[k][j]) & 0x7fffffffu);
        vtop = max(vtop, __float_as_uint(v[k][j]) & 0x7fffffffu);
      }
    }
  }
  unsigned mb = 0, vb = 0;
  if constexpr (BITS == 8) {
    mtop = min(__reduce_max_sync(0xffffffffu, mtop), ADAMW_TOP);
    vtop = min(__reduce_max_sync(0xffffffffu, vtop), ADAMW_TOP);
    mb = code_base(mtop, 127);
    vb = code_base(vtop, 255);
    if (lane == 0) {
      t.mb[block] = short(mb);
      t.vb[block] = short(vb);
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long e = e0 + k * 128;
    store4(t.p + e, n[k], p[k]);
    if (t.p16 != nullptr) store4(t.p16 + e, n[k], p[k]);
    if constexpr (BITS == 32) {
      store4(static_cast<float*>(t.m) + e, n[k], m[k]);
      store4(static_cast<float*>(t.v) + e, n[k], v[k]);
    } else {
      mu[k] = vu[k] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned word = adamw_hash(unsigned(e >> 1) + (j >> 1), t.seed);
        const unsigned dither = (j & 1 ? word >> 16 : word & 0xffffu) << 4 | 8u;
        const unsigned mbits = __float_as_uint(m[k][j]), vbits = min(__float_as_uint(v[k][j]) & 0x7fffffffu, ADAMW_TOP);
        const unsigned mag = min(mbits & 0x7fffffffu, ADAMW_TOP);
        const int mc = int((mag + dither) >> 20) - int(mb), vc = int((vbits + dither) >> 20) - int(vb);
        mu[k] |= (unsigned(mag && mc > 0 ? mc : 0) | mbits >> 31 << 7) << (8 * j);
        vu[k] |= unsigned(vbits ? max(vc, 1) : 0) << (8 * j);
      }
      store_codes(static_cast<unsigned char*>(t.m) + e, n[k], mu[k]);
      store_codes(static_cast<unsigned char*>(t.v) + e, n[k], vu[k]);
    }
  }
}

template <int N, int BITS>
__global__ void __launch_bounds__(256) adamw_list_kernel(const __grid_constant__ AdamwList<N> list) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int i = 0;
  for (long tile = blockIdx.x; tile < list.end[list.count - 1]; tile += gridDim.x) {
    while (tile >= list.end[i]) ++i;
    const AdamwTensor& t = list.t[i];
    const long block = (tile - (i > 0 ? list.end[i - 1] : 0)) * 8 + warp;
    if (block * ADAMW_BLOCK >= t.n) continue;
    if (t.grad_f32) adamw_block<BITS, float>(t, list.h, block, lane);
    else adamw_block<BITS, __nv_bfloat16>(t, list.h, block, lane);
  }
}

// out = what a tensor's codes stand for
template <typename T>
__global__ void __launch_bounds__(256) moment_values_kernel(const unsigned char* m, const short* mb, const unsigned char* v,
                                                            const short* vb, T* m_out, T* v_out, long n) {
  for (long e = (blockIdx.x * 256L + threadIdx.x) * 4; e < n; e += gridDim.x * 1024L) {
    const int k = n - e >= 4 ? 4 : int(n - e);
    const unsigned mu = load_codes(m + e, k), vu = load_codes(v + e, k);
    const unsigned bm = unsigned(mb[e / ADAMW_BLOCK]), bv = unsigned(vb[e / ADAMW_BLOCK]);
    float a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = decode_m(mu >> (8 * j) & 0xffu, bm);
      b[j] = __uint_as_float(decode_bits(vu >> (8 * j) & 0xffu, bv));
    }
    store4(m_out + e, k, a);
    store4(v_out + e, k, b);
  }
}

template <int N, int BITS>
static int adamw_launch(const AdamwTensor* t, int count, const AdamwHyper& h, cudaStream_t stream) {
  AdamwList<N> list;
  list.count = count;
  list.h = h;
  long tiles = 0;
  for (int i = 0; i < count; ++i) {
    list.t[i] = t[i];
    tiles += (t[i].n + ADAMW_TILE - 1) / ADAMW_TILE;
    list.end[i] = tiles;
  }
  if (tiles == 0) return 0;
  const long cap = long(num_sms()) * 8;
  adamw_list_kernel<N, BITS><<<int(tiles < cap ? tiles : cap), 256, 0, stream>>>(list);
  ZB_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // namespace zb

extern "C" {

// table: `count` AdamwTensor.  A launch takes up to 256 of them as its parameters, longer lists go in several.
int zb_adamw_list(const void* table, int count, int bits, float beta1, float c1, float beta2, float c2, float eps, float keep,
                  float grad_scale, cudaStream_t stream) {
  using namespace zb;
  const AdamwTensor* t = static_cast<const AdamwTensor*>(table);
  if (bits != 8 && bits != 32) ZB_FAIL(-1, "adamw: moments in %d bits", bits);
  for (int i = 0; i < count; ++i) {
    const uintptr_t wide = reinterpret_cast<uintptr_t>(t[i].p) | (t[i].grad_f32 ? reinterpret_cast<uintptr_t>(t[i].g) : 0) |
                           (bits == 32 ? reinterpret_cast<uintptr_t>(t[i].m) | reinterpret_cast<uintptr_t>(t[i].v) : 0);
    const uintptr_t narrow = reinterpret_cast<uintptr_t>(t[i].p16) | (t[i].grad_f32 ? 0 : reinterpret_cast<uintptr_t>(t[i].g));
    const uintptr_t codes = bits == 8 ? reinterpret_cast<uintptr_t>(t[i].m) | reinterpret_cast<uintptr_t>(t[i].v) : 0;
    if ((wide & 15) || (narrow & 7) || (codes & 3))
      ZB_FAIL(-1, "adamw: tensor %d is not aligned (fp32 16 bytes, bf16 8, codes 4)", i);
  }
  const AdamwHyper h = {beta1, c1, beta2, c2, eps, keep, grad_scale};
  for (int i = 0; i < count; i += 256) {
    const int n = count - i < 256 ? count - i : 256;
    const int rc = bits == 8 ? (n <= 32 ? adamw_launch<32, 8>(t + i, n, h, stream) : adamw_launch<256, 8>(t + i, n, h, stream))
                             : (n <= 32 ? adamw_launch<32, 32>(t + i, n, h, stream) : adamw_launch<256, 32>(t + i, n, h, stream));
    if (rc) return rc;
  }
  return 0;
}

int zb_moment_values(const void* m, const void* mb, const void* v, const void* vb, void* m_out, void* v_out, long n, int out_f32,
                     cudaStream_t stream) {
  using namespace zb;
  if (n <= 0) return 0;
  if (((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 3) ||
      ((reinterpret_cast<uintptr_t>(m_out) | reinterpret_cast<uintptr_t>(v_out)) & 15))
    ZB_FAIL(-1, "moment_values: codes must be 4-byte aligned, values 16");
  const long ctas = (n + 1023) / 1024, cap = long(num_sms()) * 16;
  const int grid = int(ctas < cap ? ctas : cap);
  const unsigned char *mc = static_cast<const unsigned char*>(m), *vc = static_cast<const unsigned char*>(v);
  const short *bm = static_cast<const short*>(mb), *bv = static_cast<const short*>(vb);
  if (out_f32)
    moment_values_kernel<float><<<grid, 256, 0, stream>>>(mc, bm, vc, bv, static_cast<float*>(m_out), static_cast<float*>(v_out), n);
  else
    moment_values_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(mc, bm, vc, bv, static_cast<__nv_bfloat16*>(m_out),
                                                                  static_cast<__nv_bfloat16*>(v_out), n);
  ZB_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // extern "C"
