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
//
// Bound by memory: 8 x 61 million parameters, fp32 gradients, 1.42 ms with moments in 8 bits (18 bytes a parameter, 6.2 TB/s or
// 96 % of a copy's rate); the units of a 125M model, bf16 gradients, 0.755 ms with moments in fp32 (28 bytes, 94 %).  The 8-bit form
// is near the issue limit as well (70 % of its slots are taken; with scalar arithmetic, codes handled one by one and no block ahead it
// took 1.6 ms).
// Blocks go to warps round robin, so that all warps work in one part of the tensors: in a stretch of its own for each warp, the
// same kernel took 1.58 ms.
#include "../common/host.h"
#include "../common/ptx.cuh"

namespace zb {

constexpr int ADAMW_BLOCK = 256;                     // values with one base; a warp's work at a time
constexpr int ADAMW_CTAS = 3;                        // on an SM

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
  long end[N];                                       // blocks up to and with this tensor
  int count;
  AdamwHyper h;
};

// Two values an instruction, every operation rounded to nearest by itself, subnormals kept.  (A packed product and a packed sum
// behind it come out as one fma in spite of their rounding modifiers; a scalar sum does not join a packed product.)
struct Pair {
  float a, b;
};
__device__ __forceinline__ Pair operator*(Pair x, Pair y) {
  Pair r;
  fmul2(r.a, r.b, x.a, x.b, y.a, y.b);
  return r;
}
__device__ __forceinline__ Pair operator+(Pair x, Pair y) {
  Pair r;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(r.a) : "f"(x.a), "f"(y.a));
  asm("add.rn.f32 %0, %1, %2;" : "=f"(r.b) : "f"(x.b), "f"(y.b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair x, Pair y, Pair z) {
  Pair r;
  ffma2(r.a, r.b, x.a, x.b, y.a, y.b, z.a, z.b);
  return r;
}
__device__ __forceinline__ Pair both(float v) { return {v, v}; }
// The square root to 2^-23.  sqrtf of a build with fast mathematics takes subnormals as 0; with FINE they have their roots.
template <bool FINE>
__device__ __forceinline__ float root(float v) {
  if constexpr (!FINE) return sqrtf(v);
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ unsigned adamw_hash(unsigned pair_times_weyl_plus_seed) {
  unsigned x = pair_times_weyl_plus_seed;
  x = (x ^ (x >> 15)) * 0x6A09E667u;
  x = (x ^ (x >> 13)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}
constexpr unsigned ADAMW_WEYL = 0x9E3779B1u;

// Byte J of a word of codes, shifted to bits 20 .. 27
template <int J>
__device__ __forceinline__ unsigned code_at_20(unsigned word, unsigned mask) {
  const unsigned t = word & (mask << (8 * J));
  return J < 3 ? t << (20 - 8 * J) : t >> 4;
}
__device__ __forceinline__ bool has_zero_byte(unsigned w) { return ((w - 0x01010101u) & ~w & 0x80808080u) != 0; }
// The patterns of four values from their codes; base20: the block's base, shifted.  ZEROS: some code may be 0
template <bool ZEROS>
__device__ __forceinline__ void decode4(unsigned word, unsigned mask, unsigned base20, unsigned (&u)[4]) {
  u[0] = code_at_20<0>(word, mask); u[1] = code_at_20<1>(word, mask); u[2] = code_at_20<2>(word, mask); u[3] = code_at_20<3>(word, mask);
#pragma unroll
  for (int j = 0; j < 4; ++j) u[j] = ZEROS && u[j] == 0 ? 0 : u[j] + base20;
}
__device__ __forceinline__ void decode_v4(unsigned word, unsigned base20, float (&f)[4]) {
  unsigned u[4];
  if (has_zero_byte(word)) decode4<true>(word, 0xffu, base20, u);
  else decode4<false>(word, 0xffu, base20, u);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(u[j]);
}
__device__ __forceinline__ void decode_m4(unsigned word, unsigned base20, float (&f)[4]) {
  unsigned u[4];
  if (has_zero_byte(word & 0x7f7f7f7fu)) decode4<true>(word, 0x7fu, base20, u);
  else decode4<false>(word, 0x7fu, base20, u);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(u[j] | (word << (24 - 8 * j) & 0x80000000u));
}
// The base of a block whose largest pattern is `top`: the highest code that a dither can give still fits
__device__ __forceinline__ int code_base(unsigned top, int most) {
  const int b = int((top + 0xfffffu) >> 20) - most;
  return b > 0 ? b : 0;
}
constexpr unsigned ADAMW_INF = 0x7f800000u, ADAMW_TOP = 0x7fe00000u;   // NaNs are held as the second one, clear of the sign bit

__device__ __forceinline__ unsigned bytes4(const int (&c)[4]) {
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
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

// What a lane has of a block of 256: elements 4 l .. 4 l + 3 and 128 + 4 l .., n of either there
template <int BITS>
struct AdamwLane {
  int n[2];
  float p[2][4], g[2][4], m[2][4], v[2][4];
  unsigned mu[2], vu[2];
};
template <int BITS, typename GT>
__device__ __forceinline__ void adamw_load(AdamwLane<BITS>& x, const AdamwTensor& t, long e0) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long e = e0 + k * 128, left = t.n - e;
    x.n[k] = left >= 4 ? 4 : left > 0 ? int(left) : 0;
    load4(t.p + e, x.n[k], x.p[k]);
    load4(static_cast<const GT*>(t.g) + e, x.n[k], x.g[k]);
    if constexpr (BITS == 32) {
      load4(static_cast<const float*>(t.m) + e, x.n[k], x.m[k]);
      load4(static_cast<const float*>(t.v) + e, x.n[k], x.v[k]);
    } else {
      x.mu[k] = load_codes(static_cast<const unsigned char*>(t.m) + e, x.n[k]);
      x.vu[k] = load_codes(static_cast<const unsigned char*>(t.v) + e, x.n[k]);
    }
  }
}

// Every lane copies its parts of its warp's next block into its own places in shared memory while it works on this one: with the
// loads in registers, too few bytes were on their way behind the arithmetic of the 8-bit form.  The last block of a tensor, if it
// is not whole, is loaded when it is its turn.
template <int BITS>
struct AdamwRing {
  uint4 wide[2][BITS == 8 ? 4 : 8][256];      // p, g (8 bytes of bf16), and m, v in fp32
  unsigned code[BITS == 8 ? 2 : 1][4][256];   // m, v in 8 bits
};
template <int BITS>
__device__ __forceinline__ void adamw_request(AdamwRing<BITS>& ring, int slot, const AdamwTensor& t, long e0) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long e = e0 + k * 128;
    ring_load16(&ring.wide[slot][k][tid], t.p + e);
    if (t.grad_f32) ring_load16(&ring.wide[slot][2 + k][tid], static_cast<const float*>(t.g) + e);
    else ring_load8(&ring.wide[slot][2 + k][tid], static_cast<const __nv_bfloat16*>(t.g) + e);
    if constexpr (BITS == 32) {
      ring_load16(&ring.wide[slot][4 + k][tid], static_cast<const float*>(t.m) + e);
      ring_load16(&ring.wide[slot][6 + k][tid], static_cast<const float*>(t.v) + e);
    } else {
      ring_load4(&ring.code[slot][k][tid], static_cast<const unsigned char*>(t.m) + e);
      ring_load4(&ring.code[slot][2 + k][tid], static_cast<const unsigned char*>(t.v) + e);
    }
  }
}
__device__ __forceinline__ void floats4(const uint4& u, float (&f)[4]) {
  f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}
template <int BITS>
__device__ __forceinline__ void adamw_take(AdamwLane<BITS>& x, const AdamwRing<BITS>& ring, int slot, bool grad_f32) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    x.n[k] = 4;
    floats4(ring.wide[slot][k][tid], x.p[k]);
    if (grad_f32) {
      floats4(ring.wide[slot][2 + k][tid], x.g[k]);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(&ring.wide[slot][2 + k][tid]);
      const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
      x.g[k][0] = a.x; x.g[k][1] = a.y; x.g[k][2] = b.x; x.g[k][3] = b.y;
    }
    if constexpr (BITS == 32) {
      floats4(ring.wide[slot][4 + k][tid], x.m[k]);
      floats4(ring.wide[slot][6 + k][tid], x.v[k]);
    } else {
      x.mu[k] = ring.code[slot][k][tid];
      x.vu[k] = ring.code[slot][2 + k][tid];
    }
  }
}

// The step of one block by one warp; mb0, vb0: the block's bases
template <int BITS, bool FINE, bool WHOLE>
__device__ __forceinline__ void adamw_block(AdamwLane<BITS>& x, const AdamwTensor& t, const AdamwHyper& h, long block, int lane, int mb0,
                                            int vb0) {
  const long e0 = block * ADAMW_BLOCK + lane * 4;
  auto &p = x.p, &g = x.g, &m = x.m, &v = x.v;
  int n[2] = {WHOLE ? 4 : x.n[0], WHOLE ? 4 : x.n[1]};
  if constexpr (BITS == 8) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      decode_m4(x.mu[k], unsigned(mb0) << 20, m[k]);
      decode_v4(x.vu[k], unsigned(vb0) << 20, v[k]);
    }
  }
  unsigned mtop = 0, vtop = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const Pair gs = Pair{g[k][j], g[k][j + 1]} * both(h.grad_scale);
      const Pair mm = Pair{m[k][j], m[k][j + 1]} * both(h.beta1) + gs * both(h.c1);
      const Pair vv = Pair{v[k][j], v[k][j + 1]} * both(h.beta2) + gs * both(h.c2) * gs;
      m[k][j] = mm.a; m[k][j + 1] = mm.b;
      v[k][j] = vv.a; v[k][j + 1] = vv.b;
      const Pair denom = fma2({root<FINE>(vv.a), root<FINE>(vv.b)}, both(t.inv_bc2), both(h.eps));
      const Pair up = {__fdividef(mm.a, denom.a), __fdividef(mm.b, denom.b)};
      const Pair pp = fma2(up, both(-t.step), Pair{p[k][j], p[k][j + 1]} * both(h.keep));
      p[k][j] = pp.a; p[k][j + 1] = pp.b;
    }
    if constexpr (BITS == 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mtop = max(mtop, __float_as_uint(m[k][j]) & 0x7fffffffu);
        vtop = max(vtop, __float_as_uint(v[k][j]));           // (never negative; NaN as the canonical one)
      }
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
    }
  }
  if constexpr (BITS == 8) {
    mtop = __reduce_max_sync(0xffffffffu, mtop);
    vtop = __reduce_max_sync(0xffffffffu, vtop);
    if (max(mtop, vtop) > ADAMW_INF) {                        // a NaN somewhere in the block
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if ((__float_as_uint(m[k][j]) & 0x7fffffffu) > ADAMW_INF) m[k][j] = __uint_as_float(ADAMW_TOP);
          if (__float_as_uint(v[k][j]) > ADAMW_INF) v[k][j] = __uint_as_float(ADAMW_TOP);
        }
      }
      mtop = min(mtop, ADAMW_TOP);
      vtop = min(vtop, ADAMW_TOP);
    }
    const int mb = code_base(mtop, 127), vb = code_base(vtop, 255);
    if (lane == 0) {
      t.mb[block] = short(mb);
      t.vb[block] = short(vb);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const long e = e0 + k * 128;
      const unsigned x = unsigned(e >> 1) * ADAMW_WEYL + t.seed, w0 = adamw_hash(x), w1 = adamw_hash(x + ADAMW_WEYL);
      const unsigned dither[4] = {(w0 << 4 & 0xffff0u) | 8u, (w0 >> 12 & 0xffff0u) | 8u, (w1 << 4 & 0xffff0u) | 8u,
                                  (w1 >> 12 & 0xffff0u) | 8u};
      int mc[4], vc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned vbits = __float_as_uint(v[k][j]), mag = __float_as_uint(m[k][j]) & 0x7fffffffu;
        mc[j] = max(int((mag + dither[j]) >> 20) - mb, 0);
        vc[j] = max(int((vbits + dither[j]) >> 20) - vb, int(min(vbits, 1u)));
      }
      // (the signs are the top bits of the patterns)
      const unsigned tops = __byte_perm(__byte_perm(__float_as_uint(m[k][0]), __float_as_uint(m[k][1]), 0x0073),
                                        __byte_perm(__float_as_uint(m[k][2]), __float_as_uint(m[k][3]), 0x0073), 0x5410);
      store_codes(static_cast<unsigned char*>(t.m) + e, n[k], bytes4(mc) | (tops & 0x80808080u));
      store_codes(static_cast<unsigned char*>(t.v) + e, n[k], bytes4(vc));
    }
  }
}

template <int N, int BITS, bool FINE>
__global__ void __launch_bounds__(256, ADAMW_CTAS) adamw_list_kernel(const __grid_constant__ AdamwList<N> list) {
  chain_trigger();
  chain_wait();
  extern __shared__ __align__(16) unsigned char raw[];
  AdamwRing<BITS>& ring = *reinterpret_cast<AdamwRing<BITS>*>(raw);
  const int lane = threadIdx.x & 31;
  const long all = list.end[list.count - 1], stride = gridDim.x * 8L, first = blockIdx.x * 8L + (threadIdx.x >> 5);
  // a block on its way: its tensor, its number in it, and its bases (m's below, v's above)
  struct Asked {
    int i, bases;
    long block;
  };
  long ask = first;
  int ask_i = 0;
  // the tensor of the first block, looked for by halves; of later ones from there on
  for (int top = list.count - 1; ask_i < top;) {
    const int mid = (ask_i + top) >> 1;
    if (ask >= list.end[mid]) ask_i = mid + 1;
    else top = mid;
  }
  auto request = [&](int slot) {
    Asked x = {0, 0, 0};
    if (ask < all) {
      while (ask >= list.end[ask_i]) ++ask_i;
      const AdamwTensor& t = list.t[ask_i];
      x.i = ask_i;
      x.block = ask - (ask_i > 0 ? list.end[ask_i - 1] : 0);
      if ((x.block + 1) * ADAMW_BLOCK <= t.n) adamw_request<BITS>(ring, slot, t, x.block * ADAMW_BLOCK + lane * 4);
      if (BITS == 8) x.bases = int(static_cast<unsigned short>(t.mb[x.block])) | int(t.vb[x.block]) << 16;
      ask += stride;
    }
    ring_commit();
    return x;
  };
  Asked next = request(0);
  int slot = 0;
  for (long at = first; at < all; at += stride) {
    const Asked now = next;
    next = request(slot ^ 1);
    ring_wait<1>();
    const AdamwTensor& t = list.t[now.i];
    AdamwLane<BITS> x;
    if ((now.block + 1) * ADAMW_BLOCK <= t.n) {
      adamw_take<BITS>(x, ring, slot, t.grad_f32);
      adamw_block<BITS, FINE, true>(x, t, list.h, now.block, lane, now.bases & 0xffff, now.bases >> 16);
    } else {
      if (t.grad_f32) adamw_load<BITS, float>(x, t, now.block * ADAMW_BLOCK + lane * 4);
      else adamw_load<BITS, __nv_bfloat16>(x, t, now.block * ADAMW_BLOCK + lane * 4);
      adamw_block<BITS, FINE, false>(x, t, list.h, now.block, lane, now.bases & 0xffff, now.bases >> 16);
    }
    slot ^= 1;
  }
}

// out = what a tensor's codes stand for; eight of them a thread, n of the last thread's
template <typename T>
__global__ void __launch_bounds__(256) moment_values_kernel(const unsigned char* m, const short* mb, const unsigned char* v,
                                                            const short* vb, T* m_out, T* v_out, long n) {
  chain_trigger();
  chain_wait();
  const long e = (blockIdx.x * 256L + threadIdx.x) * 8;
  if (e >= n) return;
  const unsigned bm = unsigned(mb[e / ADAMW_BLOCK]) << 20, bv = unsigned(vb[e / ADAMW_BLOCK]) << 20;
  const int k[2] = {n - e >= 4 ? 4 : int(n - e), n - e >= 8 ? 4 : n - e > 4 ? int(n - e - 4) : 0};
  unsigned mu[2], vu[2];
  if (k[1] == 4) {
    const uint2 a = *reinterpret_cast<const uint2*>(m + e), b = *reinterpret_cast<const uint2*>(v + e);
    mu[0] = a.x; mu[1] = a.y; vu[0] = b.x; vu[1] = b.y;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mu[i] = load_codes(m + e + 4 * i, k[i]);
      vu[i] = load_codes(v + e + 4 * i, k[i]);
    }
  }
  float a[2][4], b[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    decode_m4(mu[i], bm, a[i]);
    decode_v4(vu[i], bv, b[i]);
  }
  if (sizeof(T) == 2 && k[1] == 4) {
    *reinterpret_cast<uint4*>(m_out + e) = make_uint4(pack_bf16x2(a[0][0], a[0][1]), pack_bf16x2(a[0][2], a[0][3]),
                                                      pack_bf16x2(a[1][0], a[1][1]), pack_bf16x2(a[1][2], a[1][3]));
    *reinterpret_cast<uint4*>(v_out + e) = make_uint4(pack_bf16x2(b[0][0], b[0][1]), pack_bf16x2(b[0][2], b[0][3]),
                                                      pack_bf16x2(b[1][0], b[1][1]), pack_bf16x2(b[1][2], b[1][3]));
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    store4(m_out + e + 4 * i, k[i], a[i]);
    store4(v_out + e + 4 * i, k[i], b[i]);
  }
}

template <int N, int BITS, bool FINE>
static int adamw_launch(const AdamwTensor* t, int count, const AdamwHyper& h, cudaStream_t stream) {
  AdamwList<N> list;
  list.count = count;
  list.h = h;
  long blocks = 0;
  for (int i = 0; i < count; ++i) {
    list.t[i] = t[i];
    blocks += (t[i].n + ADAMW_BLOCK - 1) / ADAMW_BLOCK;
    list.end[i] = blocks;
  }
  if (blocks == 0) return 0;
  const long want = (blocks + 7) / 8, cap = long(num_sms()) * ADAMW_CTAS;
  auto kern = adamw_list_kernel<N, BITS, FINE>;
  static SharedLimit limit;
  ZB_CUDA_OK(limit.raise(kern, sizeof(AdamwRing<BITS>)));
  ZB_CUDA_OK(launch_pass(kern, int(want < cap ? want : cap), 256, sizeof(AdamwRing<BITS>), stream, list));
  return 0;
}

// The fast root takes a v below 2^-126 as 0, which takes at most 2^-63 / sqrt(1 - b2^k) from the divisor: no more than half an fp32
// step of an eps of ordinary size.  Where it may be more, the root that keeps subnormals is taken; moments in 32 bits, bound by memory,
// always take that one (8 bits, 8 x 61 million parameters: 1.455 ms instead of 1.41).
static bool fine_root(const AdamwTensor* t, int count, float eps) {
  for (int i = 0; i < count; ++i)
    if (!(t[i].inv_bc2 * 0x1p-39f <= eps)) return true;
  return false;
}
template <int N>
static int adamw_launch(int bits, const AdamwTensor* t, int count, const AdamwHyper& h, cudaStream_t stream) {
  if (bits == 32) return adamw_launch<N, 32, true>(t, count, h, stream);
  return fine_root(t, count, h.eps) ? adamw_launch<N, 8, true>(t, count, h, stream) : adamw_launch<N, 8, false>(t, count, h, stream);
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
    const int rc = n <= 32 ? adamw_launch<32>(bits, t + i, n, h, stream) : adamw_launch<256>(bits, t + i, n, h, stream);
    if (rc) return rc;
  }
  return 0;
}

int zb_moment_values(const void* m, const void* mb, const void* v, const void* vb, void* m_out, void* v_out, long n, int out_f32,
                     cudaStream_t stream) {
  using namespace zb;
  if (n <= 0) return 0;
  if (((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 7) ||
      ((reinterpret_cast<uintptr_t>(m_out) | reinterpret_cast<uintptr_t>(v_out)) & 15))
    ZB_FAIL(-1, "moment_values: codes must be 8-byte aligned, values 16");
  if ((n + 2047) / 2048 > 0x7fffffffL) ZB_FAIL(-1, "moment_values: %ld values", n);
  const int grid = int((n + 2047) / 2048);
  const unsigned char *mc = static_cast<const unsigned char*>(m), *vc = static_cast<const unsigned char*>(v);
  const short *bm = static_cast<const short*>(mb), *bv = static_cast<const short*>(vb);
  if (out_f32)
    ZB_CUDA_OK(launch_pass(moment_values_kernel<float>, grid, 256, 0, stream, mc, bm, vc, bv, static_cast<float*>(m_out),
                           static_cast<float*>(v_out), n));
  else
    ZB_CUDA_OK(launch_pass(moment_values_kernel<__nv_bfloat16>, grid, 256, 0, stream, mc, bm, vc, bv,
                           static_cast<__nv_bfloat16*>(m_out), static_cast<__nv_bfloat16*>(v_out), n));
  return 0;
}

}  // extern "C"
