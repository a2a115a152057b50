// What the attention kernels know of a packed batch: sequences of different lengths, one after another, in one stream of T
// tokens.  bounds[t] = {begin, end} of the sequence that token t belongs to; tokens behind the last sequence, up to the next
// multiple of 256, have {total, total}, `total` being the end of the last sequence.  Both numbers never fall from a token
// to the next, so the first and the last row of a tile tell which tiles of the other side it meets.
#pragma once
#include <cuda_runtime.h>
#include "../common/host.h"
#include "../common/ptx.cuh"

namespace zb {

constexpr int PACK_PAD = 256;
#define PACKED_NAN __uint_as_float(0x7fc00000u)

// A tile (or pair of tiles) as it is dealt out, with all that a CTA needs before it knows its loads: read in one go.
struct alignas(16) PackedTile {
  int2 first, last;         // bounds of its first and last row
  int tile, total;          // total: the end of the last sequence; -1: the offsets did not rise, and results are NaN
  int unused[2];
};
struct alignas(16) PackedPair {
  int2 first[2], last[2];   // of the two tiles
  int pair, total;
  int unused[2];
};
struct PackedView {
  const int2* bounds;
  const PackedPair* pairs;  // pairs of query tiles in the order of the plan
  const PackedTile* tiles;  // query or key tiles likewise
};
template <typename T>
__device__ __forceinline__ T load_packed(const T* p) {
  T r;
  uint4* to = reinterpret_cast<uint4*>(&r);
#pragma unroll
  for (int i = 0; i < int(sizeof(T) / 16); ++i) to[i] = ld_v4(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
inline int packed_rows(int T) { return (T + PACK_PAD - 1) / PACK_PAD * PACK_PAD; }   // entries of bounds

// Sizes that the packed kernels take: tiles are the grid's second dimension, at most 65535 of 128 rows.
inline int packed_check(int T, int Hq, int Hkv, int D) {
  if (Hkv <= 0 || Hq % Hkv != 0) ZB_FAIL(-1, "attention: Hq=%d not a multiple of Hkv=%d", Hq, Hkv);
  if (D != 64 && D != 128) ZB_FAIL(-1, "attention: head dim %d unsupported (64 or 128)", D);
  if (T > 65535 * 128) ZB_FAIL(-1, "attention: %d packed tokens, at most %d", T, 65535 * 128);
  if (Hq > 65535) ZB_FAIL(-1, "attention: %d heads", Hq);
  return 0;
}

struct KeyRange {
  int lo, hi;
};
// Keys that the rows [q0, q0 + 128) of a query tile see between them; `first`, `last`: bounds of its first and last row.
__device__ __forceinline__ KeyRange key_range(int2 first, int2 last, int q0, int causal, int window) {
  KeyRange r;
  r.lo = window > 0 ? max(first.x, q0 - window + 1) : first.x;
  r.hi = causal ? min(q0 + 128, last.y) : last.y;
  return r;
}
// Queries that see the keys [k0, k0 + 128) of a key tile.
__device__ __forceinline__ KeyRange query_range(int2 first, int2 last, int k0, int causal, int window) {
  KeyRange r;
  r.lo = causal ? k0 : first.x;
  r.hi = window > 0 ? min(last.y, k0 + 127 + window) : last.y;
  return r;
}

// Rows [from, ROWS) of a tile of ROWS rows (64-column blocks of 128-byte rows) become zeros, for the products that a whole warp is
// about to issue.  Only the tile that the last sequence ends in has any: what lies behind it may be anything.
template <int D, int ROWS = 128>
__device__ __forceinline__ void clear_tail_rows(uint32_t tile, int from, int lane) {
  if (from >= ROWS) return;   // (the same for the whole warp)
#pragma unroll 1
  for (int i = max(from, 0) * 8 + lane; i < ROWS * 8; i += 32)
#pragma unroll
    for (int b = 0; b < D / 64; ++b) st_shared_v4(tile + uint32_t(b * ROWS * 128 + i * 16), 0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  __syncwarp();
}

}  // namespace zb
