// Plan of a packed batch, made once and used by every layer: bounds and position of each token, and the order in which
// tiles are dealt to the SMs.
//
// bounds[t] is found by halves in the offsets (12 dependent loads for 4096 sequences), one thread a token.  The work of a tile
// follows from the bounds of its first and last token; a tile's place in an order is the number of tiles with more work (or
// as much and a lower index), counted against all of them.  With sequences of mixed lengths the tiles with the most
// work lie anywhere; whoever is dealt one of them last keeps the GPU waiting for it.
//
// Offsets are clamped to [0, T] and a token counts as one of a sequence only if it lies between the sequence's offsets,
// so offsets that do not rise give tiles of no meaning but no access outside the batch.
#include "packed.cuh"

namespace zb {

// The sequence of token t: the last offset that is not behind it.
__device__ __forceinline__ int2 bounds_of(const int* offsets, int n, int T, int total, int t) {
  if (t >= total) return make_int2(total, total);
  int lo = 0, hi = n;   // offsets[lo] <= t < offsets[hi], if they rise
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= t) lo = mid; else hi = mid;
  }
  const int b = min(max(offsets[lo], 0), T), e = min(max(offsets[hi], 0), T);
  return b <= t && t < e ? make_int2(b, e) : make_int2(total, total);
}

constexpr int PACK_THREADS = 256;

// Blocks [0, token_blocks): tokens.  The rest: places in the three orders, one tile a thread.
__global__ void __launch_bounds__(PACK_THREADS)
pack_sequences_kernel(const int* offsets, int n, int T, int padded, int token_blocks, int2* bounds, int* positions, int* order_pairs,
                      int* order_tiles, int* order_keys) {
  chain_trigger();
  chain_wait();
  const int total = n > 0 ? min(max(offsets[n], 0), T) : 0;
  if (int(blockIdx.x) < token_blocks) {
    const int t = int(blockIdx.x) * PACK_THREADS + int(threadIdx.x);
    const int2 b = bounds_of(offsets, n, T, total, t);
    bounds[t] = b;
    if (t < T) positions[t] = b.x < b.y ? t - b.x : 0;
    return;
  }
  const int pairs = padded / 256, tiles = (T + 127) / 128;
  int block = int(blockIdx.x) - token_blocks;
  const int pair_blocks = (pairs + PACK_THREADS - 1) / PACK_THREADS, tile_blocks = (tiles + PACK_THREADS - 1) / PACK_THREADS;
  int which = 0, count = pairs, rows = 256;
  if (block >= pair_blocks) {
    block -= pair_blocks;
    which = 1 + block / tile_blocks;
    block %= tile_blocks;
    count = tiles;
    rows = 128;
  }
  // keys of a causal query tile, queries of a causal key tile
  auto work = [&](int i) {
    const int first = i * rows, last = min(first + rows, T);
    return which == 2 ? max(bounds_of(offsets, n, T, total, min(last, total) - 1).y - first, 0)
                      : max(last - bounds_of(offsets, n, T, total, first).x, 0);
  };
  __shared__ int others[PACK_THREADS];
  const int mine = block * PACK_THREADS + int(threadIdx.x);
  const int my_work = mine < count ? work(mine) : 0;
  int place = 0;
  for (int base = 0; base < count; base += PACK_THREADS) {
    __syncthreads();
    if (base + int(threadIdx.x) < count) others[threadIdx.x] = work(base + int(threadIdx.x));
    __syncthreads();
    const int m = min(PACK_THREADS, count - base);
    for (int j = 0; j < m; ++j) place += others[j] > my_work || (others[j] == my_work && base + j < mine);
  }
  if (mine < count) (which == 0 ? order_pairs : which == 1 ? order_tiles : order_keys)[place] = mine;
}

}  // namespace zb

// offsets [n + 1] on the device: where the sequences begin, and the last one's end.  bounds [2 padded] with padded = T rounded up to a
// multiple of 256, positions [T], order_pairs [padded / 256], order_tiles and order_keys [(T + 127) / 128].
extern "C" int zb_pack_sequences(const int* offsets, int n, int T, void* bounds, int* positions, int* order_pairs, int* order_tiles,
                                 int* order_keys, cudaStream_t stream) {
  using namespace zb;
  if (T <= 0) return 0;
  if (T > 65535 * 128) ZB_FAIL(-1, "attention: %d packed tokens, at most %d", T, 65535 * 128);
  const int padded = packed_view(nullptr, T).padded, token_blocks = padded / PACK_THREADS;
  const int tile_blocks = ((T + 127) / 128 + PACK_THREADS - 1) / PACK_THREADS, pair_blocks = (padded / 256 + PACK_THREADS - 1) / PACK_THREADS;
  ZB_CUDA_OK(launch_pass(pack_sequences_kernel, dim3(token_blocks + pair_blocks + 2 * tile_blocks), PACK_THREADS, 0, stream, offsets, n, T,
                         padded, token_blocks, static_cast<int2*>(bounds), positions, order_pairs, order_tiles, order_keys));
  return 0;
}
