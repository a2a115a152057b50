// Plan of a packed batch, made once and used by every layer: bounds and position of each token, and the order in which
// tiles are dealt to the SMs.
//
// bounds[t] is found by halves in the offsets (12 dependent loads for 4096 sequences), one thread a token.  Tiles are dealt sequence by
// sequence, the longest first, and within one by falling work: whoever is dealt a long tile last keeps the GPU waiting for it, and
// what neighbours in the order read lies in one sequence and stays in L2.  (By falling work alone, all sequences side by side, 16 x
// 1024 tokens with 32 / 8 heads of 128 took 705 us backward and 224 forward.)  A tile's place is the number of tiles ahead of it,
// counted against all of them.
//
// Offsets that do not rise from 0 to at most T cannot be refused without a wait for the GPU.  Their plan has no sequences and -1 for their end, at
// which the attention kernels write NaN: a result that nobody takes for one.  Every block looks at all offsets for itself (one comparison a thread for
// 256 sequences); of more than PACK_SCAN a block of their own does, ahead of the plan.
#include "packed.cuh"

namespace zb {

// The sequence of token t: the last offset that is not behind it.  (total: 0 for offsets that do not rise, whose other values are not used)
__device__ __forceinline__ int2 bounds_of(const int* offsets, int n, int total, int t) {
  if (t >= total) return make_int2(total, total);
  int lo = 0, hi = n;   // offsets[lo] <= t < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= t) lo = mid; else hi = mid;
  }
  return make_int2(offsets[lo], offsets[hi]);
}

constexpr int PACK_THREADS = 256, PACK_SCAN = 4096;

// Whether offsets [n + 1] are anything but rising from 0 to at most T; for all threads of a block.
__device__ __forceinline__ bool offsets_wrong(const int* offsets, int n, int T) {
  bool wrong = false;
  for (int i = int(threadIdx.x); i <= n; i += int(blockDim.x)) {
    const int o = offsets[i];
    wrong = wrong || o > T || (i == 0 ? o != 0 : o < offsets[i - 1]);
  }
  return __syncthreads_or(wrong);
}
__global__ void __launch_bounds__(1024) offsets_wrong_kernel(const int* offsets, int n, int T, int* found) {
  chain_trigger();
  chain_wait();
  const bool wrong = offsets_wrong(offsets, n, T);
  if (threadIdx.x == 0) *found = wrong;
}

// Blocks [0, token_blocks): tokens.  The rest: places in the three orders, one tile a thread.
__global__ void __launch_bounds__(PACK_THREADS)
pack_sequences_kernel(const int* offsets, int n, int T, int padded, int token_blocks, int2* bounds, int* positions, PackedPair* pairs_out,
                      PackedTile* tiles_out, PackedTile* keys_out, const int* found) {
  chain_trigger();
  chain_wait();
  const bool wrong = n > PACK_SCAN ? *found != 0 : offsets_wrong(offsets, n, T);
  const int total = n > 0 && !wrong ? offsets[n] : 0, end = wrong ? -1 : total;
  if (int(blockIdx.x) < token_blocks) {
    const int t = int(blockIdx.x) * PACK_THREADS + int(threadIdx.x);
    const int2 b = bounds_of(offsets, n, total, t);
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
  // A query tile reads most from the sequence of its first row, whose earlier tiles read less; a key tile is read most by that of its last
  // row, whose later tiles are read less.
  auto key = [&](int i) {
    const int row = which == 2 ? min(i * rows + rows, max(total, 1)) - 1 : i * rows;
    const int2 b = bounds_of(offsets, n, total, which == 2 ? max(row, i * rows) : row);
    return (static_cast<unsigned long long>(0xffffff - (b.y - b.x)) << 40) | (static_cast<unsigned long long>(b.x) << 16) |
           static_cast<unsigned long long>(which == 2 ? i : 0xffff - i);
  };
  __shared__ unsigned long long others[PACK_THREADS];
  const int mine = block * PACK_THREADS + int(threadIdx.x);
  const unsigned long long my_key = mine < count ? key(mine) : 0;
  int place = 0;
  for (int base = 0; base < count; base += PACK_THREADS) {
    __syncthreads();
    if (base + int(threadIdx.x) < count) others[threadIdx.x] = key(base + int(threadIdx.x));
    __syncthreads();
    const int m = min(PACK_THREADS, count - base);
    for (int j = 0; j < m; ++j) place += others[j] < my_key;
  }
  if (mine >= count) return;
  if (which == 0) {
    PackedPair r = {};
    r.pair = mine;
    r.total = end;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      r.first[c] = bounds_of(offsets, n, total, mine * 256 + c * 128);
      r.last[c] = bounds_of(offsets, n, total, mine * 256 + c * 128 + 127);
    }
    pairs_out[place] = r;
  } else {
    PackedTile r = {};
    r.tile = mine;
    r.total = end;
    r.first = bounds_of(offsets, n, total, mine * 128);
    r.last = bounds_of(offsets, n, total, mine * 128 + 127);
    (which == 1 ? tiles_out : keys_out)[place] = r;
  }
}

}  // namespace zb

// offsets [n + 1] on the device: where the sequences begin, and the last one's end.  bounds [2 padded] with padded = T rounded up to a
// multiple of 256, positions [T], order_pairs [padded / 256] PackedPair, order_tiles and order_keys [(T + 127) / 128] PackedTile; scratch: an int.
extern "C" int zb_pack_sequences(const int* offsets, int n, int T, void* bounds, int* positions, void* order_pairs, void* order_tiles,
                                 void* order_keys, int* scratch, cudaStream_t stream) {
  using namespace zb;
  if (T <= 0) return 0;
  if (T > 65535 * 128) ZB_FAIL(-1, "attention: %d packed tokens, at most %d", T, 65535 * 128);
  const int padded = packed_rows(T), token_blocks = padded / PACK_THREADS;
  const int tile_blocks = ((T + 127) / 128 + PACK_THREADS - 1) / PACK_THREADS, pair_blocks = (padded / 256 + PACK_THREADS - 1) / PACK_THREADS;
  if (n > PACK_SCAN) ZB_CUDA_OK(launch_pass(offsets_wrong_kernel, dim3(1), 1024, 0, stream, offsets, n, T, scratch));
  ZB_CUDA_OK(launch_pass(pack_sequences_kernel, dim3(token_blocks + pair_blocks + 2 * tile_blocks), PACK_THREADS, 0, stream, offsets, n, T,
                         padded, token_blocks, static_cast<int2*>(bounds), positions, static_cast<PackedPair*>(order_pairs),
                         static_cast<PackedTile*>(order_tiles), static_cast<PackedTile*>(order_keys), static_cast<const int*>(scratch)));
  return 0;
}
