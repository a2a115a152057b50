// Token embedding with a scale, and its gradient summed token by token:
//   forward   out[t] = scale table[id_t] (+ pos[t mod S + off])
//   backward  gtable[v] += scale sum over t with id_t = v of dout[t],  gpos[p + off] += sum over t with t mod S = p of dout[t]
// The gradient without atomics: the ids are sorted together with their positions (equal ids keep the order of their
// positions), and every row of the table that occurs is read, added to and written once, by the sum of its terms in a fixed
// order, in fp32.  So the result is the same on each run, a token that occurs thousands of times does not queue up at one
// address, and in a bf16 bucket a row is rounded once and not once for every occurrence.
// Ids outside [0, V) count as the nearest inside, as in the gather without a scale.
// The gather of 32768 rows of 2048 columns takes 36 us: 134 MB written and as many read, most of them from L2, 7.5 TB/s.  The
// gradient of 16384 tokens of 4096 columns into an fp32 table of 32000, a fifth of them one token, takes 71 us: 45 the sums
// themselves (296 MB, 6.5 TB/s), the rest the order of the ids and the runs over several pieces, both bound by latency.
// Against atomics, in a graph, us by atomics / by token: into fp32 tables 16384 tokens of 4096 columns with ids spread evenly 130 / 103,
// 16384 of 256 with a fifth one token 66 / 29, but 8192 of 2048 spread evenly 22 / 26 and 16384 of 64 3.1 / 15.5; into bf16 tables, where
// atomics take half the traffic and round at every occurrence, 16384 of 4096 56 / 71 and 16384 of 64 2.3 / 16.8.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../norm/norm_common.cuh"

namespace zb {

__device__ __forceinline__ int clamp_id(long id, int V) {
  return static_cast<unsigned long>(id) < static_cast<unsigned long>(V) ? int(id) : id < 0 ? 0 : V - 1;
}

// ------------------------------- forward -------------------------------
// 2^shift lanes share a row (all 32 from 256 columns up), every lane up to four chunks of it at once: an id is read once for a
// row and not for every chunk, and nothing is divided.
template <bool POS>
__global__ void __launch_bounds__(128) embedding_scaled_kernel(const long* ids, const __nv_bfloat16* table, const __nv_bfloat16* pos,
                                                               __nv_bfloat16* out, int T, int H, int V, int S, int off, float scale,
                                                               int shift) {
  chain_trigger();
  chain_wait();
  constexpr int U = 4;
  const int lane = threadIdx.x & 31, lanes = 1 << shift;
  const long t = ((blockIdx.x * 4L + (threadIdx.x >> 5)) << (5 - shift)) + (lane >> shift);
  if (t >= T) return;
  const __nv_bfloat16* src = table + long(clamp_id(ids[t], V)) * H;
  const __nv_bfloat16* add = POS ? pos + long(int(t) % S + off) * H : nullptr;
  for (int c0 = (lane & (lanes - 1)) * 8; c0 < H; c0 += U * lanes * 8) {
    uint4 row[U], at[POS ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * lanes * 8;
      if (c >= H) break;
      row[u] = ld_v4(src + c);
      if constexpr (POS) at[u] = ld_v4(add + c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * lanes * 8;
      if (c >= H) break;
      float a[8];
      unpack8(row[u], a);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] *= scale;
      if constexpr (POS) {
        float b[8];
        unpack8(at[u], b);
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] += b[j];
      }
      *reinterpret_cast<uint4*>(out + t * H + c) = pack8(a);
    }
  }
}

// ------------------------------- order of the ids -------------------------------
// Sorts the ids of a chunk together with their positions, equal ids in the order of their positions.  A CTA has `width` neighbouring
// ids of the vocabulary and looks at the whole chunk: its own are ranked among those of the same id (by a warp's match, and counts
// added over the warps), and how many ids are lower is counted on the way.  So no CTA needs another one, and there is one pass
// over the chunk, from L2: 11 us for 16384 ids of 32000; a cluster of CTAs that sorted in their shared memory digit by digit took 15.
// ROUNDS: ids of a thread (a chunk has at most 1024 times as many).
constexpr int SORT_BINS = 1024, SORT_CHUNK = 32 * 1024;
struct SortShared {
  unsigned short count[32][SORT_BINS];   // ids of a warp; then those of its CTA in warps before it
  int base[SORT_BINS];                   // where a bin begins in the chunk
  int scan[32], lower;
};
// order, sorted: [T]
template <int ROUNDS>
__global__ void __launch_bounds__(1024) embedding_sort_kernel(const long* ids, int* order, int* sorted, int T, int V, int width, int ctas) {
  chain_trigger();
  chain_wait();
  extern __shared__ __align__(16) unsigned char raw[];
  SortShared& sh = *reinterpret_cast<SortShared*>(raw);
  const int chunk = blockIdx.x / ctas, lo = (blockIdx.x - chunk * ctas) * width, first = chunk * SORT_CHUNK, n = min(T - first, SORT_CHUNK);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rounds = (n + 1023) >> 10, e0 = warp * rounds * 32 + lane;     // 32 ids a round, a warp's rounds in a row
  const int end = min(n, (warp + 1) * rounds * 32);
  const long* from = ids + first + e0;
  for (int i = lane * 8; i < width; i += 256) *reinterpret_cast<uint4*>(&sh.count[warp][i]) = make_uint4(0, 0, 0, 0);
  if (tid == 0) sh.lower = 0;
  int key[ROUNDS], below = 0;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int e = e0 + r * 32;
    key[r] = 1 << 30;
    if (e < end) key[r] = clamp_id(from[r * 32], V) - lo;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    if (r >= rounds) break;
    below += unsigned(key[r]) >> 31;
    const bool mine = unsigned(key[r]) < unsigned(width);
    const unsigned all = __ballot_sync(0xffffffffu, mine);
    if (all == 0) {
      key[r] = -1;
      continue;
    }
    int place = 0;
    if (mine) {
      const unsigned same = __match_any_sync(all, key[r]), lower = same & ((1u << lane) - 1);
      const int before = sh.count[warp][key[r]];
      place = before + __popc(lower);
      __syncwarp(all);
      if (lower == 0) sh.count[warp][key[r]] = static_cast<unsigned short>(before + __popc(same));
    }
    __syncwarp();
    key[r] = mine ? key[r] | place << 10 : -1;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
  if (lane == 0 && below) atomicAdd(&sh.lower, below);      // (whole numbers: the order does not matter)
  __syncthreads();
  // bin `tid`: over the warps, then over the bins
  int sum = 0;
  if (tid < width) {
#pragma unroll 8
    for (int w = 0; w < 32; ++w) {
      const int c = sh.count[w][tid];
      sh.count[w][tid] = static_cast<unsigned short>(sum);
      sum += c;
    }
  }
  int run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += v;
  }
  if (lane == 31) sh.scan[warp] = run;
  __syncthreads();
  if (warp == 0) {
    const int self = sh.scan[lane];
    int t = self;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += v;
    }
    sh.scan[lane] = t - self;
  }
  __syncthreads();
  sh.base[tid] = sh.lower + sh.scan[warp] + run - sum;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    if (r >= rounds) break;
    if (key[r] >= 0) {
      const int bin = key[r] & (SORT_BINS - 1), pos = sh.base[bin] + sh.count[warp][bin] + (key[r] >> 10);
      order[first + pos] = first + e0 + r * 32;
      sorted[first + pos] = lo + bin;
    }
  }
}

// More ids than a chunk: the chunks' orders become one.  An id's place is its place in its own chunk and, for each of the others, how many
// ids there come before it: the lower ones, and the equal ones of earlier chunks, found by halves.  (Neighbours in a chunk's order
// look for neighbouring ids, so their steps read the same lines.)
// Then every row of the table is rounded once, and read once: sums and runs chunk by chunk, each added to the table, took 243 us
// instead of 223 for 65536 tokens of 2048 columns of 128256 rows, 251 instead of 188 for 131072 of 768, a fifth of them one token, and
// 112 instead of 116 for 32769 of 2048, where the second chunk is one id.
__global__ void __launch_bounds__(256) embedding_merge_kernel(const int* order, const int* sorted, int* order_out, int* sorted_out, int T) {
  chain_trigger();
  chain_wait();
  const long i = blockIdx.x * 256L + threadIdx.x;
  if (i >= T) return;
  const int id = sorted[i], mine = int(i / SORT_CHUNK), chunks = (T + SORT_CHUNK - 1) / SORT_CHUNK;
  int place = int(i) - mine * SORT_CHUNK;
  for (int c = 0; c < chunks; ++c) {
    if (c == mine) continue;
    const int* ids = sorted + long(c) * SORT_CHUNK;
    const long most = c < mine ? long(id) + 1 : id;       // ids below this one come before
    int from = 0, to = min(T - c * SORT_CHUNK, SORT_CHUNK);
    while (from < to) {
      const int mid = (from + to) >> 1;
      if (ids[mid] < most) from = mid + 1;
      else to = mid;
    }
    place += from;
  }
  order_out[place] = order[i];
  sorted_out[place] = id;
}

// ------------------------------- sums by token -------------------------------
// The sorted rows are cut into pieces of K; a warp sums a piece over 256 columns.  A run of equal ids that lies within a piece
// goes straight to the table.  Of a run over several pieces, the first one leaves its part in `tail`, every further one in
// `head`, and embedding_join_kernel adds those up.
struct ByToken {
  const __nv_bfloat16* dout;
  const int *order, *sorted;      // n of them
  float *head, *tail;             // [pieces, H]
  int n, H;
  float scale;
};

// A lane's columns of a slice of 256: eight neighbours for a bf16 table, twice four for an fp32 one, 128 apart, so that every
// access of a warp is to whole 32-byte sectors (with eight fp32 neighbours a lane, sectors went by halves).
template <typename GT>
constexpr int VEC = sizeof(GT) == 4 ? 4 : 8;
template <typename GT>
constexpr int PARTS = 8 / VEC<GT>;

template <typename GT>
__device__ __forceinline__ int parts_of(int col, int H) {       // of a lane whose first column is col
  return col >= H ? 0 : PARTS<GT> == 2 && col + 128 < H ? 2 : 1;
}
__device__ __forceinline__ void unpack4(const uint4& u, float* f) {
  f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack4(const uint2& u, float* f) {
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
// A part of a table's row is 16 bytes; of a row of dout 8 or 16
template <typename GT>
__device__ __forceinline__ void unpack_grad(const uint4& u, float* f) {
  if constexpr (sizeof(GT) == 4) unpack4(u, f);
  else unpack8(u, f);
}
__device__ __forceinline__ void unpack_row(const uint2& u, float* f) { unpack4(u, f); }
__device__ __forceinline__ void unpack_row(const uint4& u, float* f) { unpack8(u, f); }
__device__ __forceinline__ void store_part(float* p, const float* f) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
__device__ __forceinline__ void store_part(__nv_bfloat16* p, const float* f) { *reinterpret_cast<uint4*>(p) = pack8(f); }
template <typename GT>
struct RowPart;
template <>
struct RowPart<float> {
  using type = uint2;
};
template <>
struct RowPart<__nv_bfloat16> {
  using type = uint4;
};
__device__ __forceinline__ void ring_load(uint4* to, const void* from) { ring_load16(to, from); }
__device__ __forceinline__ void ring_load(uint2* to, const void* from) { ring_load8(to, from); }
__device__ __forceinline__ uint2 ld_v2(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ void load_row(uint2& u, const void* p) { u = ld_v2(p); }
__device__ __forceinline__ void load_row(uint4& u, const void* p) { u = ld_v4(p); }
// VEC sums in fp32, in shared memory or a workspace
template <typename GT>
__device__ __forceinline__ void store_sums(float* p, const float* f) {
#pragma unroll
  for (int k = 0; k < VEC<GT>; k += 4) store_part(p + k, f + k);
}

// Rows lie anywhere, so what bounds a warp is how many of them are on their way: every lane copies its parts of the rows to come
// (and of the table's, which a run's end will add to) into its own places of a ring in shared memory.
constexpr int PIECE_RING = 4;
template <typename GT>
struct PieceRing {
  typename RowPart<GT>::type row[PIECE_RING][PARTS<GT>][256];
  uint4 old[PIECE_RING][PARTS<GT>][256];
};
template <int K, typename GT>
__global__ void __launch_bounds__(256) embedding_pieces_kernel(const ByToken a, GT* table) {
  chain_trigger();
  chain_wait();
  extern __shared__ __align__(16) unsigned char raw[];
  PieceRing<GT>& ring = *reinterpret_cast<PieceRing<GT>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, slices = (a.H + 255) >> 8, pieces = (a.n - 1) / K + 1;
  const int item = blockIdx.x * 8 + (tid >> 5);
  if (item >= pieces * slices) return;
  constexpr int V = VEC<GT>, P = PARTS<GT>;
  const int piece = item / slices, from = piece * K, rows = min(K, a.n - from);
  const int col = (item - piece * slices) * 256 + lane * V, parts = parts_of<GT>(col, a.H);
  const int id = lane < rows ? a.sorted[from + lane] : -1, at = lane < rows ? a.order[from + lane] : 0;
  const int prev = from > 0 ? a.sorted[from - 1] : -1, next = from + rows < a.n ? a.sorted[from + rows] : -1;
  int after = __shfl_down_sync(0xffffffffu, id, 1);
  if (lane == rows - 1) after = next;
  const unsigned ends = __ballot_sync(0xffffffffu, lane < rows && id != after);
  const bool goes_on = prev >= 0 && prev == __shfl_sync(0xffffffffu, id, 0);   // the first run began in an earlier piece
  const int first_end = goes_on ? __ffs(ends) - 1 : -1;
  auto request = [&](int j, int slot) {
    if (j < rows) {
      const __nv_bfloat16* row = a.dout + size_t(__shfl_sync(0xffffffffu, at, j)) * a.H + col;
#pragma unroll
      for (int k = 0; k < P; ++k)
        if (k < parts) ring_load(&ring.row[slot][k][tid], row + 128 * k);
      if ((ends >> j & 1) && j != first_end) {
        const GT* old = table + size_t(__shfl_sync(0xffffffffu, id, j)) * a.H + col;
#pragma unroll
        for (int k = 0; k < P; ++k)
          if (k < parts) ring_load16(&ring.old[slot][k][tid], old + 128 * k);
      }
    }
    ring_commit();
  };
#pragma unroll
  for (int j = 0; j < PIECE_RING - 1; ++j) request(j, j);
  float acc[8] = {};
  auto leave = [&](float* to) {
#pragma unroll
    for (int k = 0; k < P; ++k)
      if (k < parts) store_sums<GT>(to + size_t(piece) * a.H + col + 128 * k, acc + V * k);
  };
  for (int j0 = 0; j0 < rows; j0 += PIECE_RING) {
#pragma unroll
    for (int slot = 0; slot < PIECE_RING; ++slot) {
      const int j = j0 + slot;
      request(j + PIECE_RING - 1, (slot + PIECE_RING - 1) % PIECE_RING);
      ring_wait<PIECE_RING - 1>();
      if (j >= rows) break;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        if (k >= parts) break;
        float f[V];
        unpack_row(ring.row[slot][k][tid], f);
#pragma unroll
        for (int i = 0; i < V; i += 2) fadd2(acc[V * k + i], acc[V * k + i + 1], acc[V * k + i], acc[V * k + i + 1], f[i], f[i + 1]);
      }
      if (!(ends >> j & 1)) continue;
      if (j == first_end) {
        leave(a.head);
      } else {
        GT* dst = table + size_t(__shfl_sync(0xffffffffu, id, j)) * a.H + col;
#pragma unroll
        for (int k = 0; k < P; ++k) {
          if (k >= parts) break;
          float old[V];
          unpack_grad<GT>(ring.old[slot][k][tid], old);
#pragma unroll
          for (int i = 0; i < V; ++i) old[i] += a.scale * acc[V * k + i];
          store_part(dst + 128 * k, old);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    }
  }
  if (!(ends >> (rows - 1) & 1)) leave(goes_on && ends == 0 ? a.head : a.tail);
}

// Runs over several pieces: a CTA looks at eight pieces and 256 columns, a warp at one piece.  What begins in it and goes on is
// its tail and the heads that follow, up to the run's last piece; runs over more than JOIN_ALONE pieces are added by the whole CTA,
// each warp a stretch of the heads, the stretches in order.
constexpr int JOIN_ALONE = 16;
template <typename GT>
__device__ __forceinline__ void add_to_row(GT* dst, const uint4 (&old)[2], int parts, float scale, const float (&acc)[8]) {
#pragma unroll
  for (int k = 0; k < PARTS<GT>; ++k) {
    if (k >= parts) break;
    float f[VEC<GT>];
    unpack_grad<GT>(old[k], f);
#pragma unroll
    for (int i = 0; i < VEC<GT>; ++i) f[i] += scale * acc[VEC<GT> * k + i];
    store_part(dst + 128 * k, f);
  }
}
template <typename GT>
__device__ __forceinline__ void load_old(const GT* src, int parts, uint4 (&old)[2]) {
#pragma unroll
  for (int k = 0; k < PARTS<GT>; ++k)
    if (k < parts) old[k] = ld_v4(src + 128 * k);
}
template <int K, typename GT>
__global__ void __launch_bounds__(256, 3) embedding_join_kernel(const ByToken a, GT* table) {
  chain_trigger();
  chain_wait();
  constexpr int P = PARTS<GT>;
  __shared__ int run_last[8];
  __shared__ __align__(16) float part[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slices = (a.H + 255) >> 8, pieces = (a.n - 1) / K + 1;
  const int group = blockIdx.x / slices, col = (blockIdx.x - group * slices) * 256 + lane * VEC<GT>, parts = parts_of<GT>(col, a.H);
  // a lane's columns of a row of sums
  auto load_sums = [&](const float* rows, int q, uint4 (&u)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      u[k] = make_uint4(0, 0, 0, 0);
      if (P == 2 ? k < parts : parts > 0) u[k] = ld_v4(rows + size_t(q) * a.H + col + (P == 2 ? 128 : 4) * k);
    }
  };
  int piece = group * 8 + warp, last = -1;
  uint4 old[2], tail[2], head[2];
  if (piece < pieces - 1) {
    const int end = (piece + 1) * K, id = a.sorted[end - 1], next = a.sorted[end], prev = piece == 0 ? -1 : a.sorted[piece * K - 1];
    if (next == id && prev != id) {
      load_old(table + size_t(id) * a.H + col, parts, old);
      load_sums(a.tail, piece, tail);
      load_sums(a.head, piece + 1, head);
      // the run's last piece: the first one behind this that the run does not leave, 32 looked at together
      for (last = piece + 1;; last += 32) {
        const long behind = long(last + lane + 1) * K;
        const unsigned stops = __ballot_sync(0xffffffffu, behind >= a.n || a.sorted[behind] != id);
        if (stops) {
          last += __ffs(stops) - 1;
          break;
        }
      }
    }
  }
  auto add_sums = [&](const uint4 (&u)[2], float (&acc)[8]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float f[4];
      unpack4(u[k], f);
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[4 * k + x] += f[x];
    }
  };
  auto add_heads = [&](int from, int to, float (&acc)[8]) {
    constexpr int U = 4;
    for (int q = from; q < to; q += U) {
      uint4 u[U][2];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (q + i < to) load_sums(a.head, q + i, u[i]);
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (q + i < to) add_sums(u[i], acc);
    }
  };
  const bool together = last - piece > JOIN_ALONE;
  if (last >= 0 && !together) {
    float acc[8] = {};
    add_sums(tail, acc);
    add_sums(head, acc);
    add_heads(piece + 2, last + 1, acc);
    add_to_row(table + size_t(a.sorted[(piece + 1) * K]) * a.H + col, old, parts, a.scale, acc);
  }
  if (lane == 0) run_last[warp] = together && last >= 0 ? last : -1;
  __syncthreads();
  for (int w = 0; w < 8; ++w) {
    const int end = run_last[w];
    if (end < 0) continue;
    piece = group * 8 + w;
    const int heads = end - piece, stretch = (heads + 7) / 8, from = piece + 1 + warp * stretch;
    float acc[8] = {};
    if (warp == 0) {
      load_sums(a.tail, piece, tail);
      add_sums(tail, acc);
    }
    add_heads(from, min(from + stretch, end + 1), acc);
#pragma unroll
    for (int k = 0; k < 8; ++k) part[warp][k * 32 + lane] = acc[k];
    __syncthreads();
    if (warp == 0) {
      GT* dst = table + size_t(a.sorted[(piece + 1) * K]) * a.H + col;
      load_old(dst, parts, old);
      for (int v = 1; v < 8; ++v) {
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] += part[v][k * 32 + lane];
      }
      add_to_row(dst, old, parts, a.scale, acc);
    }
    __syncthreads();
  }
}

// Few tokens: no order is needed.  A CTA has one token and 256 columns, looks for the token's id among all ids and, where the token is
// the first with it, adds up the rows of all, each warp a stretch of them.  One launch: in a graph 256 tokens of 512 columns 3.0 us
// against 10.0 by sorting, 1024 of 512, a fifth of them one token, 6.9 against 12.4; 1024 of 2048, four times as many CTAs, 16.1
// against 12.1.
constexpr int SMALL_T = 1024, SMALL_CTAS = 2048;
template <typename GT>
__global__ void __launch_bounds__(256) embedding_small_kernel(const long* ids, const __nv_bfloat16* dout, GT* table, int T, int H, int V,
                                                              float scale) {
  chain_trigger();
  chain_wait();
  constexpr int W = VEC<GT>, P = PARTS<GT>;
  __shared__ unsigned found[SMALL_T / 32];
  __shared__ unsigned short list[SMALL_T];
  __shared__ __align__(16) float part[8][256];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, slices = (H + 255) >> 8;
  const int t = blockIdx.x / slices, col = (blockIdx.x - t * slices) * 256 + lane * W, parts = parts_of<GT>(col, H);
  const int id = clamp_id(ids[t], V);
#pragma unroll
  for (int r = 0; r < SMALL_T / 256; ++r) {
    const int e = r * 256 + tid;
    const unsigned m = __ballot_sync(0xffffffffu, e < T && clamp_id(ids[e < T ? e : 0], V) == id);
    if (lane == 0) found[r * 8 + warp] = m;
  }
  __syncthreads();
  // (every warp by itself) how many there are, and whether one lies before t
  const unsigned word = found[lane];
  const int at = lane * 32;
  const unsigned early = at + 32 <= t ? word : at <= t ? word & ((1u << (t - at)) - 1) : 0;
  if (__any_sync(0xffffffffu, early != 0)) return;                 // the same for the whole CTA
  int run = __popc(word);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += v;
  }
  const int m = __shfl_sync(0xffffffffu, run, 31);
  if (warp == 0) {
    int k = run - __popc(word);
    for (unsigned w = word; w; w &= w - 1) list[k++] = static_cast<unsigned short>(at + __ffs(w) - 1);
  }
  GT* dst = table + size_t(id) * H + col;
  uint4 old[2];
  if (warp == 0) load_old(dst, parts, old);
  __syncthreads();
  const int stretch = (m + 7) / 8, to = min((warp + 1) * stretch, m);
  float acc[8] = {};
  constexpr int U = 4;
  for (int q = warp * stretch; q < to; q += U) {
    typename RowPart<GT>::type u[U][P];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const __nv_bfloat16* row = dout + size_t(list[min(q + i, m - 1)]) * H + col;
#pragma unroll
      for (int k = 0; k < P; ++k)
        if (k < parts) load_row(u[i][k], row + 128 * k);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
#pragma unroll
      for (int k = 0; k < P; ++k) {
        if (k >= parts || q + i >= to) break;
        float f[W];
        unpack_row(u[i][k], f);
#pragma unroll
        for (int x = 0; x < W; ++x) acc[W * k + x] += f[x];
      }
    }
  }
  if (m > 1) {
#pragma unroll
    for (int k = 0; k < 8; ++k) part[warp][k * 32 + lane] = acc[k];
    __syncthreads();
  }
  if (warp != 0) return;
  for (int v = 1; v < 8 && v * stretch < m; ++v) {
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] += part[v][k * 32 + lane];
  }
  add_to_row(dst, old, parts, scale, acc);
}

// gpos[p + off] += sum over the sequences of dout[b S + p], in order
template <typename GT>
__global__ void __launch_bounds__(256) position_grad_kernel(const __nv_bfloat16* dout, GT* gpos, int T, int H, int S, int off) {
  chain_trigger();
  chain_wait();
  constexpr int W = VEC<GT>;
  const int cpr = H / W, rows = min(S, T);
  const long total = long(rows) * cpr;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    const int p = int(i / cpr), c = int(i - long(p) * cpr) * W;
    GT* dst = gpos + size_t(p + off) * H + c;
    const uint4 old = ld_v4(dst);
    float acc[W] = {}, f[W];
#pragma unroll 4
    for (long t = p; t < T; t += S) {
      typename RowPart<GT>::type u;
      load_row(u, dout + t * H + c);
      unpack_row(u, f);
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k] += f[k];
    }
    unpack_grad<GT>(old, f);
#pragma unroll
    for (int k = 0; k < W; ++k) f[k] += acc[k];
    store_part(dst, f);
  }
}

// Rows to a piece: 4 to 32, as many as leave about as many warps as fit on the GPU at once.  Longer pieces cut fewer runs, shorter ones
// wait for fewer rows one behind the other.  us with pieces of 4 / 8 / 16 / 32, fp32 table: 4096 tokens of 1024 columns 14.8 / 17.1 /
// 18.9 / 32.5, 8192 of 2048 31.3 / 27.4 / 26.7 / 37.7, 16384 of 4096 104.8 / 82.3 / 72.6 / 69.9.  From 12288 tokens on not 4, however narrow the
// rows: the parts of a token that occurs often would be too many for the CTA that adds them (16384 of 64, a fifth of them one token,
// 36.5 / 28.9).
static int piece_rows(int n, int H) {
  const long k = long(n) * ((H + 255) / 256) / (27L * num_sms());
  return k >= 32 ? 32 : k >= 16 ? 16 : k >= 8 || n >= 12288 ? 8 : 4;
}

template <int K, typename GT>
static int by_token(const ByToken& a, GT* table, cudaStream_t stream) {
  const int slices = (a.H + 255) / 256, pieces = (a.n - 1) / K + 1;
  auto kern = embedding_pieces_kernel<K, GT>;
  static SharedLimit limit;
  ZB_CUDA_OK(limit.raise(kern, sizeof(PieceRing<GT>)));
  ZB_CUDA_OK(launch_pass(kern, (pieces * slices + 7) / 8, 256, sizeof(PieceRing<GT>), stream, a, table));
  if (pieces > 1) ZB_CUDA_OK(launch_pass(embedding_join_kernel<K, GT>, (pieces + 7) / 8 * slices, 256, 0, stream, a, table));
  return 0;
}

template <typename GT>
static int by_token(int K, const ByToken& a, GT* table, cudaStream_t stream) {
  switch (K) {
    case 4: return by_token<4>(a, table, stream);
    case 8: return by_token<8>(a, table, stream);
    case 16: return by_token<16>(a, table, stream);
    default: return by_token<32>(a, table, stream);
  }
}

template <typename GT>
static int small(const long* ids, const __nv_bfloat16* dout, GT* table, int T, int H, int V, float scale, cudaStream_t stream) {
  ZB_CUDA_OK(launch_pass(embedding_small_kernel<GT>, T * ((H + 255) / 256), 256, 0, stream, ids, dout, table, T, H, V, scale));
  return 0;
}
// (columns and positions are counted in 32 bits, some way beyond the last one)
static int embedding_check(int H, int V, int S, int off) {
  if (H < 8 || H % 8 != 0) ZB_FAIL(-1, "embedding: H=%d not a multiple of 8", H);
  if (H > 1 << 30) ZB_FAIL(-1, "embedding: H=%d above 2^30", H);
  if (V < 0 || S < 0 || off < 0) ZB_FAIL(-1, "embedding: a vocabulary of %d, sequences of %d, positions from %d", V, S, off);
  return 0;
}

static bool is_small(int T, int H) { return T <= SMALL_T && long(T) * ((H + 255) / 256) <= SMALL_CTAS; }

static long order_bytes(int T) { return ((T > SORT_CHUNK ? 16L : 8L) * T + 15) / 16 * 16; }

static int blocks_for(long items) {
  const long b = (items + 255) / 256, cap = long(num_sms()) * 16;
  return int(b < cap ? b : cap);
}

}  // namespace zb

extern "C" {

int zb_embedding_scaled(const long* ids, const void* table, const void* pos, void* out, int T, int H, int V, int S, int pos_offset,
                        float scale, cudaStream_t stream) {
  using namespace zb;
  if (int rc = embedding_check(H, V, S, pos_offset)) return rc;
  if ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(pos) | reinterpret_cast<uintptr_t>(out)) & 15)
    ZB_FAIL(-1, "embedding: operands must be 16-byte aligned");
  if (T <= 0) return 0;
  int shift = 0;
  while (shift < 5 && (8 << shift) < H) ++shift;
  const long warps = (long(T) + (32 >> shift) - 1) >> (5 - shift);
  auto kern = embedding_scaled_kernel<true>;
  if (pos == nullptr) kern = embedding_scaled_kernel<false>;
  ZB_CUDA_OK(launch_pass(kern, int((warps + 3) / 4), 128, 0, stream, ids, static_cast<const __nv_bfloat16*>(table),
                         static_cast<const __nv_bfloat16*>(pos), static_cast<__nv_bfloat16*>(out), T, H, V, S, pos_offset, scale, shift));
  return 0;
}

// *bytes: what zb_embedding_by_token wants as workspace: order and sorted ids (of more than one chunk twice), and two rows of sums
// for each piece
int zb_embedding_by_token_workspace(int T, int H, long* bytes) {
  using namespace zb;
  if (int rc = embedding_check(H, 0, 0, 0)) return rc;
  const int K = piece_rows(T, H);
  *bytes = T > 0 && !is_small(T, H) ? order_bytes(T) + 8L * ((T - 1L) / K + 1) * H : 0;
  return 0;
}

int zb_embedding_by_token(const long* ids, const void* dout, void* gtable, void* gpos, void* workspace, int T, int H, int V, int S,
                          int pos_offset, float scale, int grad_f32, cudaStream_t stream) {
  using namespace zb;
  if (int rc = embedding_check(H, V, S, pos_offset)) return rc;
  if ((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(gtable) | reinterpret_cast<uintptr_t>(gpos) |
       reinterpret_cast<uintptr_t>(workspace)) & 15)
    ZB_FAIL(-1, "embedding: operands must be 16-byte aligned");
  if (T <= 0) return 0;
  const __nv_bfloat16* rows = static_cast<const __nv_bfloat16*>(dout);
  int rc = 0;
  if (is_small(T, H)) {
    rc = grad_f32 ? small(ids, rows, static_cast<float*>(gtable), T, H, V, scale, stream)
                  : small(ids, rows, static_cast<__nv_bfloat16*>(gtable), T, H, V, scale, stream);
    if (rc) return rc;
  } else {
    int* order = static_cast<int*>(workspace);
    int* sorted = order + T;
    const int most = T < SORT_CHUNK ? T : SORT_CHUNK, K = piece_rows(T, H), chunks = (T - 1) / SORT_CHUNK + 1;
    float* head = reinterpret_cast<float*>(static_cast<char*>(workspace) + order_bytes(T));
    float* tail = head + ((T - 1L) / K + 1) * H;
    // ids of a CTA: about as many CTAs as SMs, of at least 8 ids and at most SORT_BINS
    int width = (V + num_sms() - 1) / num_sms();
    width = width < 8 ? 8 : width > SORT_BINS ? SORT_BINS : width;
    const int ctas = (V - 1) / width + 1;
    if (long(ctas) * chunks > 0x7fffffffL) ZB_FAIL(-1, "embedding: %d tokens of a vocabulary of %d", T, V);
    auto kern = embedding_sort_kernel<32>;
    if (most <= 4 * 1024) kern = embedding_sort_kernel<4>;
    else if (most <= 16 * 1024) kern = embedding_sort_kernel<16>;
    static SharedLimit limit[3];
    ZB_CUDA_OK(limit[most <= 4 * 1024 ? 0 : most <= 16 * 1024 ? 1 : 2].raise(kern, sizeof(SortShared)));
    ZB_CUDA_OK(launch_pass(kern, chunks * ctas, 1024, sizeof(SortShared), stream, ids, order, sorted, T, V, width, ctas));
    if (chunks > 1) {
      ZB_CUDA_OK(launch_pass(embedding_merge_kernel, (T - 1) / 256 + 1, 256, 0, stream, order, sorted, order + 2L * T, sorted + 2L * T, T));
      order += 2L * T;
      sorted += 2L * T;
    }
    const ByToken a = {rows, order, sorted, head, tail, T, H, scale};
    rc = grad_f32 ? by_token(K, a, static_cast<float*>(gtable), stream) : by_token(K, a, static_cast<__nv_bfloat16*>(gtable), stream);
    if (rc) return rc;
  }
  if (gpos != nullptr) {
    const int grid = blocks_for(long(S < T ? S : T) * (H / (grad_f32 ? 4 : 8)));
    if (grad_f32) ZB_CUDA_OK(launch_pass(position_grad_kernel<float>, grid, 256, 0, stream, rows, static_cast<float*>(gpos), T, H, S, pos_offset));
    else ZB_CUDA_OK(launch_pass(position_grad_kernel<__nv_bfloat16>, grid, 256, 0, stream, rows, static_cast<__nv_bfloat16*>(gpos), T, H, S, pos_offset));
  }
  return 0;
}

}  // extern "C"
