// Token embedding with a scale, and its gradient summed token by token:
//   forward   out[t] = scale table[id_t] (+ pos[t mod S + off])
//   backward  gtable[v] += scale sum over t with id_t = v of dout[t],  gpos[p + off] += sum over t with t mod S = p of dout[t]
// The gradient without atomics: the ids are sorted together with their positions (equal ids keep the order of their
// positions), and every row of the table that occurs is read, added to and written once, by the sum of its terms in a fixed
// order, in fp32.  So the result is the same on each run, a token that occurs thousands of times does not queue up at one
// address, and in a bf16 bucket a row is rounded once and not once for every occurrence.
// Ids outside [0, V) count as the nearest inside, as in the gather without a scale.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../norm/norm_common.cuh"
#include <cooperative_groups.h>

namespace zb {
namespace cg = cooperative_groups;

__device__ __forceinline__ int clamp_id(long id, int V) { return int(id < 0 ? 0 : id >= V ? V - 1 : id); }

// ------------------------------- forward -------------------------------
__global__ void __launch_bounds__(256) embedding_scaled_kernel(const long* ids, const __nv_bfloat16* table, const __nv_bfloat16* pos,
                                                               __nv_bfloat16* out, int T, int H, int V, int S, int off, float scale) {
  chain_trigger();
  chain_wait();
  const int cpr = H >> 3;
  const long total = long(T) * cpr;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    const int t = int(i / cpr), c = int(i - long(t) * cpr) * 8;
    float a[8];
    unpack8(ld_v4(table + size_t(clamp_id(ids[t], V)) * H + c), a);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] *= scale;
    if (pos != nullptr) {
      float b[8];
      unpack8(ld_v4(pos + size_t(t % S + off) * H + c), b);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] += b[j];
    }
    *reinterpret_cast<uint4*>(out + size_t(t) * H + c) = pack8(a);
  }
}

// ------------------------------- order of the ids -------------------------------
// Stable radix sort of up to CLUSTER * SORT_MOST ids and their positions by one cluster, which holds them in the shared memory
// of its CTAs: one launch, whatever the number of passes.  A pass: every warp ranks its ids among those of the same digit
// (match), counts are added over warps and CTAs, and every id goes to its place in the CTA that owns it.
constexpr int SORT_BITS = 9, SORT_BINS = 1 << SORT_BITS, SORT_MOST = 4096, SORT_CTAS = 8, SORT_CHUNK = SORT_CTAS * SORT_MOST;

struct SortShared {
  int key[2][SORT_MOST], at[2][SORT_MOST];
  unsigned short count[32][SORT_BINS];          // of a warp's ids; then how many of its CTA's are in warps before it
  int total[SORT_CTAS][SORT_BINS];              // of every CTA of the cluster
  int base[SORT_BINS];
  int scan[32];
};

// order, sorted: [T]; chunk k of the ids (SORT_CHUNK of them) is sorted by cluster k.  `own`: ids per CTA, a multiple of 1024.
__global__ void __launch_bounds__(1024) embedding_sort_kernel(const long* ids, int* order, int* sorted, int T, int V, int own, int passes,
                                                              int bits) {
  chain_trigger();
  chain_wait();
  extern __shared__ __align__(16) unsigned char raw[];
  SortShared& sh = *reinterpret_cast<SortShared*>(raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int first = int(blockIdx.x / ctas) * SORT_CHUNK, n = min(T - first, SORT_CHUNK);
  const int mine = max(0, min(n - rank * own, own));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, per = own >> 10;   // 32 `per` ids in a row for each warp
  cluster.sync();                               // no CTA writes to another that has not started
  for (int i = tid; i < mine; i += 1024) {
    sh.key[0][i] = clamp_id(ids[first + rank * own + i], V);
    sh.at[0][i] = first + rank * own + i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int from = pass & 1, shift = pass * bits, bins = 1 << bits;
    for (int i = tid; i < 32 * SORT_BINS / 2; i += 1024) reinterpret_cast<unsigned*>(sh.count)[i] = 0;
    __syncthreads();
    int digit[4], place[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int e = (warp * per + k) * 32 + lane;
      const bool there = k < per && e < mine;
      const unsigned all = __ballot_sync(0xffffffffu, there);
      digit[k] = there ? sh.key[from][e] >> shift & (bins - 1) : 0;
      if (there) {
        const unsigned same = __match_any_sync(all, digit[k]);
        const int before = sh.count[warp][digit[k]];
        place[k] = before + __popc(same & ((1u << lane) - 1));
        __syncwarp(all);
        if ((same & ((1u << lane) - 1)) == 0) sh.count[warp][digit[k]] = static_cast<unsigned short>(before + __popc(same));
        __syncwarp(all);
      }
      __syncwarp();
    }
    __syncthreads();
    if (tid < bins) {
      int sum = 0;
      for (int w = 0; w < 32; ++w) {
        const int c = sh.count[w][tid];
        sh.count[w][tid] = static_cast<unsigned short>(sum);
        sum += c;
      }
      for (int r = 0; r < ctas; ++r) cluster.map_shared_rank(&sh, r)->total[rank][tid] = sum;
    }
    cluster.sync();
    // base of a bin: everything of lower bins, and of this one in the CTAs before
    int sum = 0, before = 0;
    if (tid < bins) {
      for (int r = 0; r < ctas; ++r) {
        const int c = sh.total[r][tid];
        sum += c;
        before += r < rank ? c : 0;
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
      int s = sh.scan[lane];
      const int self = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += v;
      }
      sh.scan[lane] = s - self;
    }
    __syncthreads();
    if (tid < bins) sh.base[tid] = sh.scan[warp] + run - sum + before;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int e = (warp * per + k) * 32 + lane;
      if (k < per && e < mine) {
        const int pos = sh.base[digit[k]] + sh.count[warp][digit[k]] + place[k];
        const int key = sh.key[from][e], at = sh.at[from][e];
        if (pass + 1 == passes) {
          order[first + pos] = at;
          sorted[first + pos] = key;
        } else {
          const int r = pos / own;
          SortShared* to = cluster.map_shared_rank(&sh, r);
          to->key[from ^ 1][pos - r * own] = key;
          to->at[from ^ 1][pos - r * own] = at;
        }
      }
    }
    if (pass + 1 < passes) cluster.sync();
  }
}

// ------------------------------- sums by token -------------------------------
// The sorted rows are cut into pieces of K; a warp sums a piece over 256 columns.  A run of equal ids that lies within a piece
// goes straight to the table.  Of a run over several pieces, the first one leaves its part in `tail`, every further one in
// `head`, and embedding_join_kernel adds those up.
struct ByToken {
  const __nv_bfloat16* dout;
  const int *order, *sorted;      // of this chunk, n of them
  float *head, *tail;             // [pieces, H]
  int n, H;
  float scale;
};

template <typename GT>
__device__ __forceinline__ void load_grad8(const GT* p, float (&f)[8]) {
  if constexpr (sizeof(GT) == 4) {
    const uint4 a = ld_v4(p), b = ld_v4(p + 4);
    f[0] = __uint_as_float(a.x); f[1] = __uint_as_float(a.y); f[2] = __uint_as_float(a.z); f[3] = __uint_as_float(a.w);
    f[4] = __uint_as_float(b.x); f[5] = __uint_as_float(b.y); f[6] = __uint_as_float(b.z); f[7] = __uint_as_float(b.w);
  } else {
    unpack8(ld_v4(p), f);
  }
}
__device__ __forceinline__ void store_grad8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store_grad8(__nv_bfloat16* p, const float (&f)[8]) { *reinterpret_cast<uint4*>(p) = pack8(f); }

template <int K, typename GT>
__global__ void __launch_bounds__(256) embedding_pieces_kernel(const ByToken a, GT* table) {
  chain_trigger();
  chain_wait();
  constexpr int U = 4;
  const int lane = threadIdx.x & 31, slices = (a.H + 255) >> 8, pieces = (a.n + K - 1) / K;
  const int item = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= pieces * slices) return;
  const int piece = item / slices, col = (item - piece * slices) * 256 + lane * 8, j0 = piece * K, rows = min(K, a.n - j0);
  const bool used = col < a.H;
  const int id = lane < rows ? a.sorted[j0 + lane] : -1, at = lane < rows ? a.order[j0 + lane] : 0;
  const int prev = j0 > 0 ? a.sorted[j0 - 1] : -1, next = j0 + rows < a.n ? a.sorted[j0 + rows] : -1;
  int after = __shfl_down_sync(0xffffffffu, id, 1);
  if (lane == rows - 1) after = next;
  const unsigned ends = __ballot_sync(0xffffffffu, lane < rows && id != after);
  const bool goes_on = prev >= 0 && prev == __shfl_sync(0xffffffffu, id, 0);   // the first run began in an earlier piece
  const int first_end = goes_on ? __ffs(ends) - 1 : -1;
  float acc[8] = {};
  for (int j = 0; j < rows; j += U) {
    uint4 row[U];
    float old[U][8];
    int to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int src = __shfl_sync(0xffffffffu, at, (j + u) & 31);
      to[u] = __shfl_sync(0xffffffffu, id, (j + u) & 31);
      row[u] = make_uint4(0, 0, 0, 0);
      if (j + u < rows && used) {
        row[u] = ld_v4(a.dout + size_t(src) * a.H + col);
        if ((ends >> (j + u) & 1) && j + u != first_end) load_grad8(table + size_t(to[u]) * a.H + col, old[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[8];
      unpack8(row[u], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] += f[k];
      if (j + u < rows && (ends >> (j + u) & 1)) {
        if (j + u == first_end) {
          if (used) store_grad8(a.head + size_t(piece) * a.H + col, acc);
        } else if (used) {
#pragma unroll
          for (int k = 0; k < 8; ++k) old[u][k] += a.scale * acc[k];
          store_grad8(table + size_t(to[u]) * a.H + col, old[u]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = 0.f;
      }
    }
  }
  if (used && !(ends >> (rows - 1) & 1))
    store_grad8((goes_on && ends == 0 ? a.head : a.tail) + size_t(piece) * a.H + col, acc);
}

// Runs over several pieces: a CTA looks at eight pieces and 256 columns, a warp at one piece.  What begins in it and goes on is
// its tail and the heads that follow, up to the run's last piece; runs over more than JOIN_ALONE pieces are added by the whole CTA,
// each warp a stretch of the heads, the stretches in order.
constexpr int JOIN_ALONE = 16;
template <int K, typename GT>
__global__ void __launch_bounds__(256) embedding_join_kernel(const ByToken a, GT* table) {
  chain_trigger();
  chain_wait();
  __shared__ int run_last[8];
  __shared__ __align__(16) float part[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slices = (a.H + 255) >> 8, pieces = (a.n + K - 1) / K;
  const int group = blockIdx.x / slices, col = (blockIdx.x - group * slices) * 256 + lane * 8;
  const bool used = col < a.H;
  int piece = group * 8 + warp, last = -1;
  if (piece < pieces - 1) {
    const int end = (piece + 1) * K, id = a.sorted[end - 1];
    if (a.sorted[end] == id && (piece == 0 || a.sorted[piece * K - 1] != id)) {
      int lo = end, hi = a.n;                  // sorted[lo] == id; the first place behind the run is in (lo, hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.sorted[mid] == id) lo = mid;
        else hi = mid;
      }
      last = lo / K;
    }
  }
  auto sum_heads = [&](int from, int to, float (&acc)[8]) {
    int q = from;
    for (; q + 4 <= to; q += 4) {
      float f[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) load_grad8(a.head + size_t(q + u) * a.H + col, f[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] += f[u][k];
      }
    }
    for (; q < to; ++q) {
      float f[8];
      load_grad8(a.head + size_t(q) * a.H + col, f);
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] += f[k];
    }
  };
  auto add_to_table = [&](int p, const float (&acc)[8]) {
    GT* dst = table + size_t(a.sorted[(p + 1) * K]) * a.H + col;
    float f[8];
    load_grad8(dst, f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] += a.scale * acc[k];
    store_grad8(dst, f);
  };
  const bool together = last - piece > JOIN_ALONE;
  if (last >= 0 && !together && used) {
    float acc[8];
    load_grad8(a.tail + size_t(piece) * a.H + col, acc);
    sum_heads(piece + 1, last + 1, acc);
    add_to_table(piece, acc);
  }
  if (lane == 0) run_last[warp] = together && last >= 0 ? last : -1;
  __syncthreads();
  for (int w = 0; w < 8; ++w) {
    const int end = run_last[w];
    if (end < 0) continue;
    piece = group * 8 + w;
    const int heads = end - piece, stretch = (heads + 7) / 8, from = piece + 1 + warp * stretch;
    float acc[8] = {};
    if (used) sum_heads(from, min(from + stretch, end + 1), acc);
    if (used) store_grad8(&part[warp][lane * 8], acc);
    __syncthreads();
    if (warp == 0 && used) {
      load_grad8(a.tail + size_t(piece) * a.H + col, acc);
      for (int v = 0; v < 8; ++v) {
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] += part[v][lane * 8 + k];
      }
      add_to_table(piece, acc);
    }
    __syncthreads();
  }
}

// gpos[p + off] += sum over the sequences of dout[b S + p], in order
template <typename GT>
__global__ void __launch_bounds__(256) position_grad_kernel(const __nv_bfloat16* dout, GT* gpos, int T, int H, int S, int off) {
  chain_trigger();
  chain_wait();
  const int cpr = H >> 3, rows = min(S, T);
  const long total = long(rows) * cpr;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    const int p = int(i / cpr), c = int(i - long(p) * cpr) * 8;
    float acc[8] = {}, f[8];
    for (long t = p; t < T; t += S) {
      unpack8(ld_v4(dout + t * H + c), f);
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] += f[k];
    }
    GT* dst = gpos + size_t(p + off) * H + c;
    load_grad8(dst, f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] += acc[k];
    store_grad8(dst, f);
  }
}

// Rows to a piece.  Many rows: 32, so that few runs are cut; few: 4, so that there are warps enough.
static int piece_rows(int n, int H) { return long(n) * ((H + 255) / 256) >= 32L * 8 * num_sms() ? 32 : 4; }

template <int K, typename GT>
static int by_token(const ByToken& a, GT* table, cudaStream_t stream) {
  const int slices = (a.H + 255) / 256, pieces = (a.n + K - 1) / K;
  ZB_CUDA_OK(launch_pass(embedding_pieces_kernel<K, GT>, (pieces * slices + 7) / 8, 256, 0, stream, a, table));
  if (pieces > 1) ZB_CUDA_OK(launch_pass(embedding_join_kernel<K, GT>, (pieces + 7) / 8 * slices, 256, 0, stream, a, table));
  return 0;
}

static int blocks_for(long items) {
  const long b = (items + 255) / 256, cap = long(num_sms()) * 16;
  return int(b < cap ? b : cap);
}

}  // namespace zb

extern "C" {

int zb_embedding_scaled(const long* ids, const void* table, const void* pos, void* out, int T, int H, int V, int S, int pos_offset,
                        float scale, cudaStream_t stream) {
  using namespace zb;
  if (H % 8 != 0) ZB_FAIL(-1, "embedding: H=%d not a multiple of 8", H);
  if ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(pos) | reinterpret_cast<uintptr_t>(out)) & 15)
    ZB_FAIL(-1, "embedding: operands must be 16-byte aligned");
  if (T <= 0) return 0;
  ZB_CUDA_OK(launch_pass(embedding_scaled_kernel, blocks_for(long(T) * (H / 8)), 256, 0, stream, ids,
                         static_cast<const __nv_bfloat16*>(table), static_cast<const __nv_bfloat16*>(pos),
                         static_cast<__nv_bfloat16*>(out), T, H, V, S, pos_offset, scale));
  return 0;
}

// *bytes: what zb_embedding_by_token wants as workspace: order and sorted ids, and two rows of sums for each piece of a chunk
int zb_embedding_by_token_workspace(int T, int H, long* bytes) {
  using namespace zb;
  const int n = T < SORT_CHUNK ? T : SORT_CHUNK, K = piece_rows(n, H);
  *bytes = T > 0 ? ((8L * T + 15) / 16) * 16 + 8L * ((n + K - 1) / K) * H : 0;
  return 0;
}

int zb_embedding_by_token(const long* ids, const void* dout, void* gtable, void* gpos, void* workspace, int T, int H, int V, int S,
                          int pos_offset, float scale, int grad_f32, cudaStream_t stream) {
  using namespace zb;
  if (H % 8 != 0) ZB_FAIL(-1, "embedding: H=%d not a multiple of 8", H);
  if ((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(gtable) | reinterpret_cast<uintptr_t>(gpos) |
       reinterpret_cast<uintptr_t>(workspace)) & 15)
    ZB_FAIL(-1, "embedding: operands must be 16-byte aligned");
  if (T <= 0) return 0;
  int* order = static_cast<int*>(workspace);
  int* sorted = order + T;
  const int most = T < SORT_CHUNK ? T : SORT_CHUNK, K = piece_rows(most, H);
  float* head = reinterpret_cast<float*>(static_cast<char*>(workspace) + ((8L * T + 15) / 16) * 16);
  float* tail = head + long((most + K - 1) / K) * H;
  int bits = 1;
  while (bits < 31 && (1L << bits) < V) ++bits;
  const int passes = (bits + SORT_BITS - 1) / SORT_BITS, chunks = (T + SORT_CHUNK - 1) / SORT_CHUNK;
  const int ctas = most >= SORT_CTAS * 1024 ? SORT_CTAS : (most + 1023) / 1024, own = ((most + ctas - 1) / ctas + 1023) / 1024 * 1024;
  ZB_CUDA_OK(cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(SortShared))));
  ZB_CUDA_OK(launch_chained(embedding_sort_kernel, chunks * ctas, 1024, sizeof(SortShared), stream, ctas, ids, order, sorted, T, V, own,
                            passes, (bits + passes - 1) / passes));
  for (int c = 0; c < chunks; ++c) {
    ByToken a = {static_cast<const __nv_bfloat16*>(dout), order + c * SORT_CHUNK, sorted + c * SORT_CHUNK, head, tail,
                 T - c * SORT_CHUNK < SORT_CHUNK ? T - c * SORT_CHUNK : SORT_CHUNK, H, scale};
    int rc;
    if (grad_f32)
      rc = K == 32 ? by_token<32>(a, static_cast<float*>(gtable), stream) : by_token<4>(a, static_cast<float*>(gtable), stream);
    else
      rc = K == 32 ? by_token<32>(a, static_cast<__nv_bfloat16*>(gtable), stream)
                   : by_token<4>(a, static_cast<__nv_bfloat16*>(gtable), stream);
    if (rc) return rc;
  }
  if (gpos != nullptr) {
    const int grid = blocks_for(long(S < T ? S : T) * (H / 8));
    const __nv_bfloat16* d = static_cast<const __nv_bfloat16*>(dout);
    if (grad_f32) ZB_CUDA_OK(launch_pass(position_grad_kernel<float>, grid, 256, 0, stream, d, static_cast<float*>(gpos), T, H, S, pos_offset));
    else ZB_CUDA_OK(launch_pass(position_grad_kernel<__nv_bfloat16>, grid, 256, 0, stream, d, static_cast<__nv_bfloat16*>(gpos), T, H, S, pos_offset));
  }
  return 0;
}

}  // extern "C"
