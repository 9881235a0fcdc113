// K5: eviction from a paged cache by accumulated attention weight. Of every sequence longer than `keep`, each KV head
// keeps its first keep_first tokens, its last keep_last and the heaviest of those between, `keep` in all (equal weights:
// the earlier token); the kept cells and their weights move, in order, to positions 0 .. keep - 1 of the sequence's
// pages, or of other pages (a sequence whose pages others share). Cells are moved as bytes: any format, any head size.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "qp_api_internal.h"
#include "qp_common.cuh"

namespace qp {

struct EvictParams {
  uint8_t* cache;
  FastDiv block_size;
  int64_t block_stride, head_stride, slot_stride;  // bytes
  int cell;                                        // bytes, a multiple of 8
  float* weights;
  int64_t w_block, w_slot, w_head;  // element strides
  int nkv, num_seqs;
  const int32_t* seqused;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* out_table;  // null: in place
  int64_t out_stride;
  int max_n, keep, first, last;
  int32_t* kept;         // [seqs][nkv][keep]: token of each kept position, -1 behind them
  int32_t* seqused_out;  // [seqs]
  // workspace, written by the selection: new length and whether anything may move, ticket, chunk flags
  int2* lens;       // [seqs]
  uint32_t* ticket;
  uint32_t* flags;  // [seqs][nkv][chunks]
  int chunks, chunk;  // chunks of `chunk` kept positions of a pair
  int smem_weights;   // weights a CTA of the selection holds in shared memory
};

// order of the weights as unsigned integers: NaN first (it goes first), -0 = +0
__device__ __forceinline__ uint32_t weight_rank(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float* weight_at(const EvictParams& p, const int32_t* table, int kvh, int i) {
  const int b = p.block_size.div(i);
  return p.weights + static_cast<int64_t>(table[b]) * p.w_block +
         static_cast<int64_t>(i - b * p.block_size.d) * p.w_slot + kvh * p.w_head;
}
__device__ __forceinline__ uint8_t* cell_at(const EvictParams& p, const int32_t* table, int kvh, int i) {
  const int b = p.block_size.div(i);
  return p.cache + static_cast<int64_t>(table[b]) * p.block_stride +
         static_cast<int64_t>(i - b * p.block_size.d) * p.slot_stride + static_cast<int64_t>(kvh) * p.head_stride;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// the word at shared-memory address `p` of CTA `rank` of the cluster
__device__ __forceinline__ uint32_t ld_cluster(const void* p, uint32_t rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ void add_cluster(void* p, uint32_t rank, uint32_t v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

// ---------------------------------------------------------------------------------------------------- selection
// The threshold weight of a (sequence, KV head) by radix selection (digits of 11, 11 and 10 bits), then the kept tokens
// in order. A cluster of 1 to 16 CTAs shares a pair: each reads its part of the weights once, from HBM into shared
// memory (4 bytes a token are the floor of this kernel; what does not fit is read again from L2), the digits'
// histograms and the counts meet over distributed shared memory. One launch; nothing comes back to the host. Measured:
// 96 pairs of up to 16,384 tokens 24 us, 4 pairs of 262,143 about 30 us: the barriers of the digits, not the bytes.
constexpr int EV_THREADS = 1024, EV_WARPS = EV_THREADS / 32, EV_BINS = 2048;

struct EvictShared {
  uint32_t hist[EV_BINS];      // this CTA's
  uint32_t total[3][EV_BINS];  // in the first CTA: the cluster's, one for each digit
  uint32_t bin, left;      // the digit found, and how many of its weights stay
  uint32_t warp_sum[EV_WARPS];
  uint32_t gt[EV_WARPS], tie[EV_WARPS];  // per warp: tokens that stay for sure, tokens at the threshold
  uint32_t gt_all, tie_all;              // this CTA's, read by the others
};

__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(const EvictParams p) {
  asm volatile("griddepcontrol.launch_dependents;");  // the move's launch may begin; it waits for this grid's end
  extern __shared__ __align__(16) uint8_t raw[];
  EvictShared& sh = *reinterpret_cast<EvictShared*>(raw);
  uint32_t* ranks = reinterpret_cast<uint32_t*>(raw + sizeof(EvictShared));  // of this CTA's first smem_weights tokens
  uint32_t rank, ctas;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const auto sync = [&]() {
    if (ctas == 1) __syncthreads();
    else cluster_sync();
  };
  const int kvh = blockIdx.x / ctas, seq = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int32_t* table = p.table + seq * p.table_stride;
  const int n = min(max(p.seqused[seq], 0), p.max_n);
  const int64_t pair = static_cast<int64_t>(seq) * p.nkv + kvh;
  int32_t* kept = p.kept + pair * p.keep;
  if (rank == 0) {
    if (kvh == 0 && tid == 0) p.lens[seq] = make_int2(min(n, p.keep), n > p.keep || p.out_table != nullptr);
    if (pair == 0 && tid == 0) *p.ticket = 0u;
    for (int c = tid; c < p.chunks; c += EV_THREADS) p.flags[pair * p.chunks + c] = 0u;
  }
  if (n <= p.keep) {  // the whole cluster leaves
    for (int j = rank * EV_THREADS + tid; j < p.keep; j += ctas * EV_THREADS) kept[j] = j < n ? j : -1;
    return;
  }
  // this CTA's tokens
  const int part = (n + ctas - 1) / ctas, c0 = min(static_cast<int>(rank) * part, n), c1 = min(c0 + part, n);
  const int lo = p.first, hi = n - p.last;
  const auto rank_of = [&](int i) {
    const int k = i - c0;
    return k < p.smem_weights ? ranks[k] : weight_rank(*weight_at(p, table, kvh, i));
  };
  for (int i = tid; i < 3 * EV_BINS; i += EV_THREADS) (&sh.total[0][0])[i] = 0;
#pragma unroll 8
  for (int i = c0 + tid; i < min(c1, c0 + p.smem_weights); i += EV_THREADS)
    ranks[i - c0] = weight_rank(*weight_at(p, table, kvh, i));

  sync();  // the first CTA's totals are zero before anyone adds to them
  uint32_t thr = 0, mask = 0, want = p.keep - p.first - p.last;  // of the tokens [lo, hi)
  const int b0 = max(c0, lo), b1 = min(c1, hi);
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : EV_BINS;
    for (int i = tid; i < EV_BINS; i += EV_THREADS) sh.hist[i] = 0;
    __syncthreads();
    for (int i = b0 + tid; i < b1; i += EV_THREADS) {
      const uint32_t r = rank_of(i);
      if ((r & mask) == thr) atomicAdd(&sh.hist[(r >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int i = tid; i < EV_BINS; i += EV_THREADS)  // few bins hold anything
      if (sh.hist[i] != 0u) {
        if (rank == 0) atomicAdd(&sh.total[pass][i], sh.hist[i]);
        else add_cluster(&sh.total[pass][i], 0, sh.hist[i]);
      }
    sync();
    if (rank == 0) {  // the bin in which the want-th heaviest lies, from the highest on (2 bins a thread)
      const int top = EV_BINS - 1 - 2 * tid;
      const uint32_t h0 = sh.total[pass][top], h1 = sh.total[pass][top - 1];
      uint32_t incl = h0 + h1;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
      }
      if (lane == 31) sh.warp_sum[warp] = incl;
      __syncthreads();
      uint32_t before = sh.warp_sum[lane];  // EV_WARPS = 32
      before = __reduce_add_sync(0xffffffffu, lane < warp ? before : 0u);
      const uint32_t above = before + incl - h0 - h1;
      if (above < want && want <= above + h0) {
        sh.bin = top;
        sh.left = want - above;
      } else if (above + h0 < want && want <= above + h0 + h1) {
        sh.bin = top - 1;
        sh.left = want - above - h0;
      }
      if (want == 0 && tid == 0) {  // none stays: all bits 1, above every weight
        sh.bin = bins - 1;
        sh.left = 0;
      }
    }
    sync();
    thr |= ld_cluster(&sh.bin, 0) << shift;
    mask |= static_cast<uint32_t>(bins - 1) << shift;
    want = ld_cluster(&sh.left, 0);
  }
  // Tokens above the threshold stay, and of those at it the first `want`. Each warp takes a run of tokens: it counts,
  // the counts are summed over the warps and the CTAs before it, and it writes its tokens in order.
  const int run = (part + EV_WARPS - 1) / EV_WARPS, w0 = min(c0 + warp * run, c1), w1 = min(w0 + run, c1);
  uint32_t gt = 0, tie = 0;
  for (int i = w0 + lane; i < w1; i += 32) {
    const bool sure = i < lo || i >= hi;
    const uint32_t r = sure ? 0u : rank_of(i);
    gt += sure || r > thr;
    tie += !sure && r == thr;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    gt += __shfl_xor_sync(0xffffffffu, gt, d);
    tie += __shfl_xor_sync(0xffffffffu, tie, d);
  }
  if (lane == 0) {
    sh.gt[warp] = gt;
    sh.tie[warp] = tie;
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t g = 0, t = 0;
    for (int w = 0; w < EV_WARPS; ++w) {
      g += sh.gt[w];
      t += sh.tie[w];
    }
    sh.gt_all = g;
    sh.tie_all = t;
  }
  sync();
  gt = tie = 0;
  for (uint32_t c = 0; c < rank; ++c) {
    gt += ld_cluster(&sh.gt_all, c);
    tie += ld_cluster(&sh.tie_all, c);
  }
  for (int w = 0; w < warp; ++w) {
    gt += sh.gt[w];
    tie += sh.tie[w];
  }
  uint32_t at = gt + min(tie, want);
  const uint32_t below = (1u << lane) - 1u;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int i = i0 + lane;
    const bool in = i < w1, sure = in && (i < lo || i >= hi);
    const uint32_t r = in && !sure ? rank_of(i) : 0u;
    const bool eq = in && !sure && r == thr;
    const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
    const bool stay = sure || (in && !sure && r > thr) || (eq && tie + __popc(eqs & below) < want);
    const uint32_t stays = __ballot_sync(0xffffffffu, stay);
    if (stay) kept[at + __popc(stays & below)] = i;
    at += __popc(stays);
    tie += __popc(eqs);
  }
  sync();  // no CTA leaves while another may still read its counts
}

// ---------------------------------------------------------------------------------------------------- move
// The kept cells to their places, `chunk` positions of a pair at a time, each cell read once and written once. In place,
// position j gets token kept[j] >= j, so the cells a chunk overwrites are wanted by chunks before it at most: a CTA
// reads its cells into shared memory, says so in its flag, and before it writes waits (bounded) for the chunks that take
// a cell from its range. Chunks are handed out by a ticket, a pair's lower ones first, so those it waits for have been
// taken by CTAs that run already and wait for still lower ones only. Measured: 96 pairs of 4096 cells of 392 bytes 63 us,
// 4.4 TB/s of DRAM traffic (40 registers and 7 reads of 8 bytes in flight a thread; with 90 registers and 8 reads 108).
constexpr int MV_THREADS = 256, MV_BATCH = 7, MV_CTAS = 6;  // 86 KB in flight an SM

__device__ __forceinline__ int lower_bound(const int32_t* kept, int len, int token) {
  int lo = 0, hi = len;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (kept[mid] < token) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(MV_THREADS, MV_CTAS) evict_move_kernel(const EvictParams p, const FastDiv words) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ uint32_t ticket;
  const int tid = threadIdx.x;
  const uint8_t** src = reinterpret_cast<const uint8_t**>(raw);  // of each position; null: it stays
  uint8_t** dst = reinterpret_cast<uint8_t**>(raw) + p.chunk;
  uint2* cells = reinterpret_cast<uint2*>(dst + p.chunk);  // in place only
  if (p.out_table == nullptr) {
    if (tid == 0) ticket = atomicAdd(p.ticket, 1u);
    __syncthreads();
  }
  const int unit = p.out_table ? blockIdx.x : ticket;
  const int pairs = p.num_seqs * p.nkv, chunk = unit / pairs, pair = unit % pairs;
  const int seq = pair / p.nkv, kvh = pair % p.nkv;
  const int2 len = p.lens[seq];
  if (chunk == 0 && kvh == 0 && tid == 0) p.seqused_out[seq] = len.x;
  const int j0 = chunk * p.chunk, m = min(p.chunk, len.x - j0);
  if (m <= 0 || !len.y) return;
  const int32_t* from = p.table + seq * p.table_stride;
  const int32_t* to = p.out_table ? p.out_table + seq * p.out_stride : from;
  const int32_t* kept = p.kept + static_cast<int64_t>(pair) * p.keep;
  float w = 0.f;
  float* w_to = nullptr;
  bool moves = false;
  for (int k = tid; k < m; k += MV_THREADS) {  // at most one a thread: chunk <= MV_THREADS
    const int i = kept[j0 + k];
    moves = p.out_table != nullptr || i != j0 + k;
    src[k] = moves ? cell_at(p, from, kvh, i) : nullptr;
    dst[k] = cell_at(p, to, kvh, j0 + k);
    if (moves) {
      w = *weight_at(p, from, kvh, i);
      w_to = weight_at(p, to, kvh, j0 + k);
    }
  }
  if (!__syncthreads_or(moves)) return;  // nobody else takes a cell from a range that stays
  // 8 bytes a lane (cells are 8-byte aligned), MV_BATCH of them in flight; the pointers come out of shared memory before
  // anything is written there
  const int total = m * words.d;
  const auto batch = [&](int e0, auto&& store) {
    uint2 v[MV_BATCH];
    uint32_t has = 0;
#pragma unroll
    for (int u = 0; u < MV_BATCH; ++u) {
      const int e = e0 + u * MV_THREADS + tid, k = words.div(e);
      const uint8_t* from_cell = e < total ? src[k] : nullptr;
      if (from_cell != nullptr) {
        has |= 1u << u;
        v[u] = __ldcs(reinterpret_cast<const uint2*>(from_cell) + (e - k * words.d));
      }
    }
#pragma unroll
    for (int u = 0; u < MV_BATCH; ++u)
      if (has & (1u << u)) store(e0 + u * MV_THREADS + tid, v[u]);
  };
  if (p.out_table != nullptr) {  // nothing that is written is read by anyone
    for (int e0 = 0; e0 < total; e0 += MV_BATCH * MV_THREADS)
      batch(e0, [&](int e, const uint2& v) {
        const int k = words.div(e);
        reinterpret_cast<uint2*>(dst[k])[e - k * words.d] = v;
      });
    if (w_to != nullptr) *w_to = w;
    return;
  }
  for (int e0 = 0; e0 < total; e0 += MV_BATCH * MV_THREADS)
    batch(e0, [&](int e, const uint2& v) { cells[e] = v; });
  bool ok = true;
  {
    // this CTA's reads are done (their values are in shared memory, the weight in the word below)
    uint32_t* flags = p.flags + static_cast<int64_t>(pair) * p.chunks;
    __shared__ float w_seen[MV_THREADS];
    w_seen[tid] = w;
    __syncthreads();
    w = w_seen[tid];
    if (tid == 0) {
      __threadfence();
      asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(flags + chunk), "r"(1u) : "memory");
    }
    // tokens [j0, j0 + m) lie at kept positions [r0, r1) of chunks up to this one
    const int r0 = lower_bound(kept, len.x, j0), r1 = lower_bound(kept, len.x, j0 + m);
    for (int c = r0 / p.chunk + tid; r1 > r0 && c <= (r1 - 1) / p.chunk && c < chunk; c += MV_THREADS) {
      const uint64_t t0 = global_timer_ns();
      uint32_t v;
      do {
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(flags + c) : "memory");
        if (v == 0u && global_timer_ns() - t0 > 2000000000ull) {
          atomicCAS(&g_device_error, DEV_ERR_NONE, DEV_ERR_WAIT_TIMEOUT);
          ok = false;
        }
      } while (v == 0u && ok);
    }
  }
  if (__syncthreads_or(!ok)) return;
#pragma unroll 8
  for (int e = tid; e < total; e += MV_THREADS) {
    const int k = words.div(e);
    if (src[k] != nullptr) reinterpret_cast<uint2*>(dst[k])[e - k * words.d] = cells[e];
  }
  if (w_to != nullptr) *w_to = w;
}

// CTAs of a pair's cluster: about EV_PART tokens each, 16 at most (24 requests of up to 16,384 tokens: 24 us in one CTA a
// pair, 32 in clusters of two); EV_HELD tokens of a part fit its shared memory
constexpr int EV_PART = 16384, EV_HELD = 46 * 1024;
static int evict_cluster(int max_n) {
  int c = 1;
  while (c < 16 && c * EV_PART < max_n) c *= 2;
  return c;
}
// Kept positions a CTA of the move takes: 16 to 24 KB of cells
static int evict_chunk(int cell) { return cell <= 200 ? 128 : cell <= 392 ? 64 : 32; }

}  // namespace qp

using namespace qp;

// [int2 lens (seqs)][ticket, 16 bytes][uint32 flags: one a chunk of every pair], the chunks counted at their smallest
extern "C" int64_t qp_evict_workspace_bytes(int num_seqs, int num_kv_heads, int max_seqlen_k, int keep) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || keep <= 0) return 256;
  const int64_t chunks = (std::min(keep, std::max(max_seqlen_k, 1)) + 31) / 32;
  return (num_seqs * 8ll + 15) / 16 * 16 + 16 + static_cast<int64_t>(num_seqs) * num_kv_heads * chunks * 4 + 256;
}

extern "C" int qp_evict_cache(void* cache, int cell_bytes, int block_size, int64_t block_stride, int64_t head_stride,
                              int64_t slot_stride, int num_kv_heads, float* weights, int64_t weights_stride_block,
                              int64_t weights_stride_slot, int64_t weights_stride_head, int num_seqs,
                              const int32_t* seqused_k, int max_seqlen_k, const int32_t* block_table,
                              int64_t block_table_stride, const int32_t* out_block_table,
                              int64_t out_block_table_stride, int keep, int keep_first, int keep_last, int32_t* kept,
                              int32_t* seqused_out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (num_seqs < 0 || num_kv_heads <= 0 || block_size <= 0 || max_seqlen_k < 0)
    return set_error(QP_ERR_INVALID, "evict: bad sizes (seqs %d, kv heads %d, block %d)", num_seqs, num_kv_heads,
                     block_size);
  if (keep < 1 || keep_first < 0 || keep_last < 0 || keep_first > keep || keep_last > keep - keep_first)
    return set_error(QP_ERR_INVALID, "evict: keep %d with the first %d and the last %d", keep, keep_first, keep_last);
  if (num_seqs == 0) return QP_OK;
  if (num_seqs > 65535 || num_kv_heads > 65535) return set_error(QP_ERR_UNSUPPORTED, "evict: grid too large");
  if (cell_bytes <= 0 || cell_bytes % 8 || cell_bytes > 1024)
    return set_error(QP_ERR_UNSUPPORTED, "evict: cells of %d bytes (a multiple of 8 up to 1024)", cell_bytes);
  if (((block_stride | head_stride | slot_stride) & 7) || (reinterpret_cast<uintptr_t>(cache) & 7))
    return set_error(QP_ERR_LAYOUT, "evict: cells must be 8-byte aligned");
  if (!cache || !weights || !seqused_k || !block_table || !kept || !seqused_out || !workspace)
    return set_error(QP_ERR_INVALID, "evict: null pointer");
  const int64_t need = qp_evict_workspace_bytes(num_seqs, num_kv_heads, max_seqlen_k, keep);
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need)
    return set_error(QP_ERR_WORKSPACE, "evict: workspace of %lld bytes < %lld", (long long)workspace_bytes,
                     (long long)need);
  const int chunk = evict_chunk(cell_bytes);
  const int chunks = (std::min(keep, std::max(max_seqlen_k, 1)) + chunk - 1) / chunk;
  const int64_t tickets = static_cast<int64_t>(num_seqs) * num_kv_heads * chunks;
  if (tickets > 0x7fffffff) return set_error(QP_ERR_UNSUPPORTED, "evict: grid too large");
  const int cluster = evict_cluster(max_seqlen_k);
  const int part = (max_seqlen_k + cluster - 1) / cluster;
  const int held = std::min(part, EV_HELD);
  int2* lens = static_cast<int2*>(workspace);
  uint32_t* ticket = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + (num_seqs * 8ll + 15) / 16 * 16);
  const EvictParams p{static_cast<uint8_t*>(cache), FastDiv(block_size), block_stride, head_stride, slot_stride,
                      cell_bytes, weights, weights_stride_block, weights_stride_slot, weights_stride_head,
                      num_kv_heads, num_seqs, seqused_k, block_table, block_table_stride, out_block_table,
                      out_block_table_stride, max_seqlen_k, keep, keep_first, keep_last, kept, seqused_out, lens,
                      ticket, ticket + 4, chunks, chunk, held};
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(sizeof(EvictShared)) + EV_HELD * 4);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return set_error(QP_ERR_CUDA, "evict attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(num_kv_heads * cluster), static_cast<unsigned>(num_seqs));
  cfg.blockDim = dim3(EV_THREADS);
  cfg.dynamicSmemBytes = sizeof(EvictShared) + static_cast<size_t>(held) * 4;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, evict_select_kernel, p);
  if (e != cudaSuccess) return set_error(QP_ERR_CUDA, "evict select launch: %s", cudaGetErrorString(e));
  cfg.gridDim = dim3(static_cast<unsigned>(tickets));
  cfg.blockDim = dim3(MV_THREADS);
  cfg.dynamicSmemBytes = static_cast<size_t>(chunk) * (2 * sizeof(void*) + (out_block_table ? 0 : cell_bytes));
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  e = cudaLaunchKernelEx(&cfg, evict_move_kernel, p, FastDiv(cell_bytes / 8));
  if (e != cudaSuccess) return set_error(QP_ERR_CUDA, "evict move launch: %s", cudaGetErrorString(e));
  return QP_OK;
}
