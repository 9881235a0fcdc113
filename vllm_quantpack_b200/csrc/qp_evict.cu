// K5: eviction from a paged cache by accumulated attention weight. Of every sequence longer than `keep`, each KV head
// keeps its first keep_first tokens, its last keep_last and the heaviest of those between, `keep` in all (equal weights:
// the earlier token); the kept cells and their weights move, in order, to positions 0 .. keep - 1 of the sequence's
// pages, or of other pages (a sequence whose pages others share). Cells are moved as bytes: any format, any head size.
#include <math.h>

#include <algorithm>

#include "qp_api_internal.h"
#include "qp_common.cuh"

namespace qp {

struct EvictParams {
  uint8_t* cache;
  int block_size;
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
};

// order of the weights as unsigned integers: NaN first (it goes first), -0 = +0
__device__ __forceinline__ uint32_t weight_rank(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float* weight_at(const EvictParams& p, const int32_t* table, int kvh, int i) {
  return p.weights + static_cast<int64_t>(table[i / p.block_size]) * p.w_block +
         static_cast<int64_t>(i % p.block_size) * p.w_slot + kvh * p.w_head;
}
__device__ __forceinline__ uint8_t* cell_at(const EvictParams& p, const int32_t* table, int kvh, int i) {
  return p.cache + static_cast<int64_t>(table[i / p.block_size]) * p.block_stride +
         static_cast<int64_t>(i % p.block_size) * p.slot_stride + static_cast<int64_t>(kvh) * p.head_stride;
}

constexpr int EV_THREADS = 1024;

__device__ __forceinline__ int block_scan(int x, int* sm, int* total) {  // exclusive; all threads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  __syncthreads();
  if (lane == 31) sm[warp] = incl;
  __syncthreads();
  int base = 0, all = 0;
  for (int w = 0; w < EV_THREADS / 32; ++w) {
    if (w < warp) base += sm[w];
    all += sm[w];
  }
  *total = all;
  return base + incl - x;
}

__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(const EvictParams p) {
  __shared__ int hist[256], sm[32];
  __shared__ uint32_t sel[2];
  const int kvh = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
  const int32_t* table = p.table + seq * p.table_stride;
  const int n = min(max(p.seqused[seq], 0), p.max_n);
  int32_t* kept = p.kept + (static_cast<int64_t>(seq) * p.nkv + kvh) * p.keep;
  if (n <= p.keep) {
    for (int j = tid; j < p.keep; j += EV_THREADS) kept[j] = j < n ? j : -1;
    return;
  }
  const int lo = p.first, hi = n - p.last;
  int want = p.keep - p.first - p.last;  // of [lo, hi)
  uint32_t thr = 0, mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += EV_THREADS) {
      const uint32_t r = weight_rank(*weight_at(p, table, kvh, i));
      if ((r & mask) == thr) atomicAdd(&hist[(r >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int b = 255, left = want;
      while (b > 0 && hist[b] < left) left -= hist[b--];
      sel[0] = b;
      sel[1] = left;
    }
    __syncthreads();
    thr |= sel[0] << shift;
    mask |= 255u << shift;
    want = sel[1];
    __syncthreads();
  }
  // want of the weights equal to the threshold stay, the earliest ones
  int eq = 0, out = 0;
  for (int i0 = 0; i0 < n; i0 += EV_THREADS) {
    const int i = i0 + tid;
    bool stay = i < n && (i < lo || i >= hi), tie = false;
    if (i < n && !stay) {
      const uint32_t r = weight_rank(*weight_at(p, table, kvh, i));
      stay = r > thr;
      tie = r == thr;
    }
    int total;
    const int rank = block_scan(tie, sm, &total);
    if (tie && eq + rank < want) stay = true;
    eq += total;
    const int at = block_scan(stay, sm, &total);
    if (stay) kept[out + at] = i;
    out += total;
  }
}

// One CTA per (KV head, sequence), 64 cells at a time: a position's token is never before it, so what a tile overwrites
// has been read by then.
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p) {
  extern __shared__ __align__(16) uint8_t buf[];
  const int kvh = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
  const int32_t* from = p.table + seq * p.table_stride;
  const int32_t* to = p.out_table ? p.out_table + seq * p.out_stride : from;
  const int32_t* kept = p.kept + (static_cast<int64_t>(seq) * p.nkv + kvh) * p.keep;
  const int words = p.cell / 8;
  uint2* cells = reinterpret_cast<uint2*>(buf);
  float* w = reinterpret_cast<float*>(buf + 64 * p.cell);
  for (int j0 = 0; j0 < p.keep; j0 += 64) {
    const int m = min(64, p.keep - j0);
    for (int e = tid; e < m * words; e += 256) {
      const int i = kept[j0 + e / words];
      if (i >= 0) cells[e] = reinterpret_cast<const uint2*>(cell_at(p, from, kvh, i))[e % words];
    }
    if (tid < m && kept[j0 + tid] >= 0) w[tid] = *weight_at(p, from, kvh, kept[j0 + tid]);
    __syncthreads();
    for (int e = tid; e < m * words; e += 256)
      if (kept[j0 + e / words] >= 0) reinterpret_cast<uint2*>(cell_at(p, to, kvh, j0 + e / words))[e % words] = cells[e];
    if (tid < m && kept[j0 + tid] >= 0) *weight_at(p, to, kvh, j0 + tid) = w[tid];
    __syncthreads();
  }
}

__global__ void evict_lens_kernel(const EvictParams p) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < p.num_seqs) p.seqused_out[b] = min(min(max(p.seqused[b], 0), p.max_n), p.keep);
}

}  // namespace qp

using namespace qp;

extern "C" int64_t qp_evict_workspace_bytes(int num_seqs, int num_kv_heads, int max_seqlen_k, int keep) { return 256; }

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
  const EvictParams p{static_cast<uint8_t*>(cache), block_size, block_stride, head_stride, slot_stride, cell_bytes,
                      weights, weights_stride_block, weights_stride_slot, weights_stride_head, num_kv_heads, num_seqs,
                      seqused_k, block_table, block_table_stride, out_block_table, out_block_table_stride, max_seqlen_k,
                      keep, keep_first, keep_last, kept, seqused_out};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(num_kv_heads), static_cast<unsigned>(num_seqs));
  evict_select_kernel<<<grid, EV_THREADS, 0, st>>>(p);
  int rc = check_launch("evict select");
  if (rc) return rc;
  const int smem = 64 * cell_bytes + 64 * 4;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(evict_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return set_error(QP_ERR_CUDA, "evict attribute: %s", cudaGetErrorString(e));
  }
  evict_move_kernel<<<grid, 256, smem, st>>>(p);
  rc = check_launch("evict move");
  if (rc) return rc;
  evict_lens_kernel<<<(num_seqs + 255) / 256, 256, 0, st>>>(p);
  return check_launch("evict lengths");
}
