// K4: the softmax weight every cached key got from this call's query rows, added to a paged fp32 score:
//   w_k += sum over the query tokens i of the sequence and the query heads of k's KV head of 2^(t_ik - lse_i)
//   t_ik = (softmax_scale / hs) log2(e) q_i . k_k      (RHT domain; softcap and sliding window as in the attention)
// with lse the base-2 log-sum-exp the attention call returned for the row, so the weights a row hands out sum to one
// (less what a sink took). A key a row does not see gets nothing from it.
#include <math.h>

#include <algorithm>

#include "qp_api_internal.h"
#include "qp_common.cuh"
#include "qp_decode.cuh"

namespace qp {

struct WeightParams {
  DecodeParams d;      // queries, lengths, block table, cache, features (num_splits and the partials unused)
  const float* lse;    // [tokens][nq]
  float* weights;
  int64_t w_block, w_slot, w_head;  // element strides
  int head_size;
};

// One thread a key, the query rows rotated into shared memory one by one.
template <int FMT, int DT, int HS>
__global__ void __launch_bounds__(128) weights_kernel(const WeightParams wp) {
  const DecodeParams& p = wp.d;
  using EL = Elem<DT>;
  using CL = Cell<FMT, HS>;
  constexpr int E = HS / 32;
  __shared__ float qrow[8][HS];
  __shared__ float row_lse[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = blockIdx.y;
  const DecodeSpan sp = decode_span(p, blockIdx.z);
  const int key = blockIdx.x * 128 + threadIdx.x;
  if (sp.qlen <= 0 || blockIdx.x * 128 >= sp.n) return;
  const bool valid = key < sp.n;
  const uint8_t* cell = nullptr;
  float ks = 0.f, zp = 0.f;
  int64_t at = 0;
  if (valid) {
    const int64_t blk = sp.btab[key / p.block_size];
    cell = p.cache + blk * p.block_stride + static_cast<int64_t>(kvh) * p.head_stride +
           static_cast<int64_t>(key % p.block_size) * CL::BYTES;
    at = blk * wp.w_block + static_cast<int64_t>(key % p.block_size) * wp.w_slot + kvh * wp.w_head;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(cell + CL::KS);
    ks = __uint_as_float(FMT == FMT_INT4 ? w & 0xFFFFFFF0u : w);
    zp = FMT == FMT_INT4 ? static_cast<float>(w & 0xFu) : 0.f;
  }
  const int rows = sp.qlen * p.group;
  const float capl = p.softcap * LOG2E, cap_k = capl > 0.f ? 2.f * LOG2E / capl : 0.f;
  float sum = 0.f;
  for (int r0 = 0; r0 < rows; r0 += 8) {
    __syncthreads();
    for (int r = warp; r < 8 && r0 + r < rows; r += 4) {
      const int tok = sp.q0 + (r0 + r) / p.group, qh = kvh * p.group + (r0 + r) % p.group;
      const typename EL::T* src = reinterpret_cast<const typename EL::T*>(p.q) + tok * p.q_st + qh * p.q_sh + lane * E;
      float x[E];
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = EL::to_f(src[i]);
      if (!p.q_rotated) {
        apply_signs<E>(x, p.sign_bits, lane);
        warp_wht<E>(x, lane);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) qrow[r][lane * E + i] = x[i] * p.qk_scale;
      if (lane == 0) row_lse[r] = wp.lse[static_cast<int64_t>(tok) * p.nq + qh];
    }
    __syncthreads();
    if (!valid) continue;
    float s[8] = {};
    for (int c = 0; c < HS; c += 2) {
      float k0, k1;
      if constexpr (FMT == FMT_INT4) {
        const uint8_t b = cell[c / 2];
        k0 = (b & 15) - zp;
        k1 = (b >> 4) - zp;
      } else {
        k0 = static_cast<int8_t>(cell[c]);
        k1 = static_cast<int8_t>(cell[c + 1]);
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] = fmaf(k1, qrow[r][c + 1], fmaf(k0, qrow[r][c], s[r]));
    }
    for (int r = 0; r < 8 && r0 + r < rows; ++r) {
      const int vis = sp.vis_base + (r0 + r) / p.group;
      float t = s[r] * ks;
      if (capl > 0.f) t = softcap_log2(t, capl, cap_k);
      if (key <= vis && (p.window <= 0 || key > vis - p.window) && row_lse[r] != -INFINITY)
        sum += exp2f(t - row_lse[r]);
    }
  }
  if (!valid) return;
  if (key >= sp.vis_base) wp.weights[at] = sum;  // the call's own tokens: no earlier weight
  else atomicAdd(wp.weights + at, sum);          // a page may be shared by sequences of the call
}

template <int FMT, int DT>
static int launch_weights(const WeightParams& wp, const dim3& grid, cudaStream_t st) {
  switch (wp.head_size) {
    case 128: weights_kernel<FMT, DT, 128><<<grid, 128, 0, st>>>(wp); break;
    case 256: weights_kernel<FMT, DT, 256><<<grid, 128, 0, st>>>(wp); break;
    default: weights_kernel<FMT, DT, 512><<<grid, 128, 0, st>>>(wp); break;
  }
  return check_launch("attention weights");
}

}  // namespace qp

using namespace qp;

extern "C" int64_t qp_attn_weights_workspace_bytes(int64_t num_q_tokens, int num_seqs, int num_q_heads,
                                                   int num_kv_heads, int head_size) {
  return 256;
}

extern "C" int qp_accumulate_attn_weights(int fmt, int dtype, const void* q, int64_t q_stride_token,
                                          int64_t q_stride_head, int64_t num_q_tokens, int num_seqs,
                                          const int32_t* cu_seqlens_q, const int32_t* seqused_k, int max_seqlen_q,
                                          int max_seqlen_k, const int32_t* block_table, int64_t block_table_stride,
                                          const void* cache, int block_size, int64_t block_stride,
                                          int64_t head_stride, int64_t slot_stride, int64_t k_off, int64_t ks_off,
                                          int64_t v_off, int64_t vs_off, int num_q_heads, int num_kv_heads,
                                          int head_size, float softmax_scale, const uint32_t* rht_sign_bits,
                                          int q_rotated, int tokens_after_keys, int sliding_window, float softcap,
                                          const float* lse, float* weights, int64_t weights_stride_block,
                                          int64_t weights_stride_slot, int64_t weights_stride_head, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  int rc = decode_check_cache("attention weights", fmt, dtype, head_size, cache, block_size, block_stride, head_stride,
                              slot_stride, k_off, ks_off, v_off, vs_off);
  if (rc) return rc;
  if (num_seqs < 0 || num_q_tokens < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      max_seqlen_q < 0 || max_seqlen_k < 0)
    return set_error(QP_ERR_INVALID, "attention weights: bad sizes (seqs %d, tokens %lld, heads %d/%d)", num_seqs,
                     (long long)num_q_tokens, num_q_heads, num_kv_heads);
  if (tokens_after_keys < 0)
    return set_error(QP_ERR_INVALID, "attention weights: tokens_after_keys %d", tokens_after_keys);
  if (sliding_window < 0) return set_error(QP_ERR_INVALID, "attention weights: sliding_window %d", sliding_window);
  if (!(softcap >= 0.f) || isinf(softcap)) return set_error(QP_ERR_INVALID, "attention weights: softcap %g", softcap);
  if (num_seqs == 0 || num_q_tokens == 0 || max_seqlen_q == 0 || max_seqlen_k == 0) return QP_OK;
  if (num_seqs > 65535 || num_kv_heads > 65535) return set_error(QP_ERR_UNSUPPORTED, "attention weights: grid too large");
  if (!q || !cu_seqlens_q || !seqused_k || !block_table || !cache || !rht_sign_bits || !lse || !weights || !workspace)
    return set_error(QP_ERR_INVALID, "attention weights: null pointer");
  const int64_t need = qp_attn_weights_workspace_bytes(num_q_tokens, num_seqs, num_q_heads, num_kv_heads, head_size);
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need)
    return set_error(QP_ERR_WORKSPACE, "attention weights: workspace of %lld bytes < %lld", (long long)workspace_bytes,
                     (long long)need);
  WeightParams wp{};
  DecodeParams& dp = wp.d;
  dp.q = q;
  dp.q_st = q_stride_token;
  dp.q_sh = q_stride_head;
  dp.cu_seqlens_q = cu_seqlens_q;
  dp.seqused_k = seqused_k;
  dp.num_seqs = num_seqs;
  dp.block_table = block_table;
  dp.bt_stride = block_table_stride;
  dp.cache = static_cast<const uint8_t*>(cache);
  dp.block_size = block_size;
  dp.block_stride = block_stride;
  dp.head_stride = head_stride;
  dp.nq = num_q_heads;
  dp.nkv = num_kv_heads;
  dp.group = num_q_heads / num_kv_heads;
  dp.qk_scale = softmax_scale / static_cast<float>(head_size) * LOG2E;
  dp.sign_bits = rht_sign_bits;
  dp.q_rotated = q_rotated;
  dp.num_tokens = num_q_tokens;
  dp.window = sliding_window >= (1 << 30) ? 0 : sliding_window;
  // as in the decode: tokens further after the keys than this change no mask
  dp.tokens_after = static_cast<int>(std::min<int64_t>(tokens_after_keys, static_cast<int64_t>(max_seqlen_q) + dp.window));
  dp.softcap = softcap;
  wp.lse = lse;
  wp.weights = weights;
  wp.w_block = weights_stride_block;
  wp.w_slot = weights_stride_slot;
  wp.w_head = weights_stride_head;
  wp.head_size = head_size;
  const dim3 grid(static_cast<unsigned>((max_seqlen_k + 127) / 128), static_cast<unsigned>(num_kv_heads),
                  static_cast<unsigned>(num_seqs));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fmt == FMT_INT4)
    return dtype == DT_BF16 ? launch_weights<FMT_INT4, DT_BF16>(wp, grid, st) : launch_weights<FMT_INT4, DT_F16>(wp, grid, st);
  return dtype == DT_BF16 ? launch_weights<FMT_K8V4, DT_BF16>(wp, grid, st) : launch_weights<FMT_K8V4, DT_F16>(wp, grid, st);
}
