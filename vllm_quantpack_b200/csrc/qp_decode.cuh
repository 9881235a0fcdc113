// What the split-KV decode kernels share: the launch parameters and the span of a sequence (qp_decode.cu: head 256 and
// 512 on tcgen05; qp_decode128.cu: head 128), the cell layout, the softcap and the merge's partial layout.
#pragma once
#include <math.h>

#include "qp_common.cuh"

namespace qp {

constexpr int DEC_MAX_ROWS = 32;  // query rows (tokens x query heads per KV head) a CTA holds at most
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_SLACK = 8.f;  // log2 units a row's scores may pass its running maximum by before a rescale

struct DecodeParams {
  const void* q;
  int64_t q_st, q_sh;  // element strides of q (token, head)
  const int32_t* cu_seqlens_q;
  const int32_t* seqused_k;
  const int32_t* block_table;
  int64_t bt_stride;
  const uint8_t* cache;
  int block_size;
  int64_t block_stride, head_stride;  // bytes; cells of one (block, head) are contiguous (slot stride == cell)
  int nq, nkv, group;  // query heads, KV heads, query heads per KV head
  float qk_scale;      // softmax_scale / head_size * log2(e)
  const uint32_t* sign_bits;
  int q_rotated;        // q already in the RHT domain
  const uint8_t* qrec;  // prepared query rows: [kv head][token][query head of the group] x q_rec_bytes(HS)
  int64_t num_tokens;
  int tokens_after;  // sequence tokens after this call's keys (held by other ranks), clamped to the query tokens
  // chunk_q > 0: the num_tokens query tokens are ONE sequence's chunk (its last positions, causal among themselves)
  // over chunk_n cached keys through block-table row 0, served as sub-sequences of chunk_q tokens (grid z), each
  // reading only the keys its last token sees. cu_seqlens_q / seqused_k are not read.
  int chunk_q, chunk_n;
  // subseq != null: sequence z of the grid is subseq[z] = {first query token, query tokens, keys its last token
  // sees, block-table row}, causal inside it (built on the device by varlen_table_kernel; entries past the real ones
  // hold 0 query tokens). cu_seqlens_q / seqused_k are not read.
  const int4* subseq;
  // window > 0: vLLM's SLIDING_WINDOW (1 + window_size[0]): a query token whose last visible key is p sees the keys
  // [p - window + 1, p] only (vllm/v1/attention/ops/triton_attention_helpers.py:196-218, vLLM 0.22)
  int window;
  // softcap > 0: every score S (natural units) becomes softcap x tanh(S / softcap) before the softmax, vLLM's
  // apply_softcap (vllm/v1/attention/ops/triton_attention_helpers.py:28-36, triton_unified_attention.py:513-514)
  float softcap;
  // head 128 only: the num_seqs sequences of cu_seqlens_q / seqused_k share the grid's CTAs by their lengths (set by
  // launch_decode128), each cut into num_splits parts at most, instead of num_splits equal parts of each
  int num_seqs, balanced;
  int num_splits;
  float* part_o;    // [tokens][nq][splits][HS]
  float* part_lse;  // [tokens][nq][splits], log2 units
};

// A grid's sequence: its query tokens [q0, q0 + qlen), its keys [0, n), the last key its first token sees (before
// clamping to n - 1) and its block-table row.
struct DecodeSpan {
  int q0, qlen, n, vis_base;
  const int32_t* btab;
};

__device__ __forceinline__ DecodeSpan decode_span(const DecodeParams& p, int seq) {
  DecodeSpan s;
  if (p.subseq != nullptr) {
    const int4 e = p.subseq[seq];
    s.q0 = e.x;
    s.qlen = e.y;
    s.n = e.z;
    s.vis_base = s.n - s.qlen;
    s.btab = p.block_table + static_cast<int64_t>(e.w) * p.bt_stride;
  } else if (p.chunk_q > 0) {
    s.q0 = seq * p.chunk_q;
    s.qlen = min(p.chunk_q, static_cast<int>(p.num_tokens) - s.q0);
    s.vis_base = p.chunk_n - static_cast<int>(p.num_tokens) + s.q0 + p.tokens_after;
    s.n = min(p.chunk_n, s.vis_base + s.qlen);
    s.btab = p.block_table;
  } else {
    s.q0 = p.cu_seqlens_q[seq];
    s.qlen = p.cu_seqlens_q[seq + 1] - s.q0;
    s.n = p.seqused_k[seq];
    s.vis_base = s.n - s.qlen + p.tokens_after;
    s.btab = p.block_table + static_cast<int64_t>(seq) * p.bt_stride;
  }
  return s;
}

template <int FMT, int HS>
struct Cell {
  static constexpr int KB = FMT == FMT_INT4 ? HS / 2 : HS;  // key bytes
  static constexpr int BYTES = KB + 8 + HS / 2;
  static constexpr int KS = KB, V = KB + 4, VS = KB + 4 + HS / 2;  // field offsets
};

// capl x tanh(t / capl) for a score t in log2 units (capl = softcap x log2 e, cap_k = 2 log2 e / capl), from
// tanh(y) = 1 - 2 / (e^{2y} + 1) taken on |y| and given t's sign: absolute error ~1e-7 x capl, which is what a softmax
// argument needs (no cancellation matters once it is multiplied back by capl); e^{2|y|} = 2^{|t| cap_k}, its exponent
// held below 64 so the quotient stays finite.
__device__ __forceinline__ float softcap_log2(float t, float capl, float cap_k) {
  const float a = fast_exp2(fminf(fabsf(t) * cap_k, 64.f));
  return copysignf(capl * (1.f - __fdividef(2.f, a + 1.f)), t);
}

// k index (0..HS-1) of the QK operand that carries channel c. int4: column j = 4 w + m of a key's TMEM lane holds
// the pair lop3'd from word w (shifted right 8 for m >= 2; low nibbles for even m, high for odd), i.e. channels
// 8 w + m (low half) and 8 w + m + 4 (high half); k8v4: the natural order (prmt takes bytes 0, 1 then 2, 3).
template <int FMT>
__host__ __device__ __forceinline__ int qk_k_of_channel(int c) {
  if constexpr (FMT == FMT_INT4) return 8 * (c >> 3) + 2 * (c & 3) + ((c >> 2) & 1);
  else return c;
}

// The merge of split partials (K2, and its head-128 form).
struct MergeParams {
  const float* part_o;
  const float* part_lse;     // log2 units
  int64_t po_t, po_h, po_s;  // element strides of part_o (token, head, part); channel stride 1
  int64_t pl_t, pl_h, pl_s;
  int num_splits;
  int nq;
  int mode;  // 0: inverse RHT / head, cast to the model dtype; 1: fp32 RHT-domain O and lse (log2) out
  void* out;
  int64_t out_st, out_sh;  // element strides of out
  float* lse_out;          // base 2, the sinks included (may be null)
  int64_t lo_t, lo_h;
  const uint32_t* sign_bits;
  float out_scale;  // multiplies the output (mode 0: 1 / head)
  // mode 0, may be null: per query head, a sink logit (natural units) whose exp joins every row's softmax
  // denominator once, vLLM's attention sinks (vllm/v1/attention/ops/triton_attention_helpers.py:108-138: the row
  // maximum starts at the sink with sum 1 in one segment only; triton_unified_attention.py:356-359)
  const float* sinks;
  // head 128, may be null: rows outside the query tokens [cu_seqlens_q[0], cu_seqlens_q[num_seqs]) are left alone (a
  // padded batch: nothing wrote their partials)
  const int32_t* cu_seqlens_q;
  int num_seqs;
};

// Launches the head-128 kernel (qp_decode128.cu) on the parameters of launch_decode, `rows` query rows per KV head at
// most, and its merge.
int launch_decode128(int fmt, int dtype, DecodeParams dp, int rows, int grid_z, cudaStream_t st);
// Partials a row of a head-128 decode batch may have.
int decode128_num_splits(int rows, int num_seqs, int num_kv_heads, int max_seqlen_k, int sm_count);
int launch_merge128(const MergeParams& mp, int dtype, int num_tokens, cudaStream_t st);

}  // namespace qp
