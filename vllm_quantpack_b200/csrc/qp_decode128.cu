// K1 at head size 128: split-KV paged decode of up to 32 query rows (qlen x query heads per KV head) per KV head over
// an int4 / k8v4 cache, with the query preparation inside; the merge (K2, qp_decode.cu) follows it. It takes the
// launch parameters of the head 256 / 512 kernel, so the decode, the static-scratch decode, the varlen launch and the
// chunk prefill serve head 128 through it.
//
//   t_rk = (softmax_scale / 128) log2(e) q_r . k_k      q_r: the row in the RHT domain
//   o_r  = sum_k 2^(t_rk - M_r) v_k / sum_k 2^(t_rk - M_r)
//
// What bounds it: a cell is 136 bytes (int4) or 200 (k8v4) and the rows are few, so the cache's bytes are the floor;
// the work to keep below it is the conversion of the codes, 2 MMAs' worth of tensor work per 8 rows and key pair and
// the softmax. A wide tcgen05 tile would take its operands through TMEM (at head 256 that conversion and its
// hand-offs bound the kernel, not the cache), so here each warp works alone on its own keys with register operands:
//   - a warp has its own ring of raw stages (32 cells each), filled by bulk copies that its own lanes issue: no
//     barrier between warps until the end, no producer warp;
//   - the keys are the M of mma.m16n8k16 and the query rows its N (8 at a time), so few rows waste nothing:
//       S^T (16 keys x 8 rows)      = K (codes as fp16 subnormals, 128 channels) x Q^T
//       O^T (16 channels x 8 rows) += V^T (codes as fp16 subnormals, 16 keys)    x P^T
//     a code is one AND away from an operand register (u x 2^-24; a high nibble 16 u x 2^-24, its channel's query
//     divided by 16, or its output: exact). The key zero point comes off the score in fp32 (row sum of q times zp);
//     the value zero point is one more channel row of V^T, subtracted at the end. S^T becomes P^T by movmatrix;
//   - a reference maximum per row and a power of two per row that keeps P x value scale inside fp16, both set at the
//     row's first keys and changed only when a bound is passed (one vote per 32 keys); the row sums stay in each lane.
// The warps' O^T, maxima and sums meet once in shared memory at the end.
// Measured (int4, 32 requests of 32,768 keys, 4 KV heads): 8 rows 115 us = 5.0 TB/s, 76 % of HBM; 12 rows 157 us; 16
// rows k8v4 over 16 ragged requests 75 us = 3.8 TB/s. Bound by issue (the conversions' AND and PRMT run at half rate) at
// 8 rows, with the tensor pipe (8 cycles an m16n8k16 and sub-partition) and three warps a sub-partition above that. Three
// CTAs of 80 registers at 8 rows measured 136 us, 16 warps of 128 registers at 16 rows 235 against 218 us (spills).
#include <math.h>

#include <algorithm>
#include <atomic>

#include "qp_api_internal.h"
#include "qp_common.cuh"
#include "qp_decode.cuh"
#include "qp_tcgen05.cuh"

namespace qp {

constexpr int D1_KEYS = 32;      // keys of a raw stage: two 16-cell runs, each inside one page
// P x value scale x row factor (the fp16 operand) and a lane's row sum (fp32) may grow to these before the row's
// maximum and factor change
constexpr float D1_P_LIMIT = 8192.f, D1_L_LIMIT = 0x1p60f;

template <int FMT, int NT>
struct D1 {
  using CL = Cell<FMT, 128>;
  static constexpr int WARPS = NT == 2 ? 12 : 8;
  static constexpr int CTAS = NT == 1 ? 2 : 1;  // per SM: 128 registers a thread, or 168 (16 rows) / 255
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int ROWS = 8 * NT;
  static constexpr int START = NT == 1 ? 32 : 64;  // what starting on a pair costs, in tiles (find_share)
  static constexpr int RUNS = NT <= 2 ? 2 : 1;  // 16-key runs taken at a time (registers)
  static constexpr int STAGE = D1_KEYS * CL::BYTES;
  static constexpr int STAGES = FMT == FMT_INT4 ? (NT >= 3 ? 4 : 3) : (NT >= 3 ? 3 : 2);
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int RED = WARPS * ROWS * 128 * 4;  // the warps' O^T at the end, in the ring's place
  static constexpr int OFF_Q = RING > RED ? RING : RED;  // B operand of QK: [NT][4][32 lanes] x 16 bytes
  static constexpr int OFF_ROW = OFF_Q + NT * 4 * 32 * 16;  // [ROWS / 2] float4: two score scales, two -sums x scale
  static constexpr int OFF_LIM = OFF_ROW + ROWS * 8;        // [ROWS] int2: first and last key the row sees
  static constexpr int OFF_ST = OFF_LIM + ROWS * 8;         // [WARPS][ROWS] float4: maximum, sum, row factor
  static constexpr int OFF_BAR = OFF_ST + WARPS * ROWS * 16;
  static constexpr int BYTES = OFF_BAR + WARPS * STAGES * 8;
  static_assert(STAGE % 16 == 0 && OFF_Q % 16 == 0 && OFF_BAR % 8 == 0, "alignment");
  static_assert(CTAS * (BYTES + 1024) <= 233472, "shared memory of an SM");
};

// transpose of an 8 x 8 b16 matrix held as an MMA accumulator pair (lane 4 g + t: row g, columns 2 t, 2 t + 1)
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint2 lds64(const uint8_t* p) { return *reinterpret_cast<const uint2*>(p); }
__device__ __forceinline__ uint32_t lds32(const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(p); }
__device__ __forceinline__ uint32_t h2_pack(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// a power of two at or below 1 / x for finite x > 0 (1 / 2 < x p <= 1 up to the ends of the exponent range)
__device__ __forceinline__ float pow2_below_inverse(float x) {
  int e = static_cast<int>((__float_as_uint(x) >> 23) & 0xFFu) - 127;  // x < 2^(e + 1)
  e = min(max(-(e + 1), -126), 126);
  return exp2_int(e);
}

// maximum over the lanes that hold the same rows (lane % 4)
__device__ __forceinline__ float column_max(float x) {
#pragma unroll
  for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
  return x;
}
// A operand of QK from cells ca (rows g) and cb (rows g + 8): this lane's quarter of the channels, step s at ka[s]
template <int FMT>
__device__ __forceinline__ void key_operand(const uint8_t* ca, const uint8_t* cb, int t4, uint32_t (&ka)[8][4]) {
  if constexpr (FMT == FMT_INT4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint2 a = lds64(ca + t4 * 16 + h * 8), b = lds64(cb + t4 * 16 + h * 8);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t xa = w ? a.y : a.x, xb = w ? b.y : b.x;
        const int s = 4 * h + 2 * w;
        ka[s][0] = xa & 0x000F000Fu;
        ka[s][1] = xb & 0x000F000Fu;
        ka[s][2] = xa & 0x00F000F0u;
        ka[s][3] = xb & 0x00F000F0u;
        ka[s + 1][0] = (xa >> 8) & 0x000F000Fu;
        ka[s + 1][1] = (xb >> 8) & 0x000F000Fu;
        ka[s + 1][2] = (xa >> 8) & 0x00F000F0u;
        ka[s + 1][3] = (xb >> 8) & 0x00F000F0u;
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const uint2 a = lds64(ca + t4 * 32 + h * 8), b = lds64(cb + t4 * 32 + h * 8);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t xa = (w ? a.y : a.x) ^ 0x80808080u, xb = (w ? b.y : b.x) ^ 0x80808080u;
        const int s = 2 * h + w;
        ka[s][0] = prmt(xa, 0u, 0x4140);
        ka[s][1] = prmt(xb, 0u, 0x4140);
        ka[s][2] = prmt(xa, 0u, 0x4342);
        ka[s][3] = prmt(xb, 0u, 0x4342);
      }
    }
  }
}

// first tile that any row of the sequence sees (0 without a sliding window)
__device__ __forceinline__ int first_tile(const DecodeParams& p, const DecodeSpan& sp) {
  return p.window > 0 ? max(0, sp.vis_base - p.window + 1) / D1_KEYS : 0;
}
// tiles of a sequence of a balanced batch
__device__ __forceinline__ int tiles_of(const DecodeParams& p, int seq) {
  const int qlen = p.cu_seqlens_q[seq + 1] - p.cu_seqlens_q[seq], n = p.seqused_k[seq];
  const int lo = p.window > 0 ? max(0, n - qlen + p.tokens_after - p.window + 1) / D1_KEYS : 0;
  return qlen > 0 ? max(0, (n + D1_KEYS - 1) / D1_KEYS - lo) : 0;
}
// partials [from, to) of a KV head's rows hold nothing
__device__ __forceinline__ void close_slots(const DecodeParams& p, const DecodeSpan& sp, int kvh, int rows, int from,
                                            int to, int tid, int threads) {
  const int m = to - from;
  for (int e = tid; e < rows * m; e += threads) {
    const int r = e / m, tok = sp.q0 + r / p.group, qh = kvh * p.group + r % p.group;
    p.part_lse[(static_cast<int64_t>(tok) * p.nq + qh) * p.num_splits + from + e % m] = -INFINITY;
  }
}

// A balanced launch: the tiles of all (sequence, KV head) pairs in a row, sequence by sequence, head by head, each pair
// led by C::START units that stand for what starting on it costs a CTA (its query rows, the first copies' latency, the
// merge of the warps), cut into shares of `share` units; CTA c takes the c-th. Measured in one sweep (us; START 32 / 64
// / 128): 12 rows over 131,072 keys 39.0 / 35.0 / 35.4 (now 36), a ragged k8v4 batch of 16 rows 81.4 / 75.4 / 79.9, 8
// rows over 1000 keys 12.4 / 14.4 / 14.4; without it, CTAs that meet two pairs end last (n 131,072: 45). The
// shares with tiles of a pair are its partials, in order. share: as even as the grid allows, at least a tile a warp,
// and so long that no pair meets more than num_splits shares (T <= share (num_splits - 1) tiles meet at most
// num_splits): a request much longer than the others, cut into num_splits shares at most, leaves CTAs without work.
struct Share {
  int64_t share, hi;  // units of a share, end of this CTA's
  int64_t unit;       // where the pair of (seq, kvh) starts
  int seq, kvh;
  int tiles;          // the pair's tiles
};

// False when this CTA has nothing to do. Sequences with queries but no tile get their partials closed here.
template <class C>
__device__ __forceinline__ bool find_share(const DecodeParams& p, uint8_t* smem, Share& out) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x, ctas = gridDim.x;
  int64_t* found = reinterpret_cast<int64_t*>(smem);  // sequence, its first unit, its tiles
  int64_t* tot = found + 4;                           // [WARPS]
  int* top = reinterpret_cast<int*>(tot + C::WARPS);  // [WARPS]
  const auto units_of = [&](int t) { return t > 0 ? static_cast<int64_t>(t + C::START) * p.nkv : 0; };
  int64_t total = 0;
  int most = 0, mine = 0;
  for (int b = tid; b < p.num_seqs; b += C::THREADS) {
    mine = tiles_of(p, b);
    total += units_of(mine);
    most = max(most, mine);
    if (mine == 0 && b % ctas == cta) {
      const DecodeSpan sp = decode_span(p, b);
      for (int h = 0; h < p.nkv && sp.qlen > 0; ++h)
        close_slots(p, sp, h, min(sp.qlen * p.group, C::ROWS), 0, p.num_splits, 0, 1);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, d);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
  }
  if (lane == 0) {
    tot[warp] = total;
    top[warp] = most;
  }
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < C::WARPS; ++w) {
    total += tot[w];
    most = max(most, top[w]);
  }
  // (shares of under 2^31 units: a cache of 2^36 keys)
  const uint32_t even = static_cast<uint32_t>((total + ctas - 1) / ctas);
  const uint32_t room = static_cast<uint32_t>(most + C::START + p.num_splits - 2) / (p.num_splits - 1);
  const int64_t share = max(max(even, room), static_cast<uint32_t>(C::WARPS));
  const int64_t lo = cta * share, hi = min(lo + share, total);
  if (lo >= hi) return false;
  // the sequence that unit lo lies in: the warps scan 32 sequences each at a time
  int64_t before = 0;
  for (int b0 = 0;; b0 += C::THREADS) {
    const int b = b0 + tid, t = p.num_seqs <= C::THREADS ? mine : b < p.num_seqs ? tiles_of(p, b) : 0;
    const int64_t u = units_of(t);
    int64_t incl = u;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    __syncthreads();
    if (lane == 31) tot[warp] = incl;
    __syncthreads();
    int64_t base = before;
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) {
      if (w < warp) base += tot[w];
      before += tot[w];
    }
    const int64_t start = base + incl - u;
    if (start <= lo && lo < start + u) {
      found[0] = b;
      found[1] = start;
      found[2] = t;
    }
    if (lo < before) break;
  }
  __syncthreads();
  out.seq = static_cast<int>(found[0]);
  out.tiles = static_cast<int>(found[2]);
  out.kvh = static_cast<int>(static_cast<uint32_t>(lo - found[1]) / static_cast<uint32_t>(out.tiles + C::START));
  out.unit = found[1] + static_cast<int64_t>(out.kvh) * (out.tiles + C::START);
  out.share = share;
  out.hi = hi;
  __syncthreads();
  fence_async_smem();  // the scratch lies in the ring's place
  return true;
}

// Tiles [tile0, tile0 + ntl) of (sequence, KV head) into partial `slot` of its rows. Returns false when a copy never
// landed (in every thread). at_stage, phase: where the warp's ring stands.
template <int FMT, int DT, int NT, bool FEAT>
__device__ __forceinline__ bool decode128_segment(const DecodeParams& p, const DecodeSpan& sp, uint8_t* smem, int kvh,
                                                  int tile0, int ntl, int slot, int& at_stage, uint32_t& phase) {
  using C = D1<FMT, NT>;
  using CL = typename C::CL;
  using EL = Elem<DT>;
  constexpr int WARPS = C::WARPS, CELL = CL::BYTES, ROWS = C::ROWS, STAGES = C::STAGES;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int n = sp.n, rows = min(sp.qlen * p.group, ROWS);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR) + warp * STAGES;
  uint8_t* ring = smem + warp * STAGES * C::STAGE;

  // the warp's first query row and its signs are on their way while the copies are set up
  const auto load_row = [&](int r, float (&x)[4]) {
    const int tok = sp.q0 + r / p.group, qh = kvh * p.group + r % p.group;
    const typename EL::T* src = reinterpret_cast<const typename EL::T*>(p.q) + tok * p.q_st + qh * p.q_sh + lane * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = r < rows ? EL::to_f(src[i]) : 0.f;
  };
  float x[4];
  load_row(warp, x);
  const uint32_t signs = p.q_rotated ? 0u : p.sign_bits[lane >> 3] >> ((lane & 7) * 4);

  // ---- raw stages: this warp's i-th tile is tile0 + warp + i WARPS. Lane l holds the address of run l & 1 of tile
  // 16 w + l / 2 for the current window w of 16 tiles (the page numbers are read one window ahead) and issues that
  // run's copy when its turn comes; the even lane of a pair also announces the tile's bytes.
  const int my_tiles = ntl > warp ? (ntl - warp + WARPS - 1) / WARPS : 0;
  const auto run_key = [&](int i) { return (tile0 + warp + i * WARPS) * D1_KEYS + (lane & 1) * 16; };
  const auto page_of = [&](int w) {
    const int i = 16 * w + (lane >> 1), k = run_key(i);
    return i < my_tiles && k < n ? sp.btab[k / p.block_size] : -1;
  };
  const uint8_t* src = nullptr;  // null: no such run
  const auto set_src = [&](int w, int page) {
    const int k = run_key(16 * w + (lane >> 1));
    src = page < 0 ? nullptr
                   : p.cache + static_cast<int64_t>(page) * p.block_stride +
                         static_cast<int64_t>(kvh) * p.head_stride + static_cast<int64_t>(k % p.block_size) * CELL;
  };
  set_src(0, page_of(0));
  int page_next = page_of(1);
  int to_issue = 0, issue_stage = at_stage;  // a segment leaves no copy in flight: the ring goes on where it was read
  const auto issue = [&]() {  // the next tile's copies, if there is one
    if (to_issue > 0 && (to_issue & 15) == 0) {
      set_src(to_issue >> 4, page_next);
      page_next = page_of((to_issue >> 4) + 1);
    }
    if ((lane >> 1) == (to_issue & 15) && src != nullptr) {
      uint8_t* dst = ring + issue_stage * C::STAGE + (lane & 1) * 16 * CELL;
      if ((lane & 1) == 0)
        mbar_arrive_expect_tx(&bars[issue_stage], (run_key(to_issue) + 16 < n ? 32 : 16) * CELL);
      bulk_g2s(dst, src, 16 * CELL, &bars[issue_stage]);
    }
    ++to_issue;
    if (++issue_stage == STAGES) issue_stage = 0;
  };
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) issue();

  // ---- query rows: one warp per row, rotated, scaled by a power of two to |q| < 2^14 and rounded to fp16 in the
  // operand's order. The rounding (2^-12 of a value) is what the head 256 / 512 kernel takes too: through the scores it
  // is 4e-4 of an output (P's to fp16 is 2e-4), below a bf16 output's own rounding (1.6e-3) and twice an fp16 output's
  // (2.1e-4): 4.8e-4 in all. A second fp16 term for fp16 rows would leave 2.9e-4, in a chain of products of its own, and
  // was measured at 8 % more time for 8 rows, 20 to 28 % for 12 and 16, 42 to 52 % for 32: not taken, the values
  // themselves hold 4 bits.
  float4* rowp = reinterpret_cast<float4*>(smem + C::OFF_ROW);
  int4* lim = reinterpret_cast<int4*>(smem + C::OFF_LIM);
  for (int r = warp; r < ROWS; r += WARPS) {
    if (r > warp) load_row(r, x);
    if (!p.q_rotated) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((signs >> i) & 1u) x[i] = -x[i];
      warp_wht<4>(x, lane);
    }
    const float am = warp_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
    int ex = 0;
    if (am > 0.f) {
      frexpf(am, &ex);
      ex = 14 - ex;
    }
    float sum = 0.f;
    __half* qf = reinterpret_cast<__half*>(smem + C::OFF_Q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = lane * 4 + i;
      const bool hi = FMT == FMT_INT4 && (c & 1);
      const __half h = __float2half_rn(ldexpf(x[i], hi ? ex - 4 : ex));
      sum += hi ? 16.f * __half2float(h) : __half2float(h);
      const int k = qk_k_of_channel<FMT>(c), pair = k >> 1;  // lane t of the operand holds pairs 16 t .. 16 t + 15
      qf[(((r >> 3) * 4 + ((pair >> 2) & 3)) * 32 + (r & 7) * 4 + (pair >> 4)) * 8 + (pair & 3) * 2 + (k & 1)] = h;
    }
    sum = warp_sum(sum);
    if (lane == 0) {
      float* rw = reinterpret_cast<float*>(rowp + (r >> 1)) + (r & 1);
      const float a = r < rows ? ldexpf(p.qk_scale, 24 - ex) : 0.f;  // the codes enter as u x 2^-24
      rw[0] = a;
      rw[2] = -ldexpf(sum, -24) * a;
      const int vis = sp.vis_base + r / p.group;
      const bool all = r >= rows;  // a padding row (q = 0) sees every key
      reinterpret_cast<int2*>(lim)[r] = make_int2((FEAT && p.window > 0 && !all) ? vis - p.window + 1 : 0,
                                                  all ? n - 1 : min(vis, n - 1));
    }
  }
  __syncthreads();

  const float capl = FEAT ? p.softcap * LOG2E : 0.f;
  const float cap_k = capl > 0.f ? 2.f * LOG2E / capl : 0.f;
  // keys below `open` hide nothing from any row; with a window keys from `shut` on are inside every row's
  const int open = min(sp.vis_base, n - 1);
  const int shut = (FEAT && p.window > 0) ? sp.vis_base + sp.qlen - p.window : 0;
  // the key of MMA row g is 16-cell run's key kap (row g + 8: kap + 2): with it the lanes' reads of key words (8
  // bytes at 4 t words) and of value words (word g of keys 4 apart) touch every bank once at the int4 cell's stride
  const int kap = (g & 1) | ((g & 2) << 2) | (g & 4);
  const int kv4 = ((t4 & 1) << 3) | ((t4 & 2) << 1);  // first of the four keys whose values the lane pairs up
  const uint32_t zmask = g == 0 ? 0x000F000Fu : 0u;    // the zero points are channel row 0 of one more A tile
  const uint4* qfrag = reinterpret_cast<const uint4*>(smem + C::OFF_Q) + lane;
  uint4 qreg[NT == 1 ? 4 : 1];
  if constexpr (NT == 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) qreg[j] = qfrag[j * 32];
  }
  float o[NT][8][4] = {}, z[NT][4] = {};
  // per pair of rows 2 t, 2 t + 1: -maximum, value factor, row sum
  float2 nM[NT], F[NT], L[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    nM[nt] = make_float2(0.f, 0.f);
    F[nt] = make_float2(1.f, 1.f);
    L[nt] = make_float2(0.f, 0.f);
  }

  uint32_t opened_rows = 0;  // bit 2 nt + e: row 2 t + e of row block nt has seen a key
  bool open_all = false, ok = true;
  int i = 0, key_t = (tile0 + warp) * D1_KEYS;
#pragma unroll 1
  for (; i < my_tiles; ++i, key_t += WARPS * D1_KEYS) {
    issue();
    ok = !__any_sync(0xffffffffu, !mbar_wait_spin(&bars[at_stage], phase));
    if (!ok) break;
    const uint8_t* stage = ring + at_stage * C::STAGE;
    if (++at_stage == STAGES) {
      at_stage = 0;
      phase ^= 1u;
    }
    // the runs past the sequence hold whatever the stage held before: masked like the keys behind n in the last run
#pragma unroll 1
    for (int r0 = 0; r0 < 2; r0 += C::RUNS) {
      const int key0 = key_t + r0 * 16;
      const uint8_t* run0 = stage + r0 * 16 * CELL;
      // S^T - M in log2 units: s[u][nt][0]: key kap, rows 2 t and 2 t + 1; [1]: key kap + 2
      float2 s[C::RUNS][NT][2];
      float vs[C::RUNS][2];
      const bool masked = key0 + 16 * C::RUNS - 1 > open || (FEAT && key0 < shut);
#pragma unroll
      for (int u = 0; u < C::RUNS; ++u) {
        const uint8_t* ca = run0 + u * 16 * CELL + kap * CELL;
        const uint8_t* cb = ca + 2 * CELL;
        uint32_t ka[8][4];
        key_operand<FMT>(ca, cb, t4, ka);
        // scales carry their zero point in the low 4 mantissa bits: kept (2^-19 of the scale, below P's 2^-12)
        const uint32_t wa = lds32(ca + CL::KS), wb = lds32(cb + CL::KS);
        const float ks[2] = {__uint_as_float(wa), __uint_as_float(wb)};
        float kz[2];
        if constexpr (FMT == FMT_INT4) {
          kz[0] = ks[0] * static_cast<float>(wa & 0xFu);
          kz[1] = ks[1] * static_cast<float>(wb & 0xFu);
        } else {
          kz[0] = ks[0] * 128.f;
          kz[1] = ks[1] * 128.f;
        }
        vs[u][0] = __uint_as_float(lds32(ca + CL::VS));
        vs[u][1] = __uint_as_float(lds32(cb + CL::VS));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 q;
            if constexpr (NT == 1) q = qreg[j];
            else q = qfrag[(nt * 4 + j) * 32];
            mma_f16_16816(c, ka[2 * j], q.x, q.y);
            mma_f16_16816(c, ka[2 * j + 1], q.z, q.w);
          }
          const float4 rp = rowp[nt * 4 + t4];  // scale of rows 2 t, 2 t + 1, then -(row sum) x scale
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 kr = __fmul2_rn(make_float2(ks[h], ks[h]), make_float2(rp.x, rp.y));
            const float2 c2 = make_float2(c[2 * h], c[2 * h + 1]), z2 = make_float2(kz[h], kz[h]);
            if constexpr (!FEAT) {
              s[u][nt][h] = __ffma2_rn(c2, kr, __ffma2_rn(z2, make_float2(rp.z, rp.w), nM[nt]));
            } else {
              float2 t = __ffma2_rn(c2, kr, __fmul2_rn(z2, make_float2(rp.z, rp.w)));
              if (capl > 0.f) t = make_float2(softcap_log2(t.x, capl, cap_k), softcap_log2(t.y, capl, cap_k));
              s[u][nt][h] = __fadd2_rn(t, nM[nt]);
            }
          }
        }
      }
      bool odd = false;  // a value scale that 0 x P would not take out, in front of a window or of a later token
      if (masked) {
#pragma unroll
        for (int u = 0; u < C::RUNS; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int key = key0 + 16 * u + kap + 2 * h;
            if (key >= n) vs[u][h] = 0.f;  // any bits, NaN too
            odd = odd || !(fabsf(vs[u][h]) < INFINITY);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const int4 l = lim[nt * 4 + t4];  // first and last key of row 2 t, then of row 2 t + 1
              if (key < l.x || key > l.y) s[u][nt][h].x = -INFINITY;
              if (key < l.z || key > l.w) s[u][nt][h].y = -INFINITY;
            }
          }
      }
      // P = 2^s and P x value scale x row factor; the row sums take P before its rounding
      float2 pr[C::RUNS][NT][2], pv[C::RUNS][NT][2];
      bool slow = !open_all || odd;
      float2 l[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float big = 0.f;
        l[nt] = L[nt];
#pragma unroll
        for (int u = 0; u < C::RUNS; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 x = s[u][nt][h];
            pr[u][nt][h] = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            pv[u][nt][h] = __fmul2_rn(pr[u][nt][h], __fmul2_rn(make_float2(vs[u][h], vs[u][h]), F[nt]));
            l[nt] = __fadd2_rn(l[nt], pr[u][nt][h]);
            big = fmaxf(big, fmaxf(pv[u][nt][h].x, pv[u][nt][h].y));
          }
        slow = slow || big > D1_P_LIMIT || fmaxf(l[nt].x, l[nt].y) > D1_L_LIMIT;
      }
      if (__any_sync(0xffffffffu, slow)) {
        bool opened = true;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float2 of;  // what O^T and the zero-point row are multiplied by
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const auto at = [e](float2& v) -> float& { return e ? v.y : v.x; };
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < C::RUNS; ++u) mx = fmaxf(mx, fmaxf(at(s[u][nt][0]), at(s[u][nt][1])));
            mx = column_max(mx);
            const bool opening = !((opened_rows >> (2 * nt + e)) & 1u);
            // an unopened row has maximum 0, no sum and no output yet
            const float up = opening ? (mx == -INFINITY ? 0.f : mx) : fmaxf(mx, 0.f);
            const float sc = opening ? 0.f : fast_exp2(-up);
            at(nM[nt]) -= up;
            at(l[nt]) = at(L[nt]) * sc;
            float pm = 0.f;
#pragma unroll
            for (int u = 0; u < C::RUNS; ++u)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                at(pr[u][nt][h]) = fast_exp2(at(s[u][nt][h]) - up);
                at(l[nt]) += at(pr[u][nt][h]);
                // (a masked key's value scale may be NaN)
                at(pv[u][nt][h]) = at(s[u][nt][h]) == -INFINITY ? 0.f : at(pr[u][nt][h]) * vs[u][h];
                pm = fmaxf(pm, at(pv[u][nt][h]));
              }
            pm = column_max(pm);
            // Where the maximum has moved up, what is left of the output and the products of these keys may be far below
            // 1 (value scales that fell while the scores rose), where fp16 has no digits for what comes: the factor
            // is raised, by as much as leaves the largest output (2^20 o: up to 15, a code, times the sum over the
            // keys) below 2^9, so that keys like the old ones stay within D1_P_LIMIT.
            float om = fmaxf(z[nt][e], z[nt][e + 2]);
#pragma unroll
            for (int ti = 0; ti < 8; ++ti) om = fmaxf(om, fmaxf(o[nt][ti][e], o[nt][ti][e + 2]));
            const float most = fmaxf(pm * at(F[nt]), column_max(om) * sc * 0x1p11f);
            at(of) = sc;
            if (pm > 0.f && (opening || pm * at(F[nt]) > D1_P_LIMIT)) {
              const float fn = pow2_below_inverse(pm);
              at(of) = sc * (fn / at(F[nt]));
              at(F[nt]) = fn;
            } else if (most > 0.f && most < 0.015625f) {
              const float raise = fminf(pow2_below_inverse(most), 0x1p126f / at(F[nt]));
              at(of) = sc * raise;
              at(F[nt]) *= raise;
            }
#pragma unroll
            for (int u = 0; u < C::RUNS; ++u)
#pragma unroll
              for (int h = 0; h < 2; ++h) at(pv[u][nt][h]) *= at(F[nt]);
            if (mx != -INFINITY) opened_rows |= 1u << (2 * nt + e);
            opened = opened && ((opened_rows >> (2 * nt + e)) & 1u);
          }
#pragma unroll
          for (int ti = 0; ti < 8; ++ti)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][ti][e] *= (e & 1) ? of.y : of.x;
#pragma unroll
          for (int e = 0; e < 4; ++e) z[nt][e] *= (e & 1) ? of.y : of.x;
        }
        open_all = __all_sync(0xffffffffu, opened);
      }
      uint32_t pb[C::RUNS][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        L[nt] = l[nt];
#pragma unroll
        for (int u = 0; u < C::RUNS; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) pb[u][nt][h] = movmatrix_trans(h2_pack(pv[u][nt][h].x, pv[u][nt][h].y));
      }
      // O^T: words g and g + 8 of four keys; tile ti takes nibble ti of each (channels 8 g + ti, 64 + 8 g + ti)
#pragma unroll
      for (int u = 0; u < C::RUNS; ++u) {
        const uint8_t* cv = run0 + u * 16 * CELL + kv4 * CELL;
        const uint8_t* vc = cv + CL::V + 4 * g;
        uint32_t v[4][2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // a0: word g, keys 0-1; a1: word g + 8; a2, a3: keys 2-3
          v[e][0] = lds32(vc + (e & 2) * CELL + (e & 1) * 32);
          v[e][1] = lds32(vc + ((e & 2) + 1) * CELL + (e & 1) * 32);
        }
#pragma unroll
        for (int hw = 0; hw < 2; ++hw) {  // low, then high half of the words: nibbles 0-3, 4-7
          uint32_t y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = prmt(v[e][0], v[e][1], hw ? 0x7632u : 0x5410u);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t a[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = ((q & 2) ? (y[e] >> 8) : y[e]) & ((q & 1) ? 0x00F000F0u : 0x000F000Fu);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16_16816(o[nt][4 * hw + q], a, pb[u][nt][0], pb[u][nt][1]);
          }
        }
        const uint32_t a[4] = {prmt(lds32(cv + CL::VS), lds32(cv + CELL + CL::VS), 0x5410u) & zmask, 0u,
                               prmt(lds32(cv + 2 * CELL + CL::VS), lds32(cv + 3 * CELL + CL::VS), 0x5410u) & zmask, 0u};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16_16816(z[nt], a, pb[u][nt][0], pb[u][nt][1]);
      }
    }
    __syncwarp();  // every lane has read the stage before it is filled again
  }
  if (!ok) {  // a copy never landed (the error word says so): leave once the others in flight have
    for (const int end = min(i + STAGES, my_tiles); i < end; ++i) {
      mbar_wait_bounded(&bars[at_stage], phase);
      if (++at_stage == STAGES) {
        at_stage = 0;
        phase ^= 1u;
      }
    }
  }
  if (__syncthreads_or(!ok)) return false;

  // ---- the warps' partials meet: O^T (channels of a row contiguous), maximum, sum and factor of each row
  float* red = reinterpret_cast<float*>(smem);
  float4* st = reinterpret_cast<float4*>(smem + C::OFF_ST);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = e ? L[nt].y : L[nt].x;
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      const float zz = __shfl_sync(0xffffffffu, z[nt][e], t4);  // channel row 0 lies in lanes 0-3
      const int r = nt * 8 + 2 * t4 + e;
      float* dst = red + (warp * ROWS + r) * 128 + 8 * g;
#pragma unroll
      for (int b = 0; b < 2; ++b) {  // channels 8 g .. 8 g + 7, then 64 + 8 g ..
        float v[8];
#pragma unroll
        for (int ti = 0; ti < 8; ++ti) v[ti] = o[nt][ti][2 * b + e] * ((ti & 1) ? 0.0625f : 1.f) - zz;
        *reinterpret_cast<float4*>(dst + 64 * b) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(dst + 64 * b + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
      if (g == 0) st[warp * ROWS + r] = make_float4(e ? -nM[nt].y : -nM[nt].x, l, e ? F[nt].y : F[nt].x, 0.f);
    }
  }
  __syncthreads();
  for (int r = warp; r < rows; r += WARPS) {  // one warp per row: lane l holds channels 4 l .. 4 l + 3
    float mx = -INFINITY, sum = 0.f;  // a warp with sum 0 saw no key of the row: its maximum says nothing
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, st[w * ROWS + r].y != 0.f ? st[w * ROWS + r].x : -INFINITY);
    if (mx == -INFINITY) mx = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
      if (st[w * ROWS + r].y != 0.f) sum += st[w * ROWS + r].y * fast_exp2(st[w * ROWS + r].x - mx);
    const float inv = sum > 0.f ? 16777216.f / sum : 0.f;  // 2^24: the codes entered as subnormals
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float4 s = st[w * ROWS + r];
      const float f1 = s.y != 0.f ? fast_exp2(s.x - mx) * inv : 0.f, f2 = 1.f / s.z;
      const float4 v = *reinterpret_cast<const float4*>(red + (w * ROWS + r) * 128 + 4 * lane);
      a.x += v.x * f1 * f2;
      a.y += v.y * f1 * f2;
      a.z += v.z * f1 * f2;
      a.w += v.w * f1 * f2;
    }
    const int tok = sp.q0 + r / p.group, qh = kvh * p.group + r % p.group;
    const int64_t at = (static_cast<int64_t>(tok) * p.nq + qh) * p.num_splits + slot;
    *reinterpret_cast<float4*>(p.part_o + at * 128 + 4 * lane) = a;
    // a NaN sum (NaN scores) stays NaN in the partial's lse, so the merge passes it on
    if (lane == 0) p.part_lse[at] = sum == 0.f ? -INFINITY : mx + log2f(sum);
  }
  return true;
}

template <int FMT, int DT, int NT, bool FEAT>
__global__ void __launch_bounds__((D1<FMT, NT>::THREADS), (D1<FMT, NT>::CTAS)) decode128_kernel(const DecodeParams p) {
  using C = D1<FMT, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x;
  asm volatile("griddepcontrol.launch_dependents;");  // the merge's launch may begin; it waits for this grid's end

  if ((tid & 31) == 0) {
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR) + (tid >> 5) * C::STAGES;
    for (int s = 0; s < C::STAGES; ++s) mbar_init(&bars[s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  int at_stage = 0;  // each warp's ring runs on from one segment to the next
  uint32_t phase = 0;

  // plain grid (split, KV head, sequence): num_splits equal parts of every sequence, one segment a CTA
  int seq = blockIdx.z, kvh = blockIdx.y, slot = blockIdx.x;
  Share sh{};
  if (p.balanced) {
    if (!find_share<C>(p, smem, sh)) return;
    seq = sh.seq;
    kvh = sh.kvh;
  }
#pragma unroll 1
  for (;;) {
    const DecodeSpan sp = decode_span(p, seq);
    const int rows = min(sp.qlen * p.group, C::ROWS);
    const int tile_lo = FEAT ? first_tile(p, sp) : 0;
    int at, ntl, close = slot + 1;  // the partials [slot + 1, close) get no keys
    if (p.balanced) {
      const int64_t first = sh.unit + C::START;  // unit of the pair's tile 0
      const int64_t lo = max(blockIdx.x * sh.share, first), hi = min(sh.hi, first + sh.tiles);
      at = static_cast<int>(lo - first);
      ntl = static_cast<int>(hi - lo);  // 0 or less: the share ends inside the pair's lead
      slot = blockIdx.x - static_cast<int>(first / sh.share);
      close = at + ntl == sh.tiles ? p.num_splits : slot + 1;  // the pair's last share
    } else {
      if (sp.qlen <= 0) return;
      const int tiles = max(0, (sp.n + D1_KEYS - 1) / D1_KEYS - tile_lo);
      const int tps = (tiles + p.num_splits - 1) / p.num_splits;
      at = slot * tps;
      ntl = max(0, min(tps, tiles - at));
      if (ntl == 0) close_slots(p, sp, kvh, rows, slot, slot + 1, tid, C::THREADS);
    }
    if (ntl > 0) {
      if (!decode128_segment<FMT, DT, NT, FEAT>(p, sp, smem, kvh, tile_lo + at, ntl, slot, at_stage, phase)) return;
      close_slots(p, sp, kvh, rows, slot + 1, close, tid, C::THREADS);
    }
    if (!p.balanced) return;
    sh.unit += C::START + sh.tiles;  // on to the next pair
    if (sh.unit >= sh.hi) return;
    if (++kvh == p.nkv) {
      kvh = 0;
      do sh.tiles = tiles_of(p, ++seq);
      while (sh.tiles == 0);
    }
    fence_async_smem();  // the partials lay in the ring's place: the next copies come after them
    __syncthreads();
  }
}

template <int FMT, int DT, int NT, bool FEAT>
static int launch_d1(DecodeParams dp, int grid_z, cudaStream_t st) {
  using C = D1<FMT, NT>;
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(decode128_kernel<FMT, DT, NT, FEAT>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES);
    if (e != cudaSuccess) return set_error(QP_ERR_CUDA, "decode 128 attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  dim3 grid(static_cast<unsigned>(dp.num_splits), static_cast<unsigned>(dp.nkv), static_cast<unsigned>(grid_z));
  // a decode batch is balanced over the CTAs the GPU holds at a time; one partial a row, a chunk's and a varlen
  // launch's sub-sequences keep the plain grid
  dp.balanced = dp.subseq == nullptr && dp.chunk_q == 0 && dp.num_splits > 1;
  if (dp.balanced)
    grid = dim3(static_cast<unsigned>(std::min<int64_t>(static_cast<int64_t>(device_sm_count()) * C::CTAS,
                                                        static_cast<int64_t>(dp.num_splits) * dp.nkv * grid_z)));
  decode128_kernel<FMT, DT, NT, FEAT><<<grid, C::THREADS, C::BYTES, st>>>(dp);
  return check_launch("decode 128");
}

template <int FMT, int DT, bool FEAT>
static int launch_d1_rows(const DecodeParams& dp, int rows, int grid_z, cudaStream_t st) {
  if (rows <= 8) return launch_d1<FMT, DT, 1, FEAT>(dp, grid_z, st);
  if (rows <= 16) return launch_d1<FMT, DT, 2, FEAT>(dp, grid_z, st);
  if (rows <= 24) return launch_d1<FMT, DT, 3, FEAT>(dp, grid_z, st);
  return launch_d1<FMT, DT, 4, FEAT>(dp, grid_z, st);
}

template <int FMT>
static int launch_d1_fmt(int dtype, const DecodeParams& dp, int rows, int grid_z, cudaStream_t st) {
  const bool feat = dp.window > 0 || dp.softcap > 0.f;
  if (dtype == DT_BF16)
    return feat ? launch_d1_rows<FMT, DT_BF16, true>(dp, rows, grid_z, st)
                : launch_d1_rows<FMT, DT_BF16, false>(dp, rows, grid_z, st);
  return feat ? launch_d1_rows<FMT, DT_F16, true>(dp, rows, grid_z, st)
              : launch_d1_rows<FMT, DT_F16, false>(dp, rows, grid_z, st);
}

int launch_decode128(int fmt, int dtype, DecodeParams dp, int rows, int grid_z, cudaStream_t st) {
  return fmt == FMT_INT4 ? launch_d1_fmt<FMT_INT4>(dtype, dp, rows, grid_z, st)
                         : launch_d1_fmt<FMT_K8V4>(dtype, dp, rows, grid_z, st);
}

// Partials a row of a decode batch may have: twice the shares a longest sequence would meet were all as long (shorter
// ones leave the GPU's CTAs to it), one where a sequence is no longer than a CTA's warps take at a time.
template <int NT>
static int d1_num_splits(int64_t pairs, int tiles, int sms) {
  using C = D1<FMT_INT4, NT>;  // warps and CTAs do not depend on the format
  if (tiles <= C::WARPS) return 1;
  const int64_t ctas = static_cast<int64_t>(sms) * C::CTAS;
  const int64_t share = std::max<int64_t>((pairs * tiles + ctas - 1) / ctas, C::WARPS);
  const int64_t met = (tiles + share - 1) / share, most = (tiles + C::WARPS - 1) / C::WARPS;
  return static_cast<int>(std::min<int64_t>(std::min(2 * met, most) + 1, 512));
}

int decode128_num_splits(int rows, int num_seqs, int num_kv_heads, int max_seqlen_k, int sm_count) {
  if (sm_count <= 0) sm_count = device_sm_count();
  const int64_t pairs = std::max<int64_t>(1, static_cast<int64_t>(num_seqs) * num_kv_heads);
  const int tiles = std::max(1, (max_seqlen_k + D1_KEYS - 1) / D1_KEYS);
  if (rows <= 8) return d1_num_splits<1>(pairs, tiles, sm_count);
  if (rows <= 16) return d1_num_splits<2>(pairs, tiles, sm_count);
  if (rows <= 24) return d1_num_splits<3>(pairs, tiles, sm_count);
  return d1_num_splits<4>(pairs, tiles, sm_count);
}

// ---------------------------------------------------------------------------------------------------- merge
// K2 at head 128: one warp per row (lane l: channels 4 l .. 4 l + 3) for up to 32 partials, eight warps per row, every
// eighth partial each, for more. A partial is one 512-byte read of a warp, eight in flight: the partials lie in L2, so
// the reads' latency is what there is to hide.
constexpr int MG_WARPS = 8;

template <int DT, int WPR>
__global__ void __launch_bounds__(32 * MG_WARPS) merge128_kernel(const MergeParams p, int64_t rows) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int NC = WPR == 1 ? 1 : 4;  // 32 partials a warp each: 32, or 1024 in all
  __shared__ __align__(16) float acc[WPR > 1 ? MG_WARPS : 1][128];
  __shared__ float wmax[MG_WARPS], wsum[MG_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % WPR;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (MG_WARPS / WPR) + warp / WPR;
  if (r >= rows) return;  // only where a warp is a row
  const int64_t tok = r / p.nq;
  const int qh = static_cast<int>(r % p.nq);
  if (p.cu_seqlens_q != nullptr && (tok < p.cu_seqlens_q[0] || tok >= p.cu_seqlens_q[p.num_seqs])) return;
  const float* lse = p.part_lse + tok * p.pl_t + qh * p.pl_h;
  float w[NC], M = -INFINITY;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int s = part + WPR * (32 * c + lane);
    w[c] = s < p.num_splits ? lse[s * p.pl_s] : -INFINITY;
    M = fmaxf(M, w[c]);
  }
  M = warp_max(M);
  if constexpr (WPR > 1) {
    if (lane == 0) wmax[warp] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPR; ++i) M = fmaxf(M, wmax[i]);
  }
  const float sink = p.sinks != nullptr ? p.sinks[qh] * LOG2E : -INFINITY;  // base 2, like the partials' lse
  M = fmaxf(M, sink);
  const float* po = p.part_o + tok * p.po_t + qh * p.po_h + 4 * lane;
  float x[4] = {0.f, 0.f, 0.f, 0.f}, T = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    w[c] = w[c] == -INFINITY ? 0.f : exp2f(w[c] - M);
    T += w[c];
#pragma unroll 1
    for (int k = 0; k < 32 && part + WPR * (32 * c + k) < p.num_splits; k += 8) {
      float4 v[8];
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = __shfl_sync(0xffffffffu, w[c], k + j);  // 0: absent, its partial is never read
        v[j] = f[j] != 0.f ? *reinterpret_cast<const float4*>(po + (part + WPR * (32 * c + k + j)) * p.po_s)
                           : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[0] = fmaf(f[j], v[j].x, x[0]);
        x[1] = fmaf(f[j], v[j].y, x[1]);
        x[2] = fmaf(f[j], v[j].z, x[2]);
        x[3] = fmaf(f[j], v[j].w, x[3]);
      }
    }
  }
  T = warp_sum(T);
  if constexpr (WPR > 1) {
    *reinterpret_cast<float4*>(&acc[warp][4 * lane]) = make_float4(x[0], x[1], x[2], x[3]);
    if (lane == 0) wsum[warp] = T;
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int i = 1; i < WPR; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(&acc[i][4 * lane]);
      x[0] += v.x;
      x[1] += v.y;
      x[2] += v.z;
      x[3] += v.w;
      T += wsum[i];
    }
  }
  if (sink != -INFINITY) T += exp2f(sink - M);  // in the denominator only
  if (lane == 0 && p.lse_out) p.lse_out[tok * p.lo_t + qh * p.lo_h] = T == 0.f ? -INFINITY : M + log2f(T);  // NaN stays
  const float inv = T == 0.f ? 0.f : 1.f / T;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] *= inv;
  if (p.mode == 1) {
    float* dst = reinterpret_cast<float*>(p.out) + tok * p.out_st + qh * p.out_sh + 4 * lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = x[i];
    return;
  }
  warp_wht<4>(x, lane);
  apply_signs<4>(x, p.sign_bits, lane);
  using EL = Elem<DT>;
  typename EL::T* dst = reinterpret_cast<typename EL::T*>(p.out) + tok * p.out_st + qh * p.out_sh + 4 * lane;
#pragma unroll
  for (int i = 0; i < 4; ++i) dst[i] = EL::from_f(x[i] * p.out_scale);
}

template <int DT, int WPR>
static int launch_merge128_t(const MergeParams& mp, int64_t rows, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((rows + MG_WARPS / WPR - 1) / (MG_WARPS / WPR)));
  cfg.blockDim = dim3(32 * MG_WARPS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, merge128_kernel<DT, WPR>, mp, rows);
  if (e != cudaSuccess) return set_error(QP_ERR_CUDA, "merge 128 launch: %s", cudaGetErrorString(e));
  return QP_OK;
}

int launch_merge128(const MergeParams& mp, int dtype, int num_tokens, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(num_tokens) * mp.nq;
  if (rows > 0x7fffffff) return set_error(QP_ERR_UNSUPPORTED, "merge: too many rows");
  if (mp.num_splits > 32)
    return dtype == DT_BF16 ? launch_merge128_t<DT_BF16, 8>(mp, rows, st) : launch_merge128_t<DT_F16, 8>(mp, rows, st);
  return dtype == DT_BF16 ? launch_merge128_t<DT_BF16, 1>(mp, rows, st) : launch_merge128_t<DT_F16, 1>(mp, rows, st);
}

}  // namespace qp
