// K4: the softmax weight every cached key got from this call's query rows, added to a paged fp32 score:
//   w_k += sum over the query tokens i of the sequence and the query heads of k's KV head of 2^(t_ik - lse_i)
//   t_ik = (softmax_scale / hs) log2(e) q_i . k_k      (RHT domain; softcap and sliding window as in the attention)
// with lse the base-2 log-sum-exp the attention call returned for the row, so the weights a row hands out sum to one
// (less what a sink took). A key a row does not see gets nothing from it.
//
// The result is fp32, and its relative error is the score's absolute one: a query row rounded to fp16 (2^-12 of a
// score of several units) would leave three digits. So a row enters as the sum of two fp16 terms (2^-22; K4q writes
// them with the RHT applied) and a score takes twice the products; the key codes are exact (u - zp, int8).
//
// The keys are the M of the MMA and the query rows its N, so a key is a TMEM lane and its sum over rows stays in one
// thread:  S^T (128 keys x N rows) = K_op (TMEM) x [Q_hi; Q_lo]^T (shared memory)  ->  sum_n 2^(k_scale S + ...)
// One persistent CTA per SM; roles:
//   warp 0        query tiles: one bulk copy of a prepared record (both terms in the operand's swizzled layout, the
//                 rows' -lse and mask bounds) into a ring; a tile that the next keys use again is not copied again;
//   2 warps       (the second and the last, on different SM sub-partitions) issue HS / 8 MMAs of K 16 per 128 keys and
//                 query tile, each into its own S^T buffer, so that one's waits pass while the other's MMAs run;
//   4 or 8 warps  key operand: thread = key, its codes to exact fp16 in TMEM (two sets on alternate tiles where few rows
//                 make the conversion the longest role);
//   8 warps       thread = key: exponentials, the sum over the rows, one add to global memory per key; two sets, one
//                 for each S^T buffer;
//   1 or 4 warps  cp.async of the key part of the cells, 8 bytes a lane (a cell's key part is not 16-byte aligned),
//                 into a ring of raw stages. With the 64-byte fetch hint the values in between mostly stay in HBM:
//                 75 % of the cells' bytes are read at int4 and head 256, 62 % at head 512, 94 % at head 128 (without
//                 the hint, in 128-byte fetches, all of them).
// Few rows (up to 32, decoding): a tile of 128 keys meets one query tile, two key tiles alternate in TMEM. 262,144 keys,
// 24 rows x 4 KV heads, int4, head 256: 75 us for 214 MB of DRAM traffic (2.9 TB/s; 22 us would be the keys' bytes at
// full rate); held by the hand-offs between the roles, no one of them alone (without the second term 71 us, without the
// conversion 68, with an eighth of the copies 62). Many rows (prompts): a group of two key tiles stays in TMEM while all
// query tiles that see it stream through L2, so a query tile's bytes serve 256 keys; bound by the MMAs of the two terms
// at head 256 (1024 queries x 40,960 keys, 24 / 4 heads: 0.68 ms at full clocks, 1,500 TFLOP/s with both terms, 91 % of
// the library product's peak; 0.78 ms, 79 %, when calls follow one another under the power cap). At head 128 no pipe is
// full (three whole prompts to 2,777 tokens: 0.28 ms, of it 0.19 this kernel and most of the rest K4q; tensor 44 %, XU
// 44 %): two summing warps a scheduler wait for their score reads.
// The (key group, query tile) steps of all sequences and KV heads are cut evenly over the CTAs; where a cut falls
// inside a group its parts go to the workspace and K4f adds them in order, so the sum does not depend on timing.
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "qp_api_internal.h"
#include "qp_common.cuh"
#include "qp_decode.cuh"
#include "qp_tcgen05.cuh"

namespace qp {

struct WeightParams {
  DecodeParams d;    // queries, lengths, block table, cache, features (num_splits and the partials unused)
  const float* lse;  // [tokens][nq]
  float* weights;
  int64_t w_block, w_slot, w_head;  // element strides
  FastDiv block_size;
  int max_q, max_k;  // bounds of the lengths that the launch was sized for
  // workspace: prepared query tiles; per CTA the sums of a group's parts and what they are
  uint8_t* qrec;
  float* part;    // [CTAs][2][256]: a group begun by an earlier CTA, a group that goes on in the next
  int4* records;  // [CTAs][2]: {valid, goes on}, {valid, sequence, KV head, group}
};

constexpr int WT_KEYS = 128;     // keys of a tile (TMEM lanes)
constexpr int WT_SMALL_ROWS = 32;  // query rows of a KV head up to which a sequence is one query tile

// NR: rows of a query tile; KT: key tiles of a group; MANY: a sequence may have several query tiles
template <int FMT, int HS, int NR, int KT, bool MANY>
struct WT {
  using CL = Cell<FMT, HS>;
  static constexpr int SLOTS = HS == 512 ? 1 : 2;  // key tiles in TMEM
  static constexpr int ACOLS = HS / 2;             // TMEM columns of one
  static constexpr int S = SLOTS * ACOLS;          // S^T: two buffers of NR columns
  static constexpr int COLS = S + 2 * NR <= 256 ? 256 : 512;
  static_assert(KT <= SLOTS && S + 2 * NR <= 512, "TMEM");
  static constexpr int PIECES = CL::KB / 8 + 1;    // 8-byte pieces of a key's codes and scale
  static constexpr int KEY = PIECES * 8;           // bytes of a key in a raw stage (an odd multiple of 8: no conflicts)
  static constexpr int STAGE = WT_KEYS * KEY;
  static constexpr int ATOM = NR * 128;            // 64 channels of a query tile's term
  static constexpr int TERM = HS / 64 * ATOM;
  static constexpr int ROWS = 2 * TERM;            // then [NR] float -lse, [NR] int last key, [NR] int first key,
  static constexpr int HEAD = ROWS + 12 * NR;      // then {score scale, least last key, greatest first key}
  static constexpr int QREC = (HEAD + 16 + 1023) / 1024 * 1024;
  static constexpr int QS = HS == 512 && (!MANY || FMT == FMT_K8V4) ? 1 : 2;
  // warps: 0 query tiles, 1 MMA, then the key operand, the weights, the raw keys (many rows keep a key tile long enough
  // for one converting set and one loading warp) and the second MMA warp
  static constexpr int CSETS = MANY || SLOTS == 1 ? 1 : 2;
  // where a TMEM slot is not always the same MMA warp's, both follow every tile (so that neither misses a phase)
  static constexpr bool BOTH = MANY || SLOTS == 1;
  static constexpr int W_SUM = 2 + 4 * CSETS, W_LOAD = W_SUM + 8;
  static constexpr int RUN_STEPS = (16 * PIECES + 31) / 32;  // cp.asyncs of a lane for 16 keys
  static constexpr int MISC = 4 * 128 * 4 + 2 * 128 * 4 + 32 * 8 + 64;
  static constexpr int RS0 = (231000 - QS * QREC - MISC) / STAGE;
  // raw stages, and loading warps (tiles in turn): a stage is always filled by the same warp and emptied by the same
  // converting set, which so see all of its phases
  static constexpr int RS = RS0 >= 8 ? 8 : RS0 >= 4 ? 4 : 2;
  static constexpr int LOADERS = MANY ? 1 : RS < 4 ? 2 : 4;
  static constexpr int W_MMA1 = W_LOAD + LOADERS, THREADS = 32 * (W_MMA1 + 1);
  static constexpr int OFF_RAW = QS * QREC;
  static constexpr int OFF_KP = OFF_RAW + RS * STAGE;  // [4][128] float: key scale of the last tiles
  static constexpr int OFF_RED = OFF_KP + 4 * 128 * 4;  // [2][128] float: the second half's sums
  static constexpr int OFF_BAR = OFF_RED + 2 * 128 * 4;
  static constexpr int OFF_TMEM = OFF_BAR + 32 * 8;
  static constexpr int BYTES = OFF_TMEM + 64;  // the TMEM address, then where the share starts
  static_assert(RS0 >= 2 && BYTES <= 232448, "shared memory");
};

enum { T_Q_FULL = 0, T_Q_EMPTY = 2, T_K_FULL = 4, T_K_FREE = 6, T_S_FULL = 8, T_S_FREE = 10, T_FINAL = 12,
       T_RAW_FULL = 13, T_RAW_EMPTY = 21 };  // [RS <= 8] each

// ---- the steps of a sequence: for each key group, the query tiles [first, end) with a row that sees one of its keys
struct Steps {
  int qlen, n, vis_base, group, window, ntq, groups;
};
template <int NR, int GK>
__device__ __forceinline__ Steps steps_of(const WeightParams& wp, int seq) {
  const DecodeParams& p = wp.d;
  Steps s;
  s.qlen = p.cu_seqlens_q[seq + 1] - p.cu_seqlens_q[seq];
  s.n = min(p.seqused_k[seq], wp.max_k);
  s.vis_base = p.seqused_k[seq] - s.qlen + p.tokens_after;
  s.group = p.group;
  s.window = p.window;
  s.ntq = (min(s.qlen, wp.max_q) * p.group + NR - 1) / NR;
  if (s.qlen <= 0 || s.n < 0) s.n = s.ntq = 0;
  s.groups = (s.n + GK - 1) / GK;
  return s;
}
template <int NR, int GK>
__device__ __forceinline__ void tiles_seeing(const Steps& s, int g, int& first, int& end) {
  const int lo = g * GK, hi = min(lo + GK, s.n) - 1;  // the group's keys
  if (s.window == 0 && lo <= s.vis_base) {
    first = 0;
    end = s.ntq;
    return;
  }
  const int tok = max(0, lo - s.vis_base);
  first = tok >= s.qlen ? s.ntq : static_cast<int>(static_cast<int64_t>(tok) * s.group / NR);
  end = s.ntq;
  if (s.window > 0) {
    const int last = min(s.qlen - 1, hi + s.window - 1 - s.vis_base);
    end = last < 0 ? first : max(first, static_cast<int>((static_cast<int64_t>(last + 1) * s.group - 1) / NR) + 1);
  }
}
// group from which the steps of a group are not all ntq any more (no window)
template <int GK>
__device__ __forceinline__ int full_groups(const Steps& s) {
  return s.window > 0 ? 0 : max(0, min(s.groups, s.vis_base < 0 ? 0 : s.vis_base / GK + 1));
}
template <int NR, int GK>
__device__ __forceinline__ int64_t count_steps(const Steps& s) {
  const int full = full_groups<GK>(s), groups = s.groups;
  int64_t t = static_cast<int64_t>(full) * s.ntq;
  for (int g = full; g < groups; ++g) {
    int a, b;
    tiles_seeing<NR, GK>(s, g, a, b);
    t += b - a;
  }
  return t;
}

// Few rows: a sequence's one query tile sees the groups [first_group, s.groups) (all of them without a window).
template <int GK>
__device__ __forceinline__ int first_group(const Steps& s) {
  if (s.ntq == 0) return s.groups;
  if (s.window == 0) return 0;
  const int lo = max(0, s.vis_base - s.window + 1);
  return lo >= s.n ? s.groups : lo / GK;
}
template <int NR, int GK, bool MANY>
__device__ __forceinline__ int64_t steps_in(const Steps& s) {
  if constexpr (MANY) return count_steps<NR, GK>(s);
  else return s.groups - first_group<GK>(s);
}

// Walks a CTA's share in order; every role runs its own. Many rows: a segment is a group and the query tiles [qa, qb) of
// its [first, end). Few rows: the groups [g, g1) of a (sequence, KV head).
template <int NR, int GK, bool MANY>
struct Walk {
  int seq, kvh, g, g1, qa, qb, first, end;
  int qbase;  // query tiles of the sequences before
  int left;   // steps of the share not yet handed out
  Steps s;

  __device__ __forceinline__ bool next(const WeightParams& wp) {
    if (left <= 0) return false;
    for (;;) {
      if constexpr (MANY) {
        if (qb < end) {  // the group's tiles from qb on
          qa = qb;
          qb = min(end, qa + left);
          left -= qb - qa;
          return true;
        }
        ++g;
      } else if (g1 < s.groups) {
        g = g1;
        g1 = min(s.groups, g + left);
        left -= g1 - g;
        return true;
      }
      if (!MANY || g >= s.groups) {
        if (++kvh == wp.d.nkv) {
          kvh = 0;
          do {
            qbase += s.ntq;
            s = steps_of<NR, GK>(wp, ++seq);
          } while (s.n == 0);
        }
        g = MANY ? 0 : first_group<GK>(s);
      }
      g1 = MANY ? g + 1 : g;
      if constexpr (MANY) {
        tiles_seeing<NR, GK>(s, g, first, end);
        qb = first;
      }
    }
  }
};

// What every CTA works out before it starts: the whole of the steps, its share and where that begins. In shared memory.
struct ShareStart {
  int64_t lo, hi;
  int seq, kvh, g, q, qbase;
};
static_assert(sizeof(ShareStart) <= 48, "room beside the TMEM address");

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// The sequence that unit `at` lies in, units(b) units a sequence, and what comes before it of units and tiles(b).
// scratch: 2 x 24 words of 64 bits. All `threads` threads call it and get the same answer in found[0..2].
template <class U, class T>
__device__ __forceinline__ void find_sequence(int num_seqs, int threads, int64_t at, U&& units, T&& tiles,
                                              int64_t* scratch, int64_t* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = threads / 32;
  int64_t before_u = 0, before_t = 0;
  for (int b0 = 0; b0 < num_seqs; b0 += threads) {
    const int b = b0 + tid;
    const int64_t u = b < num_seqs ? units(b) : 0, t = b < num_seqs ? tiles(b) : 0;
    int64_t iu = u, it = t;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t ou = __shfl_up_sync(0xffffffffu, iu, d), ot = __shfl_up_sync(0xffffffffu, it, d);
      if (lane >= d) {
        iu += ou;
        it += ot;
      }
    }
    __syncthreads();
    if (lane == 31) {
      scratch[warp] = iu;
      scratch[24 + warp] = it;
    }
    __syncthreads();
    int64_t bu = before_u, bt = before_t;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) {
        bu += scratch[w];
        bt += scratch[24 + w];
      }
      before_u += scratch[w];
      before_t += scratch[24 + w];
    }
    const int64_t start = bu + iu - u;
    if (start <= at && at < start + u) {
      found[0] = b;
      found[1] = start;
      found[2] = bt + it - t;
    }
    if (at < before_u) break;
  }
  __syncthreads();
}

template <int NR, int GK, bool MANY, int THREADS>
__device__ __forceinline__ void find_start(const WeightParams& wp, int64_t* scratch, ShareStart* out) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const auto units = [&](int b) { return steps_in<NR, GK, MANY>(steps_of<NR, GK>(wp, b)) * wp.d.nkv; };
  int64_t total = 0;
  for (int b = tid; b < wp.d.num_seqs; b += THREADS) total += units(b);
  total = warp_sum64(total);
  if (lane == 0) scratch[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < THREADS / 32; ++w) total += scratch[w];
  const int64_t share = (total + gridDim.x - 1) / gridDim.x, lo = blockIdx.x * share, hi = min(lo + share, total);
  int64_t* found = scratch + 48;
  if (lo < hi)
    find_sequence(wp.d.num_seqs, THREADS, lo, units, [&](int b) { return steps_of<NR, GK>(wp, b).ntq; }, scratch,
                  found);
  if (tid == 0) {
    out->lo = lo;
    out->hi = max(lo, hi);
    if (lo < hi) {
      out->seq = static_cast<int>(found[0]);
      out->qbase = static_cast<int>(found[2]);
      const Steps s = steps_of<NR, GK>(wp, out->seq);
      const int64_t each = steps_in<NR, GK, MANY>(s);
      out->kvh = static_cast<int>((lo - found[1]) / each);
      int64_t u = (lo - found[1]) % each;
      const int full = full_groups<GK>(s);
      int g, a = 0, b;
      if (!MANY) {
        g = first_group<GK>(s) + static_cast<int>(u);
      } else if (u < static_cast<int64_t>(full) * s.ntq) {
        g = static_cast<int>(u / s.ntq);
        u -= static_cast<int64_t>(g) * s.ntq;
      } else {
        u -= static_cast<int64_t>(full) * s.ntq;
        for (g = full;; ++g) {
          tiles_seeing<NR, GK>(s, g, a, b);
          if (u < b - a) break;
          u -= b - a;
        }
      }
      out->g = g;
      out->q = a + static_cast<int>(u);
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------------------------------- K4q
// One CTA per query tile: NR rows of a (sequence, KV head), rotated and scaled by a power of two common to the tile
// (|q| < 2^14 at its largest finite value: a row far smaller keeps the tile's absolute accuracy, which is what an
// exponent needs), as two fp16 terms in the operand's layout; -lse (a row without keys, and a padding row: -inf) and
// the first and last key of each row.
template <int FMT, int DT, int HS, int NR, bool MANY>
__global__ void __launch_bounds__(256) weights_qprep_kernel(const WeightParams wp) {
  asm volatile("griddepcontrol.launch_dependents;");
  using W = WT<FMT, HS, NR, 1, MANY>;
  using EL = Elem<DT>;
  constexpr int E = HS / 32, RW = NR / 8;  // channels a lane, rows a warp
  const DecodeParams& p = wp.d;
  __shared__ int64_t scratch[52];
  __shared__ float wmax[8];
  __shared__ int wvis[8], wlo[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kvh = blockIdx.y;
  int seq = blockIdx.x, qt = 0;
  if constexpr (MANY) {
    if (p.num_seqs == 1) {
      seq = 0;
      qt = blockIdx.x;
    } else {
      if (tid == 0) scratch[48] = -1;
      const auto tiles = [&](int b) { return static_cast<int64_t>(steps_of<NR, WT_KEYS>(wp, b).ntq); };
      find_sequence(p.num_seqs, 256, blockIdx.x, tiles, tiles, scratch, scratch + 48);
      if (scratch[48] < 0) return;
      seq = static_cast<int>(scratch[48]);
      qt = static_cast<int>(blockIdx.x - scratch[49]);
    }
  }
  const Steps s = steps_of<NR, WT_KEYS>(wp, seq);
  if (qt >= s.ntq) return;
  // the record's place: the sequences' tiles in a row (one place each where none has more), KV heads inside
  uint8_t* rec = wp.qrec + (static_cast<int64_t>(blockIdx.x) * p.nkv + kvh) * W::QREC;
  const int q0 = p.cu_seqlens_q[seq], rows = s.qlen * p.group;
  float x[RW][E];
  float am = 0.f;
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const int r = qt * NR + warp * RW + i;
#pragma unroll
    for (int e = 0; e < E; ++e) x[i][e] = 0.f;
    if (r < rows) {
      const int tok = q0 + r / p.group, qh = kvh * p.group + r % p.group;
      const typename EL::T* src = reinterpret_cast<const typename EL::T*>(p.q) + tok * p.q_st + qh * p.q_sh + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] = EL::to_f(src[e]);
      if (!p.q_rotated) {
        apply_signs<E>(x[i], p.sign_bits, lane);
        warp_wht<E>(x[i], lane);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) am = fmaxf(am, fabsf(x[i][e]) < INFINITY ? fabsf(x[i][e]) : 0.f);
    }
  }
  am = warp_max(am);
  int vis_min = INT_MAX, lo_max = INT_MIN;
  if (lane < RW) {  // this lane's row of the warp: its bounds and -lse
    const int rt = warp * RW + lane, r = qt * NR + rt;
    float nl = -INFINITY;
    int vis = INT_MIN, lo = INT_MIN;  // a padding row sees no key: where a tile is masked it adds 0, whatever a cell holds
    if (r < rows) {
      const int tok = r / p.group;
      const float l = wp.lse[static_cast<int64_t>(q0 + tok) * p.nq + kvh * p.group + r % p.group];
      if (l != -INFINITY) nl = -l;
      vis = s.vis_base + tok;
      if (p.window > 0) lo = vis - p.window + 1;
      vis_min = vis;
      lo_max = lo;
    }
    reinterpret_cast<float*>(rec + W::ROWS)[rt] = nl;
    reinterpret_cast<int*>(rec + W::ROWS)[NR + rt] = vis;
    reinterpret_cast<int*>(rec + W::ROWS)[2 * NR + rt] = lo;
  }
  vis_min = __reduce_min_sync(0xffffffffu, vis_min);
  lo_max = __reduce_max_sync(0xffffffffu, lo_max);
  if (lane == 0) {
    wmax[warp] = am;
    wvis[warp] = vis_min;
    wlo[warp] = lo_max;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    am = fmaxf(am, wmax[w]);
    vis_min = min(vis_min, wvis[w]);
    lo_max = max(lo_max, wlo[w]);
  }
  int ex = 0;
  if (am > 0.f) {
    frexpf(am, &ex);
    ex = 14 - ex;
  }
  if (tid == 0)
    *reinterpret_cast<float4*>(rec + W::HEAD) =
        make_float4(ldexpf(p.qk_scale, -ex), __int_as_float(vis_min), __int_as_float(lo_max), 0.f);
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const int rt = warp * RW + i;
    __half hi[E], lo[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float y = ldexpf(x[i][e], ex);
      hi[e] = __float2half_rn(y);
      lo[e] = __float2half_rn(y - __half2float(hi[e]));
    }
    // byte of channel pair k, k + 1 of a term: atom k / 64, row rt, swizzled 16-byte chunk
    const auto put = [&](int term, int chunk, const uint4& v) {
      *reinterpret_cast<uint4*>(rec + term * W::TERM + (chunk >> 3) * W::ATOM + sw128_off(rt, chunk & 7)) = v;
    };
    const auto two = [](__half a, __half b) {
      return static_cast<uint32_t>(__half_as_ushort(a)) | (static_cast<uint32_t>(__half_as_ushort(b)) << 16);
    };
    if constexpr (E == 4) {
      // two lanes hold a chunk's eight channels: the even lane writes the first term's, the odd lane the second's
      const bool odd = lane & 1;
      const uint32_t a0 = odd ? two(lo[0], lo[1]) : two(hi[0], hi[1]), a1 = odd ? two(lo[2], lo[3]) : two(hi[2], hi[3]);
      const uint32_t g0 = odd ? two(hi[0], hi[1]) : two(lo[0], lo[1]), g1 = odd ? two(hi[2], hi[3]) : two(lo[2], lo[3]);
      const uint32_t b0 = __shfl_xor_sync(0xffffffffu, g0, 1), b1 = __shfl_xor_sync(0xffffffffu, g1, 1);
      const uint32_t e0 = odd ? b0 : a0, e1 = odd ? b1 : a1, o0 = odd ? a0 : b0, o1 = odd ? a1 : b1;
      if constexpr (FMT == FMT_INT4)  // k order: channels 0 4 1 5 2 6 3 7
        put(odd, lane >> 1, make_uint4(prmt(e0, o0, 0x5410u), prmt(e0, o0, 0x7632u), prmt(e1, o1, 0x5410u),
                                       prmt(e1, o1, 0x7632u)));
      else put(odd, lane >> 1, make_uint4(e0, e1, o0, o1));
    } else {
#pragma unroll
      for (int c = 0; c < E / 8; ++c) {
#pragma unroll
        for (int term = 0; term < 2; ++term) {
          const __half* h = (term ? lo : hi) + 8 * c;
          if constexpr (FMT == FMT_INT4)
            put(term, lane * (E / 8) + c, make_uint4(two(h[0], h[4]), two(h[1], h[5]), two(h[2], h[6]), two(h[3], h[7])));
          else
            put(term, lane * (E / 8) + c, make_uint4(two(h[0], h[1]), two(h[2], h[3]), two(h[4], h[5]), two(h[6], h[7])));
        }
      }
    }
  }
}

__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global.L2::64B [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

// 32 TMEM columns (64 channels) of a key's exact codes from 32 (int4) or 64 (k8v4) bytes
template <int FMT>
__device__ __forceinline__ void key_columns(const uint8_t* codes, uint32_t lo_bias, uint32_t hi_bias, uint32_t (&a)[32]) {
  if constexpr (FMT == FMT_INT4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint2 w2 = *reinterpret_cast<const uint2*>(codes + 8 * k);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t w = e ? w2.y : w2.x, w8 = w >> 8;
        const int j = 8 * k + 4 * e;
        // 1024 + u minus 1024 + zp; (1024 + 16 u) / 16 minus 64 + zp: channels 8 w + {0, 4}, {1, 5}, {2, 6}, {3, 7}
        a[j] = hsub2_u32(lop3_and_or(w, 0x000F000Fu, 0x64006400u), lo_bias);
        a[j + 1] = hfma2_u32(lop3_and_or(w, 0x00F000F0u, 0x64006400u), 0x2C002C00u, hi_bias);
        a[j + 2] = hsub2_u32(lop3_and_or(w8, 0x000F000Fu, 0x64006400u), lo_bias);
        a[j + 3] = hfma2_u32(lop3_and_or(w8, 0x00F000F0u, 0x64006400u), 0x2C002C00u, hi_bias);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint2 w2 = *reinterpret_cast<const uint2*>(codes + 8 * k);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t x = (e ? w2.y : w2.x) ^ 0x80808080u;  // 1024 + (c + 128) minus 1152
        a[4 * k + 2 * e] = hsub2_u32(prmt(x, 0x64646464u, 0x4140u), 0x64806480u);
        a[4 * k + 2 * e + 1] = hsub2_u32(prmt(x, 0x64646464u, 0x4342u), 0x64806480u);
      }
    }
  }
}

// The call's own tokens have no earlier weight; a page of the others may be shared by sequences of the call.
__device__ __forceinline__ void add_weight(const WeightParams& wp, int32_t page, int block, int kvh, int key,
                                           int vis_base, float w) {
  float* at = wp.weights + page * wp.w_block + static_cast<int64_t>(key - block * wp.block_size.d) * wp.w_slot +
              kvh * wp.w_head;
  if (key >= vis_base) *at = w;
  else atomicAdd(at, w);
}

// ---------------------------------------------------------------------------------------------------- K4
template <int FMT, int HS, int NR, int KT, bool MANY, bool CAP>
__global__ void __launch_bounds__((WT<FMT, HS, NR, KT, MANY>::THREADS), 1) weights_kernel(const WeightParams wp) {
  using W = WT<FMT, HS, NR, KT, MANY>;
  using CL = typename W::CL;
  constexpr int GK = WT_KEYS * KT, SLOTS = W::SLOTS, RS = W::RS, QS = W::QS;
  const DecodeParams& p = wp.d;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + W::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + W::OFF_TMEM);
  // (no static shared memory: the operand's swizzle wants the dynamic part at a multiple of 1024 bytes)
  ShareStart& start = *reinterpret_cast<ShareStart*>(smem + W::OFF_TMEM + 16);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.launch_dependents;");
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[T_Q_FULL + i], 1);
      mbar_init(&bars[T_Q_EMPTY + i], 2 + 8);
      mbar_init(&bars[T_K_FULL + i], 4);
      mbar_init(&bars[T_K_FREE + i], W::BOTH ? 2 : 1);
      mbar_init(&bars[T_S_FULL + i], 1);
      mbar_init(&bars[T_S_FREE + i], 4);
    }
    for (int i = 0; i < RS; ++i) {
      mbar_init(&bars[T_RAW_FULL + i], 32);
      mbar_init(&bars[T_RAW_EMPTY + i], 4);
    }
    mbar_init(&bars[T_FINAL], 2);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, W::COLS);
    tmem_relinquish();
  }
  find_start<NR, GK, MANY, W::THREADS>(wp, reinterpret_cast<int64_t*>(smem + W::OFF_RAW), &start);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Walk<NR, GK, MANY> walk;
  walk.left = static_cast<int>(start.hi - start.lo);
  if (walk.left > 0) {
    walk.seq = start.seq;
    walk.kvh = start.kvh;
    walk.g = start.g;
    walk.g1 = MANY ? start.g + 1 : start.g;
    walk.qbase = start.qbase;
    walk.s = steps_of<NR, GK>(wp, start.seq);
    if constexpr (MANY) {
      tiles_seeing<NR, GK>(walk.s, walk.g, walk.first, walk.end);
      walk.qb = start.q;
    }
  }
  const auto tiles_in = [&](int g) {  // key tiles of group g that hold keys
    return KT == 1 ? 1 : min(KT, (walk.s.n - g * GK + WT_KEYS - 1) / WT_KEYS);
  };
  const auto tile_id = [&](int qt) { return static_cast<int64_t>(MANY ? walk.qbase + qt : walk.seq) * p.nkv + walk.kvh; };
  bool ok = true;
  const auto wait = [&](int bar, uint32_t parity) {
    if (ok) ok = !__any_sync(0xffffffffu, !mbar_wait_spin(&bars[bar], parity));
  };
  // Jobs (one key tile, one query tile) and key tiles are counted alike in every role: job j uses S^T buffer j & 1, key
  // tile i raw stage i % RS and TMEM slot i % SLOTS. With few rows a tile is one job, of the same number.

  if (warp == 0) {
    // ------------------------------------------------------------------ query tiles
    asm volatile("griddepcontrol.wait;" ::: "memory");  // K4q's records
    int64_t cur = -1;
    int loads = 0;
    while (ok && walk.next(wp)) {
      for (int qt = MANY ? walk.qa : 0; qt < (MANY ? walk.qb : 1) && ok; ++qt) {
        const int64_t id = tile_id(qt);
        if (id == cur) continue;
        cur = id;
        const int st = loads % QS;
        if (loads >= QS) wait(T_Q_EMPTY + st, (loads / QS - 1) & 1);
        if (ok && lane == 0) {
          mbar_arrive_expect_tx(&bars[T_Q_FULL + st], W::QREC);
          bulk_g2s(smem + st * W::QREC, wp.qrec + id * W::QREC, W::QREC, &bars[T_Q_FULL + st]);
        }
        __syncwarp();
        loads += ok;
      }
    }
    // the copies in flight land before the CTA's shared memory can go away
    for (int k = max(0, loads - QS); k < loads; ++k) mbar_wait_bounded(&bars[T_Q_FULL + k % QS], (k / QS) & 1);
  } else if (warp == 1 || warp == W::W_MMA1) {
    // ------------------------------------------------------------------ MMAs (this warp's: the jobs of its S^T buffer)
    constexpr uint32_t ID = f16_idesc(128, NR, false);
    const int buf = warp == 1 ? 0 : 1;
    int64_t cur = -1;
    int loads = 0, jobs = 0, tiles = 0;
    uint64_t qd = 0;
    const auto enter = [&](int64_t id) {  // the jobs from here on are of query tile id
      if (id == cur) return;
      cur = id;
      if (loads > 0 && elect_one()) umma_commit(&bars[T_Q_EMPTY + (loads - 1) % QS]);
      __syncwarp();
      wait(T_Q_FULL + loads % QS, (loads / QS) & 1);
      qd = sw128_desc(smem_u32(smem + (loads % QS) * W::QREC), 16, 1024);
      ++loads;
    };
    const auto job = [&](int j, int sl) {
      if (j >= 2) wait(T_S_FREE + buf, (j / 2 - 1) & 1);
      if (!ok) return;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t ak = tmem + sl * W::ACOLS, sd = tmem + W::S + buf * NR;
        // the small term first: each accumulation rounds the sum so far toward zero, and so only the HS / 16 of the
        // large term meet a large sum (the other order: errors of the weights 2 to 3 times as large)
#pragma unroll
        for (int term = 1; term >= 0; --term)
#pragma unroll
          for (int c = 0; c < HS / 16; ++c)
            umma_f16_ts(sd, ak + 8 * c,
                        qd + static_cast<uint64_t>((term * W::TERM + (c >> 2) * W::ATOM + (c & 3) * 32) >> 4), ID,
                        (term == 0 || c > 0) ? 1u : 0u);
        umma_commit(&bars[T_S_FULL + buf]);
      }
      __syncwarp();
    };
    const auto release = [&](int sl) {  // this warp's MMAs on the tile are all issued
      if (ok && elect_one()) umma_commit(&bars[T_K_FREE + sl]);
      __syncwarp();
    };
    while (ok && walk.next(wp)) {
      if constexpr (!MANY) {
        enter(tile_id(0));
        for (int n = walk.g1 - walk.g; n > 0 && ok; --n, ++tiles) {
          const bool own = (tiles & 1) == buf;
          if (!own && !W::BOTH) continue;
          const int sl = tiles % SLOTS;
          wait(T_K_FULL + sl, (tiles / SLOTS) & 1);
          if (own) job(tiles, sl);
          release(sl);
        }
      } else {
        const int kt = tiles_in(walk.g);
        for (int qt = walk.qa; qt < walk.qb && ok; ++qt) {
          enter(tile_id(qt));
          for (int t = 0; t < kt && ok; ++t, ++jobs) {
            const int sl = (tiles + t) % SLOTS;
            if (qt == walk.qa) wait(T_K_FULL + sl, ((tiles + t) / SLOTS) & 1);
            if ((jobs & 1) == buf) job(jobs, sl);
            if (qt == walk.qb - 1) release(sl);
          }
        }
        tiles += kt;
      }
    }
    if (elect_one()) umma_commit(&bars[T_FINAL]);
    __syncwarp();
    mbar_wait_spin(&bars[T_FINAL], 0);  // every MMA has completed before TMEM goes
  } else if (warp < W::W_SUM) {
    // ------------------------------------------------------------------ key operand (thread = key = TMEM lane)
    const int quarter = warp & 3, set = (warp - 2) >> 2, kl = 32 * quarter + lane;
    float* kp = reinterpret_cast<float*>(smem + W::OFF_KP);
    int tile = 0;
    while (ok && walk.next(wp)) {
      for (int g = walk.g; g < walk.g1 && ok; ++g) {
        const int kt = tiles_in(g);
        for (int t = 0; t < kt && ok; ++t, ++tile) {
          if (W::CSETS == 2 && (tile & 1) != set) continue;
          const int sl = tile % SLOTS, st = tile % RS;
          wait(T_RAW_FULL + st, (tile / RS) & 1);
          if (tile >= SLOTS) wait(T_K_FREE + sl, (tile / SLOTS - 1) & 1);
          if (!ok) break;
          tc_fence_after();
          const uint8_t* raw = smem + W::OFF_RAW + st * W::STAGE + kl * W::KEY;
          const uint32_t word = *reinterpret_cast<const uint32_t*>(raw + CL::KB);
          const uint32_t zp = FMT == FMT_INT4 ? word & 0xFu : 0u;
          const uint32_t lo1 = 0x6400u | zp, hi1 = 0xD400u | (zp << 4);  // 1024 + zp, -(64 + zp)
          const uint32_t ta = tmem + sl * W::ACOLS + (static_cast<uint32_t>(32 * quarter) << 16);
#pragma unroll 1
          for (int c = 0; c < HS / 64; ++c) {
            uint32_t a[32];
            key_columns<FMT>(raw + c * (CL::KB / (HS / 64)), lo1 | (lo1 << 16), hi1 | (hi1 << 16), a);
            tmem_st32u(ta + 32 * c, a);
          }
          const bool valid = g * GK + t * WT_KEYS + kl < walk.s.n;
          kp[(tile & 3) * 128 + kl] = !valid ? 0.f : __uint_as_float(FMT == FMT_INT4 ? word & 0xFFFFFFF0u : word);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bars[T_RAW_EMPTY + st]);
            mbar_arrive(&bars[T_K_FULL + sl]);
          }
        }
      }
    }
  } else if (warp < W::W_LOAD) {
    // ------------------------------------------------------------------ weights (thread = key)
    // Set b takes the jobs of S^T buffer b: every other tile (few rows), one tile of each pair of a group, or every other
    // job of a lone tile.
    constexpr int CH = NR < 16 ? NR : 16;  // columns at a time
    const int quarter = warp & 3, set = (warp - W::W_SUM) >> 2, kl = 32 * quarter + lane;
    const uint32_t ta = tmem + W::S + set * NR + (static_cast<uint32_t>(32 * quarter) << 16);
    const float* kp = reinterpret_cast<const float*>(smem + W::OFF_KP);
    float* red = reinterpret_cast<float*>(smem + W::OFF_RED);
    const float capl = CAP ? p.softcap * LOG2E : 0.f, cap_k = CAP ? 2.f * LOG2E / capl : 0.f;
    int64_t cur = -1;
    int loads = 0, jobs = 0, tiles = 0;
    int4 rec_head = make_int4(0, 0, 0, 0), rec_tail = make_int4(0, 0, 0, 0);
    const uint8_t* rec = smem;
    const auto enter = [&](int64_t id) {
      if (id == cur) return;
      cur = id;
      __syncwarp();  // the lanes read the record's rows past the score buffer's hand-off, each at its own pace
      if (loads > 0 && lane == 0) mbar_arrive(&bars[T_Q_EMPTY + (loads - 1) % QS]);
      wait(T_Q_FULL + loads % QS, (loads / QS) & 1);
      rec = smem + (loads % QS) * W::QREC;
      ++loads;
    };
    // job j's scores: the sum over the rows of the key's weights, k0 the tile's first key, ks the key's scale
    const auto job = [&](int j, int tile, int k0) {
      float2 sum = make_float2(0.f, 0.f);
      wait(T_S_FULL + set, (j / 2) & 1);
      if (!ok) return sum;
      tc_fence_after();
      const float ks = kp[(tile & 3) * 128 + kl];
      const float4 hd = *reinterpret_cast<const float4*>(rec + W::HEAD);
      const float* nl = reinterpret_cast<const float*>(rec + W::ROWS);
      const int* vis = reinterpret_cast<const int*>(rec + W::ROWS) + NR;
      const float k1 = ks * hd.x;
      const bool masked = k0 + WT_KEYS - 1 > __float_as_int(hd.y) || k0 < __float_as_int(hd.z);
#pragma unroll
      for (int c0 = 0; c0 < NR; c0 += CH) {
        float sc[CH];
        tmem_ld_cols<CH>(ta + c0, sc);
        if (c0 + CH == NR) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[T_S_FREE + set]);
        }
        float2 x[CH / 2];
#pragma unroll
        for (int c = 0; c < CH; c += 4) {
          const float4 l4 = *reinterpret_cast<const float4*>(nl + c0 + c);
          if constexpr (!CAP) {
            x[c / 2] = __ffma2_rn(make_float2(sc[c], sc[c + 1]), make_float2(k1, k1), make_float2(l4.x, l4.y));
            x[c / 2 + 1] = __ffma2_rn(make_float2(sc[c + 2], sc[c + 3]), make_float2(k1, k1), make_float2(l4.z, l4.w));
          } else {
            x[c / 2] = make_float2(softcap_log2(sc[c] * k1, capl, cap_k) + l4.x,
                                   softcap_log2(sc[c + 1] * k1, capl, cap_k) + l4.y);
            x[c / 2 + 1] = make_float2(softcap_log2(sc[c + 2] * k1, capl, cap_k) + l4.z,
                                       softcap_log2(sc[c + 3] * k1, capl, cap_k) + l4.w);
          }
        }
        if (masked) {
          const int key = k0 + kl;
#pragma unroll
          for (int c = 0; c < CH; c += 4) {
            const int4 v = *reinterpret_cast<const int4*>(vis + c0 + c);
            const int4 f = *reinterpret_cast<const int4*>(vis + NR + c0 + c);
            if (key > v.x || key < f.x) x[c / 2].x = -INFINITY;
            if (key > v.y || key < f.y) x[c / 2].y = -INFINITY;
            if (key > v.z || key < f.z) x[c / 2 + 1].x = -INFINITY;
            if (key > v.w || key < f.w) x[c / 2 + 1].y = -INFINITY;
          }
        }
#pragma unroll
        for (int c = 0; c < CH / 2; ++c) sum = __fadd2_rn(sum, make_float2(fast_exp2(x[c].x), fast_exp2(x[c].y)));
      }
      return sum;
    };
    // A prompt's query tiles: a key that every row gives about the same weight rounds the same way at every addition, so
    // the tiles' sums are added with their rounding error carried along (Kahan). One running sum over 131,072 rows was
    // off by 8.3e-5, this is by 2.4e-6 at most whatever the rows (a tile's own 32 additions, the exponential).
    const auto add_tile = [](float& sum, float& lost, float w) {
      const float y = __fsub_rn(w, lost), t = __fadd_rn(sum, y);
      lost = __fsub_rn(__fsub_rn(t, sum), y);
      sum = t;
    };
    while ((ok || MANY) && walk.next(wp)) {  // (with many rows a set that gave up still meets the barrier below)
      if constexpr (!MANY) {
        enter(tile_id(0));
        const int32_t* table = p.block_table + static_cast<int64_t>(walk.seq) * p.bt_stride;
        for (int g = walk.g; g < walk.g1 && ok; ++g, ++tiles) {
          if ((tiles & 1) != set) continue;
          const int key = g * GK + kl, block = wp.block_size.div(key);
          int32_t page = 0;  // on its way while the scores are made
          if (key < walk.s.n) page = table[block];
          const float2 sum = job(tiles, tiles, g * GK);
          if (ok && key < walk.s.n) add_weight(wp, page, block, walk.kvh, key, walk.s.vis_base, sum.x + sum.y);
        }
      } else {
        const int kt = tiles_in(walk.g), mine = kt == 2 ? (set - jobs) & 1 : 0;  // this set's tile of the group
        const int k0 = walk.g * GK + mine * WT_KEYS, key = k0 + kl;
        const bool writes = kt == 2 || (jobs & 1) == set;  // a lone tile is the set's that has its first job
        float2 sum = make_float2(0.f, 0.f), lost = make_float2(0.f, 0.f);
        for (int qt = walk.qa; qt < walk.qb && ok; ++qt, jobs += kt) {
          enter(tile_id(qt));
          const int j = jobs + (kt == 2 ? (set - jobs) & 1 : 0);  // this set's job of the query tile, if it has one
          if ((j & 1) == set) {
            const float2 w = job(j, tiles + mine, k0);
            add_tile(sum.x, lost.x, w.x);
            add_tile(sum.y, lost.y, w.y);
          }
        }
        // whole groups go to the weights, parts of one to the workspace
        const bool head = walk.qa > walk.first, tail = walk.qb < walk.end;
        float w = sum.x + sum.y;
        if (kt == 1) {  // both sets had jobs of the tile
          if (!writes) red[kl] = w;
          if (named_bar_or(1, 256, !ok)) break;
          if (writes) w += red[kl];
          named_bar_or(1, 256, false);  // read before the next lone tile's
        }
        if (ok && writes && key < walk.s.n) {
          if (head || tail) {
            wp.part[(static_cast<int64_t>(blockIdx.x) * 2 + (head ? 0 : 1)) * 256 + mine * WT_KEYS + kl] = w;
          } else {
            const int block = wp.block_size.div(key);
            add_weight(wp, p.block_table[static_cast<int64_t>(walk.seq) * p.bt_stride + block], block, walk.kvh, key,
                       walk.s.vis_base, w);
          }
        }
        if (head) rec_head = make_int4(1, tail, 0, 0);
        else if (tail) rec_tail = make_int4(1, walk.seq, walk.kvh, walk.g);
        tiles += kt;
      }
    }
    if (MANY && warp == W::W_SUM && lane == 0) {
      wp.records[2 * blockIdx.x] = rec_head;
      wp.records[2 * blockIdx.x + 1] = rec_tail;
    }
  } else {
    // ------------------------------------------------------------------ raw keys
    // A warp copies every LOADERS-th tile: lane l the 8-byte pieces l, l + 32, ... of each 16-cell run's key parts.
    const int me = warp - W::W_LOAD;
    uint32_t at[W::RUN_STEPS];  // of each piece: key << 16 | byte from the run's first cell
#pragma unroll
    for (int e = 0; e < W::RUN_STEPS; ++e) {
      const int idx = e * 32 + lane, key = idx / W::PIECES;
      at[e] = static_cast<uint32_t>(key << 16 | (key * CL::BYTES + (idx - key * W::PIECES) * 8));
    }
    int tile = 0;
    while (ok && walk.next(wp)) {
      const int32_t* table = p.block_table + static_cast<int64_t>(walk.seq) * p.bt_stride;
      const uint8_t* head_base = p.cache + walk.kvh * p.head_stride;
      const int tiles = MANY ? tiles_in(walk.g) : walk.g1 - walk.g, k0 = walk.g * GK;
      // lane r < 8 reads the page of run r of the warp's next tile while the present one is copied
      const auto first_key = [&](int t) { return k0 + t * WT_KEYS + 16 * (lane & 7); };
      const auto page_of = [&](int t) {
        const int k = first_key(t);
        return t < tiles && k < walk.s.n ? table[wp.block_size.div(k)] : 0;
      };
      int t = (me - tile % W::LOADERS + W::LOADERS) % W::LOADERS;
      int32_t page = page_of(t);
      for (; t < tiles && ok; t += W::LOADERS) {
        const int k = first_key(t), i = tile + t, st = i % RS;
        const uint8_t* const src = head_base + page * p.block_stride +
                                   static_cast<int64_t>(k - wp.block_size.div(k) * wp.block_size.d) * CL::BYTES;
        page = page_of(t + W::LOADERS);
        if (i >= RS) wait(T_RAW_EMPTY + st, (i / RS - 1) & 1);
        if (!ok) break;
        const uint32_t dst = smem_u32(smem + W::OFF_RAW + st * W::STAGE) + lane * 8;
        const int have = walk.s.n - (k0 + t * WT_KEYS);
#pragma unroll 1
        for (int r = 0; r < 8; ++r) {
          const uint8_t* base = reinterpret_cast<const uint8_t*>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), r));
          const int keys_r = min(have - 16 * r, 16);  // a run past the sequence is not there
          if (keys_r <= 0) break;
#pragma unroll
          for (int e = 0; e < W::RUN_STEPS; ++e)
            if (static_cast<int>(at[e] >> 16) < keys_r)
              cp_async8(dst + r * 16 * W::KEY + e * 256, base + (at[e] & 0xFFFFu));
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bars[T_RAW_FULL + st]))
                     : "memory");
      }
      tile += tiles;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, W::COLS);
}

// ---------------------------------------------------------------------------------------------------- K4f
// One CTA per CTA of K4 that began a group it did not finish: the parts of the group, in order (in 64 bits: up to one
// part a CTA, all alike where the rows are).
template <int GK>
__global__ void __launch_bounds__(GK) weights_fold_kernel(const WeightParams wp) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 rec = wp.records[2 * blockIdx.x + 1];
  if (!rec.x) return;
  double w = wp.part[(static_cast<int64_t>(blockIdx.x) * 2 + 1) * 256 + threadIdx.x];
  for (int c = blockIdx.x + 1; c < gridDim.x; ++c) {
    const int4 r = wp.records[2 * c];
    if (!r.x) break;
    w += wp.part[static_cast<int64_t>(c) * 512 + threadIdx.x];
    if (!r.y) break;
  }
  const Steps s = steps_of<16, GK>(wp, rec.y);
  const int key = rec.w * GK + threadIdx.x;
  if (key >= s.n) return;
  const int block = wp.block_size.div(key);
  add_weight(wp, wp.d.block_table[static_cast<int64_t>(rec.y) * wp.d.bt_stride + block], block, rec.z, key, s.vis_base,
             static_cast<float>(w));
}

// ---------------------------------------------------------------------------------------------------- host
static cudaLaunchConfig_t wt_config(const dim3& grid, int threads, int smem, cudaStream_t st, cudaLaunchAttribute* pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  pdl->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl->val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  return cfg;
}

template <int FMT, int DT, int HS, int NR, int KT, bool MANY, bool CAP>
static int launch_weights_t(const WeightParams& wp, int64_t tiles, int ctas, cudaStream_t st) {
  using W = WT<FMT, HS, NR, KT, MANY>;
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(weights_kernel<FMT, HS, NR, KT, MANY, CAP>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, W::BYTES);
    if (e != cudaSuccess) return set_error(QP_ERR_CUDA, "attention weights attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  weights_qprep_kernel<FMT, DT, HS, NR, MANY><<<dim3(static_cast<unsigned>(tiles), wp.d.nkv), 256, 0, st>>>(wp);
  int rc = check_launch("attention weights q prep");
  if (rc) return rc;
  cudaLaunchAttribute pdl[1];
  cudaLaunchConfig_t cfg = wt_config(dim3(ctas), W::THREADS, W::BYTES, st, pdl);
  cudaError_t e = cudaLaunchKernelEx(&cfg, weights_kernel<FMT, HS, NR, KT, MANY, CAP>, wp);
  if (e == cudaSuccess && MANY) {
    cfg = wt_config(dim3(ctas), WT_KEYS * KT, 0, st, pdl);
    e = cudaLaunchKernelEx(&cfg, weights_fold_kernel<WT_KEYS * KT>, wp);
  }
  if (e != cudaSuccess) return set_error(QP_ERR_CUDA, "attention weights launch: %s", cudaGetErrorString(e));
  return QP_OK;
}

// rows of a query tile: all of a sequence's where they are few, else what keeps a tile at 64 KB or two S^T buffers
// beside two key tiles in TMEM
static int wt_tile_rows(int rows, int head_size) {
  if (rows <= 16) return 16;
  if (rows <= WT_SMALL_ROWS || head_size == 512) return 32;
  return 64;
}
// query tiles (of one KV head) that a call may have at most
static int64_t wt_tiles(int64_t num_q_tokens, int num_seqs, int max_seqlen_q, int group, int head_size) {
  const int64_t rows = static_cast<int64_t>(max_seqlen_q) * group;
  if (rows <= WT_SMALL_ROWS) return num_seqs;
  const int nr = wt_tile_rows(WT_SMALL_ROWS + 1, head_size);
  return std::min(num_q_tokens * group / nr + num_seqs, num_seqs * ((rows + nr - 1) / nr));
}

template <int FMT, int DT, int HS, bool CAP>
static int launch_weights_hs(const WeightParams& wp, int64_t rows, int64_t tiles, int ctas, cudaStream_t st) {
  if (rows <= 16) return launch_weights_t<FMT, DT, HS, 16, 1, false, CAP>(wp, tiles, ctas, st);
  if (rows <= WT_SMALL_ROWS) return launch_weights_t<FMT, DT, HS, 32, 1, false, CAP>(wp, tiles, ctas, st);
  if constexpr (HS == 512) return launch_weights_t<FMT, DT, HS, 32, 1, true, CAP>(wp, tiles, ctas, st);
  else return launch_weights_t<FMT, DT, HS, 64, 2, true, CAP>(wp, tiles, ctas, st);
}

template <int FMT, int DT, bool CAP>
static int launch_weights_cap(const WeightParams& wp, int head_size, int64_t rows, int64_t tiles, int ctas,
                              cudaStream_t st) {
  if (head_size == 128) return launch_weights_hs<FMT, DT, 128, CAP>(wp, rows, tiles, ctas, st);
  if (head_size == 256) return launch_weights_hs<FMT, DT, 256, CAP>(wp, rows, tiles, ctas, st);
  return launch_weights_hs<FMT, DT, 512, CAP>(wp, rows, tiles, ctas, st);
}

template <int FMT, int DT>
static int launch_weights(const WeightParams& wp, int head_size, int64_t rows, int64_t tiles, int ctas,
                          cudaStream_t st) {
  return wp.d.softcap > 0.f ? launch_weights_cap<FMT, DT, true>(wp, head_size, rows, tiles, ctas, st)
                            : launch_weights_cap<FMT, DT, false>(wp, head_size, rows, tiles, ctas, st);
}

static int64_t wt_record_bytes(int rows, int head_size) {
  return (rows * head_size * 4ll + 12 * rows + 16 + 1023) / 1024 * 1024;
}

}  // namespace qp

using namespace qp;

// [per CTA: two sums of 256 keys, fp32][per CTA: two records of 16 bytes][prepared query tiles]
static int64_t wt_tiles_offset(int ctas) { return (static_cast<int64_t>(ctas) * (2 * 256 * 4 + 32) + 1023) / 1024 * 1024; }

extern "C" int64_t qp_attn_weights_workspace_bytes(int64_t num_q_tokens, int num_seqs, int max_seqlen_q,
                                                   int num_q_heads, int num_kv_heads, int head_size) {
  if (num_q_tokens <= 0 || num_seqs <= 0 || max_seqlen_q <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads)
    return 1024;
  const int group = num_q_heads / num_kv_heads;
  const int64_t rows = std::min<int64_t>(static_cast<int64_t>(max_seqlen_q) * group, 1 << 20);
  return wt_tiles_offset(device_sm_count()) +
         wt_tiles(num_q_tokens, num_seqs, max_seqlen_q, group, head_size) * num_kv_heads *
             wt_record_bytes(wt_tile_rows(static_cast<int>(rows), head_size), head_size);
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
  if (num_seqs > 65535 || num_kv_heads > 65535 ||
      static_cast<int64_t>(max_seqlen_q) * (num_q_heads / num_kv_heads) > 0x3fffffff)
    return set_error(QP_ERR_UNSUPPORTED, "attention weights: grid too large");
  if (!q || !cu_seqlens_q || !seqused_k || !block_table || !cache || !rht_sign_bits || !lse || !weights || !workspace)
    return set_error(QP_ERR_INVALID, "attention weights: null pointer");
  const int64_t need = qp_attn_weights_workspace_bytes(num_q_tokens, num_seqs, max_seqlen_q, num_q_heads,
                                                       num_kv_heads, head_size);
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need)
    return set_error(QP_ERR_WORKSPACE, "attention weights: workspace of %lld bytes < %lld", (long long)workspace_bytes,
                     (long long)need);
  WeightParams wp{{}, nullptr, nullptr, 0, 0, 0, FastDiv(block_size)};
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
  wp.max_q = max_seqlen_q;
  wp.max_k = max_seqlen_k;
  const int sms = device_sm_count();
  wp.part = static_cast<float*>(workspace);
  wp.records = reinterpret_cast<int4*>(wp.part + static_cast<int64_t>(sms) * 2 * 256);
  wp.qrec = static_cast<uint8_t*>(workspace) + wt_tiles_offset(sms);
  const int64_t rows = static_cast<int64_t>(max_seqlen_q) * dp.group;
  const int64_t tiles = wt_tiles(num_q_tokens, num_seqs, max_seqlen_q, dp.group, head_size);
  if (tiles > 0x7fffffff) return set_error(QP_ERR_UNSUPPORTED, "attention weights: too many query rows");
  // no more CTAs than there may be steps
  const int64_t steps = static_cast<int64_t>(num_kv_heads) * ((max_seqlen_k + WT_KEYS - 1) / WT_KEYS) *
                        std::max<int64_t>(tiles, num_seqs);
  const int ctas = static_cast<int>(std::min<int64_t>(sms, steps));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fmt == FMT_INT4)
    return dtype == DT_BF16 ? launch_weights<FMT_INT4, DT_BF16>(wp, head_size, rows, tiles, ctas, st)
                            : launch_weights<FMT_INT4, DT_F16>(wp, head_size, rows, tiles, ctas, st);
  return dtype == DT_BF16 ? launch_weights<FMT_K8V4, DT_BF16>(wp, head_size, rows, tiles, ctas, st)
                          : launch_weights<FMT_K8V4, DT_F16>(wp, head_size, rows, tiles, ctas, st);
}
