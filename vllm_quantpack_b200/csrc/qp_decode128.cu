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
//   - a running maximum per row that may be passed by 2^8 before anything is rescaled (RESCALE_SLACK), and a power
//     of two per row that keeps P x value scale inside fp16, changed as rarely; the row sums stay in each lane.
// The warps' O^T, maxima and sums meet once in shared memory at the end.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "qp_api_internal.h"
#include "qp_common.cuh"
#include "qp_decode.cuh"

namespace qp {

constexpr int D1_KEYS = 32;      // keys of a raw stage: two 16-cell runs, each inside one page
constexpr float D1_NONE = -1e30f;  // running maximum of a row that has seen no key (finite: t - D1_NONE is large, not NaN)
constexpr float D1_P_LIMIT = 8192.f;  // P x value scale x row factor may grow to this before the factor changes

template <int FMT, int NT>
struct D1 {
  using CL = Cell<FMT, 128>;
  static constexpr int WARPS = NT == 2 ? 12 : 8;
  static constexpr int CTAS = NT == 1 ? 2 : 1;  // per SM: 128 registers a thread, or 168 / 255
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int ROWS = 8 * NT;
  static constexpr int STAGE = D1_KEYS * CL::BYTES;
  static constexpr int STAGES = FMT == FMT_INT4 ? (NT >= 3 ? 4 : 3) : (NT >= 3 ? 3 : 2);
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int RED = WARPS * ROWS * 128 * 4;  // the warps' O^T at the end, in the ring's place
  static constexpr int OFF_Q = RING > RED ? RING : RED;  // B operand of QK: [NT][4][32 lanes] x 16 bytes
  static constexpr int OFF_ROW = OFF_Q + NT * 4 * 32 * 16;  // [ROWS] float2: score scale, row sum x 2^-24
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

template <int FMT, int DT, int NT, bool FEAT>
__global__ void __launch_bounds__((D1<FMT, NT>::THREADS), (D1<FMT, NT>::CTAS)) decode128_kernel(const DecodeParams p) {
  using C = D1<FMT, NT>;
  using CL = typename C::CL;
  using EL = Elem<DT>;
  constexpr int WARPS = C::WARPS, CELL = CL::BYTES, ROWS = C::ROWS, STAGES = C::STAGES;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int split = blockIdx.x, kvh = blockIdx.y;
  asm volatile("griddepcontrol.launch_dependents;");  // the merge's launch may begin; it waits for this grid's end

  const DecodeSpan sp = decode_span(p, blockIdx.z);
  if (sp.qlen <= 0) return;
  const int rows = min(sp.qlen * p.group, ROWS), n = sp.n;
  // 32-key tiles of this split; with a sliding window from the first token's first key on
  const int win_lo = (FEAT && p.window > 0) ? max(0, sp.vis_base - p.window + 1) : 0;
  const int tile_lo = win_lo / D1_KEYS, n_tiles = (n + D1_KEYS - 1) / D1_KEYS;
  const int tps = max(0, (n_tiles - tile_lo + p.num_splits - 1) / p.num_splits);
  const int tile0 = tile_lo + split * tps;
  const int ntl = max(0, min(tile0 + tps, n_tiles) - tile0);
  if (ntl == 0) {  // empty segment: lse = -inf
    for (int r = tid; r < rows; r += C::THREADS) {
      const int tok = sp.q0 + r / p.group, qh = kvh * p.group + r % p.group;
      p.part_lse[(static_cast<int64_t>(tok) * p.nq + qh) * p.num_splits + split] = -INFINITY;
    }
    return;
  }

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR) + warp * STAGES;
  uint8_t* ring = smem + warp * STAGES * C::STAGE;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(&bars[s], 1);
    fence_mbar_init();
  }
  __syncwarp();

  // ---- raw stages: this warp's i-th tile is tile0 + warp + i WARPS. Lane l looks up the page of run l & 1 of tile
  // 16 w + l / 2 for window w of 16 tiles (one window ahead) and issues that run's copy when its turn comes.
  const int my_tiles = ntl > warp ? (ntl - warp + WARPS - 1) / WARPS : 0;
  const auto run_key = [&](int i) { return (tile0 + warp + i * WARPS) * D1_KEYS + (lane & 1) * 16; };
  const auto page_of = [&](int w) {
    const int i = 16 * w + (lane >> 1), k = run_key(i);
    return i < my_tiles && k < n ? sp.btab[k / p.block_size] : 0;
  };
  int page = page_of(0), page_next = page_of(1);
  const auto issue = [&](int i) {
    if (i >= my_tiles) return;
    if (i > 0 && (i & 15) == 0) {
      page = page_next;
      page_next = page_of((i >> 4) + 1);
    }
    if ((lane >> 1) == (i & 15)) {
      const int k = run_key(i), s = i % STAGES;
      if ((lane & 1) == 0) mbar_arrive_expect_tx(&bars[s], (k + 16 < n ? 32 : 16) * CELL);
      if (k < n)
        bulk_g2s(ring + s * C::STAGE + (lane & 1) * 16 * CELL,
                 p.cache + static_cast<int64_t>(page) * p.block_stride + static_cast<int64_t>(kvh) * p.head_stride +
                     static_cast<int64_t>(k % p.block_size) * CELL,
                 16 * CELL, &bars[s]);
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i);

  // ---- query rows: one warp per row, rotated, scaled by a power of two to |q| < 2^14 and rounded to fp16 in the
  // operand's order; the rounding (2^-12 of a value) is the size of the model dtype's own
  float2* rowp = reinterpret_cast<float2*>(smem + C::OFF_ROW);
  int2* lim = reinterpret_cast<int2*>(smem + C::OFF_LIM);
  for (int r = warp; r < ROWS; r += WARPS) {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < rows) {
      const int tok = sp.q0 + r / p.group, qh = kvh * p.group + r % p.group;
      const typename EL::T* src = reinterpret_cast<const typename EL::T*>(p.q) + tok * p.q_st + qh * p.q_sh + lane * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = EL::to_f(src[i]);
      if (!p.q_rotated) {
        apply_signs<4>(x, p.sign_bits, lane);
        warp_wht<4>(x, lane);
      }
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
      rowp[r] = make_float2(r < rows ? ldexpf(p.qk_scale, 24 - ex) : 0.f, ldexpf(sum, -24));
      const int vis = sp.vis_base + r / p.group;
      lim[r] = make_int2((FEAT && p.window > 0) ? vis - p.window + 1 : 0, r < rows ? min(vis, n - 1) : n - 1);
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
  float M[NT][2], F[NT][2], L[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    M[nt][0] = M[nt][1] = D1_NONE;
    F[nt][0] = F[nt][1] = 1.f;
    L[nt][0] = L[nt][1] = 0.f;
  }

  bool ok = true;
  int i = 0;
#pragma unroll 1
  for (; i < my_tiles; ++i) {
    issue(i + STAGES - 1);
    ok = !__any_sync(0xffffffffu, !mbar_wait_spin(&bars[i % STAGES], (i / STAGES) & 1));
    if (!ok) break;
    const uint8_t* stage = ring + (i % STAGES) * C::STAGE;
    const int key_t = (tile0 + warp + i * WARPS) * D1_KEYS;
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      const int key0 = key_t + half * 16;
      if (key0 >= n) break;
      const uint8_t* run = stage + half * 16 * CELL;
      const uint8_t* ca = run + kap * CELL;
      const uint8_t* cb = ca + 2 * CELL;
      // S^T
      uint32_t ka[8][4];
      float ksa, ksb, za, zb;
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
        const uint32_t wa = lds32(ca + CL::KS), wb = lds32(cb + CL::KS);
        ksa = __uint_as_float(wa & 0xFFFFFFF0u);
        ksb = __uint_as_float(wb & 0xFFFFFFF0u);
        za = static_cast<float>(wa & 0xFu);
        zb = static_cast<float>(wb & 0xFu);
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
        ksa = __uint_as_float(lds32(ca + CL::KS));
        ksb = __uint_as_float(lds32(cb + CL::KS));
        za = zb = 128.f;
      }
      float s4[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float* c = s4[nt];
        c[0] = c[1] = c[2] = c[3] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 q;
          if constexpr (NT == 1) q = qreg[j];
          else q = qfrag[(nt * 4 + j) * 32];
          mma_f16_16816(c, ka[2 * j], q.x, q.y);
          mma_f16_16816(c, ka[2 * j + 1], q.z, q.w);
        }
      }
      // scores in log2 units, then P and P x value scale x row factor
      const float vsa = __uint_as_float(lds32(ca + CL::VS) & 0xFFFFFFF0u);
      const float vsb = __uint_as_float(lds32(cb + CL::VS) & 0xFFFFFFF0u);
      const bool masked = key0 + 15 > open || (FEAT && key0 < shut);
      float pr[NT][4], pv[NT][4];
      bool slow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float4 rp = *reinterpret_cast<const float4*>(rowp + nt * 8 + 2 * t4);  // rows 2 t, 2 t + 1: scale, sum
        float* c = s4[nt];
        c[0] = fmaf(-za, rp.y, c[0]) * (ksa * rp.x);
        c[1] = fmaf(-za, rp.w, c[1]) * (ksa * rp.z);
        c[2] = fmaf(-zb, rp.y, c[2]) * (ksb * rp.x);
        c[3] = fmaf(-zb, rp.w, c[3]) * (ksb * rp.z);
        if (FEAT && capl > 0.f) {
#pragma unroll
          for (int e = 0; e < 4; ++e) c[e] = softcap_log2(c[e], capl, cap_k);
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int2 l = lim[nt * 8 + 2 * t4 + (e & 1)];
            const int key = key0 + kap + (e & 2);
            if (key > l.y || key < l.x) c[e] = -INFINITY;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pr[nt][e] = fast_exp2(c[e] - M[nt][e & 1]);
          pv[nt][e] = pr[nt][e] * ((e < 2 ? vsa : vsb) * F[nt][e & 1]);
        }
        slow = slow || fmaxf(c[0], c[2]) > M[nt][0] + RESCALE_SLACK || fmaxf(c[1], c[3]) > M[nt][1] + RESCALE_SLACK ||
               fmaxf(fmaxf(pv[nt][0], pv[nt][2]), fmaxf(pv[nt][1], pv[nt][3])) > D1_P_LIMIT;
      }
      if (masked) {  // a cell past the sequence may hold any scale: its product is dropped, not multiplied by 0
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (s4[nt][e] == -INFINITY) pv[nt][e] = 0.f;
      }
      if (__any_sync(0xffffffffu, slow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float of[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(s4[nt][e], s4[nt][e + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const bool opening = M[nt][e] == D1_NONE;
            const float mn = fmaxf(M[nt][e], mx), sc = fast_exp2(M[nt][e] - mn);
            M[nt][e] = mn;
            L[nt][e] *= sc;
            pr[nt][e] = fast_exp2(s4[nt][e] - mn);
            pr[nt][e + 2] = fast_exp2(s4[nt][e + 2] - mn);
            const float va = s4[nt][e] == -INFINITY ? 0.f : pr[nt][e] * vsa;
            const float vb = s4[nt][e + 2] == -INFINITY ? 0.f : pr[nt][e + 2] * vsb;
            float pm = fmaxf(va, vb);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, d));
            of[e] = sc;
            if (pm > 0.f && (opening || pm * F[nt][e] > D1_P_LIMIT)) {
              const float fn = pow2_below_inverse(pm);
              of[e] = opening ? 0.f : sc * (fn / F[nt][e]);
              F[nt][e] = fn;
            }
            pv[nt][e] = va * F[nt][e];
            pv[nt][e + 2] = vb * F[nt][e];
          }
#pragma unroll
          for (int ti = 0; ti < 8; ++ti)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][ti][e] *= of[e & 1];
#pragma unroll
          for (int e = 0; e < 4; ++e) z[nt][e] *= of[e & 1];
        }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        L[nt][0] += pr[nt][0] + pr[nt][2];
        L[nt][1] += pr[nt][1] + pr[nt][3];
        pb[nt][0] = movmatrix_trans(h2_pack(pv[nt][0], pv[nt][1]));
        pb[nt][1] = movmatrix_trans(h2_pack(pv[nt][2], pv[nt][3]));
      }
      // O^T: words g and g + 8 of four keys; tile ti takes nibble ti of each (channels 8 g + ti, 64 + 8 g + ti)
      const uint8_t* vc = run + kv4 * CELL + CL::V + 4 * g;
#pragma unroll
      for (int hw = 0; hw < 2; ++hw) {  // low, then high half of the words: nibbles 0-3, 4-7
        const uint32_t sel = hw ? 0x7632u : 0x5410u;
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // a0: word g, keys 0-1; a1: word g + 8; a2, a3: keys 2-3
          const uint8_t* at = vc + (e & 2) * CELL + (e & 1) * 32;
          y[e] = prmt(lds32(at), lds32(at + CELL), sel);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t a[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = ((q & 2) ? (y[e] >> 8) : y[e]) & ((q & 1) ? 0x00F000F0u : 0x000F000Fu);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16_16816(o[nt][4 * hw + q], a, pb[nt][0], pb[nt][1]);
        }
      }
      {
        const uint8_t* at = run + kv4 * CELL + CL::VS;
        const uint32_t a[4] = {prmt(lds32(at), lds32(at + CELL), 0x5410u) & zmask, 0u,
                               prmt(lds32(at + 2 * CELL), lds32(at + 3 * CELL), 0x5410u) & zmask, 0u};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16_16816(z[nt], a, pb[nt][0], pb[nt][1]);
      }
    }
    __syncwarp();  // every lane has read the stage before it is filled again
  }
  if (!ok) {  // a copy never landed (the error word says so): leave once the others in flight have
    for (const int end = min(i + STAGES, my_tiles); i < end; ++i)
      mbar_wait_bounded(&bars[i % STAGES], (i / STAGES) & 1);
  }
  if (__syncthreads_or(!ok)) return;

  // ---- the warps' partials meet: O^T (channels of a row contiguous), maximum, sum and factor of each row
  float* red = reinterpret_cast<float*>(smem);
  float4* st = reinterpret_cast<float4*>(smem + C::OFF_ST);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = L[nt][e];
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
      if (g == 0) st[warp * ROWS + r] = make_float4(M[nt][e], l, F[nt][e], 0.f);
    }
  }
  __syncthreads();
  for (int r = warp; r < rows; r += WARPS) {  // one warp per row: lane l holds channels 4 l .. 4 l + 3
    float mx = D1_NONE, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, st[w * ROWS + r].x);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum += st[w * ROWS + r].y * fast_exp2(st[w * ROWS + r].x - mx);
    const float inv = sum > 0.f ? 16777216.f / sum : 0.f;  // 2^24: the codes entered as subnormals
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float4 s = st[w * ROWS + r];
      const float f1 = fast_exp2(s.x - mx) * inv, f2 = 1.f / s.z;
      const float4 v = *reinterpret_cast<const float4*>(red + (w * ROWS + r) * 128 + 4 * lane);
      a.x += v.x * f1 * f2;
      a.y += v.y * f1 * f2;
      a.z += v.z * f1 * f2;
      a.w += v.w * f1 * f2;
    }
    const int tok = sp.q0 + r / p.group, qh = kvh * p.group + r % p.group;
    const int64_t at = (static_cast<int64_t>(tok) * p.nq + qh) * p.num_splits + split;
    *reinterpret_cast<float4*>(p.part_o + at * 128 + 4 * lane) = a;
    // a NaN sum (NaN scores) stays NaN in the partial's lse, so the merge passes it on
    if (lane == 0) p.part_lse[at] = sum == 0.f ? -INFINITY : mx + log2f(sum);
  }
}

template <int FMT, int DT, int NT, bool FEAT>
static int launch_d1(const DecodeParams& dp, int grid_z, cudaStream_t st) {
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
  const dim3 grid(static_cast<unsigned>(dp.num_splits), static_cast<unsigned>(dp.nkv), static_cast<unsigned>(grid_z));
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

int launch_decode128(int fmt, int dtype, const DecodeParams& dp, int rows, int grid_z, cudaStream_t st) {
  return fmt == FMT_INT4 ? launch_d1_fmt<FMT_INT4>(dtype, dp, rows, grid_z, st)
                         : launch_d1_fmt<FMT_K8V4>(dtype, dp, rows, grid_z, st);
}

}  // namespace qp
