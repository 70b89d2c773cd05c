// Packed causal attention for gfx950: sequences of different lengths laid end to end on one
// token axis, grouped heads, forward and atomics-free backward.
//
//   s_ij = scale q_i . k_j   for start(i) <= j <= i,   p_i = softmax_j(s_ij),   o_i = sum_j p_ij v_j
//   ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = do_i . o_i
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// start(t) / end(t) are the bounds of the sequence of row t (packed_plan_kernel, from the
// cumulative lengths).  The kernels tile the PACKED axis, not each sequence: a 128-row block
// takes the keys [start(first row), last row], so a block may hold the end of one sequence and
// the beginning of others and many short sequences cost no padding; a 32 x 32 subtile is skipped,
// taken whole, or masked per element (start(i) <= j <= i is one unsigned compare).  Rows behind
// the last sequence (a batch padded to a fixed size) never matter, whatever they hold.
//
// A masked score has p = 0, but 0 * NaN = NaN inside a matrix product: a masked subtile whose
// V (dQ: K; dK / dV: Q, dO) rows hold a non-finite value marks its wave, and the wave's rows are
// redone one by one over their visible terms alone, so one sequence's infinities and NaN never
// reach another's rows, nor a later row's an earlier one.
#include "flash_common.h"
#include "gemm_common.h"

#include <type_traits>

using namespace mx;
using namespace mx::flash;
using mx::gemm::i32x4_t;

namespace {

// ------------------------------------------------------------------------------ plan
// start / end / position of every row from the cumulative lengths cu[0..n] (one binary search per
// row: the last i with cu[i] <= t, so sequences of length zero are passed over).  Every value is
// clamped into [0, T], so a table that breaks its contract gives wrong sequences, never an access
// out of range.  meta[0] = rows that belong to a sequence.  Rows behind them: start = end = t.
template <typename IT>
__global__ __launch_bounds__(256) void packed_plan_kernel(const IT* __restrict__ cu, int n, int T,
                                                          int* __restrict__ start, int* __restrict__ end,
                                                          int* __restrict__ meta, int64_t* __restrict__ pos) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  const long long last = (long long)cu[n];
  const int nv = (int)(last < 0 ? 0 : last > T ? T : last);
  if (t == 0) meta[0] = nv;
  if (t >= T) return;
  int s = t, e = t;
  if (t < nv) {
    int lo = 0, hi = n;   // cu[lo] <= t < cu[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((long long)cu[mid] <= t) lo = mid;
      else hi = mid;
    }
    const long long a = (long long)cu[lo], b = (long long)cu[lo + 1];
    s = (int)(a < 0 ? 0 : a > t ? t : a);
    e = (int)(b < t + 1 ? t + 1 : b > nv ? nv : b);
  }
  start[t] = s;
  end[t] = e;
  pos[t] = t - s;
}

// Dispatch order of the 128-row query blocks, the 128-key and the 256-key blocks: most work first
// (ties: query blocks from the back, key blocks from the front), so that the longest blocks of a batch
// of mixed lengths do not start last.  One workgroup counts each block's rank; above ORDER_MAX blocks
// the lists are left in sequence order.  meta[1]: query tiles of all 128-key blocks (how much a split
// key block should hold).  Behind the lists (order_base), the query tiles of all 256-key blocks before
// each, which the D = 128 dK / dV kernel cuts into shares.
constexpr int ORDER_MAX = 2048;
__host__ __device__ inline int64_t order_base(int T) { return (2 * ((int64_t)(T + 127) / 128) + (T + 255) / 256 + 1) & ~1ll; }
__global__ __launch_bounds__(1024) void packed_order_kernel(int T, const int* __restrict__ start,
                                                            const int* __restrict__ end, int* __restrict__ meta,
                                                            int* __restrict__ order) {
  __shared__ int work[ORDER_MAX];
  __shared__ int sum;
  __shared__ int64_t scan[2][1024];
  const int nv = meta[0], tid = threadIdx.x;
  if (tid == 0) sum = 0;
  __syncthreads();
  int* list0 = order;
#pragma unroll 1
  for (int list = 0; list < 3; ++list) {
    const int B = list == 2 ? 256 : 128, nb = (T + B - 1) / B;
    int tiles = 0;
    for (int b = tid; b < nb; b += 1024) {
      const int b0 = b * B, b1 = min(b0 + B, nv);
      const int w = b0 >= nv ? 0 : list == 0 ? b1 - start[b0] : end[b1 - 1] - b0;
      tiles += (w + 63) / 64;
      if (nb <= ORDER_MAX) work[b] = w;
      else order[b] = list == 0 ? nb - 1 - b : b;
    }
    if (list == 1) atomicAdd(&sum, tiles);
    __syncthreads();
    if (list == 1 && tid == 0) meta[1] = sum;
    if (nb <= ORDER_MAX) {
      for (int b = tid; b < nb; b += 1024) {
        const int w = work[b];
        int rank = 0;
#pragma unroll 16
        for (int o = 0; o < nb; ++o)
          rank += (int)(work[o] > w) | ((int)(work[o] == w) & (int)(list == 0 ? o > b : o < b));
        order[rank] = b;
      }
    }
    __syncthreads();
    order += nb;
  }
  int64_t* before = reinterpret_cast<int64_t*>(list0 + order_base(T));
  const int nb2 = (T + 255) / 256;
  int64_t base = 0;
#pragma unroll 1
  for (int c0 = 0; c0 < nb2; c0 += 1024) {
    const int b0 = (c0 + tid) * 256;
    int64_t x = c0 + tid < nb2 && b0 < nv ? (end[min(b0 + 256, nv) - 1] - b0 + 63) / 64 : 0;
    scan[0][tid] = x;
    __syncthreads();
    int p = 0;
#pragma unroll 1
    for (int d = 1; d < 1024; d *= 2, p ^= 1) {
      scan[p ^ 1][tid] = scan[p][tid] + (tid >= d ? scan[p][tid - d] : 0);
      __syncthreads();
    }
    if (c0 + tid < nb2) before[c0 + tid + 1] = base + scan[p][tid];
    base += scan[p][1023];
    __syncthreads();
  }
  if (tid == 0) before[0] = 0;
}

struct PArgs {
  const uint16_t *q, *k, *v, *dout, *o;
  uint16_t *out, *dk, *dv;      // forward: O; backward: dQ, dK, dV
  float *lse, *nlse, *delta;    // [Hq][T]: log-sum-exp; backward: -lse / c and -delta
  const int *start, *end, *meta;
  const int* order;             // the launched kernel's dispatch order
  int ldq, ldk, ldv, lddo, ldo, ldout, lddk, lddv;
  int T, Hq, Hkv;
  float c, scale;               // scale log2(e), scale
  float* part;                  // partial dK / dV of split blocks
  int nsplit;                   // most splits of a key block
  int nshare;                   // most shares (see KeyShare; 0: blocks are split by themselves)
  const int64_t* before;        // query tiles of the 256-key blocks before each
  int fill;                     // zero the rows behind the last sequence (else leave them)
};

__device__ __forceinline__ uint32_t nonfinite(bf16x8 x) {   // high bit set in a half whose exponent is all ones
  const uint4 u = __builtin_bit_cast(uint4, x);
  constexpr uint32_t M = 0x7f807f80u, A = 0x00800080u;
  return (((u.x & M) + A) | ((u.y & M) + A) | ((u.z & M) + A) | ((u.w & M) + A)) & 0x80008000u;
}

// Whether one of the lane's 16 rows (d: their -delta, 4 in 8) has a non-finite q or do.  delta = do . o
// is not finite if do is not; nor if q is not, for then every score of the row, and so o, is not.
__device__ __forceinline__ uint32_t bad_rows(const float* d) {
  uint32_t bad = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const float4 v = *reinterpret_cast<const float4*>(d + 8 * x);
    bad |= !(fabsf(v.x) < INFINITY) | !(fabsf(v.y) < INFINITY) | !(fabsf(v.z) < INFINITY) | !(fabsf(v.w) < INFINITY);
  }
  return bad;
}

// Row-at-a-time forms for a wave whose masked subtiles met a non-finite operand: every lane holds
// columns lane (+ 64) of the row, and only visible terms are ever formed.
template <int D>
struct RowVec {
  float x[D / 64];
  __device__ __forceinline__ RowVec() {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) x[i] = 0.f;
  }
  __device__ __forceinline__ RowVec(const uint16_t* p, int lane) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) x[i] = bf2f(p[lane + 64 * i]);
  }
  __device__ __forceinline__ float dot(const RowVec& y) const {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) s += x[i] * y.x[i];
    return wave_sum(s);
  }
  __device__ __forceinline__ void axpy(float w, const RowVec& y) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) x[i] = __builtin_fmaf(w, y.x[i], x[i]);
  }
  __device__ __forceinline__ void store(uint16_t* p, int lane, float sc) const {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) p[lane + 64 * i] = f2bf(x[i] * sc);
  }
};

// one 1-KiB LDS-DMA piece through a buffer resource: rows past its size read zeros
__device__ __forceinline__ void dma16_buf(i32x4_t rsrc, uint32_t voff, char* lds_base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :: "v"(voff), "s"(rsrc), "s"(lds_u32(lds_base)) : "memory", "m0");
}
// resource over `rows` rows of D values at `base` (row stride ld); rows <= 0: everything reads zero
template <int D>
__device__ __forceinline__ i32x4_t rows_rsrc(const uint16_t* base, int rows, int ld) {
  const uint64_t b = (uint64_t)(uintptr_t)base;
  const uint32_t bytes = rows > 0 ? ((uint32_t)(rows - 1) * (uint32_t)ld + D) * 2u : 0u;
  return i32x4_t{uni((int)(uint32_t)b), uni((int)(uint32_t)(b >> 32)), uni((int)bytes), 0x00020000};
}

template <int D>
__device__ __forceinline__ void zero_row(uint16_t* row, int hh) {   // the lane's half of a D-wide row
#pragma unroll
  for (int i = 0; i < D / 16; ++i) *reinterpret_cast<uint4*>(row + 16 * i + 8 * hh) = make_uint4(0, 0, 0, 0);
}

// When every workgroup is resident at once (two on each of the 256 CUs), the CU that got the heaviest
// gets its second from the light end; else the hardware's dispatch in descending order balances.
__device__ __forceinline__ int pair_rank(int rank, int n) {
  const int half = (n + 1) / 2;
  return gridDim.x <= 512 && rank >= half ? n - 1 - (rank - half) : rank;
}

// ============================================================================ query-major
// Forward, and dQ of the backward.  Four waves of 32 query rows; query on the MFMA lane
// (S^T = K Q^T, O^T = V^T P^T), so the softmax statistics are lane-local plus one half exchange.
// K / V tiles of BK keys arrive by LDS-DMA into a two-slot ring, one barrier per tile.  Two workgroups a
// CU, so that one's exponentials run beside the other's products: 16384 tokens in one, 32 heads of 128,
// forward 2.15 ms (1.03 PFLOP/s), dQ 2.95 (1.12); 16 heads of 64, 0.72 ms (0.76) and 0.76 (1.08), bound by vector issue (busy
// 67 and 62 % of the time, the matrix pipe 41 and 53 %: a score costs as many vector operations as with 128
// columns, for half the products); 4096 of ~300, 16 heads of 64, bound by the latency of a block's few tiles,
// 20 and 23 us.  The forward of 128 in whole blocks spills 11 registers, which its tile loop reads back.  HALF: 64
// rows, two waves for each 32 (see launch_qmajor).
template <int D, bool DQ, bool HALF>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void packed_qmajor_kernel(const PArgs a) {
  constexpr int BQ = HALF ? 64 : 128, BK = D == 64 ? 128 : 64, NSUB = BK / 32, NKK = D / 16, NDT = D / 32;
  constexpr int RB = D * 2, CPR = D / 8, RPP = 64 / CPR, TILE = BK * RB, PPW = TILE / 1024 / 4;
  __shared__ __attribute__((aligned(16))) char kbuf0[TILE];
  __shared__ __attribute__((aligned(16))) char kbuf1[TILE];
  __shared__ __attribute__((aligned(16))) char vbuf0[TILE];
  __shared__ __attribute__((aligned(16))) char vbuf1[TILE];
  const int tid = threadIdx.x, lane = tid & 63, wl = uni(tid >> 6);
  const int r = lane & 31, hh = lane >> 5, g = lane >> 4, gi = lane & 15;
  const int wq = HALF ? wl & 1 : wl, kh = HALF ? wl >> 1 : 0;   // row group; half of a key tile's subtiles
  const int T = a.T, nqb = (T + 127) / 128;
  int rank, hq;
  block_map(a.Hq, rank, hq);
  const int hk = hq / (a.Hq / a.Hkv);
  int q0 = 0;
  if constexpr (HALF) q0 = uni(a.order[rank >> 1]) * 128 + 64 * (rank & 1 ^ 1);
  else q0 = uni(a.order[pair_rank(rank, nqb)]) * 128;
  const int qw = q0 + 32 * wq, qrow = qw + r;
  uint16_t* outp = a.out + (size_t)qrow * a.ldout + hq * D;
  // the table reads depend on nothing but the block (a row behind the last sequence has start = itself)
  const int nv = uni(a.meta[0]);
  const int qrow_c = min(qrow, T - 1);
  const int kv_lo = uni(a.start[min(q0, T - 1)]) & ~31;
  const int smin = uni(a.start[min(qw, T - 1)]), smax = uni(a.start[min(qw + 31, T - 1)]);
  const int st = a.start[qrow_c];
  if (q0 >= nv) {                                    // behind the last sequence
    if (a.fill && qrow < T) {
      zero_row<D>(outp, hh);
      if (!DQ && hh == 0) a.lse[(size_t)hq * T + qrow] = INFINITY;
    }
    return;
  }
  const int q_end = min(q0 + BQ, nv);
  const int ntile = (q_end - kv_lo + BK - 1) / BK;
  // the wave's rows: visible keys of row i are start(i) .. i
  const bool wave_on = qw < nv;
  const int wlast = min(qw + 31, nv - 1);
  const int cnt = qrow < nv ? qrow - st + 1 : 0;     // visible keys

  // DMA: per-lane byte offsets inside a tile
  uint32_t voK[PPW], voV[PPW];
#pragma unroll
  for (int i = 0; i < PPW; ++i) {
    const int R = (wl + 4 * i) * RPP + lane / CPR, ch = (lane % CPR) ^ swz<D>(R);
    voK[i] = (uint32_t)(R * a.ldk + ch * 8) * 2u;
    voV[i] = (uint32_t)(R * a.ldv + ch * 8) * 2u;
  }
  const uint16_t* kbase = a.k + (size_t)kv_lo * a.ldk + hk * D;
  const uint16_t* vbase = a.v + (size_t)kv_lo * a.ldv + hk * D;
  auto issue = [&](char* kd, char* vd, int j) __attribute__((always_inline)) {
    const int rows = min(BK, nv - kv_lo - j * BK);
    const i32x4_t kr = rows_rsrc<D>(kbase + (size_t)j * BK * a.ldk, rows, a.ldk);
    const i32x4_t vr = rows_rsrc<D>(vbase + (size_t)j * BK * a.ldv, rows, a.ldv);
#pragma unroll
    for (int i = 0; i < PPW; ++i) {
      dma16_buf(kr, voK[i], kd + (wl + 4 * i) * 1024);
      dma16_buf(vr, voV[i], vd + (wl + 4 * i) * 1024);
    }
  };
  issue(kbuf0, vbuf0, 0);                            // (under the row loads)

  bf16x8 qf[NKK];
  bf16x8 dof[DQ ? NKK : 1];
  float lse2 = 0.f, dl = 0.f;
  {
    const uint16_t* qp = a.q + (size_t)qrow_c * a.ldq + hq * D + 8 * hh;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) qf[kk] = ld8(qp + 16 * kk);
    if constexpr (DQ) {
      const uint16_t* dp = a.dout + (size_t)qrow_c * a.lddo + hq * D + 8 * hh;
      const uint16_t* op = a.o + (size_t)qrow_c * a.ldo + hq * D + 8 * hh;
      float s = 0.f;
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
        dof[kk] = ld8(dp + 16 * kk);
        float x[8], y[8];
        unpack8(__builtin_bit_cast(uint4, dof[kk]), x);
        unpack8(*reinterpret_cast<const uint4*>(op + 16 * kk), y);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += x[j] * y[j];
      }
      dl = xhalf_sum(s);
      lse2 = a.lse[(size_t)hq * T + qrow_c];
      if (hh == 0 && kh == 0 && qrow < nv) {   // what the dK / dV kernel starts its products from
        a.delta[(size_t)hq * T + qrow] = -dl;
        a.nlse[(size_t)hq * T + qrow] = -lse2 / a.c;
      }
    }
  }
  float m_i = -INFINITY, l_i = 0.f;
  f32x16 acc[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) acc[dt] = f32x16{};
  // row operands complete before the loop, through the compiler-visible wait: it does not count
  // the DMA issued from asm, and would wait for these loads in front of the loop's MFMAs
  __builtin_amdgcn_s_waitcnt(0);

  int offK[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) offK[kk] = toff<D>(r, 2 * kk + hh);
  int offT[NDT][2];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    const int col = 32 * dt + 16 * (g & 1) + 4 * (gi & 3), row0 = 4 * hh + (gi >> 2);
    offT[dt][0] = toff<D>(row0, col >> 3) + (col & 7) * 2;
    offT[dt][1] = toff<D>(row0 + 8, col >> 3) + (col & 7) * 2;
  }
  const float c = a.c, slack = 8.f / c;

  auto seen = [&](int k0, int e) __attribute__((always_inline)) {   // key k0 + crow(e, hh) visible to the lane's row
    return (uint32_t)(k0 + 4 * hh - st + crow(e, 0)) < (uint32_t)cnt;
  };
  auto scores = [&](const char* Kt) __attribute__((always_inline)) {
    f32x16 s = f32x16{};
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) s = mfma32(lds8(Kt, offK[kk]), qf[kk], s);
    return s;
  };
  auto raise_max = [&](float mx) __attribute__((always_inline)) {
    mx = xhalf_max(mx);
    // m_i need not be the maximum, only near it: P = 2^(c (s - m_i)) up to 2^8 keeps its relative precision in
    // bf16 and its sums in fp32.  So the sums are rescaled only where a row's maximum rose by more than that
    // (the first visible scores raise it from -inf; 16384 tokens in one, 32 heads of 128: 2.28 -> 2.21 ms)
    if (!__all(mx <= m_i + slack)) {
      const float m_new = fmaxf(m_i, mx);
      const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_i - m_new) * c);
      l_i *= alpha;
      m_i = m_new;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] *= alpha;
    }
    return m_i == -INFINITY ? 0.f : m_i * c;
  };
  auto expo = [&](f32x16& s, float mc) __attribute__((always_inline)) {   // s -> P, row sums into l_i
    float rs0 = 0.f, rs1 = 0.f;
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -mc));
      s[e + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e + 1], c, -mc));
      rs0 += s[e];
      rs1 += s[e + 1];
    }
    l_i += rs0 + rs1;
  };
  auto tfrag = [&](const char* Xt, int h, int dt) __attribute__((always_inline)) {   // 32 columns of d x 16 rows
    return cat(tr_read(Xt + 16 * h * RB, offT[dt][0]), tr_read(Xt + 16 * h * RB, offT[dt][1]));
  };
  // acc += (weights w of the 32 rows) X, w rounded to bf16 for the matrix unit (sums stay fp32)
  auto accum = [&](const char* Xt, const f32x16& w) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bf16x8 wb = pack8(w, 8 * h);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) acc[dt] = mfma32(tfrag(Xt, h, dt), wb, acc[dt]);
    }
  };
  uint32_t bad = 0;   // a masked subtile held a non-finite value: the wave's rows are redone at the end
  auto check = [&](const char* Xt) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) bad |= nonfinite(lds8(Xt, offK[kk]));
  };
  // N adjacent 32-key subtiles from key k0: their products are independent, so one's latency runs under
  // the other's (forward of 4096 tokens of ~300-token documents, 16 heads of 64: 24.5 us one subtile at a
  // time, 22.5 in pairs; dQ of 16384 tokens, 32 heads of 128: 3.18 and 2.88 ms).  PART: some may be masked.
  auto block = [&](const char* Kt, const char* Vt, int k0, auto nc, auto partc) __attribute__((always_inline)) {
    constexpr int N = decltype(nc)::value;
    constexpr bool PART = decltype(partc)::value;
    bool masked[N];
#pragma unroll
    for (int t = 0; t < N; ++t) {
      const int kt = k0 + 32 * t;
      masked[t] = PART && uni(kt < smax || kt + 31 > qw || qw + 31 >= nv ? 1 : 0);
    }
    f32x16 s[N];
    // products before the other workgroup's vector work: forward of 16384 tokens in one, 32 heads of 128, 2.24 ->
    // 2.11 ms, 4096 tokens 168 -> 146 us; no gain for dQ (2.9 ms both ways), and 4096 .. 8000 tokens of documents
    // with heads of 64 take 2 - 5 % longer
    constexpr bool PRIO = !DQ && D == 128;
    if constexpr (PRIO) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int t = 0; t < N; ++t) s[t] = scores(Kt + 32 * t * RB);
    if constexpr (!DQ) {
      if constexpr (PRIO) __builtin_amdgcn_s_setprio(0);
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < N; ++t) {
        if (masked[t]) {
          asm volatile("" ::: "memory");   // a real branch, not per-element selects
#pragma unroll
          for (int e = 0; e < 16; ++e) s[t][e] = seen(k0 + 32 * t, e) ? s[t][e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
      }
      const float mc = raise_max(mx);
#pragma unroll
      for (int t = 0; t < N; ++t) expo(s[t], mc);
      if constexpr (PRIO) __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < N; ++t) {
        if (masked[t]) check(Vt + 32 * t * RB);
        accum(Vt + 32 * t * RB, s[t]);
      }
      if constexpr (PRIO) __builtin_amdgcn_s_setprio(0);
    } else {
      f32x16 dp[N];
#pragma unroll
      for (int t = 0; t < N; ++t) {
        dp[t] = f32x16{};
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) dp[t] = mfma32(lds8(Vt + 32 * t * RB, offK[kk]), dof[kk], dp[t]);
      }
#pragma unroll
      for (int t = 0; t < N; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], c, -lse2)) * (dp[t][e] - dl);   // dS^T
#pragma unroll
      for (int t = 0; t < N; ++t) {
        if (masked[t]) {
          asm volatile("" ::: "memory");
#pragma unroll
          for (int e = 0; e < 16; ++e) s[t][e] = seen(k0 + 32 * t, e) ? s[t][e] : 0.f;
          check(Kt + 32 * t * RB);
        }
        accum(Kt + 32 * t * RB, s[t]);
      }
    }
  };
  constexpr int NW = HALF ? NSUB / 2 : NSUB;   // subtiles of a tile for each wave
  auto compute = [&](const char* Kt, const char* Vt, int j) __attribute__((always_inline)) {
    const int k0 = kv_lo + j * BK;
    if (uni(!wave_on || k0 > wlast || k0 + BK <= smin ? 1 : 0)) return;
    if constexpr (!DQ) {   // whole tile visible to every row of the wave: straight-line code
      if (uni(k0 >= smax && k0 + BK <= qw + 1 && qw + 31 < nv ? 1 : 0)) {
        block(Kt + kh * NW * 32 * RB, Vt + kh * NW * 32 * RB, k0 + 32 * kh * NW, std::integral_constant<int, NW>{},
              std::false_type{});
        return;
      }
    }
    int t = max(kh * NW, (smin - k0) >> 5);
    const int tb = min(kh * NW + NW - 1, (wlast - k0) >> 5);
#pragma unroll 1
    for (; t < tb; t += 2)
      block(Kt + 32 * t * RB, Vt + 32 * t * RB, k0 + 32 * t, std::integral_constant<int, 2>{}, std::true_type{});
    if (t == tb)
      block(Kt + 32 * t * RB, Vt + 32 * t * RB, k0 + 32 * t, std::integral_constant<int, 1>{}, std::true_type{});
  };
  auto step = [&](char* Kc, char* Vc, char* Kn, char* Vn, int j) __attribute__((always_inline)) {
    vm_drain();
    __syncthreads();
    if (j + 1 < ntile) issue(Kn, Vn, j + 1);
    compute(Kc, Vc, j);
  };
  for (int j = 0; j < ntile; j += 2) {
    step(kbuf0, vbuf0, kbuf1, vbuf1, j);
    if (j + 1 < ntile) step(kbuf1, vbuf1, kbuf0, vbuf0, j + 1);
  }

  if constexpr (HALF) {   // the halves meet: m, l and the first columns in one buffer, the rest in the other
    __syncthreads();
    float* x = reinterpret_cast<float*>(wq ? kbuf1 : kbuf0) + lane;
    float* y = reinterpret_cast<float*>(wq ? vbuf1 : vbuf0) + lane;
    if (kh == 1) {
      x[0] = m_i;
      x[64] = l_i;
      x[128] = __any(bad != 0) ? 1.f : 0.f;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          (dt < NDT / 2 ? x + 64 * (3 + 16 * dt + e) : y + 64 * (16 * (dt - NDT / 2) + e))[0] = acc[dt][e];
    }
    __syncthreads();
    if (kh == 1) return;
    bad |= x[128] != 0.f;
    float a0 = 1.f, a1 = 1.f;
    if constexpr (!DQ) {
      // (a half that saw no finite score holds sums of 0 or NaN, whatever their scale)
      const float m1 = x[0], m = fmaxf(m_i, m1);
      a0 = m_i == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_i - m) * c);
      a1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m1 - m) * c);
      l_i = l_i * a0 + x[64] * a1;
      m_i = m;
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        acc[dt][e] = acc[dt][e] * a0 +
                     (dt < NDT / 2 ? x + 64 * (3 + 16 * dt + e) : y + 64 * (16 * (dt - NDT / 2) + e))[0] * a1;
  }
  if (a.fill && qrow >= nv && qrow < T) {
    zero_row<D>(outp, hh);
    if (!DQ && hh == 0) a.lse[(size_t)hq * T + qrow] = INFINITY;
  }
  if (__any(bad != 0)) {
#pragma unroll 1
    for (int i = qw; i <= wlast; ++i) {
      const RowVec<D> qi(a.q + (size_t)i * a.ldq + hq * D, lane);
      RowVec<D> res;
      float m = -INFINITY, l = 0.f, de = 0.f, ls = 0.f;
      RowVec<D> doi;
      if constexpr (DQ) {
        doi = RowVec<D>(a.dout + (size_t)i * a.lddo + hq * D, lane);
        de = doi.dot(RowVec<D>(a.o + (size_t)i * a.ldo + hq * D, lane));
        ls = a.lse[(size_t)hq * T + i];
      }
#pragma unroll 1
      for (int j = a.start[i]; j <= i; ++j) {
        const RowVec<D> kj(a.k + (size_t)j * a.ldk + hk * D, lane);
        const RowVec<D> vj(a.v + (size_t)j * a.ldv + hk * D, lane);
        const float sij = qi.dot(kj);
        if constexpr (!DQ) {
          const float m_new = fmaxf(m, sij), mc = m_new == -INFINITY ? 0.f : m_new * c;
          const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c);
          const float pij = __builtin_amdgcn_exp2f(__builtin_fmaf(sij, c, -mc));
          m = m_new;
          l = l * alpha + pij;
#pragma unroll
          for (int x = 0; x < D / 64; ++x) res.x[x] *= alpha;
          res.axpy(pij, vj);
        } else {
          res.axpy(__builtin_amdgcn_exp2f(__builtin_fmaf(sij, c, -ls)) * (doi.dot(vj) - de), kj);
        }
      }
      const float nan = __uint_as_float(0x7fc00000u);
      res.store(a.out + (size_t)i * a.ldout + hq * D, lane, DQ ? a.scale : l > 0.f ? 1.f / l : nan);
      if (!DQ && lane == 0) a.lse[(size_t)hq * T + i] = l > 0.f ? m * c + __log2f(l) : nan;
    }
    return;
  }
  if (qrow >= nv) return;
  float sc = a.scale;
  if constexpr (!DQ) {
    const float lt = xhalf_sum(l_i);
    // lt = 0 only where every visible score is -inf: NaN, as the definition has it
    sc = lt > 0.f ? 1.f / lt : __uint_as_float(0x7fc00000u);
    if (hh == 0) a.lse[(size_t)hq * T + qrow] = lt > 0.f ? m_i * c + __log2f(lt) : sc;
  }
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) store_row32(outp + 32 * dt, acc[dt], sc, hh);
}

// ============================================================================ key-major
constexpr int KB1 = 128, KB2 = 256, QT2 = 64;   // keys of a block (D = 64 / 128), rows of a query tile
// Splits of a key block of `items` (query head, query tile) pairs: a split holds a workgroup slot's even
// share of the batch (meta: the query tiles of all blocks of one head) and a few items more, which pay
// for its partial sums.  dQ, dK, dV of 8 query heads on one key head, 512 tokens: 73 -> 38 us (D 64),
// 156 -> 58 us (D 128); without the extra items 4096 tokens of ~300-token documents take 120 us, not 99
// (16 heads of 128); with shares twice as large 16384 tokens, 16 / 4 heads, take 4.9 ms, not 3.8.
// No split is empty (the last would fetch rows and statistics behind the last query head): 88 items in 16
// splits of 6 are 15.
__host__ __device__ inline int split_count(int64_t tiles, int Hq, int D, int nsplit, int items) {
  if (nsplit == 1) return 1;
  const int64_t share = tiles * Hq / (D == 64 ? 512 : 256) + 5, most = (items + share - 1) / share;
  const int n = most < 1 ? 1 : most < nsplit ? (int)most : nsplit, per = (items + n - 1) / n;
  return (items + per - 1) / per;
}
template <int D>
__device__ __forceinline__ int block_splits(const PArgs& a, int items) {
  return split_count(D == 64 ? (int64_t)a.meta[1] : a.before[(a.T + KB2 - 1) / KB2], a.Hq, D, a.nsplit, items);
}

// D = 128, few key blocks: the items of all of them, head by head and block by block, are one line that
// is cut into even shares, one per workgroup; a block that a cut falls into is done in pieces, whose
// fp32 sums packed_join2_kernel adds.  A block counts PIECE items beside its own (its K and V rows, its
// results); a cut within SNAP items of a block's end moves there.  (Moving cuts saves partial sums but makes
// shares uneven: 4096 tokens of ~300, 16 / 4 heads, dQ + dK + dV 153 us in the mean of three batches at 2, 163 at
// 5, 224 at 16.)
constexpr int PIECE = 3, SNAP = 2, SHARE_MIN = 8;
__device__ __forceinline__ int64_t uni64(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)uni((int)x) | (uint64_t)(uint32_t)uni((int)(x >> 32)) << 32);
}
struct KeyShare {
  const int64_t* before;    // query tiles of the blocks before each
  int nb, grp, n;           // blocks, query heads of a key head, shares
  int64_t head, total;      // length of a head's line, of all
  __device__ __forceinline__ KeyShare(const PArgs& a, int nv)
      : before(a.before), nb((nv + KB2 - 1) / KB2), grp(a.Hq / a.Hkv) {
    head = off(nb);
    total = head * a.Hkv;
    n = (int)min((int64_t)a.nshare, (total + SHARE_MIN - 1) / SHARE_MIN);
  }
  struct Pos { int64_t line; int hk, blk; int64_t f; };    // on the line; head, block, offset in the block
  __device__ __forceinline__ int64_t off(int b) const { return grp * before[b] + PIECE * (int64_t)b; }
  // where share w begins; a wave probes 64 blocks at a time
  __device__ __forceinline__ Pos first(int w, int lane) const {
    Pos p;
    p.line = total * w / n;
    p.hk = uni((int)(p.line / head));
    const int64_t q = p.line - p.hk * head;
    int lo = 0, cnt = nb;
    while (cnt > 1) {
      const int step = (cnt + 63) / 64, x = lane * step;
      const int k = __popcll(__ballot(x < cnt && off(lo + min(x, cnt - 1)) <= q)) - 1;
      lo += k * step;
      cnt = min(step, cnt - k * step);
    }
    p.blk = uni(lo);
    p.f = q - off(lo);
    if (w == n) return p;                                  // (the end of the line: never looked into)
    const int64_t left = off(lo + 1) - q;
    if (p.f <= PIECE + SNAP) {
      p.line -= p.f;
      p.f = 0;
    } else if (left <= SNAP) {
      p.line += left;
      p.f = 0;
      if (++p.blk == nb) { p.blk = 0; ++p.hk; }
    }
    return p;
  }
};

// Where a key block's dK / dV go: the results, or (pk given) fp32 partial sums, key row0 first, W floats a row
template <int D>
struct KeyOut {
  const PArgs& a;
  int hk, lane;
  float *pk, *pv;
  int row0, W;
  // the accumulators of one key per lane pair
  template <int N>
  __device__ __forceinline__ void put(int key, const f32x16 (&dk)[N], const f32x16 (&dv)[N], int hh) const {
    if (pk) {
#pragma unroll
      for (int dt = 0; dt < N; ++dt)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const size_t o = (size_t)(key - row0) * W + 32 * dt + 2 * e + 4 * hh;
          *reinterpret_cast<float4*>(pk + o) = make_float4(dk[dt][e], dk[dt][e + 1], dk[dt][e + 2], dk[dt][e + 3]);
          *reinterpret_cast<float4*>(pv + o) = make_float4(dv[dt][e], dv[dt][e + 1], dv[dt][e + 2], dv[dt][e + 3]);
        }
      return;
    }
#pragma unroll
    for (int dt = 0; dt < N; ++dt) {
      store_row32(a.dk + (size_t)key * a.lddk + hk * D + 32 * dt, dk[dt], a.scale, hh);
      store_row32(a.dv + (size_t)key * a.lddv + hk * D + 32 * dt, dv[dt], 1.f, hh);
    }
  }
  __device__ __forceinline__ void put(int key, const RowVec<D>& dk, const RowVec<D>& dv) const {
    if (pk) {
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {
        pk[(size_t)(key - row0) * W + lane + 64 * x] = dk.x[x];
        pv[(size_t)(key - row0) * W + lane + 64 * x] = dv.x[x];
      }
      return;
    }
    dk.store(a.dk + (size_t)key * a.lddk + hk * D, lane, a.scale);
    dv.store(a.dv + (size_t)key * a.lddv + hk * D, lane, 1.f);
  }
};

// keys ka .. kb one by one over the items t0 .. t1 - 1 of their block (a wave that met a non-finite operand)
template <int D>
__device__ __forceinline__ void redo_keys(const PArgs& a, const KeyOut<D>& out, int ka, int kb, int k0, int t0, int t1,
                                          int nqt, int hk, int grp, int lane) {
#pragma unroll 1
  for (int j = ka; j <= kb; ++j) {
    const RowVec<D> kj(a.k + (size_t)j * a.ldk + hk * D, lane);
    const RowVec<D> vj(a.v + (size_t)j * a.ldv + hk * D, lane);
    RowVec<D> rk, rv;
    const int je = a.end[j];
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      const int hq = hk * grp + t / nqt, qs = k0 + (t % nqt) * QT2;
#pragma unroll 1
      for (int i = max(j, qs); i < min(je, qs + QT2); ++i) {
        const RowVec<D> qi(a.q + (size_t)i * a.ldq + hq * D, lane);
        const RowVec<D> doi(a.dout + (size_t)i * a.lddo + hq * D, lane);
        const size_t li = (size_t)hq * a.T + i;
        const float pij = __builtin_amdgcn_exp2f(__builtin_fmaf(qi.dot(kj), a.c, -a.lse[li]));
        rv.axpy(pij, doi);
        rk.axpy(pij * (doi.dot(vj) + a.delta[li]), qi);
      }
    }
    out.put(j, rk, rv);
  }
}

// dK, dV: key on the MFMA lane; Q / dO tiles of QT rows (and their statistics) stream through a
// two-slot LDS-DMA ring, over the query heads of the key head's group.  Where there are few key blocks,
// those of long sequences are split along their (query head, query tile) items over up to `nsplit`
// workgroups, whose fp32 partial sums packed_join_kernel adds in order (or all are cut, see KeyShare).
//
// D = 64.  Four waves of 32 keys, two waves per SIMD.  16384 tokens in one, 16 heads: 1.22 ms (0.90 PFLOP/s), the
// matrix pipe busy 45 % of the time, the vector pipe 43: a 32-key wave reads LDS for 1.5 cycles to each of the
// matrix pipe's.
template <int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void
packed_kmajor_kernel(const PArgs a) {
  constexpr int KB = KB1, QT = QT2, NQS = QT / 32, NKK = D / 16, NDT = D / 32;
  constexpr int RB = D * 2, CPR = D / 8, RPP = 64 / CPR, TILE = QT * RB, PPW = TILE / 1024 / 4;
  __shared__ __attribute__((aligned(16))) char qb0[TILE];
  __shared__ __attribute__((aligned(16))) char qb1[TILE];
  __shared__ __attribute__((aligned(16))) char ob0[TILE];
  __shared__ __attribute__((aligned(16))) char ob1[TILE];
  __shared__ __attribute__((aligned(16))) float lb0[64];
  __shared__ __attribute__((aligned(16))) float lb1[64];
  __shared__ __attribute__((aligned(16))) float db0[64];
  __shared__ __attribute__((aligned(16))) float db1[64];
  const int tid = threadIdx.x, lane = tid & 63, wl = uni(tid >> 6);
  const int r = lane & 31, hh = lane >> 5, g = lane >> 4, gi = lane & 15;
  const int T = a.T;
  const int nblk = gridDim.x / a.nsplit, sp = blockIdx.x / nblk;
  int rank, hk;
  block_map(blockIdx.x - sp * nblk, a.Hkv, rank, hk);
  const int grp = a.Hq / a.Hkv;
  // (table reads that depend on the block alone; see packed_qmajor_kernel)
  const int k0 = uni(a.order[pair_rank(rank, (T + KB - 1) / KB)]) * KB;
  const int kw = k0 + 32 * wl, key = kw + r;
  const int nv = uni(a.meta[0]);
  const int qend = min(uni(a.end[min(k0 + KB, T) - 1]), nv);   // queries of the block: k0 .. qend - 1
  const int emin = uni(a.end[min(kw, T - 1)]), emax = min(uni(a.end[min(kw + 31, T - 1)]), nv);
  const int key_c = min(key, T - 1), kend = a.end[key_c];
  uint16_t* dkp = a.dk + (size_t)key * a.lddk + hk * D;
  uint16_t* dvp = a.dv + (size_t)key * a.lddv + hk * D;
  if (k0 >= nv) {
    if (a.fill && sp == 0 && key < T) {
      zero_row<D>(dkp, hh);
      zero_row<D>(dvp, hh);
    }
    return;
  }
  const int nqt = (qend - k0 + QT - 1) / QT, items = nqt * grp;
  const int nsp = uni(block_splits<D>(a, items)), per = (items + nsp - 1) / nsp;
  const int t0 = sp * per, t1 = min(items, t0 + per);
  if (sp >= nsp) return;
  const bool wave_on = kw < nv;
  const int cnt = key < nv ? kend - key : 0;           // rows that see this key: key .. key + cnt - 1
  uint32_t voQ[PPW], voO[PPW];
#pragma unroll
  for (int i = 0; i < PPW; ++i) {
    const int R = (wl + 4 * i) * RPP + lane / CPR, ch = (lane % CPR) ^ swz<D>(R);
    voQ[i] = (uint32_t)(R * a.ldq + ch * 8) * 2u;
    voO[i] = (uint32_t)(R * a.lddo + ch * 8) * 2u;
  }
  auto issue = [&](char* qd, char* od, float* ld, float* dd, int hq, int qs) __attribute__((always_inline)) {
    const int rows = min(QT, nv - qs);
    const i32x4_t qr = rows_rsrc<D>(a.q + (size_t)qs * a.ldq + hq * D, rows, a.ldq);
    const i32x4_t dr = rows_rsrc<D>(a.dout + (size_t)qs * a.lddo + hq * D, rows, a.lddo);
#pragma unroll
    for (int i = 0; i < PPW; ++i) {
      dma16_buf(qr, voQ[i], qd + (wl + 4 * i) * 1024);
      dma16_buf(dr, voO[i], od + (wl + 4 * i) * 1024);
    }
    if (wl < 2) {
      const size_t li = (size_t)hq * T + min(qs + lane, nv - 1);
      if (wl == 0) dma4(a.nlse + li, (char*)ld);
      else dma4(a.delta + li, (char*)dd);
    }
  };
  int hq_n = hk * grp + t0 / nqt, qs_n = k0 + (t0 % nqt) * QT;   // the item to fetch next
  int qs_c = qs_n;
  auto advance = [&]() __attribute__((always_inline)) {
    qs_n += QT;
    if (qs_n >= qend) { qs_n = k0; ++hq_n; }
  };
  issue(qb0, ob0, lb0, db0, hq_n, qs_n);             // (under the row loads)
  advance();
  bf16x8 kf[NKK], vf[NKK];
  {
    const uint16_t* kp = a.k + (size_t)key_c * a.ldk + hk * D + 8 * hh;
    const uint16_t* vp = a.v + (size_t)key_c * a.ldv + hk * D + 8 * hh;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      kf[kk] = ld8(kp + 16 * kk);
      vf[kk] = ld8(vp + 16 * kk);
    }
  }
  f32x16 dvacc[NDT], dkacc[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) { dvacc[dt] = f32x16{}; dkacc[dt] = f32x16{}; }
  __builtin_amdgcn_s_waitcnt(0);   // (see packed_qmajor_kernel)

  int offQ[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) offQ[kk] = toff<D>(r, 2 * kk + hh);
  int offT[NDT][2];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    const int col = 32 * dt + 16 * (g & 1) + 4 * (gi & 3), row0 = 4 * hh + (gi >> 2);
    offT[dt][0] = toff<D>(row0, col >> 3) + (col & 7) * 2;
    offT[dt][1] = toff<D>(row0 + 8, col >> 3) + (col & 7) * 2;
  }
  const float c = a.c;
  uint32_t bad = 0;   // (see packed_qmajor_kernel)
  auto body = [&](const char* Qt, const char* Ot, const float* Lt, const float* Dt, int qs) __attribute__((always_inline)) {
#pragma unroll 1
    for (int u = 0; u < NQS; ++u) {
      const int qsu = qs + 32 * u;
      if (uni(qsu + 31 < kw || qsu >= emax ? 1 : 0)) continue;
      // the products start from -lse / c and -delta of their rows: P = 2^(c S), dS = P dP
      f32x16 s, dp;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const float4 ls = *reinterpret_cast<const float4*>(Lt + 32 * u + 2 * e + 4 * hh);
        const float4 de = *reinterpret_cast<const float4*>(Dt + 32 * u + 2 * e + 4 * hh);
        s[e] = ls.x; s[e + 1] = ls.y; s[e + 2] = ls.z; s[e + 3] = ls.w;
        dp[e] = de.x; dp[e + 1] = de.y; dp[e + 2] = de.z; dp[e + 3] = de.w;
      }
      const char* Qu = Qt + 32 * u * RB;
      const char* Ou = Ot + 32 * u * RB;
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
        s = mfma32(lds8(Qu, offQ[kk]), kf[kk], s);
        dp = mfma32(lds8(Ou, offQ[kk]), vf[kk], dp);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(s[e] * c);
        dp[e] *= s[e];
      }
      // whole: every row of the subtile sees every key of the wave
      if (uni(qsu < kw + 31 || qsu + 32 > emin || kw + 31 >= nv ? 1 : 0)) {
        asm volatile("" ::: "memory");   // a real branch
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const bool seen = (uint32_t)(qsu + 4 * hh - key + crow(e, 0)) < (uint32_t)cnt;
          s[e] = seen ? s[e] : 0.f;
          dp[e] = seen ? dp[e] : 0.f;
        }
        bad |= bad_rows(Dt + 32 * u + 4 * hh);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16x8 pb = pack8(s, 8 * h);
        const bf16x8 sb = pack8(dp, 8 * h);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const int ro = 16 * h * RB;
          dvacc[dt] = mfma32(cat(tr_read(Ou + ro, offT[dt][0]), tr_read(Ou + ro, offT[dt][1])), pb, dvacc[dt]);
          dkacc[dt] = mfma32(cat(tr_read(Qu + ro, offT[dt][0]), tr_read(Qu + ro, offT[dt][1])), sb, dkacc[dt]);
        }
      }
    }
  };
  auto step = [&](char* Qc, char* Oc, float* Lc, float* Dc, char* Qn, char* On, float* Ln, float* Dn,
                  int t) __attribute__((always_inline)) {
    vm_drain();
    __syncthreads();
    const int qs = qs_c;
    if (t + 1 < t1) {
      issue(Qn, On, Ln, Dn, hq_n, qs_n);
      qs_c = qs_n;
      advance();
    }
    if (uni(wave_on && qs < emax && qs + QT > kw ? 1 : 0)) body(Qc, Oc, Lc, Dc, qs);
  };
  for (int t = t0; t < t1; t += 2) {
    step(qb0, ob0, lb0, db0, qb1, ob1, lb1, db1, t);
    if (t + 1 < t1) step(qb1, ob1, lb1, db1, qb0, ob0, lb0, db0, t + 1);
  }
  if (a.fill && sp == 0 && key >= nv && key < T) {
    zero_row<D>(dkp, hh);
    zero_row<D>(dvp, hh);
  }
  const int W = a.Hkv * D;                             // partials: [split][dk, dv][T][Hkv D]
  float* pk = nsp > 1 ? a.part + (size_t)sp * 2 * T * W + hk * D : nullptr;
  const KeyOut<D> out{a, hk, lane, pk, pk + (size_t)T * W, 0, W};
  if (__any(bad != 0)) {
    redo_keys<D>(a, out, kw, min(kw + 31, nv - 1), k0, t0, t1, nqt, hk, grp, lane);
    return;
  }
  if (key >= nv) return;
  out.put(key, dkacc, dvacc, hh);
}

// D = 128.  Two 32-key groups per wave, one wave per SIMD: every Q / dO fragment read from LDS feeds
// two MFMAs (a 32-key wave needs 1408 LDS cycles per 1024 MFMA cycles of the four SIMDs -- the
// transposed reads run at half rate --, this one 1408 per 2048), and the accumulators of both groups
// (256 registers), their K rows and half of V (96; the rest is read again from LDS) and S, dP (64) fit
// the 512 registers.  A workgroup holds 256 keys.  16384 tokens in one, 32 heads: 4.2 ms, 1.05 PFLOP/s,
// the matrix pipe busy 45 % of the time: no other wave runs beside a wave's own vector work.
//
// MFMA with its accumulator in ordinary registers.  The compiler gives every MFMA of a kernel that
// needs accumulation registers an accumulator there; dK and dV of 64 keys take all 256 of them, and
// it moved S and dP in and out of them at every subtile.  Written as asm, so the wait between the
// last product and the first use is mfma_v_done's: 8 passes of 4 cycles and 3 more are required,
// 24 are waited.  A product's operands are read from LDS (waited for by the compiler) or long loaded.
__device__ __forceinline__ void mfma_v(f32x16& d, bf16x8 a, bf16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_v_done(f32x16& a, f32x16& b) {
  asm volatile("s_nop 15\n\ts_nop 7" : "+v"(a), "+v"(b));
}

template <int D, bool SHARES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void packed_kmajor2_kernel(const PArgs a0) {
  constexpr int NL = 4;   // the V fragments of odd kk stay in LDS: the registers do not hold all
  constexpr int QT = QT2, NQS = QT / 32, NKK = D / 16, NDT = D / 32;
  constexpr int RB = D * 2, CPR = D / 8, RPP = 64 / CPR, TILE = QT * RB, PPW = TILE / 1024 / 4;
  __shared__ __attribute__((aligned(16))) char ring[2][2 * TILE];   // Q, dO
  __shared__ __attribute__((aligned(16))) float stat[2][2][64];     // -lse / c, -delta
  __shared__ __attribute__((aligned(16))) uint4 vlds[4][2 * NL][64];  // the waves' V fragments of odd kk
  const int lane0 = threadIdx.x & 63, wl = uni((int)threadIdx.x >> 6);
  const int nv = uni(a0.meta[0]);
  if (a0.fill)                                          // rows behind the last sequence
    for (int64_t x = (int64_t)nv * a0.Hkv + blockIdx.x * 4 + wl; x < (int64_t)a0.T * a0.Hkv; x += gridDim.x * 4) {
      const int64_t row = x / a0.Hkv;
      const int col = (int)(x - row * a0.Hkv) * D + 2 * lane0;
      *reinterpret_cast<uint32_t*>(a0.dk + row * a0.lddk + col) = 0;
      *reinterpret_cast<uint32_t*>(a0.dv + row * a0.lddv + col) = 0;
    }
  const int nbv = (nv + KB2 - 1) / KB2;                // blocks with work
  int w = 0, hk, blk, sp = 0;
  int64_t f = 0, left = 0;                             // offset in the block; what is left of the share
  if constexpr (SHARES) {                              // a share to each workgroup, neighbours on one XCD
    const KeyShare ks(a0, nv);
    if ((int)blockIdx.x >= ks.n) return;
    const int n8 = ks.n >> 3, x = (int)blockIdx.x;
    w = x < 8 * n8 ? (x & 7) * n8 + (x >> 3) : x;
    const KeyShare::Pos p = ks.first(w, lane0);
    hk = uni(p.hk); blk = uni(p.blk); f = uni64(p.f);
    left = uni64(ks.first(w + 1, lane0).line - p.line);
    if (left <= 0) return;
  } else {                                             // a block, or a split of it, to each
    const int nblk = gridDim.x / a0.nsplit;
    sp = blockIdx.x / nblk;
    block_map(blockIdx.x - sp * nblk, a0.Hkv, blk, hk);
    blk = uni(a0.order[blk]);
    if (blk >= nbv) return;
  }
#pragma unroll 1
  for (;; blk + 1 < nbv ? ++blk : (blk = 0, ++hk)) {
  // (the arguments are read again for every block: kept across blocks they and what derives from them
  // overflow the scalar registers, and those they spill to)
  const PArgs& a = a0;
  const int T = a.T, grp = a.Hq / a.Hkv;
  const int k0 = blk * KB2, kw = k0 + 64 * wl;
  const int qend = min(uni(a.end[min(k0 + KB2, T) - 1]), nv);
  const int emax = min(uni(a.end[min(kw + 63, T - 1)]), nv);
  const int nqt = (qend - k0 + QT - 1) / QT, items = nqt * grp;
  int t0, t1, nsp = 1;
  if constexpr (SHARES) {
    const int64_t take = min(left, items + PIECE - f);
    t0 = uni((int)max(f - PIECE, (int64_t)0));
    t1 = uni((int)(f + take - PIECE));
    left -= take;
    f = 0;
    if (t1 <= t0) {
      if (left <= 0) break;
      continue;
    }
  } else {
    nsp = uni(block_splits<D>(a, items));
    const int per = (items + nsp - 1) / nsp;
    t0 = sp * per;
    t1 = min(items, t0 + per);
    if (sp >= nsp) return;
  }
  int lane = lane0;                                    // (no table of it is kept across blocks: there are no registers)
  asm volatile("" : "+v"(lane));
  const int r = lane & 31, hh = lane >> 5, g = lane >> 4, gi = lane & 15;
  int key[2], cnt[2], emin[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    key[j] = kw + 32 * j + r;
    cnt[j] = a.end[min(key[j], T - 1)] - key[j];       // rows that see this key: key .. key + cnt - 1
    emin[j] = uni(a.end[min(kw + 32 * j, T - 1)]);
  }
  const bool wave_on = kw < nv;
  const int klast = min(kw + 63, nv - 1);
  uint32_t bad = 0;   // (see packed_qmajor_kernel)
  bf16x8 kf[2][NKK], vf[2][NL];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (key[j] >= nv) cnt[j] = 0;
    const int kc = min(key[j], nv - 1);
    const uint16_t* kp = a.k + (size_t)kc * a.ldk + hk * D + 8 * hh;
    const uint16_t* vp = a.v + (size_t)kc * a.ldv + hk * D + 8 * hh;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      kf[j][kk] = ld8(kp + 16 * kk);
      const bf16x8 x = ld8(vp + 16 * kk);
      if (kk & 1) vlds[wl][kk - 1 + j][lane] = __builtin_bit_cast(uint4, x);
      else vf[j][kk >> 1] = x;
    }
  }
  f32x16 dvacc[2][NDT], dkacc[2][NDT];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) { dvacc[j][dt] = f32x16{}; dkacc[j][dt] = f32x16{}; }
  __builtin_amdgcn_s_waitcnt(0);   // (see packed_qmajor_kernel)

  // LDS offsets: chunk 2 kk + hh (row reads) and 4 dt + .. (transposed reads) differ from the first
  // by bits that the swizzle only flips, so one register and a XOR stand for each table
  static_assert(D == 128, "256-B rows");
  // (made opaque where they are used, so that the XORs are not hoisted into registers there are not)
  int offQ0 = toff<D>(r, hh);
  const int tcol = 16 * (g & 1) + 4 * (gi & 3), trow = 4 * hh + (gi >> 2);
  int offT0 = toff<D>(trow, tcol >> 3) + (tcol & 7) * 2, offT1 = toff<D>(trow + 8, tcol >> 3) + (tcol & 7) * 2;
  auto rread = [&](const char* X, int kk) __attribute__((always_inline)) { return lds8(X, offQ0 ^ (kk << 5)); };
  auto tread = [&](const char* X, int dt) __attribute__((always_inline)) {
    return cat(tr_read(X, offT0 ^ (dt << 6)), tr_read(X, offT1 ^ (dt << 6)));
  };
  // DMA pieces of a wave are 16 rows apart (the same swizzle)
  const int R0 = wl * RPP + lane / CPR, ch0 = (lane % CPR) ^ swz<D>(R0);
  uint32_t voQ = (uint32_t)(R0 * a.ldq + ch0 * 8) * 2u, voO = (uint32_t)(R0 * a.lddo + ch0 * 8) * 2u;
  auto issue = [&](char* qd, char* od, float* ld, float* dd, int hq, int qs) __attribute__((always_inline)) {
    const int rows = min(QT, nv - qs);
    asm volatile("" : "+v"(voQ), "+v"(voO));
    const i32x4_t qr = rows_rsrc<D>(a.q + (size_t)qs * a.ldq + hq * D, rows, a.ldq);
    const i32x4_t dr = rows_rsrc<D>(a.dout + (size_t)qs * a.lddo + hq * D, rows, a.lddo);
#pragma unroll
    for (int i = 0; i < PPW; ++i) {
      dma16_buf(qr, voQ + (uint32_t)(8 * RPP * i * a.ldq), qd + (wl + 4 * i) * 1024);
      dma16_buf(dr, voO + (uint32_t)(8 * RPP * i * a.lddo), od + (wl + 4 * i) * 1024);
    }
    if (wl < 2) {
      const size_t li = (size_t)hq * T + min(qs + lane, nv - 1);
      if (wl == 0) dma4(a.nlse + li, (char*)ld);
      else dma4(a.delta + li, (char*)dd);
    }
  };
  const float c = a.c;
  auto body = [&](const char* Qt, const char* Ot, const float* Lt, const float* Dt, int qs) __attribute__((always_inline)) {
#pragma unroll 1
    for (int u = 0; u < NQS; ++u) {
      const int qsu = qs + 32 * u;
      if (uni(qsu + 31 < kw || qsu >= emax ? 1 : 0)) continue;
      asm volatile("" : "+v"(offQ0), "+v"(offT0), "+v"(offT1));
      f32x16 s[2], dp[2];
      const char* Qu = Qt + 32 * u * RB;
      const char* Ou = Ot + 32 * u * RB;
      const float* Lu = Lt + 32 * u + 4 * hh;
      const float* Du = Dt + 32 * u + 4 * hh;
      // part: some (row, key) pair of the subtile is masked
      const bool part = uni(qsu < kw + 63 || qsu + 32 > emin[0] || qsu + 32 > emin[1] || kw + 63 >= nv ? 1 : 0);
      // One wave per SIMD: vector work runs beside the matrix pipe only where it stands between matrix
      // instructions.  Four phases of 16 products each -- S; dP between the exponentials; dV between the
      // products P (dP - delta); dK -- over one stream of 32 LDS fragments, read PD steps (of two products,
      // 64 cycles) ahead.  The scheduling barriers keep this order (the compiler would read every fragment
      // first, for which there are no registers).
      constexpr int PD = 2, RN = PD + 1;
      bf16x8 f[RN];
      auto fetch = [&](int x) __attribute__((always_inline)) {
        if (x < 8) f[x % RN] = rread(Qu, x);
        else if (x < 16) f[x % RN] = rread(Ou, x - 8);
        else if (x < 24) f[x % RN] = tread(Ou + 16 * ((x - 16) / NDT) * RB, x % NDT);
        else if (x < 32) f[x % RN] = tread(Qu + 16 * ((x - 24) / NDT) * RB, x % NDT);
      };
      // the products start from -lse / c and -delta of their rows: P = 2^(c S), dS = P dP
      auto start = [&](f32x16& d, const float* p) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 x = *reinterpret_cast<const float4*>(p + 2 * e);
          d[e] = x.x; d[e + 1] = x.y; d[e + 2] = x.z; d[e + 3] = x.w;
        }
      };
      start(s[0], Lu);
      start(s[1], Lu);
#pragma unroll
      for (int x = 0; x < PD; ++x) fetch(x);
      start(dp[0], Du);
      start(dp[1], Du);
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
        fetch(kk + PD);
        mfma_v(s[0], f[kk % RN], kf[0][kk]);
        mfma_v(s[1], f[kk % RN], kf[1][kk]);
        __builtin_amdgcn_sched_barrier(0);
      }
      auto vread = [&](int x) __attribute__((always_inline)) { return __builtin_bit_cast(bf16x8, vlds[wl][x][lane]); };
      bf16x8 vl[2] = {vread(0), vread(1)};
      auto expo = [&](int x) __attribute__((always_inline)) {   // elements 2 x, 2 x + 1 of both groups: S -> P
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[j][2 * x] = __builtin_amdgcn_exp2f(s[j][2 * x] * c);
          s[j][2 * x + 1] = __builtin_amdgcn_exp2f(s[j][2 * x + 1] * c);
        }
      };
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
        fetch(8 + kk + PD);
        const bf16x8 v0 = kk & 1 ? vl[0] : vf[0][kk >> 1], v1 = kk & 1 ? vl[1] : vf[1][kk >> 1];
        mfma_v(dp[0], f[(8 + kk) % RN], v0);
        mfma_v(dp[1], f[(8 + kk) % RN], v1);
        if (kk == 0) mfma_v_done(s[0], s[1]);
        if ((kk & 1) && kk + 2 < NKK) {
          vl[0] = vread(kk + 1);
          vl[1] = vread(kk + 2);
        }
        expo(kk);
        __builtin_amdgcn_sched_barrier(0);
      }
      static_assert(NKK == 8 && NDT == 4, "the phases carry 16 elements in 8 steps");
      auto grad = [&](int x) __attribute__((always_inline)) {   // elements 2 x, 2 x + 1: dP -> dS
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          dp[j][2 * x] *= s[j][2 * x];
          dp[j][2 * x + 1] *= s[j][2 * x + 1];
        }
      };
      if (part) {
        // P = 0 and dP - delta = 0 where masked: do_i . v_j of finite values may overflow, and 0 times that is NaN.
        // (With the wait it costs batches of short documents 2 %: 8001 tokens of ~900, 32 / 8 heads, dQ + dK + dV 416 ->
        // 425 us.  In the shadow of the dV products instead, by a compare of every P with 0, 430.)
        asm volatile("" ::: "memory");   // a real branch
        mfma_v_done(dp[0], dp[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool seen = (uint32_t)(qsu + 4 * hh - key[j] + crow(e, 0)) < (uint32_t)cnt[j];
            s[j][e] = seen ? s[j][e] : 0.f;
            dp[j][e] = seen ? dp[j][e] : 0.f;
          }
        bad |= bad_rows(Du);
      }
      bf16x8 w[2][2];                                  // P, then dS, of both groups as MFMA operands
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) w[j][h] = pack8(s[j], 8 * h);
      auto dv_step = [&](int x) __attribute__((always_inline)) {   // (16-row half x / 4, 32 columns x % 4)
        fetch(16 + x + PD);
        dvacc[0][x % NDT] = mfma32(f[(16 + x) % RN], w[0][x / NDT], dvacc[0][x % NDT]);
        dvacc[1][x % NDT] = mfma32(f[(16 + x) % RN], w[1][x / NDT], dvacc[1][x % NDT]);
      };
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        dv_step(x);
        if (x == 0) mfma_v_done(dp[0], dp[1]);
        grad(x);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) w[j][h] = pack8(dp[j], 8 * h);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        fetch(24 + x + PD);
        dkacc[0][x % NDT] = mfma32(f[(24 + x) % RN], w[0][x / NDT], dkacc[0][x % NDT]);
        dkacc[1][x % NDT] = mfma32(f[(24 + x) % RN], w[1][x / NDT], dkacc[1][x % NDT]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  int hq_n = hk * grp + t0 / nqt, qs_n = k0 + (t0 % nqt) * QT;   // the item to fetch next
  int qs_c = qs_n;
  auto advance = [&]() __attribute__((always_inline)) {
    qs_n += QT;
    if (qs_n >= qend) { qs_n = k0; ++hq_n; }
  };
  issue(ring[0], ring[0] + TILE, stat[0][0], stat[0][1], hq_n, qs_n);
  advance();
#pragma unroll 1
  for (int t = t0; t < t1; ++t) {
    const int slot = (t - t0) & 1, nslot = slot ^ 1;
    vm_drain();
    __syncthreads();
    const int qs = qs_c;
    if (t + 1 < t1) {
      issue(ring[nslot], ring[nslot] + TILE, stat[nslot][0], stat[nslot][1], hq_n, qs_n);
      qs_c = qs_n;
      advance();
    }
    if (uni(wave_on && qs < emax && qs + QT > kw ? 1 : 0))
      body(ring[slot], ring[slot] + TILE, stat[slot][0], stat[slot][1], qs);
  }
  const int W = SHARES ? D : a.Hkv * D;                // partials: of a piece [dk, dv][KB2][D], or as of D = 64
  float *pk = nullptr, *pv = nullptr;
  if (SHARES ? t1 - t0 < items : nsp > 1) {
    pk = a.part + (SHARES ? (size_t)(2 * w + (t0 == 0 ? 1 : 0)) * 2 * KB2 * D : (size_t)sp * 2 * T * W + hk * D);
    pv = pk + (size_t)(SHARES ? KB2 : T) * W;
  }
  const KeyOut<D> out{a, hk, lane, pk, pv, SHARES ? k0 : 0, W};
  const bool redo = __any(bad != 0);
  if (redo) redo_keys<D>(a, out, kw, klast, k0, t0, t1, nqt, hk, grp, lane);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (key[j] < nv && !redo) out.put(key[j], dkacc[j], dvacc[j], hh);
  if (!SHARES || left <= 0) break;
  __syncthreads();                                     // the ring is free for the next block
  }
}

// the partial dK / dV of split blocks, in the order of the splits; 4 values per thread
template <int D>
__global__ __launch_bounds__(256) void packed_join_kernel(const PArgs a) {
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int W = a.Hkv * D, nw = W / 4;
  const int64_t t = v / nw;
  const int nv = a.meta[0];
  if (t >= nv) return;
  constexpr int KB = D == 64 ? KB1 : KB2;
  const int col = (int)(v - t * nw) * 4, k0 = (int)t / KB * KB;
  const int nqt = (min(a.end[min(k0 + KB, a.T) - 1], nv) - k0 + QT2 - 1) / QT2;
  const int nsp = block_splits<D>(a, nqt * (a.Hq / a.Hkv));
  if (nsp == 1) return;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < nsp; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(a.part + ((size_t)(2 * k + w) * a.T + t) * W + col);
      s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
    const float sc = w ? 1.f : a.scale;
    uint16_t* o = w ? a.dv + (size_t)t * a.lddv : a.dk + (size_t)t * a.lddk;
    *reinterpret_cast<uint2*>(o + col) = make_uint2(pack2(s.x * sc, s.y * sc), pack2(s.z * sc, s.w * sc));
  }
}

// D = 128: the blocks that the ends of shares cut.  JOIN workgroups for the end of each share w; the one
// where the cut block's first piece ends adds all of its pieces, in the order of the shares.
constexpr int JOIN = 16;
__global__ __launch_bounds__(256) void packed_join2_kernel(const PArgs a) {
  constexpr int D = 128;
  const int w = blockIdx.x / JOIN, lane = threadIdx.x & 63, nv = uni(a.meta[0]);
  const KeyShare ks(a, nv);
  if (w + 1 >= ks.n) return;
  const KeyShare::Pos cut = ks.first(w + 1, lane);
  if (cut.f == 0) return;                              // between two blocks
  const int64_t b0 = cut.line - cut.f;                 // the block's first item is of share w, or of one before
  if (ks.first(w, lane).line > b0) return;
  const int64_t b1 = b0 + ks.off(cut.blk + 1) - ks.off(cut.blk);
  int last = w + 1;
  while (last + 1 < ks.n && ks.first(last + 1, lane).line < b1) ++last;
  const int hk = cut.hk, blk = cut.blk;
  const int k0 = blk * KB2, n = min(KB2, nv - k0) * (D / 4);
  for (int x = (blockIdx.x % JOIN) * 256 + threadIdx.x; x < 2 * n; x += JOIN * 256) {
    const int which = x >= n, y = x - which * n, row = k0 + y / (D / 4), col = hk * D + y % (D / 4) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = w; k <= last; ++k) {
      const float* p = a.part + (size_t)((2 * k + (k == w ? 1 : 0)) * 2 + which) * KB2 * D + 4 * (size_t)y;
      const float4 v = *reinterpret_cast<const float4*>(p);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const float sc = which ? 1.f : a.scale;
    uint16_t* o = which ? a.dv + (size_t)row * a.lddv : a.dk + (size_t)row * a.lddk;
    *reinterpret_cast<uint2*>(o + col) = make_uint2(pack2(s.x * sc, s.y * sc), pack2(s.z * sc, s.w * sc));
  }
}

// most splits of a key block: until there are 1024 workgroups, or 512 where a key head has one query
// head (4096 tokens of ~300-token documents, 16 / 16 heads of 64: 53 us unsplit, 60 in two; 16 / 4 heads,
// 16384 tokens: 472 and 352)
int key_splits(int T, int Hq, int Hkv, int D) {
  const int kb = D == 64 ? KB1 : KB2;
  const int64_t blocks = (int64_t)((T + kb - 1) / kb) * Hkv;
  int n = 1;
  while (n < 16 && blocks * n < (Hq > Hkv ? 1024 : 512)) n *= 2;
  return n;
}
// Most shares, one per CU, or 0: shared heads of D = 128 have few key blocks, and shares beat splits
// once there is work enough to pay for the joining, unless there are blocks enough to keep the CUs
// evenly busy.  dQ, dK, dV in us by shares and by splits (means of three batches): 8001 tokens of ~900-token
// documents, 32 / 8 heads, 558 and 624; 16384 of ~1000, 8 / 1 heads, 381 and 547; 4096 in one, 16 / 4 heads, 319 and
// 391; 4096 of ~300, 16 / 4 heads, 150 and 162; but 4096 of ~300, 8 / 1 heads, 129 and 104; 512 in one 78 and 58; own
// heads, 8001 of ~900, 326 and 309.
int key_shares(int T, int Hq, int Hkv, int D) {
  const int64_t blocks = (int64_t)((T + KB2 - 1) / KB2) * Hkv;
  return D == 128 && Hq > Hkv && blocks < 1024 && (int64_t)T * Hq >= 60000 ? 256 : 0;
}

// At most one block for each CU: 64-row blocks whose wave pairs take half of the keys each, which halves the
// longest chain of tiles (2048 tokens in one, 16 heads of 64, forward 29.6 -> 24.7 us, of 128, 50 -> 42 and dQ + dK +
// dV 140 -> 120; 512 tokens 12.2 -> 11.5 and 17.0 -> 14.2).  With more blocks the CUs are full without it and the
// twice as many tiles cost more: 4096 of ~300, 16 heads of 64, 18.7 -> 20.2; 8000 of ~900, 32 heads of 128, 124 -> 151.
// Up to two for the forward of 128, whose half blocks need no spilled registers (4096 in one, 16 heads, 101 -> 96 us;
// 2048 of ~300, 32 heads, 32 -> 28; dQ + dK + dV of 2048 in one, 32 heads, 190 -> 197).
template <bool DQ>
int launch_qmajor(const PArgs& a, int D, hipStream_t s) {
  const unsigned n = (unsigned)((a.T + 127) / 128 * a.Hq);
  const bool half = n <= (D == 128 && !DQ ? 512 : 256);
  if (D == 64) {
    if (half) hipLaunchKernelGGL((packed_qmajor_kernel<64, DQ, true>), dim3(2 * n), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((packed_qmajor_kernel<64, DQ, false>), dim3(n), dim3(256), 0, s, a);
  } else {
    if (half) hipLaunchKernelGGL((packed_qmajor_kernel<128, DQ, true>), dim3(2 * n), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((packed_qmajor_kernel<128, DQ, false>), dim3(n), dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

bool bad_mat(const void* p, int ld, int width) {   // 16-B rows, tile offsets below 2^31 bytes
  return p == nullptr || ((uintptr_t)p & 15) || (ld & 7) || ld < width || ld > (1 << 22);
}
bool bad_shape(int T, int Hq, int Hkv, int D) {
  if (T <= 0 || T > (1 << 30) || Hq <= 0 || Hkv <= 0 || Hq % Hkv || (D != 64 && D != 128)) return true;
  return (int64_t)((T + 127) / 128) * Hq >= ((int64_t)1 << 31) || (int64_t)((T + 63) / 64) * (Hq / Hkv) >= 1 << 30;
}

}  // namespace

// Row table of a packed batch (packed_plan_kernel).  cu: n + 1 cumulative lengths (int64 when
// `wide`, else int32); start, end: int32 [T]; meta: int32 [4]; pos: int64 [T].
MX_EXPORT int mx_packed_plan(const void* cu, int wide, int n, int T, int* start, int* end, int* meta, void* pos,
                             int* order, hipStream_t s) {
  if (!cu || !start || !end || !meta || !pos || !order || n < 1 || T <= 0 || T > (1 << 30)) return hipErrorInvalidValue;
  const dim3 grid((T + 255) / 256);
  if (wide)
    hipLaunchKernelGGL((packed_plan_kernel<int64_t>), grid, dim3(256), 0, s, (const int64_t*)cu, n, T, start, end,
                       meta, (int64_t*)pos);
  else
    hipLaunchKernelGGL((packed_plan_kernel<int32_t>), grid, dim3(256), 0, s, (const int32_t*)cu, n, T, start, end,
                       meta, (int64_t*)pos);
  if (const int e = hipGetLastError(); e != hipSuccess) return e;
  hipLaunchKernelGGL(packed_order_kernel, dim3(1), dim3(1024), 0, s, T, start, end, meta, order);
  return hipGetLastError();
}

// int32 entries of `order` for T rows
MX_EXPORT int64_t mx_packed_order_len(int T) { return T > 0 ? order_base(T) + 2 * ((T + 255) / 256 + 1) : 0; }

// Q, K, V, O: bf16 [T] rows with strides ld*, head h at column h D.  lse: fp32 [Hq][T], base 2.
// fill: rows behind the last sequence get o = 0, lse = +inf; else they are left as they are.
MX_EXPORT int mx_packed_attn_fwd(const void* q, const void* k, const void* v, int ldq, int ldk, int ldv, void* o,
                                 int ldo, float* lse, const int* start, const int* end, const int* meta, const int* order,
                                 int T, int Hq, int Hkv, int D, float scale, int fill, hipStream_t s) {
  if (bad_shape(T, Hq, Hkv, D) || bad_mat(q, ldq, Hq * D) || bad_mat(k, ldk, Hkv * D) || bad_mat(v, ldv, Hkv * D) ||
      bad_mat(o, ldo, Hq * D) || !lse || !start || !end || !meta || !order || !(scale > 0.f))
    return hipErrorInvalidValue;
  PArgs a{};
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
  a.out = (uint16_t*)o;
  a.lse = lse;
  a.start = start; a.end = end; a.meta = meta; a.order = order;
  a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldout = ldo;
  a.T = T; a.Hq = Hq; a.Hkv = Hkv;
  a.c = scale * 1.4426950408889634f;
  a.scale = scale;
  a.fill = fill;
  return launch_qmajor<false>(a, D, s);
}

// splits of a key block of `items` (query head, query tile) pairs in a batch of `tiles` query tiles; 0: none (shares)
MX_EXPORT int mx_packed_block_splits(int T, int Hq, int Hkv, int D, int64_t tiles, int items) {
  if (bad_shape(T, Hq, Hkv, D) || tiles < 0 || items < 1 || key_shares(T, Hq, Hkv, D)) return 0;
  return split_count(tiles, Hq, D, key_splits(T, Hq, Hkv, D), items);
}

// floats of `part` (0: none)
MX_EXPORT int64_t mx_packed_attn_bwd_floats(int T, int Hq, int Hkv, int D) {
  if (bad_shape(T, Hq, Hkv, D)) return 0;
  if (const int n = key_shares(T, Hq, Hkv, D)) return (int64_t)n * 2 * 2 * KB2 * D;
  const int n = key_splits(T, Hq, Hkv, D);
  return n > 1 ? (int64_t)n * 2 * T * Hkv * D : 0;
}

// stats: fp32 [2][Hq][T] workspace (written by the dQ kernel, read by the dK / dV kernel).
MX_EXPORT int mx_packed_attn_bwd(const void* q, const void* k, const void* v, int ldq, int ldk, int ldv,
                                 const void* o, int ldo, const void* dout, int lddo, const float* lse, float* stats,
                                 void* dq, int lddq, void* dk, void* dv, int lddk, int lddv, const int* start,
                                 const int* end, const int* meta, const int* order, int T, int Hq, int Hkv, int D,
                                 float scale, int fill, float* part, int64_t part_floats, hipStream_t s) {
  if (bad_shape(T, Hq, Hkv, D) || bad_mat(q, ldq, Hq * D) || bad_mat(k, ldk, Hkv * D) || bad_mat(v, ldv, Hkv * D) ||
      bad_mat(o, ldo, Hq * D) || bad_mat(dout, lddo, Hq * D) || bad_mat(dq, lddq, Hq * D) ||
      bad_mat(dk, lddk, Hkv * D) || bad_mat(dv, lddv, Hkv * D) || !lse || !stats || ((uintptr_t)stats & 3) || !start ||
      !end || !meta || !order || !(scale > 0.f))
    return hipErrorInvalidValue;
  PArgs a{};
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
  a.o = (const uint16_t*)o; a.dout = (const uint16_t*)dout;
  a.out = (uint16_t*)dq; a.dk = (uint16_t*)dk; a.dv = (uint16_t*)dv;
  a.lse = const_cast<float*>(lse);
  a.nlse = stats;
  a.delta = stats + (size_t)Hq * T;
  a.start = start; a.end = end; a.meta = meta; a.order = order;
  a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo; a.lddo = lddo; a.ldout = lddq; a.lddk = lddk; a.lddv = lddv;
  a.T = T; a.Hq = Hq; a.Hkv = Hkv;
  a.c = scale * 1.4426950408889634f;
  a.scale = scale;
  a.fill = fill;
  a.nsplit = key_splits(T, Hq, Hkv, D);
  a.nshare = key_shares(T, Hq, Hkv, D);
  a.before = reinterpret_cast<const int64_t*>(order + order_base(T));
  a.part = part;
  if (const int64_t n = mx_packed_attn_bwd_floats(T, Hq, Hkv, D); n && (!part || ((uintptr_t)part & 15) || part_floats < n))
    return hipErrorInvalidValue;
  if (const int e = launch_qmajor<true>(a, D, s); e != hipSuccess) return e;   // (dK / dV read its statistics)
  const unsigned nb = (unsigned)((T + 127) / 128), nk = (unsigned)((T + KB2 - 1) / KB2);
  a.order = order + (D == 64 ? nb : 2 * nb);
  if (D == 64)
    hipLaunchKernelGGL((packed_kmajor_kernel<64>), dim3(nb * Hkv * a.nsplit), dim3(256), 0, s, a);
  else if (a.nshare)
    hipLaunchKernelGGL((packed_kmajor2_kernel<128, true>), dim3(a.nshare), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((packed_kmajor2_kernel<128, false>), dim3(nk * Hkv * a.nsplit), dim3(256), 0, s, a);
  if (const int e = hipGetLastError(); e != hipSuccess || (!a.nshare && a.nsplit == 1)) return e;
  const dim3 grid((unsigned)(((int64_t)T * Hkv * (D / 4) + 255) / 256));
  if (a.nshare) hipLaunchKernelGGL(packed_join2_kernel, dim3((a.nshare - 1) * JOIN), dim3(256), 0, s, a);
  else if (D == 64) hipLaunchKernelGGL((packed_join_kernel<64>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((packed_join_kernel<128>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}
