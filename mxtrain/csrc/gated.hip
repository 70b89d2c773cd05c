// Gated feed-forward block for gfx950 (bf16 in and out, fp32 accumulate):
//
//   pre = x W1^T + b1 = [a | b],   h = act(a) b,   y = h W2^T + b2           act: SiLU or tanh-GeLU
//   dh = dy W2,  da = dh b act'(a),  db = dh act(a),  dx = [da | db] W1,
//   dW1 = [da | db]^T x,  dW2 = dy^T h,  bias gradients = column sums of [da | db] and dy
//
// The gate and the up projection are ONE matrix product: a tile's weight image holds the same
// columns of both halves of W1, dealt so that a wave ends with a and b of the same elements, and
// the epilogue adds the biases, applies the activation and writes h (and pre, for training)
// without another pass.  dh never exists in memory: the epilogue of dy W2 reads a and b and
// writes da, db and the column partials of the bias gradient.
//
// Rounded to bf16 on the way, once each from fp32: pre and h (what backward is given; fp32 would double the
// largest tensors of the block) and [da | db] (a matrix operand of dx and dW1; its column sums are taken
// before the rounding).  Splits, partial and column sums stay fp32.
//
// All six products share one kernel.  Operands are staged by LDS-DMA through buffer resources:
// what lies past a tile's rows reads zero, so any number of tokens and any feature count that is a
// multiple of 8 is taken without padding.  16 x 16 x 32 MFMA with the weight (column) operand
// first, so that a lane holds 4 consecutive columns of a row.
//
// Large products (4096 x 4096 x 10880, forward and backward in 2.95 ms) run at 0.74 PFLOP/s (gate gradient) to 1.15
// (dx): gate 765 us, down 325, where library products of these shapes without an epilogue take 618 and 231.
// At 256 x 256 one workgroup holds a CU, so an epilogue's memory traffic (178 MB in and 178 out for the gate
// gradient) runs beside no products; and the K-contiguous loop waits for more than its LDS reads, or it would
// match the library's.  Short ones (4096 x 1024 x 2688: 0.27 ms) are bound by rounds of workgroups that fill and
// drain for 16 - 84 steps.
#include "gemm_common.h"

#include <type_traits>

using namespace mx;
using namespace mx::gemm;

namespace {

struct GArgs {
  const uint16_t* a;     // AKC: [M][lda] (K contiguous), else [K][lda]
  const uint16_t* b;     // BKC: [N][ldb] (K contiguous), else [K][ldb]
  uint16_t* c;           // [M][ldc]
  uint16_t* aux;         // EPI 2: pre out or null; EPI 3: pre in; [M][2 N]
  uint16_t* grad;        // EPI 3: [da | db] out [M][2 N]
  const uint16_t* bias;  // EPI 1: [N]; EPI 2: [2 N] or null
  float* part;           // EPI 3: column partials [row blocks][2 N] or null
  int lda, ldb, ldc;
  int M, N, K;
  int tiles_m, tiles_n, gm;
  int act, accumulate;
  int splits, nks;       // EPI 4: K-steps per split
  // EPI 5: the second product (its K and accumulate are the first's)
  const uint16_t *a2, *b2;
  uint16_t* c2;
  int lda2, ldb2, ldc2, M2, N2, tiles_m2, tiles_n2;
  int wgs1;              // workgroups of the first
};

__device__ __forceinline__ float act_fwd(int act, float x) {
  // sigmoid forms: x s(x) for SiLU, x s(2 k0 x (1 + k1 x^2)) for the tanh GeLU
  if (act == 0) return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
  return gelu_tanh(x);
}
// act(x) and act'(x).  Beyond |x| = 100 the sigmoid is 0 or 1 in fp32 and the slope with it; clamping
// there keeps x^2 from overflowing (a NaN stays one)
__device__ __forceinline__ void act_both(int act, float x, float& y, float& d) {
  const float xc = fminf(fmaxf(x, -100.f), 100.f);
  if (act == 0) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * xc));
    y = x * s;
    d = s * __builtin_fmaf(xc, 1.f - s, 1.f);
  } else {
    y = gelu_tanh(x);
    d = gelu_tanh_grad(xc);
  }
  d = x == x ? d : x;
}

// geometry: WM x WN waves of FM x FN 16 x 16 accumulators, BKT-deep steps, NSLOT-slot ring
template <bool AKC, bool BKC, int WM, int WN, int FM, int FN, int BKT, int NSLOT>
struct Geo {
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int BM = 16 * FM * WM, BN = 16 * FN * WN;
  static constexpr int RA = AKC ? BKT * 2 : BM * 2, RB = BKC ? BKT * 2 : BN * 2;   // image row bytes
  static constexpr int IA = AKC ? BM * RA : BKT * RA, IB = BKC ? BN * RB : BKT * RB;
  static constexpr int PA = IA / 1024 / NW, PB = IB / 1024 / NW;                   // DMA pieces per wave
  static constexpr int SLOT = IA + IB, LDS = NSLOT * SLOT;
  static_assert(PA * NW * 1024 == IA && PB * NW * 1024 == IB, "DMA pieces per wave");
  static_assert(BKT == 32 || BKT == 64, "K-step");
  static_assert((AKC || BM % 128 == 0) && (BKC || BN % 128 == 0), "K-major images have 256-B rows");
  static_assert(LDS <= 160 * 1024, "LDS");
};

// swizzle of the 16-B chunks of a K-contiguous image row (128-B rows: chunk ^ (row & 7); 64-B rows:
// four rows share a 256-B bank row) -- on the DMA source and on the fragment read
template <int RA>
__device__ __forceinline__ int kc_swz(int r) {
  if constexpr (RA == 128) return r & 7;
  else return (0x78 >> (2 * ((r >> 2) & 3))) & 3;
}

template <int N, int I = 0, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, I + 1>(f);
  }
}

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
// resource of `rows` rows of `cols` values at base (row stride ld); nothing if rows <= 0
__device__ __forceinline__ i32x4_t tile_rsrc(const uint16_t* base, int rows, int cols, int ld) {
  const uint64_t p = (uint64_t)(uintptr_t)base;
  const uint32_t n = rows > 0 && cols > 0 ? ((uint32_t)(rows - 1) * (uint32_t)ld + (uint32_t)cols) * 2u : 0u;
  return i32x4_t{uni((int)(uint32_t)p), uni((int)(uint32_t)(p >> 32)), uni((int)n), 0x00020000};
}

// EPI 0: C (+)= acc   1: C = acc + bias   2: gate (two column halves)   3: gate gradient
//     4: fp32 partial of one K range into part[split][M][N] (joined by gated_join_kernel)
//     5: 0 of two products in one launch, whose rounds of workgroups would each end half empty
template <bool AKC, bool BKC, int WM, int WN, int FM, int FN, int BKT, int NSLOT, int MINB, int KIND>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(MINB, MINB))) void gated_gemm_kernel(
    const GArgs g0) {
  constexpr int EPI = KIND == 5 ? 0 : KIND;
  using Gm = Geo<AKC, BKC, WM, WN, FM, FN, BKT, NSLOT>;
  constexpr int BM = Gm::BM, BN = Gm::BN, RA = Gm::RA, RB = Gm::RB, IA = Gm::IA;
  constexpr int PA = Gm::PA, PB = Gm::PB, SLOT = Gm::SLOT, PER = PA + PB;
  constexpr bool DUAL = EPI == 2;
  constexpr int BNO = DUAL ? BN / 2 : BN;          // output columns of a tile
  static_assert(FN % (DUAL ? 4 : 2) == 0, "stores pair subtiles");
  __shared__ __attribute__((aligned(1024))) char smem[Gm::LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int G = lane >> 4, i = lane & 15;
  const int wm = wave / WN, wn = wave % WN;
  // XCD-contiguous order over groups of gm row tiles
  // (the splits of a tile are adjacent ids)
  int wgs = xcd_remap(blockIdx.x, gridDim.x);
  GArgs g = g0;
  if constexpr (KIND == 5)
    if (wgs >= g0.wgs1) {
      wgs -= g0.wgs1;
      g.a = g0.a2; g.b = g0.b2; g.c = g0.c2;
      g.lda = g0.lda2; g.ldb = g0.ldb2; g.ldc = g0.ldc2;
      g.M = g0.M2; g.N = g0.N2;
      g.tiles_m = g0.tiles_m2; g.tiles_n = g0.tiles_n2;
    }
  const int split = EPI == 4 ? wgs % g.splits : 0, wg = EPI == 4 ? wgs / g.splits : wgs;
  const int per = g.gm * g.tiles_n, grp = wg / per, rem = wg - grp * per;
  const int gmr = min(g.gm, g.tiles_m - grp * g.gm);   // (the last group may be smaller)
  const int tm = grp * g.gm + rem % gmr, tn = rem / gmr;
  const int m0 = tm * BM, n0 = tn * BNO;
  const int nk_all = (g.K + BKT - 1) / BKT;
  const int kt0 = EPI == 4 ? split * g.nks : 0;     // first K-step
  const int nk = EPI == 4 ? min(g.nks, nk_all - kt0) : nk_all;
  const int K = g.K;

  // per-lane byte offsets of the DMA pieces inside one step's image source
  uint32_t voA[PA], voB[PB];
  int kcA = 0, kcB = 0;                             // first k of the lane's chunk (K-contiguous images)
#pragma unroll
  for (int j = 0; j < PA; ++j) {
    if constexpr (AKC) {
      constexpr int LPR = RA / 16;
      const int row = (PA * wave + j) * (1024 / RA) + lane / LPR;
      kcA = 8 * ((lane % LPR) ^ kc_swz<RA>(row));   // (the same for every piece)
      voA[j] = (uint32_t)(row * g.lda + kcA) * 2u;
    } else {
      constexpr int CB = RA / 16;
      const int k = (PA * wave + j) * (1024 / RA) + lane / CB;
      voA[j] = (uint32_t)(k * g.lda + 8 * pchunk(k, lane % CB)) * 2u;
    }
  }
  // gate tiles: image row r of a wave's 16 FN rows: the first half are gate columns, the second the
  // same columns of the up half
  constexpr int HB = 8 * FN;
#pragma unroll
  for (int j = 0; j < PB; ++j) {
    if constexpr (BKC) {
      constexpr int LPR = RB / 16;
      int row = (PB * wave + j) * (1024 / RB) + lane / LPR;
      kcB = 8 * ((lane % LPR) ^ kc_swz<RB>(row));
      if constexpr (DUAL) row = (row / (2 * HB)) * HB + row % HB;
      voB[j] = (uint32_t)(row * g.ldb + kcB) * 2u;
    } else {
      constexpr int CB = RB / 16;
      const int k = (PB * wave + j) * (1024 / RB) + lane / CB;
      voB[j] = (uint32_t)(k * g.ldb + 8 * pchunk(k, lane % CB)) * 2u;
    }
  }
  const int rowsA = min(BM, g.M - m0), rowsB = min(BNO, g.N - n0);
  const uint32_t lds0 = lds_addr(smem);
  const uint32_t ldsA = uni(lds0 + PA * wave * 1024), ldsB = uni(lds0 + IA + PB * wave * 1024);
  auto piece = [&](int slot, int it, int j) __attribute__((always_inline)) {
    const int k0 = (kt0 + it) * BKT;
    if (j < PA) {
      i32x4_t r;
      uint32_t vo = voA[j];
      if constexpr (AKC) {
        r = tile_rsrc(g.a + (size_t)m0 * g.lda + k0, rowsA, K - k0, g.lda);
        if (k0 + BKT > K) vo = kcA < K - k0 ? vo : kOOB;     // the chunks past K
      } else {
        r = tile_rsrc(g.a + (size_t)k0 * g.lda + m0, min(BKT, K - k0), rowsA, g.lda);
      }
      dma16_buf(r, vo, ldsA + slot * SLOT + j * 1024);
    } else {
      i32x4_t r;
      uint32_t vo = voB[j - PA];
      if constexpr (BKC) {
        const uint16_t* base = g.b + (size_t)n0 * g.ldb + k0;
        if constexpr (DUAL) {
          const int row0 = (PB * wave + j - PA) * (1024 / RB);
          if (row0 % (2 * HB) >= HB) base += (size_t)g.N * g.ldb;
        }
        r = tile_rsrc(base, rowsB, K - k0, g.ldb);
        if (k0 + BKT > K) vo = kcB < K - k0 ? vo : kOOB;
      } else {
        r = tile_rsrc(g.b + (size_t)k0 * g.ldb + n0, min(BKT, K - k0), rowsB, g.ldb);
      }
      dma16_buf(r, vo, ldsB + slot * SLOT + (j - PA) * 1024);
    }
  };

  // fragment offsets: lane (G, i) holds row i of a 16-row subtile, k 8G .. 8G + 7 (+ 32 kk)
  int offA[FM], offB[FN], cA[BKT / 32], cB[BKT / 32];
  const int krow = 8 * G + (i >> 2);
#pragma unroll
  for (int kk = 0; kk < BKT / 32; ++kk) {
    cA[kk] = AKC ? 16 * ((4 * kk + G) ^ kc_swz<AKC ? RA : 128>(i)) : 32 * RA * kk;
    cB[kk] = BKC ? 16 * ((4 * kk + G) ^ kc_swz<BKC ? RB : 128>(i)) : 32 * RB * kk;
  }
#pragma unroll
  for (int s = 0; s < FM; ++s)
    offA[s] = AKC ? (16 * (FM * wm + s) + i) * RA
                  : krow * RA + ((((FM * wm + s) ^ gsw(krow)) << 1) | ((i & 3) >> 1)) * 16 + (i & 1) * 8;
#pragma unroll
  for (int u = 0; u < FN; ++u)
    offB[u] = BKC ? (16 * (FN * wn + u) + i) * RB
                  : krow * RB + ((((FN * wn + u) ^ gsw(krow)) << 1) | ((i & 3) >> 1)) * 16 + (i & 1) * 8;

  f32x4 acc[FM][FN];
#pragma unroll
  for (int s = 0; s < FM; ++s)
#pragma unroll
    for (int u = 0; u < FN; ++u) acc[s][u] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int q = 0; q < NSLOT - 1; ++q)
    if (q < nk) {
#pragma unroll
      for (int j = 0; j < PER; ++j) piece(q, q, j);
    }
  constexpr int NS = (BKT / 32) * FN;
  constexpr int SPREAD = NS / 2 >= PER ? NS / 2 : NS;   // the next step's DMA issues spread over the MFMAs
  for (int it0 = 0; it0 < nk; it0 += NSLOT) {
    static_for<NSLOT>([&](auto qc) __attribute__((always_inline)) {
      constexpr int q = decltype(qc)::value;
      const int it = it0 + q;
      if (it >= nk) return;
      // retire step it's pieces (later steps stay in flight), then one barrier: every wave's pieces
      // have landed and every wave is done reading step it - 1's slot
      const int later = nk - 1 - it;
      if (NSLOT >= 4 && later >= 2) vm_wait<(NSLOT >= 4 ? 2 : 0) * PER>();
      else if (NSLOT >= 3 && later >= 1) vm_wait<(NSLOT >= 3 ? 1 : 0) * PER>();
      else vm_wait<0>();
      __builtin_amdgcn_s_barrier();
      const bool fetch = it + NSLOT - 1 < nk;
      constexpr int ns = (q + NSLOT - 1) % NSLOT;
      const char* As = smem + q * SLOT;
      const char* Bs = As + IA;
#pragma unroll
      for (int kk = 0; kk < BKT / 32; ++kk) {
        bf16x8 x[FM];
#pragma unroll
        for (int s = 0; s < FM; ++s) {
          if constexpr (AKC) x[s] = lds_read8(As, offA[s] + cA[kk]);
          else x[s] = cat(tr_read(As, offA[s] + cA[kk]), tr_read(As, offA[s] + cA[kk] + 4 * RA));
        }
#pragma unroll
        for (int u = 0; u < FN; ++u) {
          bf16x8 w;
          if constexpr (BKC) w = lds_read8(Bs, offB[u] + cB[kk]);
          else w = cat(tr_read(Bs, offB[u] + cB[kk]), tr_read(Bs, offB[u] + cB[kk] + 4 * RB));
          const int qq = kk * FN + u;
#pragma unroll
          for (int j = 0; j < PER; ++j)
            if (qq < SPREAD && j * SPREAD / PER == qq && fetch) piece(ns, it + NSLOT - 1, j);
#pragma unroll
          for (int s = 0; s < FM; ++s) acc[s][u] = mfma16(w, x[s], acc[s][u]);
        }
      }
    });
  }

  // ---- epilogue: lane holds C[m][n + e], m = m0 + 16 (FM wm + s) + i, n = .. + 16 u + 4 G; pairs of
  // subtiles are re-dealt so that a lane stores 8 consecutive columns (16 B)
  if constexpr (EPI == 4) {
    float* P = g.part + (size_t)split * g.M * g.N;
#pragma unroll
    for (int s = 0; s < FM; ++s) {
      const int m = m0 + 16 * (FM * wm + s) + i;
#pragma unroll
      for (int u = 0; u < FN; ++u) {
        const int col = n0 + 16 * (FN * wn + u) + 4 * G;
        if (m < g.M && col < g.N)
          *reinterpret_cast<float4*>(P + (size_t)m * g.N + col) =
              make_float4(acc[s][u][0], acc[s][u][1], acc[s][u][2], acc[s][u][3]);
      }
    }
    return;
  }
  constexpr int FO = DUAL ? FN / 2 : FN;
  const int colw = n0 + 16 * FO * wn, N = g.N;
  const int mrow = m0 + 16 * FM * wm + i;
  float bias[FN][4];
#pragma unroll
  for (int u = 0; u < FN; ++u) {
    const int col = colw + 16 * (u % FO) + 4 * G;
    uint2 v = make_uint2(0u, 0u);
    if ((EPI == 1 || EPI == 2) && g.bias && col < N)
      v = *reinterpret_cast<const uint2*>(g.bias + col + (u >= FO ? N : 0));
    bias[u][0] = lo_bf(v.x); bias[u][1] = hi_bf(v.x); bias[u][2] = lo_bf(v.y); bias[u][3] = hi_bf(v.y);
  }
  float csum[EPI == 3 ? 2 : 1][FO][4];
#pragma unroll
  for (int u = 0; u < FO; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) csum[0][u][e] = csum[EPI == 3 ? 1 : 0][u][e] = 0.f;
  auto put = [&](uint16_t* p, uint32_t (&v)[2][2], bool ok) __attribute__((always_inline)) {
    deal(v[0][0], v[0][1], v[1][0], v[1][1]);
    if (ok) *reinterpret_cast<uint4*>(p) = make_uint4(v[0][0], v[0][1], v[1][0], v[1][1]);
  };
  auto get = [&](const uint4& x, uint32_t (&v)[2][2]) __attribute__((always_inline)) {
    v[0][0] = x.x; v[0][1] = x.y; v[1][0] = x.z; v[1][1] = x.w;
    undeal(v[0][0], v[0][1], v[1][0], v[1][1]);
  };
  // what the epilogue reads (pre; C when it accumulates) is fetched a row group ahead: one group's
  // loads waited for in turn were 30 us of a 60 us launch (4096 x 1024 x 2688, 256 x 256 tiles)
  constexpr int NR = EPI == 3 ? 2 : EPI == 0 ? 1 : 0;
  uint4 pf[NR ? NR : 1][FO / 2];
  auto fetch_row = [&](int s) __attribute__((always_inline)) {
    const int m = mrow + 16 * s;
#pragma unroll
    for (int up = 0; up < FO / 2; ++up) {
      const int col = colw + 32 * up + 8 * G;
#pragma unroll
      for (int h = 0; h < NR; ++h) {
        pf[h][up] = make_uint4(0u, 0u, 0u, 0u);
        if (m < g.M && col < N && (EPI == 3 || g.accumulate))
          pf[h][up] = *reinterpret_cast<const uint4*>(EPI == 3 ? g.aux + (size_t)m * 2 * N + h * N + col
                                                               : g.c + (size_t)m * g.ldc + col);
      }
    }
  };
  fetch_row(0);
#pragma unroll
  for (int s = 0; s < FM; ++s) {
    const int m = mrow + 16 * s;
    uint4 cur[NR ? NR : 1][FO / 2];
#pragma unroll
    for (int up = 0; up < FO / 2; ++up)
#pragma unroll
      for (int h = 0; h < NR; ++h) cur[h][up] = pf[h][up];
    if (s + 1 < FM) fetch_row(s + 1);
#pragma unroll
    for (int up = 0; up < FO / 2; ++up) {
      const int col = colw + 32 * up + 8 * G;       // the lane's 8 columns after the re-deal
      const bool ok = m < g.M && col < N;
      uint32_t c[2][2], pa[2][2], pb[2][2];
      if constexpr (NR > 0) get(cur[0][up], pa);
      if constexpr (NR > 1) get(cur[NR - 1][up], pb);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int u = 2 * up + hf;
        float v[4], w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[s][u][e] + bias[u][e];
        if constexpr (EPI == 0) {   // (zeros unless it accumulates)
          v[0] += lo_bf(pa[hf][0]); v[1] += hi_bf(pa[hf][0]); v[2] += lo_bf(pa[hf][1]); v[3] += hi_bf(pa[hf][1]);
        }
        if constexpr (EPI == 2) {
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = acc[s][u + FO][e] + bias[u + FO][e];
          pa[hf][0] = pack2(v[0], v[1]); pa[hf][1] = pack2(v[2], v[3]);
          pb[hf][0] = pack2(w[0], w[1]); pb[hf][1] = pack2(w[2], w[3]);
          // (from the unrounded pre-activations; backward differentiates at the bf16 ones it keeps)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = act_fwd(g.act, v[e]) * w[e];
        }
        if constexpr (EPI == 3) {
          const float a[4] = {lo_bf(pa[hf][0]), hi_bf(pa[hf][0]), lo_bf(pa[hf][1]), hi_bf(pa[hf][1])};
          const float b[4] = {lo_bf(pb[hf][0]), hi_bf(pb[hf][0]), lo_bf(pb[hf][1]), hi_bf(pb[hf][1])};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y, d;
            act_both(g.act, a[e], y, d);
            w[e] = v[e] * y;
            v[e] = v[e] * b[e] * d;
            csum[0][u][e] += v[e];
            csum[1][u][e] += w[e];
          }
          pb[hf][0] = pack2(w[0], w[1]); pb[hf][1] = pack2(w[2], w[3]);
        }
        c[hf][0] = pack2(v[0], v[1]); c[hf][1] = pack2(v[2], v[3]);
      }
      if constexpr (EPI == 2) {
        if (g.aux) {
          put(g.aux + (size_t)m * 2 * N + col, pa, ok);
          put(g.aux + (size_t)m * 2 * N + N + col, pb, ok);
        }
      }
      if constexpr (EPI == 3) {
        put(g.grad + (size_t)m * 2 * N + col, c, ok);
        put(g.grad + (size_t)m * 2 * N + N + col, pb, ok);
      } else {
        put(g.c + (size_t)m * g.ldc + col, c, ok);
      }
    }
  }
  if constexpr (EPI == 3) {
    if (g.part) {   // column sums of the wave's 16 FM rows (rows past M added nothing)
      float* prow = g.part + (size_t)(tm * WM + wm) * 2 * N;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < FO; ++u) {
          float t[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) t[e] = row_sum16(csum[h][u][e]);
          const int col = colw + 16 * u + 4 * G;
          if (i == 0 && col < N)
            *reinterpret_cast<float4*>(prow + h * N + col) = make_float4(t[0], t[1], t[2], t[3]);
        }
    }
  }
}

// ---- few tokens (a decoding step): y^T = W x^T with the weight rows streamed once from memory.
// A workgroup takes 16 output columns (of both halves for the gate) and its NW waves split K, so
// that even a 1024-column product has hundreds of waves with all their loads in flight; no LDS on
// the way in (a weight is used once), partial sums meet in LDS.  Lane (G, i) loads row i, k 8G ..
// 8G + 7 of a 16 x 32 block; NG groups of 16 tokens.  Bound by memory latency: 1024 x 2688, one token,
// 16.5 MB of weights in 5.1 (gate) + 4.3 us, 1.8 TB/s.
template <int NG, bool DUAL, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW / 4, NW / 4))) void gated_few_kernel(const GArgs g) {
  constexpr int NH = DUAL ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float4 red[NW][NH * NG][64];
  const int lane = threadIdx.x & 63, w = uni(threadIdx.x >> 6), G = lane >> 4, i = lane & 15;
  const int n0 = blockIdx.x * 16, N = g.N, K = g.K, M = g.M;
  const int steps = (K + 31) / 32, per = (steps + NW - 1) / NW;
  const int s0 = w * per, s1 = min(steps, s0 + per);
  const uint16_t* wp[NH];
#pragma unroll
  for (int h = 0; h < NH; ++h) wp[h] = g.b + (size_t)(min(n0 + i, N - 1) + h * N) * g.ldb;
  const uint16_t* xp[NG];
#pragma unroll
  for (int t = 0; t < NG; ++t) xp[t] = g.a + (size_t)min(16 * t + i, M - 1) * g.lda;
  f32x4 acc[NH][NG];
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int t = 0; t < NG; ++t) acc[h][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto load = [&](const uint16_t* p, int k) __attribute__((always_inline)) {   // zeros past K
    const uint4 v = *reinterpret_cast<const uint4*>(p + (k < K ? k : 0));
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    return __builtin_bit_cast(bf16x8, k < K ? v : z);
  };
  auto block = [&](int s, auto unc) __attribute__((always_inline)) {   // UN steps, every load in flight
    constexpr int UN = decltype(unc)::value;
    bf16x8 a[UN][NH], b[UN][NG];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int k = 32 * (s + u) + 8 * G;
#pragma unroll
      for (int h = 0; h < NH; ++h) a[u][h] = load(wp[h], k);
#pragma unroll
      for (int t = 0; t < NG; ++t) b[u][t] = load(xp[t], k);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int t = 0; t < NG; ++t) acc[h][t] = mfma16(a[u][h], b[u][t], acc[h][t]);
  };
  int s = s0;
  for (; s + 4 <= s1; s += 4) block(s, std::integral_constant<int, 4>{});
  if (s + 2 <= s1) {
    block(s, std::integral_constant<int, 2>{});
    s += 2;
  }
  if (s < s1) block(s, std::integral_constant<int, 1>{});
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int t = 0; t < NG; ++t)
      red[w][h * NG + t][lane] = make_float4(acc[h][t][0], acc[h][t][1], acc[h][t][2], acc[h][t][3]);
  __syncthreads();
  // wave t finishes token group t: lane holds columns n0 + 4 G .. + 3 of token 16 t + i
  if (w >= NG) return;
  const int m = 16 * w + i, col = n0 + 4 * G;
  float v[NH][4];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[h][e] = 0.f;
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      const float4 x = red[q][h * NG + w][lane];
      v[h][0] += x.x; v[h][1] += x.y; v[h][2] += x.z; v[h][3] += x.w;
    }
  }
  if (m >= M || col >= N) return;
  if (g.bias) {
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const uint2 x = *reinterpret_cast<const uint2*>(g.bias + h * N + col);
      v[h][0] += lo_bf(x.x); v[h][1] += hi_bf(x.x); v[h][2] += lo_bf(x.y); v[h][3] += hi_bf(x.y);
    }
  }
  if constexpr (DUAL) {
    if (g.aux) {
#pragma unroll
      for (int h = 0; h < NH; ++h)
        *reinterpret_cast<uint2*>(g.aux + (size_t)m * 2 * N + h * N + col) =
            make_uint2(pack2(v[h][0], v[h][1]), pack2(v[h][2], v[h][3]));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[0][e] = act_fwd(g.act, v[0][e]) * v[NH - 1][e];
  }
  *reinterpret_cast<uint2*>(g.c + (size_t)m * g.ldc + col) =
      make_uint2(pack2(v[0][0], v[0][1]), pack2(v[0][2], v[0][3]));
}
// Up to 16 tokens always; up to 64 while the products are small, for every further group of 16 reads x and
// multiplies again beside the one read of the weights, where a tile of 128 rows does so for nothing (block
// without `pre`, few-token form and tiles, us: 1 token 1024 x 2688 9.4 and 23, 64 tokens 22.5 and 24.5;
// 2048 x 5504: 16 tokens 28 and 34, 32 tokens 36 and 35, 64 tokens 53 and 36; 4096 x 10880: 1 token 50 and
// 62, 16 tokens 62 and 62, 64 tokens 130 and 65).
bool few_tokens(const GArgs& g) {
  return g.M <= 16 || (g.M <= 64 && (int64_t)g.M * g.K * g.N <= 320000000);
}
template <bool DUAL>
int run_few(const GArgs& g, hipStream_t s) {
  const dim3 grid((g.N + 15) / 16);
  constexpr int NW = DUAL ? 8 : 16;
  if (g.M <= 16) hipLaunchKernelGGL((gated_few_kernel<1, DUAL, NW>), grid, dim3(64 * NW), 0, s, g);
  else if (g.M <= 32) hipLaunchKernelGGL((gated_few_kernel<2, DUAL, NW>), grid, dim3(64 * NW), 0, s, g);
  else hipLaunchKernelGGL((gated_few_kernel<4, DUAL, NW>), grid, dim3(64 * NW), 0, s, g);
  return hipGetLastError();
}

// sums the partials of EPI 4 in order: C = sum (+ bias) (+ C)
__global__ __launch_bounds__(256) void gated_join_kernel(const GArgs g) {
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int nv = g.N / 8;
  if (v >= (int64_t)g.M * nv) return;
  const int64_t m = v / nv;
  const int n = (int)(v - m * nv) * 8;
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < g.splits; ++k) {
    const float4* p = reinterpret_cast<const float4*>(g.part + ((size_t)k * g.M + m) * g.N + n);
    const float4 x = p[0], y = p[1];
    o[0] += x.x; o[1] += x.y; o[2] += x.z; o[3] += x.w;
    o[4] += y.x; o[5] += y.y; o[6] += y.z; o[7] += y.w;
  }
  uint16_t* c = g.c + (size_t)m * g.ldc + n;
  float x[8];
  if (g.bias) {
    unpack8(*reinterpret_cast<const uint4*>(g.bias + n), x);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] += x[j];
  }
  if (g.accumulate) {
    unpack8(*reinterpret_cast<const uint4*>(c), x);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] += x[j];
  }
  *reinterpret_cast<uint4*>(c) = pack8(o);
}

template <bool AKC, bool BKC, int WM, int WN, int FM, int FN, int BKT, int NSLOT, int EPI>
int launch(GArgs g, hipStream_t s) {
  using Gm = Geo<AKC, BKC, WM, WN, FM, FN, BKT, NSLOT>;
  const int bn = EPI == 2 ? Gm::BN / 2 : Gm::BN;
  g.tiles_m = (g.M + Gm::BM - 1) / Gm::BM;
  g.tiles_n = (g.N + bn - 1) / bn;
  g.gm = 8;
  const int nk = (g.K + BKT - 1) / BKT;
  g.nks = (nk + g.splits - 1) / g.splits;
  g.splits = (nk + g.nks - 1) / g.nks;              // (no empty split)
  int64_t grid = (int64_t)g.tiles_m * g.tiles_n * g.splits;
  if (EPI == 5) {
    g.wgs1 = (int)min(grid, (int64_t)INT32_MAX);
    g.tiles_m2 = (g.M2 + Gm::BM - 1) / Gm::BM;
    g.tiles_n2 = (g.N2 + Gm::BN - 1) / Gm::BN;
    grid += (int64_t)g.tiles_m2 * g.tiles_n2;
  }
  if (grid >= ((int64_t)1 << 31)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((gated_gemm_kernel<AKC, BKC, WM, WN, FM, FN, BKT, NSLOT, 2, EPI>), dim3((unsigned)grid),
                     dim3(Gm::NT), 0, s, g);
  if (EPI == 4) {
    if (const int e = hipGetLastError(); e != hipSuccess) return e;
    const int64_t vecs = (int64_t)g.M * (g.N / 8);
    hipLaunchKernelGGL(gated_join_kernel, dim3((unsigned)((vecs + 255) / 256)), dim3(256), 0, s, g);
  }
  return hipGetLastError();
}

// tiles: rows, columns of the product (the gate's two halves together), column-partial rows per tile
struct Tile {
  int bm, bn, wm;
};
constexpr Tile kTiles[] = {
    {128, 128, 2},   // 0: 4 waves of 64 x 64, 64-deep steps, 2 slots, two workgroups per CU
    {256, 256, 2},   // 1: 8 waves of 128 x 64, 32-deep steps, 4 slots
    {128, 128, 4},   // 2: 8 waves of 32 x 64, 64-deep steps, 4 slots
    {256, 128, 4},   // 3: 8 waves of 64 x 64, 64-deep steps, 3 slots
    {64, 128, 2},    // 4: 4 waves of 32 x 64, 64-deep steps, 3 slots, two per CU (not for weight gradients)
};
constexpr int kNumTiles = sizeof(kTiles) / sizeof(kTiles[0]);

template <bool AKC, bool BKC, int EPI>
int run_tile(int tile, const GArgs& g, hipStream_t s) {
  switch (tile) {
    case 0: return launch<AKC, BKC, 2, 2, 4, 4, 64, 2, EPI>(g, s);
    case 1: return launch<AKC, BKC, 2, 4, 8, 4, 32, 4, EPI>(g, s);
    case 2: return launch<AKC, BKC, 4, 2, 2, 4, 64, 4, EPI>(g, s);
    case 3: return launch<AKC, BKC, 4, 2, 4, 4, 64, 3, EPI>(g, s);
    case 4:
      if constexpr (AKC) return launch<AKC, BKC, 2, 2, 2, 4, 64, 3, EPI>(g, s);
      return hipErrorInvalidValue;
    default: return hipErrorInvalidValue;
  }
}
// splits > 1: fp32 partials in `part` (splits x M x N) and a join
template <bool AKC, bool BKC, int EPI>
int run(int tile, int splits, GArgs g, hipStream_t s) {
  if (splits < 1 || splits > 64) return hipErrorInvalidValue;
  g.splits = splits;
  if constexpr (EPI == 0 || EPI == 1) {
    if (splits > 1) {
      if (!g.part || ((uintptr_t)g.part & 15)) return hipErrorInvalidValue;
      return run_tile<AKC, BKC, 4>(tile, g, s);
    }
  } else if (splits != 1) {
    return hipErrorInvalidValue;
  }
  return run_tile<AKC, BKC, EPI>(tile, g, s);
}

bool bad_rows(const void* p, int ld, int cols) {   // 16-B rows; tile offsets stay below 2^31 bytes
  return p == nullptr || ((uintptr_t)p & 15) || (ld & 7) || ld < cols || ld > (1 << 21);
}
bool bad_dim(int n) { return n <= 0 || (n & 7) || n > (1 << 20); }

}  // namespace

// geometry of a tile: what = 0 rows, 1 columns, 2 column-partial rows (mx_gated_dgate); -1: no such tile
MX_EXPORT int mx_gated_tile(int tile, int what) {
  if (tile < 0 || tile >= kNumTiles) return -1;
  return what == 0 ? kTiles[tile].bm : what == 1 ? kTiles[tile].bn : kTiles[tile].wm;
}

// whether M tokens take the few-token form in a product of K x N weights (no tile, no splits)
MX_EXPORT int mx_gated_few(int M, int K, int N) {
  GArgs g{};
  g.M = M; g.N = N; g.K = K;
  return few_tokens(g);
}

// h[M][F] = act(x W1a^T + b1a) (x W1b^T + b1b), y[M][Ho] = h W2^T + b2: x [M][ldx] (H wide), w1 [2F][ld1], w2
// [Ho][ld2], biases or null; pre [M][2F] or null; part: splits x M x Ho floats (splits > 1)
MX_EXPORT int mx_gated_fwd(const void* x, int ldx, const void* w1, int ld1, const void* b1, void* pre, void* h,
                           const void* w2, int ld2, const void* b2, void* y, int M, int H, int F, int Ho, int act,
                           int gate_tile, int down_tile, int splits, float* part, hipStream_t s) {
  if (M <= 0 || bad_dim(H) || bad_dim(F) || bad_dim(Ho) || bad_rows(x, ldx, H) || bad_rows(w1, ld1, H) ||
      bad_rows(h, F, F) || bad_rows(w2, ld2, F) || bad_rows(y, Ho, Ho) || ((uintptr_t)pre & 15) ||
      ((uintptr_t)b1 & 15) || ((uintptr_t)b2 & 15) || act < 0 || act > 1)
    return hipErrorInvalidValue;
  GArgs g{};
  g.a = (const uint16_t*)x; g.b = (const uint16_t*)w1; g.c = (uint16_t*)h; g.aux = (uint16_t*)pre;
  g.bias = (const uint16_t*)b1;
  g.lda = ldx; g.ldb = ld1; g.ldc = F;
  g.M = M; g.N = F; g.K = H; g.act = act;
  if (const int e = few_tokens(g) ? run_few<true>(g, s) : run<true, true, 2>(gate_tile, 1, g, s); e != hipSuccess)
    return e;
  GArgs d{};
  d.a = (const uint16_t*)h; d.b = (const uint16_t*)w2; d.c = (uint16_t*)y; d.bias = (const uint16_t*)b2;
  d.lda = F; d.ldb = ld2; d.ldc = Ho; d.part = part;
  d.M = M; d.N = Ho; d.K = F;
  return few_tokens(d) ? run_few<false>(d, s) : run<true, true, 1>(down_tile, splits, d, s);
}

// dpre[M][2F] = [dh b act'(a) | dh act(a)], dh = dy W2: dy [M][lddy] (K wide), w2 [K][ldw]; part null or
// the fp32 column partials [tiles x mx_gated_tile(tile, 2)][2F]
MX_EXPORT int mx_gated_dgate(const void* dy, int lddy, const void* w2, int ldw, const void* pre, void* dpre,
                             float* part, int M, int K, int F, int act, int tile, hipStream_t s) {
  if (M <= 0 || bad_dim(K) || bad_dim(F) || bad_rows(dy, lddy, K) || bad_rows(w2, ldw, F) ||
      bad_rows(pre, 2 * F, 2 * F) || bad_rows(dpre, 2 * F, 2 * F) || ((uintptr_t)part & 15) || act < 0 || act > 1)
    return hipErrorInvalidValue;
  GArgs g{};
  g.a = (const uint16_t*)dy; g.b = (const uint16_t*)w2; g.aux = (uint16_t*)const_cast<void*>(pre);
  g.grad = (uint16_t*)dpre; g.part = part;
  g.lda = lddy; g.ldb = ldw;
  g.M = M; g.N = F; g.K = K; g.act = act;
  return run<true, false, 3>(tile, 1, g, s);
}

// dx[M][N] = dpre W1: dpre [M][K] contiguous, w1 [K][ldw]
MX_EXPORT int mx_gated_dx(const void* dpre, const void* w1, int ldw, void* dx, int M, int N, int K, int tile,
                          int splits, float* part, hipStream_t s) {
  if (M <= 0 || bad_dim(K) || bad_dim(N) || bad_rows(dpre, K, K) || bad_rows(w1, ldw, N) || bad_rows(dx, N, N))
    return hipErrorInvalidValue;
  GArgs g{};
  g.a = (const uint16_t*)dpre; g.b = (const uint16_t*)w1; g.c = (uint16_t*)dx;
  g.lda = K; g.ldb = ldw; g.ldc = N; g.part = part;
  g.M = M; g.N = N; g.K = K;
  return run<true, false, 0>(tile, splits, g, s);
}

// dw[M][N] (+)= a^T b over T rows: a [T][lda] (M wide), b [T][ldb] (N wide), dw [M][ldc]
MX_EXPORT int mx_gated_dw(const void* a, int lda, const void* b, int ldb, void* dw, int ldc, int T, int M, int N,
                          int accumulate, int tile, int splits, float* part, hipStream_t s) {
  if (T <= 0 || bad_dim(M) || bad_dim(N) || bad_rows(a, lda, M) || bad_rows(b, ldb, N) || bad_rows(dw, ldc, N))
    return hipErrorInvalidValue;
  GArgs g{};
  g.a = (const uint16_t*)a; g.b = (const uint16_t*)b; g.c = (uint16_t*)dw;
  g.lda = lda; g.ldb = ldb; g.ldc = ldc; g.part = part;
  g.M = M; g.N = N; g.K = T; g.accumulate = accumulate;
  return run<false, false, 0>(tile, splits, g, s);
}

// two such products over the same T rows in one launch
MX_EXPORT int mx_gated_dw_pair(const void* a1, int lda1, const void* b1, int ldb1, void* dw1, int ldc1, int M1, int N1,
                               const void* a2, int lda2, const void* b2, int ldb2, void* dw2, int ldc2, int M2, int N2,
                               int T, int accumulate, int tile, hipStream_t s) {
  if (T <= 0 || bad_dim(M1) || bad_dim(N1) || bad_rows(a1, lda1, M1) || bad_rows(b1, ldb1, N1) ||
      bad_rows(dw1, ldc1, N1) || bad_dim(M2) || bad_dim(N2) || bad_rows(a2, lda2, M2) || bad_rows(b2, ldb2, N2) ||
      bad_rows(dw2, ldc2, N2))
    return hipErrorInvalidValue;
  GArgs g{};
  g.a = (const uint16_t*)a1; g.b = (const uint16_t*)b1; g.c = (uint16_t*)dw1;
  g.lda = lda1; g.ldb = ldb1; g.ldc = ldc1;
  g.M = M1; g.N = N1; g.K = T; g.accumulate = accumulate;
  g.a2 = (const uint16_t*)a2; g.b2 = (const uint16_t*)b2; g.c2 = (uint16_t*)dw2;
  g.lda2 = lda2; g.ldb2 = ldb2; g.ldc2 = ldc2; g.M2 = M2; g.N2 = N2;
  g.splits = 1;
  return run_tile<false, false, 5>(tile, g, s);
}
