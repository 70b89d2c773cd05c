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
// All six products share one kernel.  Operands are staged by LDS-DMA through buffer resources:
// what lies past a tile's rows reads zero, so any number of tokens and any feature count that is a
// multiple of 8 is taken without padding.  16 x 16 x 32 MFMA with the weight (column) operand
// first, so that a lane holds 4 consecutive columns of a row.
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
template <bool AKC, bool BKC, int WM, int WN, int FM, int FN, int BKT, int NSLOT, int MINB, int EPI>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(MINB, MINB))) void gated_gemm_kernel(
    const GArgs g) {
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
  const int wg = xcd_remap(blockIdx.x, gridDim.x);
  const int per = g.gm * g.tiles_n, grp = wg / per, rem = wg - grp * per;
  const int gmr = min(g.gm, g.tiles_m - grp * g.gm);   // (the last group may be smaller)
  const int tm = grp * g.gm + rem % gmr, tn = rem / gmr;
  const int m0 = tm * BM, n0 = tn * BNO;
  const int K = g.K, nk = (K + BKT - 1) / BKT;

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
    const int k0 = it * BKT;
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
  auto get = [&](const uint16_t* p, uint32_t (&v)[2][2], bool ok) __attribute__((always_inline)) {
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (ok) x = *reinterpret_cast<const uint4*>(p);
    v[0][0] = x.x; v[0][1] = x.y; v[1][0] = x.z; v[1][1] = x.w;
    undeal(v[0][0], v[0][1], v[1][0], v[1][1]);
  };
#pragma unroll
  for (int s = 0; s < FM; ++s) {
    const int m = mrow + 16 * s;
#pragma unroll
    for (int up = 0; up < FO / 2; ++up) {
      const int col = colw + 32 * up + 8 * G;       // the lane's 8 columns after the re-deal
      const bool ok = m < g.M && col < N;
      uint32_t c[2][2], pa[2][2], pb[2][2];
      if constexpr (EPI == 0) {
        if (g.accumulate) get(g.c + (size_t)m * g.ldc + col, pa, ok);
      }
      if constexpr (EPI == 3) {
        get(g.aux + (size_t)m * 2 * N + col, pa, ok);
        get(g.aux + (size_t)m * 2 * N + N + col, pb, ok);
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int u = 2 * up + hf;
        float v[4], w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[s][u][e] + bias[u][e];
        if constexpr (EPI == 0) {
          if (g.accumulate) {
            v[0] += lo_bf(pa[hf][0]); v[1] += hi_bf(pa[hf][0]); v[2] += lo_bf(pa[hf][1]); v[3] += hi_bf(pa[hf][1]);
          }
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

template <bool AKC, bool BKC, int WM, int WN, int FM, int FN, int BKT, int NSLOT, int MINB, int EPI>
int launch(GArgs g, hipStream_t s) {
  using Gm = Geo<AKC, BKC, WM, WN, FM, FN, BKT, NSLOT>;
  const int bn = EPI == 2 ? Gm::BN / 2 : Gm::BN;
  g.tiles_m = (g.M + Gm::BM - 1) / Gm::BM;
  g.tiles_n = (g.N + bn - 1) / bn;
  g.gm = 8;
  if ((int64_t)g.tiles_m * g.tiles_n >= ((int64_t)1 << 31)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((gated_gemm_kernel<AKC, BKC, WM, WN, FM, FN, BKT, NSLOT, MINB, EPI>),
                     dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(Gm::NT), 0, s, g);
  return hipGetLastError();
}
template <bool AKC, bool BKC, int EPI>
int run(const GArgs& g, hipStream_t s) {
  return launch<AKC, BKC, 2, 2, 4, 4, 64, 2, 2, EPI>(g, s);
}
constexpr int kPartRows = 64;   // rows behind one row of column partials (16 FM)

bool bad_rows(const void* p, int ld, int cols) {   // 16-B rows; tile offsets stay below 2^31 bytes
  return p == nullptr || ((uintptr_t)p & 15) || (ld & 7) || ld < cols || ld > (1 << 21);
}
bool bad_dim(int n) { return n <= 0 || (n & 7) || n > (1 << 20); }

}  // namespace

// h[M][F] = act(x W1a^T + b1a) (x W1b^T + b1b): x [M][ldx] (K wide), w1 [2F][ldw]; pre [M][2F] or null
MX_EXPORT int mx_gated_fwd(const void* x, int ldx, const void* w1, int ldw, const void* b1, void* pre, void* h, int M,
                           int K, int F, int act, hipStream_t s) {
  if (M <= 0 || bad_dim(K) || bad_dim(F) || bad_rows(x, ldx, K) || bad_rows(w1, ldw, K) || bad_rows(h, F, F) ||
      ((uintptr_t)pre & 15) || ((uintptr_t)b1 & 15) || act < 0 || act > 1)
    return hipErrorInvalidValue;
  GArgs g{};
  g.a = (const uint16_t*)x; g.b = (const uint16_t*)w1; g.c = (uint16_t*)h; g.aux = (uint16_t*)pre;
  g.bias = (const uint16_t*)b1;
  g.lda = ldx; g.ldb = ldw; g.ldc = F;
  g.M = M; g.N = F; g.K = K; g.act = act;
  return run<true, true, 2>(g, s);
}

// y[M][N] = h W2^T (+ b2): h [M][K] contiguous, w2 [N][ldw]
MX_EXPORT int mx_gated_down(const void* h, const void* w2, int ldw, const void* b2, void* y, int M, int N, int K,
                            hipStream_t s) {
  if (M <= 0 || bad_dim(K) || bad_dim(N) || bad_rows(h, K, K) || bad_rows(w2, ldw, K) || bad_rows(y, N, N) ||
      ((uintptr_t)b2 & 15))
    return hipErrorInvalidValue;
  GArgs g{};
  g.a = (const uint16_t*)h; g.b = (const uint16_t*)w2; g.c = (uint16_t*)y; g.bias = (const uint16_t*)b2;
  g.lda = K; g.ldb = ldw; g.ldc = N;
  g.M = M; g.N = N; g.K = K;
  return run<true, true, 1>(g, s);
}

// rows of column partials mx_gated_dgate writes for M tokens
MX_EXPORT int mx_gated_parts(int M) { return (M + 127) / 128 * 2; }

// dpre[M][2F] = [dh b act'(a) | dh act(a)], dh = dy W2: dy [M][lddy] (K wide), w2 [K][ldw]; part or null
MX_EXPORT int mx_gated_dgate(const void* dy, int lddy, const void* w2, int ldw, const void* pre, void* dpre,
                             float* part, int M, int K, int F, int act, hipStream_t s) {
  if (M <= 0 || bad_dim(K) || bad_dim(F) || bad_rows(dy, lddy, K) || bad_rows(w2, ldw, F) ||
      bad_rows(pre, 2 * F, 2 * F) || bad_rows(dpre, 2 * F, 2 * F) || ((uintptr_t)part & 15) || act < 0 || act > 1)
    return hipErrorInvalidValue;
  static_assert(kPartRows * 2 == 128, "mx_gated_parts counts two partial rows per 128-row tile");
  GArgs g{};
  g.a = (const uint16_t*)dy; g.b = (const uint16_t*)w2; g.aux = (uint16_t*)const_cast<void*>(pre);
  g.grad = (uint16_t*)dpre; g.part = part;
  g.lda = lddy; g.ldb = ldw;
  g.M = M; g.N = F; g.K = K; g.act = act;
  return run<true, false, 3>(g, s);
}

// dx[M][N] = dpre W1: dpre [M][K] contiguous, w1 [K][ldw]
MX_EXPORT int mx_gated_dx(const void* dpre, const void* w1, int ldw, void* dx, int M, int N, int K, hipStream_t s) {
  if (M <= 0 || bad_dim(K) || bad_dim(N) || bad_rows(dpre, K, K) || bad_rows(w1, ldw, N) || bad_rows(dx, N, N))
    return hipErrorInvalidValue;
  GArgs g{};
  g.a = (const uint16_t*)dpre; g.b = (const uint16_t*)w1; g.c = (uint16_t*)dx;
  g.lda = K; g.ldb = ldw; g.ldc = N;
  g.M = M; g.N = N; g.K = K;
  return run<true, false, 0>(g, s);
}

// dw[M][N] (+)= a^T b over T rows: a [T][lda] (M wide), b [T][ldb] (N wide), dw [M][ldc]
MX_EXPORT int mx_gated_dw(const void* a, int lda, const void* b, int ldb, void* dw, int ldc, int T, int M, int N,
                          int accumulate, hipStream_t s) {
  if (T <= 0 || bad_dim(M) || bad_dim(N) || bad_rows(a, lda, M) || bad_rows(b, ldb, N) || bad_rows(dw, ldc, N))
    return hipErrorInvalidValue;
  GArgs g{};
  g.a = (const uint16_t*)a; g.b = (const uint16_t*)b; g.c = (uint16_t*)dw;
  g.lda = lda; g.ldb = ldb; g.ldc = ldc;
  g.M = M; g.N = N; g.K = T; g.accumulate = accumulate;
  return run<false, false, 0>(g, s);
}
