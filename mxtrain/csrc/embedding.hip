// Scaled embedding lookup and its gradient by sorted tokens (gfx950, bf16 rows, fp32 sums).
//
//   out[t] = scale wte[id_t] + wpe[pos_t]
//   dtable[v] (+)= scale sum_{t: key_t = v} dout[t]     (wte: keys = ids; wpe: keys = positions)
//
// Both are bound by memory: the lookup by its rows in and out, the gradient by reading dout once
// and writing the table once.  The gradient sorts (key, token) pairs with a stable radix sort, so
// the tokens of a row are contiguous and in token order; waves then sum fixed chunks of CH sorted
// tokens, so a token that fills half of the batch costs no more than one that never repeats, and
// the order of every sum is fixed (bit-reproducible, no float atomics).  Runs that cross a chunk
// border leave fp32 partials that a second kernel adds in order.
#include "common.h"

using namespace mx;

namespace {

constexpr int CH = 32;          // sorted tokens per wave
constexpr int SORT_NT = 1024;   // threads of a sort block (16 waves)
constexpr int SORT_NW = SORT_NT / 64;
constexpr int MAX_BITS = 9;     // digit width: at most 2^9 counters per wave

// ------------------------------------------------------------------------------ lookup
// one wave per row, 16 B per lane; 32768 rows of 4096 in 89 us, 6.0 TB/s in and out
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const int64_t* __restrict__ ids,
                                                            const uint16_t* __restrict__ wte, int64_t vstart, int V,
                                                            float scale, const int64_t* __restrict__ pos,
                                                            const uint16_t* __restrict__ wpe, int P,
                                                            uint16_t* __restrict__ out, int T, int H) {
  const int lane = threadIdx.x & 63;
  for (int t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); t < T; t += gridDim.x * 4) {
    const int64_t id = ids[t] - vstart;
    const bool in = id >= 0 && id < V;                 // (another vocabulary shard's token: zero)
    const uint16_t* row = wte + (in ? id : 0) * (int64_t)H;
    const int64_t p = pos ? pos[t] : -1;
    const uint16_t* prow = p >= 0 && p < P ? wpe + p * (int64_t)H : nullptr;
    uint16_t* orow = out + (int64_t)t * H;
#pragma unroll 4
    for (int c = lane * 8; c < H; c += 512) {
      float f[8];
      unpack8(*reinterpret_cast<const uint4*>(row + c), f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = in ? f[j] * scale : 0.f;
      if (prow) {
        float g[8];
        unpack8(*reinterpret_cast<const uint4*>(prow + c), g);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] += g[j];
      }
      *reinterpret_cast<uint4*>(orow + c) = pack8(f);
    }
  }
}

// ------------------------------------------------------------------------------ sort
// keys of the first pass come from the int64 ids (a key outside [0, V) sorts last as V), later
// passes from the previous pass's pairs
struct SortArgs {
  const int64_t* ids;
  int64_t vstart;
  int V, T, tpb;                // tokens per block (a multiple of 64 SORT_NW)
  const int* kin;
  const int* iin;
  int *kout, *iout;
  int* hist;                    // [blocks][1 << bits]
  int shift, bits;
};
__device__ __forceinline__ int sort_key(const SortArgs& a, int t) {
  if (a.kin) return a.kin[t];
  const int64_t k = a.ids[t] - a.vstart;
  return k >= 0 && k < a.V ? (int)k : a.V;
}

__global__ __launch_bounds__(SORT_NT) void sort_hist_kernel(const SortArgs a) {
  __shared__ int cnt[1 << MAX_BITS];
  const int R = 1 << a.bits, tid = threadIdx.x;
  for (int d = tid; d < R; d += SORT_NT) cnt[d] = 0;
  __syncthreads();
  const int t0 = blockIdx.x * a.tpb, t1 = min(a.T, t0 + a.tpb);
  for (int t = t0 + tid; t < t1; t += SORT_NT) atomicAdd(&cnt[(sort_key(a, t) >> a.shift) & (R - 1)], 1);
  __syncthreads();
  for (int d = tid; d < R; d += SORT_NT) a.hist[blockIdx.x * R + d] = cnt[d];
}

// lanes of the wave whose `bits`-bit digit equals this lane's (only among active lanes `live`)
__device__ __forceinline__ uint64_t match_digit(int d, int bits, uint64_t live) {
  uint64_t m = live;
  for (int b = 0; b < bits; ++b) {
    const uint64_t v = __ballot((d >> b) & 1);
    m &= (d >> b) & 1 ? v : ~v;
  }
  return m;
}

// Next output slot of every (wave, digit): wcnt holds the waves' digit counts on entry; `total` and
// `before` are the digit's count anywhere and in the blocks before this one (digit = threadIdx.x)
__device__ __forceinline__ void digit_slots(int* wcnt, int* wsum, int R, int total, int before) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int x = total;                          // inclusive scan over the digits: wave, then waves
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == 63) wsum[w] = x;
  __syncthreads();
  int off = 0;
  for (int i = 0; i < w; ++i) off += wsum[i];
  if (tid < R) {                          // R <= SORT_NT: one digit per thread
    int s = off + x - total + before;
    for (int i = 0; i < SORT_NW; ++i) {
      const int c = wcnt[i * R + tid];
      wcnt[i * R + tid] = s;
      s += c;
    }
  }
  __syncthreads();
}
// slot of this lane's digit among its wave's tokens, in token order (wcnt: the wave's slots)
__device__ __forceinline__ int take_slot(int* wcnt, int d, int bits, bool live, int lane) {
  const uint64_t peers = match_digit(d, bits, __ballot(live));
  const int rank = __popcll(peers & ((1ull << lane) - 1)), lead = __ffsll((unsigned long long)peers) - 1;
  int slot = 0;
  if (live && rank == 0) slot = atomicAdd(&wcnt[d], __popcll(peers));
  return __shfl(slot, live ? lead : lane) + rank;
}

// Stable scatter of one block's tokens: wave w owns the w-th contiguous share.
__global__ __launch_bounds__(SORT_NT) void sort_scatter_kernel(const SortArgs a) {
  extern __shared__ int wcnt[];           // [SORT_NW][R]
  __shared__ int wsum[SORT_NW];
  const int R = 1 << a.bits, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  for (int i = tid; i < SORT_NW * R; i += SORT_NT) wcnt[i] = 0;
  __syncthreads();
  const int share = a.tpb / SORT_NW;
  const int s0 = blockIdx.x * a.tpb + w * share, s1 = min(a.T, s0 + share);
  for (int t = s0 + lane; t < s1; t += 64) atomicAdd(&wcnt[w * R + ((sort_key(a, t) >> a.shift) & (R - 1))], 1);
  __syncthreads();
  int total = 0, before = 0;
  if (tid < R) {
#pragma unroll 8
    for (int b = 0; b < (int)gridDim.x; ++b) {
      const int c = a.hist[b * R + tid];
      total += c;
      before += b < (int)blockIdx.x ? c : 0;
    }
  }
  digit_slots(wcnt, wsum, R, total, before);
  for (int c0 = s0; c0 < s1; c0 += 64) {
    const int t = c0 + lane;
    const bool live = t < s1;
    const int key = live ? sort_key(a, t) : 0, d = (key >> a.shift) & (R - 1);
    const int slot = take_slot(wcnt + w * R, d, a.bits, live, lane);
    if (live) {
      a.kout[slot] = key;
      a.iout[slot] = a.iin ? a.iin[t] : t;
    }
  }
}

// Few tokens: the place of a token is the number of keys below its own, and of equal ones before it, so
// one launch counts it -- T^2 compares of keys in LDS, little at T tokens against the latency of radix
// passes (6.0 us at 4096 tokens, where a radix sort in one workgroup took 13.3 and the block form 17;
// the whole gradient of 8192 tokens, 50304 rows of 64: 28 us, and 38 by the block form, which takes no
// more at 16384, where this would take four times as many compares).  A workgroup places 16
// tokens: lane (q, i) of wave w compares token i with every 64th group of four keys.
constexpr int SMALL = 8192;
__global__ __launch_bounds__(SORT_NT) void sort_small_kernel(const SortArgs a) {
  __shared__ __attribute__((aligned(16))) int keys[SMALL];
  __shared__ int cnt[SORT_NW][16];
  const int T = a.T, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int T4 = (T + 3) & ~3;
  for (int t = tid; t < T4; t += SORT_NT) keys[t] = t < T ? sort_key(a, t) : INT32_MAX;   // (above every key)
  __syncthreads();
  const int i = min((int)blockIdx.x * 16 + (lane & 15), T - 1), mine = keys[i];
  int n = 0;
#pragma unroll 4
  for (int u = w * 4 + (lane >> 4); u < T4 / 4; u += SORT_NW * 4) {
    const int4 k = *reinterpret_cast<const int4*>(keys + 4 * u);
    const int below = mine + (4 * u + 3 < i ? 1 : 0);
    n += (int)(k.x < below) + (int)(k.y < below) + (int)(k.z < below) + (int)(k.w < below);
  }
  n += __shfl_xor(n, 16);
  n += __shfl_xor(n, 32);
  if (lane < 16) cnt[w][lane] = n;
  __syncthreads();
  if (tid >= 16 || (int)blockIdx.x * 16 + tid >= T) return;
  int place = 0;
  for (int x = 0; x < SORT_NW; ++x) place += cnt[x][tid];
  for (int t = i & ~3; t < i; ++t) place += keys[t] == mine;     // equal ones of its own four
  a.kout[place] = mine;
  a.iout[place] = i;
}

// ------------------------------------------------------------------------------ sums
struct SumArgs {
  const int *key, *idx;         // sorted
  const uint16_t* dout;
  uint16_t* table;
  float* part;                  // [chunks][2][H]: open run at the chunk's start / at its end
  int T, V, H, ldd, ncol, chunks;
  float scale;
  int accumulate;
};
__device__ __forceinline__ void emit_row(const SumArgs& a, int key, int c, const float (&acc)[8]) {
  uint16_t* p = a.table + (int64_t)key * a.H + c;
  float o[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = acc[j] * a.scale;
  if (a.accumulate) {
    float x[8];
    unpack8(*reinterpret_cast<const uint4*>(p), x);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] += x[j];
  }
  *reinterpret_cast<uint4*>(p) = pack8(o);
}
__device__ __forceinline__ void emit_part(const SumArgs& a, int chunk, int which, int c, const float (&acc)[8]) {
  float* p = a.part + ((int64_t)chunk * 2 + which) * a.H + c;
  *reinterpret_cast<float4*>(p) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
}

// blocks [0, sum_blocks): one wave per (chunk, 512 columns); the rest zero the rows of the table
// that no token has, 64 rows a block (each lane looks its row up in the sorted keys).  Bound by memory:
// 32768 rows of 4096 into 50304 in 139 us, 4.9 TB/s
__global__ __launch_bounds__(256) void embedding_sum_kernel(const SumArgs a, int sum_blocks) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= sum_blocks) {
    const int v0 = ((int)blockIdx.x - sum_blocks) * 64, v = v0 + lane;
    int lo = 0, hi = a.T;                 // first sorted position with key >= v
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.key[mid] < v) lo = mid + 1;
      else hi = mid;
    }
    const bool absent = v < a.V && !(lo < a.T && a.key[lo] == v);
    const uint64_t m = __ballot(absent);
    for (int i = w; i < 64; i += 4) {
      if (!((m >> i) & 1)) continue;
      uint16_t* row = a.table + (int64_t)(v0 + i) * a.H;
      for (int c = lane * 8; c < a.H; c += 512) *reinterpret_cast<uint4*>(row + c) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int item = blockIdx.x * 4 + w;
  const int chunk = item / a.ncol, c = (item - chunk * a.ncol) * 512 + lane * 8;
  if (chunk >= a.chunks) return;
  const int e0 = chunk * CH, n = min(CH, a.T - e0);
  // lane i < n holds sorted entry e0 + i
  const int kl = lane < n ? a.key[e0 + lane] : -1, il = lane < n ? a.idx[e0 + lane] : 0;
  const int prev = e0 > 0 ? a.key[e0 - 1] : -1, next = e0 + n < a.T ? a.key[e0 + n] : -1;
  const bool col = c < a.H;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int run = __builtin_amdgcn_readlane(kl, 0);
  bool open = run == prev;                // the current run began in an earlier chunk
  constexpr int G = 8;                    // rows in flight
  for (int b = 0; b < n; b += G) {
    uint4 x[G];
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int i = min(b + j, n - 1);
      const int t = __builtin_amdgcn_readlane(il, i), k = __builtin_amdgcn_readlane(kl, i);
      // (a key of V belongs to no row of this table: never read)
      x[j] = col && k < a.V ? *reinterpret_cast<const uint4*>(a.dout + (int64_t)t * a.ldd + c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
      if (b + j >= n) break;
      const int k = __builtin_amdgcn_readlane(kl, b + j);
      if (k != run) {                     // the run before ends here
        if (col && run < a.V) {
          if (open) emit_part(a, chunk, 0, c, acc);
          else emit_row(a, run, c, acc);
        }
        open = false;
        run = k;
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] = 0.f;
      }
      float f[8];
      unpack8(x[j], f);
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += f[q];
    }
  }
  if (!col || run >= a.V) return;
  if (open) emit_part(a, chunk, 0, c, acc);
  else if (run == next) emit_part(a, chunk, 1, c, acc);
  else emit_row(a, run, c, acc);
}

// runs that cross chunk borders: the wave of the chunk where such a run begins adds the partials
__global__ __launch_bounds__(256) void embedding_join_kernel(const SumArgs a) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x * 4 + w;
  const int chunk = item / a.ncol, c = (item - chunk * a.ncol) * 512 + lane * 8;
  if (chunk >= a.chunks - 1) return;      // (the last chunk's run ends with it)
  const int last = chunk * CH + CH - 1, run = a.key[last];
  if (run >= a.V || a.key[last + 1] != run) return;
  if (a.key[chunk * CH] == run && chunk > 0 && a.key[chunk * CH - 1] == run) return;   // began earlier
  int lo = last + 2, hi = a.T;            // first sorted position behind the run
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.key[mid] == run) lo = mid + 1;
    else hi = mid;
  }
  const int end = (lo - 1) / CH;          // last chunk that holds a part of it
  if (c >= a.H) return;
  float acc[8];
  const float* p = a.part + ((int64_t)chunk * 2 + 1) * a.H + c;
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = p[j];
#pragma unroll 8
  for (int k = chunk + 1; k <= end; ++k) {
    const float4* q = reinterpret_cast<const float4*>(a.part + (int64_t)k * 2 * a.H + c);
    const float4 x = q[0], y = q[1];
    acc[0] += x.x; acc[1] += x.y; acc[2] += x.z; acc[3] += x.w;
    acc[4] += y.x; acc[5] += y.y; acc[6] += y.z; acc[7] += y.w;
  }
  emit_row(a, run, c, acc);
}

struct SortPlan {
  int bits, passes, blocks, tpb;
};
SortPlan sort_plan(int T, int V) {
  SortPlan p;
  int total = 1;
  while (total < 31 && ((int64_t)1 << total) <= V) ++total;   // keys 0 .. V
  p.passes = (total + MAX_BITS - 1) / MAX_BITS;
  p.bits = (total + p.passes - 1) / p.passes;
  p.tpb = 2 * 64 * SORT_NW;               // 2048 tokens a block, more once there are 256 blocks
  while ((int64_t)p.tpb * 256 < T) p.tpb *= 2;
  p.blocks = (T + p.tpb - 1) / p.tpb;
  return p;
}

}  // namespace

MX_EXPORT int mx_embedding_fwd(const void* ids, const void* wte, int64_t vstart, int V, float scale, const void* pos,
                               const void* wpe, int P, void* out, int T, int H, hipStream_t s) {
  if (!ids || !wte || !out || T <= 0 || T > (1 << 30) || V <= 0 || H <= 0 || (H & 7) || (pos && (!wpe || P <= 0)))
    return hipErrorInvalidValue;
  if (((uintptr_t)wte | (uintptr_t)wpe | (uintptr_t)out) & 15) return hipErrorInvalidValue;
  // (a launch has fewer than 2^32 threads: beyond 2^25 tokens a wave takes several)
  hipLaunchKernelGGL(embedding_fwd_kernel, dim3(T > 1 << 25 ? 1 << 23 : (T + 3) / 4), dim3(256), 0, s, (const int64_t*)ids,
                     (const uint16_t*)wte, vstart, V, scale, (const int64_t*)pos, (const uint16_t*)wpe, P,
                     (uint16_t*)out, T, H);
  return hipGetLastError();
}

// int32 words of workspace: two (key, token) arrays, the block histograms, fp32 partials (16-B aligned); -1: sizes
// that the kernels do not take
MX_EXPORT int64_t mx_embedding_bwd_words(int T, int V, int H) {
  if (T <= 0 || V <= 0 || H <= 0 || T > (1 << 30) || V >= (1 << 30)) return -1;
  const SortPlan p = sort_plan(T, V);
  const int64_t t4 = ((int64_t)T + 3) & ~3ll, chunks = (T + CH - 1) / CH;
  // threads of the sums' launch
  if (256 * ((chunks * ((H + 511ll) / 512) + 3) / 4 + (V + 63) / 64) >= (int64_t)1 << 32) return -1;
  return 4 * t4 + (((int64_t)p.blocks << p.bits) + 3 & ~3ll) + chunks * 2 * H;
}

// table[V][H] (+)= scale * sums of dout rows by key; `words` is the size of ws the caller holds.
MX_EXPORT int mx_embedding_bwd(const void* ids, int64_t vstart, const void* dout, int ldd, void* table, int T, int V,
                               int H, float scale, int accumulate, void* ws, int64_t words, hipStream_t s) {
  if (!ids || !dout || !table || !ws || (H & 7) || (ldd & 7) || ldd < H) return hipErrorInvalidValue;
  const int64_t need = mx_embedding_bwd_words(T, V, H);
  if (need < 0 || words < need) return hipErrorInvalidValue;
  if (((uintptr_t)dout | (uintptr_t)table | (uintptr_t)ws) & 15) return hipErrorInvalidValue;
  const SortPlan p = sort_plan(T, V);
  const int64_t t4 = ((int64_t)T + 3) & ~3ll;
  int* b = (int*)ws;
  int *k0 = b, *i0 = b + t4, *k1 = b + 2 * t4, *i1 = b + 3 * t4, *hist = b + 4 * t4;
  float* part = (float*)(hist + (((int64_t)p.blocks << p.bits) + 3 & ~3ll));
  SortArgs a{(const int64_t*)ids, vstart, V, T, p.tpb, nullptr, nullptr, k0, i0, hist, 0, p.bits};
  // (each launch is looked at before the next: the sums read at the token numbers that the sort writes)
  hipError_t e = hipSuccess;
  if (T <= SMALL) {
    hipLaunchKernelGGL(sort_small_kernel, dim3((T + 15) / 16), dim3(SORT_NT), 0, s, a);
    e = hipGetLastError();
    a.kin = k0;
    a.iin = i0;
  }
  const size_t lds = (size_t)SORT_NW * sizeof(int) << p.bits;
  for (int q = 0; q < (T <= SMALL ? 0 : p.passes) && e == hipSuccess; ++q) {
    a.shift = q * p.bits;
    hipLaunchKernelGGL(sort_hist_kernel, dim3(p.blocks), dim3(SORT_NT), 0, s, a);
    if ((e = hipGetLastError()) != hipSuccess) break;
    hipLaunchKernelGGL(sort_scatter_kernel, dim3(p.blocks), dim3(SORT_NT), lds, s, a);
    e = hipGetLastError();
    a.kin = a.kout;
    a.iin = a.iout;
    a.kout = a.kout == k0 ? k1 : k0;
    a.iout = a.iout == i0 ? i1 : i0;
  }
  if (e != hipSuccess) return e;
  SumArgs u{a.kin, a.iin, (const uint16_t*)dout, (uint16_t*)table, part, T, V, H, ldd, (H + 511) / 512,
            (T + CH - 1) / CH, scale, accumulate};
  const int64_t items = (int64_t)u.chunks * u.ncol, sum_blocks = (items + 3) / 4;
  const int64_t zero_blocks = accumulate ? 0 : (V + 63) / 64;
  hipLaunchKernelGGL(embedding_sum_kernel, dim3((unsigned)(sum_blocks + zero_blocks)), dim3(256), 0, s, u,
                     (int)sum_blocks);
  if ((e = hipGetLastError()) != hipSuccess || u.chunks == 1) return e;
  hipLaunchKernelGGL(embedding_join_kernel, dim3((unsigned)sum_blocks), dim3(256), 0, s, u);
  return hipGetLastError();
}
