// Device helpers shared by the attention kernels (flash.hip: fixed [B, S] batches with dropout;
// packed.hip: packed sequences): LDS tile swizzle, transposed reads, 32 x 32 MFMA, LDS-DMA,
// row stores and the block -> head map.  gfx950 only.
#pragma once
#include "common.h"

#pragma clang diagnostic ignored "-Winline-asm"  // m0 is clobbered on purpose (dma16 / dma4)

namespace mx {
namespace flash {

typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

// Chunk swizzle for a [rows][D] bf16 tile (D*2-byte rows, 16-B chunks).
//  D=64 (128-B rows, two rows per 256-B bank row): f = x ^ ((x&1)<<2), x = (row>>1)&7
//  D=128 (256-B rows): f = ((row&3)<<2) | ((row>>2)&3)
// Both keep the row reads (ds_read_b128, 32 rows) and the transposed reads (4 consecutive
// rows x 32 columns per half-wave) conflict-free; f depends on row bits 0-3 only, so a
// 32-row step is an immediate offset.
template <int D>
__device__ __forceinline__ int swz(int row) {
  if constexpr (D == 64) {
    int x = (row >> 1) & 7;
    return x ^ ((x & 1) << 2);
  } else {
    return ((row & 3) << 2) | ((row >> 2) & 3);
  }
}
template <int D>
__device__ __forceinline__ int toff(int row, int chunk) {
  return row * (D * 2) + ((chunk ^ swz<D>(row)) << 4);
}
__device__ __forceinline__ bf16x4 tr_read(const char* lds, int byte_off) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_bf16x4*)(lds + byte_off));
}
__device__ __forceinline__ bf16x8 cat(bf16x4 a, bf16x4 b) {
  return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ bf16x8 ld8(const uint16_t* p) {
  return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(p));
}
__device__ __forceinline__ bf16x8 lds8(const char* base, int off) {
  return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(base + off));
}
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ int crow(int e, int hh) { return (e & 3) + 8 * (e >> 2) + 4 * hh; }
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// One 32-column group of a row-per-lane 32x32 MFMA result (lane r and r + 32 hold row r:
// columns 8 k + 4 hh .. +3 of each group k) stored as bf16 with 16-B stores: for each pair of
// groups (k, k + 1) one v_permlane32_swap per dword gives the lower half-wave columns
// 8 k .. 8 k + 7 and the upper one 8 k + 8 .. 8 k + 15 -- 2 dwordx4 stores per lane instead of
// 4 dwordx2 (the epilogue store tail is issue-bound: MI355X guide T21).  Both lanes of a row
// must be active.
__device__ __forceinline__ void store_row32(uint16_t* rowp, const f32x16& acc, float sc, int hh) {
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const uint32_t ax = pack2(acc[4 * k + 0] * sc, acc[4 * k + 1] * sc);
    const uint32_t ay = pack2(acc[4 * k + 2] * sc, acc[4 * k + 3] * sc);
    const uint32_t bx = pack2(acc[4 * k + 4] * sc, acc[4 * k + 5] * sc);
    const uint32_t by = pack2(acc[4 * k + 6] * sc, acc[4 * k + 7] * sc);
    const auto rx = __builtin_amdgcn_permlane32_swap(ax, bx, false, false);
    const auto ry = __builtin_amdgcn_permlane32_swap(ay, by, false, false);
    *reinterpret_cast<uint4*>(rowp + 8 * k + 8 * hh) = make_uint4(rx[0], ry[0], rx[1], ry[1]);
  }
}

// one 1-KiB LDS-DMA piece: lane i's 16 B from `g` land at lds_base + 16 i.  Issued from
// inline asm: for the builtin, the compiler cannot prove that a later ds_read of another
// ring slot does not alias the in-flight DMA (no alias-scope info on either access) and
// waits vmcnt(0) before the first LDS read after every issue -- the next tile's DMA was
// drained before the current tile's first MFMA, serialising load and compute.  The kernels
// order DMA and reads themselves (vm_drain + barrier at the top of every tile).  M0 = LDS
// base (wave-uniform); one wait state between the M0 write and the DMA.
__device__ __forceinline__ uint32_t lds_u32(const void* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const lds_void_t*)p);
}
__device__ __forceinline__ void dma16(const void* g, char* lds_base) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :: "v"(g), "s"(lds_u32(lds_base)) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* g, char* lds_base) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
               :: "v"(g), "s"(lds_u32(lds_base)) : "memory", "m0");
}
// vmcnt(0) through the builtin (expcnt / lgkmcnt fields at their "no wait" maxima), not asm:
// the waitcnt pass then knows every compiler-visible load (e.g. the dropout words of the
// previous step) is complete, instead of re-waiting for them mid-tile with a vmcnt(N) that
// the hardware also applies to the asm-issued DMA of the next tile.
__device__ __forceinline__ void vm_drain() { __builtin_amdgcn_s_waitcnt(0x0F70); }

__device__ __forceinline__ bf16x8 pack8(const f32x16& acc, int base) {
  uint4 u;
  u.x = pack2(acc[base + 0], acc[base + 1]);
  u.y = pack2(acc[base + 2], acc[base + 3]);
  u.z = pack2(acc[base + 4], acc[base + 5]);
  u.w = pack2(acc[base + 6], acc[base + 7]);
  return __builtin_bit_cast(bf16x8, u);
}
// workgroup id -> (block rank, head): block ranks in dispatch order (rank 0 first, so the
// caller maps rank 0 to the heaviest causal block), and, when the head count is a multiple
// of 8, every block of a head on one XCD (workgroups are dealt round-robin over the 8 XCDs,
// id % 8): its K/V (Q/dO) stream is then read once into that XCD's L2.
__device__ __forceinline__ void block_map(int L, int nheads, int& rank, int& head) {
  if ((nheads & 7) == 0) {
    const int x = L & 7, idx = L >> 3, nh8 = nheads >> 3;
    rank = idx / nh8;
    head = (idx - rank * nh8) * 8 + x;
  } else {
    rank = L / nheads;
    head = L - rank * nheads;
  }
}

__device__ __forceinline__ void block_map(int nheads, int& rank, int& head) {
  block_map((int)blockIdx.x, nheads, rank, head);
}

}  // namespace flash
}  // namespace mx
