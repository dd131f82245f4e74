// What the absorbed-MLA kernels that feed 32-row waves from an LDS ring share: the
// layout of a 32-token bf16 latent tile, the loads straight to LDS, the MFMAs with
// their accumulator in VGPRs, waits, and row stores (ws_mla_wide.h, ws_mla_rows.hip).
#pragma once

#include "ws_common.h"

namespace ws {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWideRowData = 72;  // 576 bf16 = 72 x 16 B
// LDS chunk offset of row r of a tile.
__host__ __device__ constexpr int wide_row_off(int r) {
  return kWideRowData * r + 5 * (r >> 2) + 4 * ((r >> 1) & 1);
}
constexpr int kWideTileChunks = wide_row_off(31) + kWideRowData;  // 2343
constexpr int kWideTileDma = (kWideTileChunks + 63) / 64;         // 37 instructions of 64 chunks
constexpr int kWideTileAlloc = kWideTileDma * 64;                 // 2368 chunks
constexpr int kWideTiles = 4;
constexpr int kWideDmaPerWave = 10;  // 4 x 10 = 37 + 3 into the sink
constexpr float kWideHeadroomLog2 = 64.f;
// chunk offsets of rows 16 s + 8 t + q (q < 8) are wide_row_off(q) + 1172 s + 586 t
constexpr int kWideRowsS = 1172, kWideRowsT = 586;
static_assert(wide_row_off(16) == kWideRowsS * 1 + 0 && wide_row_off(8) == kWideRowsT &&
                  wide_row_off(24 + 7) == wide_row_off(7) + kWideRowsS + kWideRowsT,
              "row offsets split into a row-group part and a per-lane part");
static_assert(kWideTileDma == 37 && 4 * (kWideDmaPerWave - 1) == kWideTileDma - 1,
              "instructions 0-8 of every wave and instruction 9 of wave 0 fill the tile");

// Row of tile chunk c (the pad chunks after a row count as that row's; c past
// the tile gives row 31).
__device__ __forceinline__ int wide_row_of(int c) {
  int r = min(c / 74, 31);  // 72 r <= wide_row_off(r) <= 74 r: the row is r or r + 1
  if (r < 31 && wide_row_off(r + 1) <= c) ++r;
  return r;
}

__device__ __forceinline__ f32x16 mfma32x32x16(const u32x4& a, const u32x4& b,
                                               const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
      __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The QK MFMAs with their 32 x 32 accumulator in VGPRs.  The output
// accumulators take all 256 AGPRs, and the compiler gives every MFMA of a
// function that uses AGPRs an AGPR accumulator: the scores would then
// compete with the outputs for AGPRs and be shuttled between the register
// files.  qk_first starts a chain (accumulator 0), qk_next continues it
// (back-to-back accumulation into the same registers needs no wait states),
// qk_last ends it with the wait states a VALU read of an XDL result needs
// (19 for a 16-pass MFMA, plus one on gfx950: 21 here), which the compiler's
// hazard tracking does not know about for inline assembly.  The memory
// clobber keeps LDS reads on the side of each MFMA where the source puts
// them (the kernel places its reads a few MFMAs ahead of their use).
__device__ __forceinline__ void qk_first(f32x16& c, const u32x4& a, const u32x4& b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b) : "memory");
}
__device__ __forceinline__ void qk_next(f32x16& c, const u32x4& a, const u32x4& b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b) : "memory");
}
__device__ __forceinline__ void qk_last(f32x16& c, const u32x4& a, const u32x4& b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0\n\ts_nop 7\n\ts_nop 7\n\ts_nop 4"
               : "+v"(c)
               : "v"(a), "v"(b)
               : "memory");
}

// One 16-byte chunk per lane from global memory into LDS, from the
// wave-uniform 64-bit base `sbase` (SGPRs) plus the lane's 32-bit byte offset:
// lane i of the wave writes lds_base + 16 i (lds_base wave-uniform, in
// bytes).  Written as inline assembly: the compiler then does not see an LDS
// write whose completion it would wait for (vmcnt(0)) before every later LDS
// read, which would drain the blocks in flight; the kernel waits for
// completion itself (wide_wait_barrier).  Vector memory loads complete in
// issue order, so the waits the compiler computes for its own loads stay
// sufficient.
__device__ __forceinline__ void wide_dma16_s(uint32_t off, const void* sbase,
                                             uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(sbase), "s"(lds_base)
               : "memory");
}

// The same with the LDS destination lds_base + imm, imm a constant once the
// caller's loop is unrolled (one scalar add into M0).
__device__ __forceinline__ void wide_dma16_add(uint32_t off, const void* sbase,
                                               uint32_t lds_base, int imm) {
  asm volatile("s_add_u32 m0, %2, %3\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(sbase), "s"(lds_base), "i"(imm)
               : "memory", "scc");
}

// The largest of three (one NaN: of the others), without the quieting operations
// the compiler puts in front of fmaxf on what inline assembly computed.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

// Waits until at most N vector memory operations of this wave are in flight
// and its LDS reads are done, then joins the workgroup barrier.
template <int N>
__device__ __forceinline__ void wide_wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// Waits for this wave's LDS operations and joins the workgroup barrier.
__device__ __forceinline__ void wide_lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
}
// Waits for this wave's LDS operations (its own LDS writes before it reads
// other lanes' values back).
__device__ __forceinline__ void wide_lds_wait() {
  asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
}

// Stores `rows` (0, 16 or 32) staged 1 KB rows (row h at src + 260 h dwords,
// lane part at src) to dst + h * row_bytes + col_byte, eight rows' LDS reads in
// flight before their stores.
__device__ __forceinline__ void wide_store_rows(char* dst, int row_bytes, const uint32_t* src,
                                                int col_byte, int rows) {
#pragma unroll
  for (int h0 = 0; h0 < 32; h0 += 8) {
    if (h0 >= rows) break;
    u32x4 v[8];
#pragma unroll
    for (int h = 0; h < 8; ++h) v[h] = *(const u32x4*)(src + (h0 + h) * 260);
#pragma unroll
    for (int h = 0; h < 8; ++h)
      *(u32x4*)(dst + (size_t)(h0 + h) * row_bytes + col_byte) = v[h];
  }
}

}  // namespace ws
