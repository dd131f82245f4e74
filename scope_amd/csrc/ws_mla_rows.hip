// Absorbed-MLA attention of any number of query rows over the latent pages (gfx950):
// prompts, chunks of them and drafted tokens over bf16 or 8-bit pages (causal, ragged),
// and decode over 8-bit pages.
//
// A sequence's rows are its (new token, head) pairs, row = i H + h, which lie one after
// the other in q_nope, q_pe, out and lse.  All of them read the same latents, so a
// workgroup takes a tile of 128 rows, a wave 32 of them, and walks the tokens in blocks
// of 32 that the four waves load to LDS together:
//   S^T[token][row] = L Q^T       576 columns, A = the latents, B = Q in registers
//   O^T[column][row] += L^T P^T   512 columns, A = the latents read transposed, B = P as
//                                 it comes out of S^T
// Token t's row sees the tokens 0 .. its own position (prompts), so a tile ends at the
// last row's and masks the blocks that its first row does not see whole.
//
// The step, its loads and the fixed reference of the softmax are ws_mla_wide.h's: block
// k + 1's scores and block k's values' product interleaved, the output in 256
// accumulator registers that nothing rescales.
//
// 8-bit pages (e4m3, a power of two per `block` tokens) lie in LDS as they are, half the
// bytes, and are never widened for the scores: v_mfma_scale_f32_32x32x64_f8f6f4 takes
// e4m3 operands with a power of two per 32 columns, so the latents enter with their
// tokens' scales as they are stored.  The query is split into two e4m3 values,
//   q = 2^e (hi + lo / 16),  hi = e4m3(q / 2^e), lo = e4m3(16 (q / 2^e - hi)),
// e the least that keeps the row's largest at 448: bf16 has 8 significant bits, e4m3 has 4,
// and the rest of a rounding to 4 of 8 bits has 4, so the split is exact for every column
// within 2^-14 of the row's largest (2^-22 of it for the smaller ones).  Two products at
// twice the bf16 rate take the time of one in bf16, without the 144 conversions that
// widening would cost a wave and block.  The values' product has P in bf16: its operand is
// read transposed in 8 bits and widened (four instructions an MFMA), and a token's scale
// goes to its probability instead of its 512 columns.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "ws_attn.h"
#include "ws_mla_ring.h"
#include "ws_plan.h"
#include "ws_reduce.h"

namespace ws {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kRowsC = 512;
constexpr int kRowsPe = 64;
constexpr int kRowsTile = 128;       // rows of a tile, 32 a wave
constexpr int kRowsMaxSplits = 256;  // of a tile
constexpr int kRowsMinShare = 4;     // blocks of a split, at the least

struct RowsParams {
  const uint16_t* q_nope;
  const uint16_t* q_pe;
  const void* latent;
  const uint8_t* scale;  // 8-bit pages
  const int32_t* page_table;
  const int32_t* kv_len;
  const int32_t* cu_new;  // nullptr: one row of tokens a sequence (decode)
  uint16_t* out_bf16;
  float* out_f32;
  float* lse;
  float* part_out;  // [pieces][piece_rows][512], with part_lse [pieces][piece_rows]
  float* part_lse;
  int N, B, H, page_size, max_pages, num_pages, cap, block_log2;
  int n_splits;  // of every tile; 0: by the lengths, about `fill` workgroups in all
  int fill;
  bool fit;       // the tiles are fewer than `fill`: all items are to fit
  int pieces;     // room for them
  int piece_rows;
  float scale_log2;  // > 0
  uint32_t q_sign;   // 0x80008000 where the caller's scale is negative
};

// ---------------------------------------------------------------------------
// which rows and tokens a workgroup takes

struct RowsSeq {
  int c0, n, len, tiles, blocks;
};
__device__ __forceinline__ RowsSeq rows_seq(const RowsParams& p, int b) {
  RowsSeq s;
  s.c0 = b;
  s.n = 1;
  if (p.cu_new) {
    s.c0 = min(max(p.cu_new[b], 0), p.N);
    s.n = min(max(p.cu_new[b + 1], s.c0), p.N) - s.c0;
  }
  s.len = p.kv_len[b];
  s.tiles = (s.n * p.H + kRowsTile - 1) / kRowsTile;
  s.blocks = len_ok(s.len, 0, p.cap) ? (s.len + 31) / 32 : 0;
  return s;
}

struct RowsPlace {
  int b;              // the sequence (< 0: past the list's end)
  int tile;           // tile of its rows
  int split, splits;  // and which of the tile's splits
  int piece;          // a split tile's piece
  int c0, n, len;
};

// Item `at` of the list of all tiles' splits (TILES: of all tiles): longest sequences
// first (up to 64 of them), their last tile first.  A tile has one split for every M of
// its sequence's blocks, M the batch's blocks over `fill` workgroups, and where the tiles
// alone are fewer than those the least M (within 2^-6) at which all items fit.  Every
// kernel of a call finds the same.  Every lane must call it; the result is uniform.
template <bool TILES>
__device__ __forceinline__ RowsPlace rows_place(const RowsParams& p, int at) {
  constexpr int kRegs = 4;  // sequences a lane holds while M is searched
  const int lane = threadIdx.x & 63;
  const int per = (p.B + 63) >> 6;
  const int b0 = lane * per;
  float rM = 0.f;
  if (p.n_splits == 0) {
    int til[kRegs] = {}, blk[kRegs] = {};
    unsigned long long total = 0;
    int tiles = 0, longest = 0;
    for (int k = 0; k < per && b0 + k < p.B; ++k) {
      const RowsSeq s = rows_seq(p, b0 + k);
#pragma unroll
      for (int j = 0; j < kRegs; ++j)
        if (k == j) {
          til[j] = s.tiles;
          blk[j] = s.blocks;
        }
      total += (unsigned long long)s.tiles * (unsigned)s.blocks;
      tiles += s.tiles;
      longest = max(longest, s.blocks);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      total += __shfl_xor(total, o);
      tiles += __shfl_xor(tiles, o);
      longest = max(longest, __shfl_xor(longest, o));
    }
    auto blocks_at = [&](int places) {
      const double m = (double)total / (double)max(places, 1);
      return (int)ceil(min(max(m, (double)kRowsMinShare), 1e9));
    };
    int M = blocks_at(p.fill);
    if (p.fit) {
      auto fits = [&](int m) {
        const float r = __builtin_amdgcn_rcpf((float)m);
        int items = 0;
        for (int j = 0; j < kRegs; ++j) {
          if (j >= per) break;
          items += til[j] * max(plan_nsplits(blk[j], r), 1);
        }
        return uniform((int)__ockl_wfred_add_u32((unsigned)items)) <= p.fill;
      };
      int lo = M;
      int hi = uniform(max(min(blocks_at(p.fill - tiles), longest), lo));
      if (!fits(lo)) {
        if (!fits(hi)) hi = max(longest, 1);  // (a split a sequence and tile)
        for (int i = 0; i < 6 && hi - lo > 1; ++i) {
          const int mid = (lo + hi) >> 1;
          if (fits(mid)) hi = mid;
          else lo = mid;
        }
        M = hi;
      }
    }
    rM = __builtin_amdgcn_rcpf((float)M);
  }
  auto splits_of = [&](const RowsSeq& s) {
    if (p.n_splits > 0) return p.n_splits;
    return min(max(plan_nsplits(s.blocks, rM), 1), kRowsMaxSplits);
  };
  // a lane's items, and the pieces before its first sequence in the batch's order
  int items = 0, units = 0, key = -1;
  for (int k = 0; k < per && b0 + k < p.B; ++k) {
    const RowsSeq s = rows_seq(p, b0 + k);
    const int splits = splits_of(s);
    units += splits > 1 ? s.tiles * splits : 0;
    items += TILES ? s.tiles : s.tiles * splits;
    key = s.blocks;
  }
  const int before = __ockl_wfscan_add_i32(units, true) - units;
  int from = lane;  // the lane whose sequences stand at this lane's place in the list
  if (!TILES && per == 1 && p.B > 1) {
    int rank = 0;
    for (int j = 0; j < p.B; ++j) {
      const int other = __builtin_amdgcn_readlane(key, j);
      rank += other > key || (other == key && j < lane) ? 1 : 0;
    }
    if (lane >= p.B) rank = lane;
    from = __builtin_amdgcn_ds_permute(4 * rank, lane);
    items = __builtin_amdgcn_ds_permute(4 * rank, items);
  }
  const int incl = __ockl_wfscan_add_i32(items, true);
  const uint64_t past = __builtin_amdgcn_ballot_w64(incl > at);
  RowsPlace r{-1, 0, 0, 1, 0, 0, 0, 0};
  if (past == 0) return r;
  const int slot = __builtin_ctzll(past);
  int left = at - __builtin_amdgcn_readlane(incl - items, slot);
  const int owner = __builtin_amdgcn_readlane(from, slot);
  int piece = __builtin_amdgcn_readlane(before, owner);
  for (int k = 0; k < per; ++k) {
    const int b = uniform(owner * per + k);
    if (b >= p.B || left < 0) break;  // (left < 0: sums past 2^31, cu_new not non-decreasing)
    const RowsSeq s = rows_seq(p, b);
    const int splits = uniform(splits_of(s));
    const int tiles = uniform(s.tiles);
    const int here = TILES ? tiles : tiles * splits;
    if (left < here) {
      const int t = TILES ? left : left / splits;
      r.b = b;
      r.tile = TILES ? t : tiles - 1 - t;
      r.split = TILES ? 0 : left - t * splits;
      r.splits = splits;
      r.piece = piece + r.tile * splits + r.split;
      r.c0 = uniform(s.c0);
      r.n = uniform(s.n);
      r.len = uniform(s.len);
      break;
    }
    left -= here;
    piece += splits > 1 ? tiles * splits : 0;
  }
  return r;
}

// ---------------------------------------------------------------------------
// the LDS ring

template <bool F8>
struct RowsRing;
// bf16: ws_mla_wide.h's tiles, three blocks ahead.
template <>
struct RowsRing<false> {
  static constexpr int kTiles = kWideTiles;
  static constexpr int kDma = kWideTileDma;  // 1 KB load instructions of a block
  static constexpr int kPer = kWideDmaPerWave;
  static constexpr int kRowBytes = 1152;
  static constexpr int kRowsS = kWideRowsS;
  __host__ __device__ static constexpr int row_off(int r) { return wide_row_off(r); }
  __device__ static int row_of(int c) { return wide_row_of(c); }
};
// 8 bits: rows of 36 chunks of 16 bytes and one chunk of padding every four rows, so that
// the score reads (16 rows, one chunk each) meet 16 chunk slots mod 16 and the transposed
// reads (rows 4 j .. 4 j + 3 and 8 more, 32 bytes of each) 8 different pairs of them.  19
// instructions fill a tile: five a wave but the last, whose fifth loads the block's scales.
template <>
struct RowsRing<true> {
  static constexpr int kTiles = 8;
  static constexpr int kDma = 19;
  static constexpr int kPer = 5;
  static constexpr int kRowBytes = 576;
  static constexpr int kRowsS = 580;  // chunks from row r to r + 16
  __host__ __device__ static constexpr int row_off(int r) { return 36 * r + (r >> 2); }
  __device__ static int row_of(int c) {
    const int g = min(c / 145, 7);
    return 4 * g + min((c - 145 * g) / 36, 3);
  }
};
static_assert(RowsRing<true>::row_off(31) + 36 <= 64 * RowsRing<true>::kDma, "a tile's chunks");
static_assert(RowsRing<true>::row_off(16 + 8 + 4 + 3) == 580 + 290 + 145 + 108, "row offsets add up");

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes a lane from sbase + off to LDS at lds + imm + 16 * lane (ws_mla_ring.h, with the
// wait state that an m0 just written asks for).
__device__ __forceinline__ void rows_dma16(uint32_t off, const void* sbase, uint32_t lds, int imm) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(sbase), "s"(lds), "i"(imm)
               : "memory", "scc", "m0");
}
// One byte a lane to the dword at lds + 4 * lane.
__device__ __forceinline__ void rows_dma1(uint32_t off, const void* sbase, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, %1"
               :
               : "v"(off), "s"(sbase), "s"(lds)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// Score products with their accumulator in VGPRs (ws_mla_ring.h qk_*).  The s_nop: the
// latents' registers may just have been moved, which the compiler does not see an MFMA
// read here.
__device__ __forceinline__ void qk8_first(f32x16& c, const i32x8& a, const i32x8& b, int sa,
                                          int sb) {
  asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, 0, %3, %4 op_sel_hi:[0,0,0]"
               : "=&v"(c)
               : "v"(a), "v"(b), "v"(sa), "v"(sb)
               : "memory");
}
__device__ __forceinline__ void qk8_next(f32x16& c, const i32x8& a, const i32x8& b, int sa,
                                         int sb) {
  asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
               : "+v"(c)
               : "v"(a), "v"(b), "v"(sa), "v"(sb)
               : "memory");
}
// The wait states that a VALU read of the last product's result asks for (16 passes and
// four).
__device__ __forceinline__ void qk_settle(f32x16& c) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(c) : : "memory");
}
// The same with two other MFMAs issued in between (each waits for the one before it).
__device__ __forceinline__ void qk_settle_short(f32x16& c) {
  asm volatile("s_nop 3" : "+v"(c) : : "memory");
}

// Has a value in registers at this point.  (A function: as a statement of the kernel itself,
// the host's compiler refuses the wider registers and leaves the kernel out.)
template <class T>
__device__ __forceinline__ void hold(T& x) {
  asm volatile("" : "+v"(x) : : "memory");
}

// Four columns of a query (bf16 pairs w0, w1) over `unit` as e4m3, and what that leaves
// over `sub`.
__device__ __forceinline__ void split_query4(uint32_t w0, uint32_t w1, float unit, float sub,
                                             int& hi, int& lo) {
  typedef short s16x2_t __attribute__((ext_vector_type(2)));
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  s16x2_t h8 = {0, 0}, l8 = {0, 0};
  h8 = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h8, __builtin_bit_cast(bf16x2_t, w0), unit, false);
  h8 = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h8, __builtin_bit_cast(bf16x2_t, w1), unit, true);
  const uint32_t hw = __builtin_bit_cast(uint32_t, h8);
  const f32x2_t b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hw, unit, false);
  const f32x2_t b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hw, unit, true);
  const float r0 = __builtin_bit_cast(float, w0 << 16) - b0[0];
  const float r1 = __builtin_bit_cast(float, w0 & 0xffff0000u) - b0[1];
  const float r2 = __builtin_bit_cast(float, w1 << 16) - b1[0];
  const float r3 = __builtin_bit_cast(float, w1 & 0xffff0000u) - b1[1];
  l8 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l8, r0, r1, sub, false);
  l8 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l8, r2, r3, sub, true);
  hi = (int)hw;
  lo = __builtin_bit_cast(int, l8);
}

template <bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
}
// Eight e4m3 values as bf16 (exact).
__device__ __forceinline__ u32x4 widen8(const uint2& w) {
  return u32x4{widen2<false>(w.x), widen2<true>(w.x), widen2<false>(w.y), widen2<true>(w.y)};
}
// ds_read_b64_tr_b8: in each 16-lane group lanes 2 e and 2 e + 1 address the halves of
// row e's 16 bytes; result lane i holds byte i of rows 0 .. 7 (measured in bounds).
__device__ __forceinline__ uint2 lds_read_tr8_b64(uint32_t addr) {
  typedef int i32x2_t __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) i32x2_t lds_i32x2_t;
  const i32x2_t v = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_t*)(uintptr_t)addr);
  return make_uint2((uint32_t)v[0], (uint32_t)v[1]);
}

// Stores `rows` staged 1 KB rows (row h at src + 260 h dwords, lane part at src) to dst + h *
// row_bytes + col_byte.
__device__ __forceinline__ void rows_store(char* dst, int row_bytes, const uint32_t* src,
                                           int col_byte, int rows) {
#pragma unroll
  for (int h0 = 0; h0 < 32; h0 += 8) {
    if (h0 >= rows) break;
    u32x4 v[8];
#pragma unroll
    for (int h = 0; h < 8; ++h) v[h] = *(const u32x4*)(src + (h0 + h) * 260);
#pragma unroll
    for (int h = 0; h < 8; ++h)
      if (h0 + h < rows) *(u32x4*)(dst + (size_t)(h0 + h) * row_bytes + col_byte) = v[h];
  }
}

// What a bf16 pair holds of infinities and NaN: their halves' bits, all set.
__device__ __forceinline__ uint32_t nonfinite_halves(uint32_t w) {
  const uint32_t hit = (((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15;
  return hit * 0xffffu;
}
// The bytes of four e4m3 values that are NaN, all set.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t hit = (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
  return hit * 0xffu;
}

template <bool F8>
__global__ __launch_bounds__(256) void mla_rows_kernel(const RowsParams p) {
  using R = RowsRing<F8>;
  constexpr int kAlloc = 64 * R::kDma;
  constexpr int kAhead = R::kTiles - 1;  // blocks requested ahead of the one whose values are taken
  constexpr int kRow = R::kRowBytes;
  constexpr int kChunks = kRow / 16;
  __shared__ u32x4 s_tile[R::kTiles][kAlloc];
  __shared__ u32x4 s_sink[F8 ? 1 : 64];
  __shared__ uint32_t s_scale[F8 ? R::kTiles : 1][64];
  __shared__ int s_redo;
  static_assert(R::kTiles * kAlloc >= kRowsTile * 65, "the queries are staged in the tiles");
  const int tid = threadIdx.x;
  const int wave = uniform(tid >> 6);
  const int lane = tid & 63;
  const int n32 = lane & 31;  // row of the wave (QK B, PV B, output) or token (A operands)
  const int j2 = lane >> 5;
  const int H = p.H;

  const RowsPlace pl = rows_place<false>(p, blockIdx.x);
  const bool piece = pl.splits > 1;
  if (pl.b < 0 || (piece && (pl.piece < 0 || pl.piece >= p.pieces))) return;
  if (tid == 0) s_redo = 0;  // read after the ring's barriers
  const int R_all = pl.n * H;
  const int row0 = pl.tile * kRowsTile;
  const int here = min(kRowsTile, R_all - row0);
  const int rows = min(max(here - 32 * wave, 0), 32);  // this wave's
  const bool len_good = len_ok(pl.len, 0, p.cap);
  const int first_pos = pl.len - pl.n;  // position of the sequence's first query
  // tokens that the tile's first row and its last one see
  const int lim_lo = first_pos + row0 / H + 1;
  const int lim_hi = len_good ? max(first_pos + (row0 + here - 1) / H + 1, 0) : 0;
  const int nb = (lim_hi + 31) / 32;
  const int blk0 = (int)((long long)pl.split * nb / pl.splits);
  const int blk1 = (int)((long long)(pl.split + 1) * nb / pl.splits);
  const int nblk = blk1 - blk0;
  const int t_begin = 32 * blk0;
  const int t_end = min(lim_hi, 32 * blk1);
  const size_t g_row0 = (size_t)pl.c0 * H + row0;  // of q, out and lse
  const size_t o_row0 = piece ? (size_t)pl.piece * p.piece_rows : g_row0;
  if (nblk <= 0) {  // nothing to see: (0, -inf), or NaN for an invalid length
    const float fill = len_good ? 0.f : qnan();
    for (int x = tid; x < here * (kRowsC / 4); x += 256) {
      const size_t at = o_row0 * (kRowsC / 4) + x;
      if (piece) {
        ((float4*)p.part_out)[at] = make_float4(fill, fill, fill, fill);
      } else {
        if (p.out_f32) ((float4*)p.out_f32)[at] = make_float4(fill, fill, fill, fill);
        if (p.out_bf16) ((uint2*)p.out_bf16)[at] = make_uint2(pack_bf16x2(fill, fill), pack_bf16x2(fill, fill));
      }
    }
    if (tid < here) {
      const float l = len_good ? neg_inf() : qnan();
      if (piece) p.part_lse[o_row0 + tid] = l;
      else if (p.lse) p.lse[o_row0 + tid] = l;
    }
    return;
  }
  // the tokens that the lane's row sees (past the rows: the last one again)
  const int lim_lane = first_pos + min(row0 + 32 * wave + n32, R_all - 1) / H + 1;

  const uint32_t tile_base0 = (uint32_t)uniform((int)(uint32_t)(uintptr_t)&s_tile[0][0]);
  const uint32_t sink_base = (uint32_t)uniform((int)(uint32_t)(uintptr_t)&s_sink[0]);
  const uint32_t scale_base = (uint32_t)uniform((int)(uint32_t)(uintptr_t)&s_scale[0][0]);
  // Byte offsets, within a block's rows in HBM, of the chunks this lane loads, two to a
  // register (the largest is 31 * 1152 + 1136).
  constexpr int kOff = (R::kPer + 1) / 2;
  uint32_t offp[kOff];
#pragma unroll
  for (int j = 0; j < kOff; ++j) {
    uint32_t v = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 64 * min(wave + 4 * (2 * j + h), R::kDma - 1) + lane;
      const int r = R::row_of(c);
      const int x = min(c - R::row_off(r), kChunks - 1);
      v |= (uint32_t)(r * kRow + 16 * x) << (16 * h);
    }
    offp[j] = v;
  }
  // Per-lane part of the transposed reads.  bf16: lane 4 e + r of a 16-lane group
  // addresses token row 4 j2 + e, columns 4 r .. 4 r + 3 of the group's 16.  8 bits: lanes 2
  // e and 2 e + 1 token row 8 (e / 4) + 4 j2 + e % 4, 8 columns each.
  const uint32_t v_lane = [&] {
    const int ch = (lane >> 4) & 1;
    if constexpr (F8) {
      const int e = (lane & 15) >> 1;
      return (uint32_t)(16 * R::row_off(8 * (e >> 2) + 4 * j2 + (e & 3)) + 16 * ch + 8 * (lane & 1));
    } else {
      const int e = (lane >> 2) & 3, r = lane & 3;
      return (uint32_t)(16 * R::row_off(4 * j2 + e) + 2 * (16 * ch + 4 * r));
    }
  }();

  // Pool token index of the first row of each block, 64 at a time (lane l: block pid_base +
  // l); a page id outside the pool is clamped and marks the index with bit 31.
  const int32_t* pt = p.page_table + (size_t)pl.b * p.max_pages;
  int pid_base = 0;
  int m_tok = 0;
  uint32_t bad_bits = 0;  // of the blocks requested last: whether their page id was bad
  auto first_tok = [&]() __attribute__((always_inline)) {
    return t_begin + 32 * min(pid_base + lane, nblk - 1);
  };
  auto set_pids = [&](int raw) __attribute__((always_inline)) {
    const int t0 = first_tok();
    const int page = t0 / p.page_size;
    const int pid = clamp_page(raw, p.num_pages);
    m_tok = (pid * p.page_size + (t0 - page * p.page_size)) | (raw == pid ? 0 : (int)0x80000000u);
  };
  auto fetch_pids = [&]() __attribute__((always_inline)) { set_pids(pt[first_tok() / p.page_size]); };
  int raw_pid = pt[first_tok() / p.page_size];

  // Q^T of this wave's rows, through LDS a 1 KB row an instruction (row slots of 65 chunks).
  // bf16: k-step u holds columns 16 u + 8 j2 .. + 8; 8 bits: 64 u + 32 j2 .. + 32, hi and lo.
  constexpr int kSteps = F8 ? 9 : 36;
  using QReg = typename std::conditional<F8, i32x8, u32x4>::type;
  QReg qb[F8 ? 18 : 36];
  float sx = p.scale_log2;  // of the raw scores
  {
    const uint16_t* qrow0 = p.q_nope + (g_row0 + 32 * wave) * kRowsC;
    const uint32_t qst = tile_base0 + (uint32_t)(32 * wave * 65 * 16);
    if (rows > 0)
      for (int h = 0; h < 32; ++h)
        rows_dma16(16 * lane, qrow0 + (size_t)min(h, rows - 1) * kRowsC, qst + (uint32_t)(h * 65 * 16), 0);
    const u32x4* pe =
        (const u32x4*)(p.q_pe + (g_row0 + min(32 * wave + n32, here - 1)) * kRowsPe);
    u32x4 pe_q[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) pe_q[c] = pe[F8 ? 4 * j2 + c : 2 * c + j2];
    asm volatile("s_waitcnt vmcnt(0)" : "+v"(raw_pid) : : "memory");
    set_pids(raw_pid);
    const u32x4* qs = &s_tile[0][0] + (32 * wave + n32) * 65;
    if constexpr (F8) {
      auto chunk = [&](int u, int c) __attribute__((always_inline)) {
        return u < 8 ? qs[8 * u + 4 * j2 + c] : pe_q[c];
      };
      uint32_t top = 0;  // the row's largest magnitude (bf16 bits)
#pragma unroll
      for (int u = 0; u < 9; ++u)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const u32x4 w = chunk(u, c);
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max(top, max(w[e] & 0x7fffu, (w[e] >> 16) & 0x7fffu));
        }
      top = max(top, (uint32_t)__shfl_xor((int)top, 32));
      // 2^e with top <= 448 2^e (and 2^(e - 4) normal); a row with an infinity or a NaN is
      // NaN whole
      const int byte = max((int)(((top << 16) + 0x1fffffu) >> 23) - 8, 5);
      const float unit = __builtin_bit_cast(float, (uint32_t)byte << 23);
      const float sub = __builtin_bit_cast(float, (uint32_t)(byte - 4) << 23);
      sx = top >= 0x7f80u ? qnan() : fmaxf(sx * unit, 1.17549435e-38f);
#pragma unroll
      for (int u = 0; u < 9; ++u) {
        int hi[8], lo[8];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const u32x4 w = chunk(u, c) ^ p.q_sign;
          split_query4(w[0], w[1], unit, sub, hi[2 * c], lo[2 * c]);
          split_query4(w[2], w[3], unit, sub, hi[2 * c + 1], lo[2 * c + 1]);
        }
        qb[2 * u] = i32x8{hi[0], hi[1], hi[2], hi[3], hi[4], hi[5], hi[6], hi[7]};
        qb[2 * u + 1] = i32x8{lo[0], lo[1], lo[2], lo[3], lo[4], lo[5], lo[6], lo[7]};
        // one k-step's registers at a time
        hold(qb[2 * u]);
        hold(qb[2 * u + 1]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < 36; ++u) qb[u] = (u < 32 ? qs[2 * u + j2] : pe_q[u - 32]) ^ p.q_sign;
    }
  }
  // the queries in registers, and every wave done with its staged rows, before the loads
#pragma unroll
  for (int u = 0; u < (F8 ? 18 : 36); ++u) hold(qb[u]);
  wide_lds_barrier();

  // Block k into tile k % kTiles: this wave's kPer instructions.  Rows past t_end read the
  // last row's last chunk; a block past the last is the last one again, in a tile that
  // nothing reads.
  const char* g0 = (const char*)p.latent;
  struct Dma {
    const char* sb;
    const uint8_t* ss;
    uint32_t wbase, last, lim, lim_s;
  };
  auto issue_begin = [&](int k) __attribute__((always_inline)) {
    const int kc = min(k, nblk - 1);
    if (kc - pid_base >= 64) {
      pid_base += 64;
      fetch_pids();
    }
    const int tok_raw = __builtin_amdgcn_readlane(m_tok, kc - pid_base);
    const uint32_t bit = 1u << (k & 31);
    bad_bits = tok_raw < 0 ? bad_bits | bit : bad_bits & ~bit;
    const uint32_t tok = (uint32_t)tok_raw & 0x7fffffffu;
    const int nt = min(t_end - (t_begin + 32 * kc), 32);
    Dma d;
    d.sb = g0 + (size_t)tok * kRow;
    d.lim = nt >= 32 ? 0xffffu : (uint32_t)((nt - 1) * kRow + 16 * (kChunks - 1));
    const int slot = k & (R::kTiles - 1);
    const uint32_t tb = tile_base0 + (uint32_t)slot * (kAlloc * 16);
    d.wbase = tb + 1024 * wave;
    if constexpr (F8) {
      d.ss = p.scale + (tok >> p.block_log2);
      d.lim_s = (uint32_t)(nt - 1) >> p.block_log2;
      d.last = scale_base + 256 * slot;
    } else {
      d.last = wave == 0 ? tb + 1024 * (R::kDma - 1) : sink_base;
    }
    // recomputed per block (not hoisted)
    asm volatile("" : "+s"(d.wbase), "+s"(d.last));
    return d;
  };
  auto dma_one = [&](const Dma& d, int i) __attribute__((always_inline)) {
    asm volatile("" : "+v"(offp[i >> 1]));  // unpacked at each use
    const uint32_t pr = offp[i >> 1];
    const uint32_t off = min((i & 1) ? pr >> 16 : pr & 0xffffu, d.lim);
    if (i < R::kPer - 1) {
      rows_dma16(off, d.sb, d.wbase, 4 * 1024 * i);
    } else if constexpr (F8) {
      if (wave == 3)
        rows_dma1(min((uint32_t)n32 >> p.block_log2, d.lim_s), d.ss, d.last);
      else
        rows_dma16(off, d.sb, d.wbase, 4 * 1024 * i);
    } else {
      rows_dma16(off, d.sb, d.last, 0);
    }
  };
  auto issue = [&](int k) __attribute__((always_inline)) {
    const Dma d = issue_begin(k);
#pragma unroll
    for (int i = 0; i < R::kPer; ++i) dma_one(d, i);
  };

  f32x16 acc[16];
  float m_run = neg_inf();  // reference of the lane's row: its largest score in the first block
  float m_max = neg_inf();  // the lane's largest raw score so far
  float l_run = 0.f;  // bf16: the lane's sum of probabilities as rounded
  float s_run = 0.f;  // and in fp32

  // QK operand u of a tile, and its product
  using KReg = QReg;
  const u32x4* arow0 = &s_tile[0][0] + R::row_off(n32) + (F8 ? 2 * j2 : j2);
  auto qk_read = [&](int tile, int u) __attribute__((always_inline)) {
    if constexpr (F8) {
      const u32x4 a = arow0[tile * kAlloc + 4 * u], b = arow0[tile * kAlloc + 4 * u + 1];
      return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
    } else {
      return arow0[tile * kAlloc + 2 * u];
    }
  };
  // link v of the chain: bf16 k-step v; 8 bits k-step v / 2, hi then lo (2^-4)
  constexpr int kLinks = F8 ? 18 : 36;
  int one = 127, sixteenth = 123;
  auto qk_link = [&](f32x16& sc, const KReg& kr, int tok_scale, int v) __attribute__((always_inline)) {
    if constexpr (F8) {
      if (v == 0) qk8_first(sc, kr, qb[0], tok_scale, one);
      else qk8_next(sc, kr, qb[v], tok_scale, (v & 1) ? sixteenth : one);
    } else {
      if (v == 0) qk_first(sc, kr, qb[0]);
      else qk_next(sc, kr, qb[v]);
    }
  };
  auto vbase = [&](int tile) __attribute__((always_inline)) {
    uint32_t vl = v_lane;
    asm volatile("" : "+v"(vl));  // (one register, the rest in the instruction's offset)
    return tile_base0 + (uint32_t)tile * (kAlloc * 16) + vl;
  };
  // V^T operand of MFMA m (tokens 16 (m / 16) .., columns 32 (m % 16) ..), as read
  using VReg = typename std::conditional<F8, uint2, u32x4>::type;
  auto vread = [&](uint32_t vt, int m) __attribute__((always_inline)) {
    const int sv = m >> 4, ct = m & 15;
    const uint32_t a = vt + 16 * R::kRowsS * sv + (F8 ? 32 : 64) * ct;
    if constexpr (F8) {
      return lds_read_tr8_b64(a);
    } else {
      const uint2 lo = lds_read_tr_b64(a);
      const uint2 hi = lds_read_tr_b64(a + 16 * kWideRowsT);
      return u32x4{lo.x, lo.y, hi.x, hi.y};
    }
  };
  auto widened = [&](const VReg& v) __attribute__((always_inline)) {
    if constexpr (F8) return widen8(v);
    else return v;
  };
  // the memory clobber keeps the operand reads where the source puts them
  auto pv_mfma = [&](const u32x4& va, const u32x4& pbs, int m) __attribute__((always_inline)) {
    f32x16& a = acc[m & 15];
    a = mfma32x32x16(va, pbs, a);
    asm volatile("" : "+a"(a));
    asm volatile("" : : : "memory");
  };
  // The scores of block kb in the log2 domain less the reference (xa: the first 16 tokens',
  // xh: the others').  In the blocks that the tile's first row does not see whole, a score
  // that a row does not see is -inf, and an infinity or a NaN in a token shows in its
  // score: a row that sees it is NaN, and where a row of the wave does not, the result is
  // true and the tile is cleaned before its values are taken.
  auto soft_x = [&](int kb, const f32x16& sc, float (&xa)[8], float (&xh)[8], bool first)
      __attribute__((always_inline)) {
    const int t0 = t_begin + 32 * kb;
    f32x16 v = sc;
    bool odd = false;
    const bool bad_page = (bad_bits >> (kb & 31)) & 1;
    if (t0 + 32 > lim_lo || bad_page) {
      int l = lane;  // recomputed here rather than kept live
      asm volatile("" : "+v"(l));
      const int lim = lim_lane - t0 - 4 * (l >> 5);
      bool hidden = false;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool seen = 8 * (i >> 2) + (i & 3) < lim;
        const bool finite = __builtin_fabsf(v[i]) < __builtin_inff();
        hidden |= !seen && !finite;
        const float x = bad_page || !finite ? qnan() : v[i];
        v[i] = seen ? x : neg_inf();
      }
      odd = __builtin_amdgcn_ballot_w64(hidden) != 0;
    }
    float r = max3(v[0], v[1], v[2]);
#pragma unroll
    for (int i = 3; i < 15; i += 2) r = max3(r, v[i], v[i + 1]);
    m_max = max3(r, v[15], m_max);
    if (first) {
      // a row that sees anything of these tokens sees the first block's first (none: 0)
      float lo, hi;
      pair_xor32(m_max * sx, lo, hi);
      m_run = m_run == neg_inf() ? fmaxf(lo, hi) : m_run;
      m_run = m_run == neg_inf() ? 0.f : m_run;
    }
    const float nm = -m_run;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      xa[i] = __builtin_fmaf(v[i], sx, nm);
      xh[i] = __builtin_fmaf(v[8 + i], sx, nm);
    }
    return odd;
  };
  // The scales of the tokens of dwords 2 g and 2 g + 1 of k-step s of P
  auto p_scales = [&](int tile, int s, int g) __attribute__((always_inline)) {
    if constexpr (F8) return *(const u32x4*)&s_scale[tile][16 * s + 8 * g + 4 * j2];
    else return u32x4{};
  };
  // One dword of a k-step's P^T (two exp2)
  auto soft_p = [&](float (&xs)[8], const u32x4& ts, u32x4& pbs, int dd) __attribute__((always_inline)) {
    xs[2 * dd] = __builtin_amdgcn_exp2f(xs[2 * dd]);
    xs[2 * dd + 1] = __builtin_amdgcn_exp2f(xs[2 * dd + 1]);
    if constexpr (F8) {
      const float s0 = __builtin_bit_cast(float, ts[2 * (dd & 1)] << 23);
      const float s1 = __builtin_bit_cast(float, ts[2 * (dd & 1) + 1] << 23);
      pbs[dd] = pack_bf16x2(xs[2 * dd] * s0, xs[2 * dd + 1] * s1);
    } else {
      typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
      const uint32_t pk = pack_bf16x2(xs[2 * dd], xs[2 * dd + 1]);
      pbs[dd] = pk;
      l_run = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pk),
                                              __builtin_bit_cast(bf16x2_t, 0x3f803f80u), l_run, false);
    }
  };
  auto soft_s = [&](const float (&xa)[8], const float (&xh)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s_run += xa[i] + xh[i];
  };
  auto token_scale = [&](int tile) __attribute__((always_inline)) {
    return F8 ? (int)s_scale[F8 ? tile : 0][n32] : 0;
  };
  auto scores = [&](int tile, f32x16& sc) __attribute__((always_inline)) {
    const int ts = token_scale(tile);
    KReg kr[2];
    kr[0] = qk_read(tile, 0);
#pragma unroll
    for (int v = 0; v < kLinks; ++v) {
      const int u = F8 ? v >> 1 : v;
      if ((!F8 || !(v & 1)) && u + 1 < kSteps) kr[(u + 1) & 1] = qk_read(tile, u + 1);
      qk_link(sc, kr[u & 1], ts, v);
    }
    qk_settle(sc);
  };
  auto probabilities = [&](int tile, float (&xa)[8], float (&xh)[8], u32x4 (&pb)[2])
      __attribute__((always_inline)) {
#pragma unroll
    for (int dd = 0; dd < 4; ++dd) soft_p(xa, p_scales(tile, 0, dd >> 1), pb[0], dd);
#pragma unroll
    for (int dd = 0; dd < 4; ++dd) soft_p(xh, p_scales(tile, 1, dd >> 1), pb[1], dd);
  };
  // A block's values' product by itself (its tile is in and synchronised)
  auto values = [&](int kk, float (&xa)[8], float (&xh)[8]) __attribute__((always_inline)) {
    const int tp = kk & (R::kTiles - 1);
    const uint32_t vt = vbase(tp);
    VReg va[4];
    u32x4 pb[2];
#pragma unroll
    for (int m = 0; m < 3; ++m) va[m] = vread(vt, m);
    probabilities(tp, xa, xh, pb);
#pragma unroll
    for (int m = 0; m < 32; ++m) {
      if (m + 3 < 32) va[(m + 3) & 3] = vread(vt, m + 3);
      pv_mfma(widened(va[m & 3]), pb[m >> 4], m);
    }
    soft_s(xa, xh);
  };
  // Takes the infinities and NaN out of block kk's tile, where some token that a row of the
  // wave does not see holds one (0 * inf would bring it into that row).  Behind the barrier
  // at which every wave has its scores of the tile; a row that sees one is NaN by its score
  // (soft_x), whatever it finds in the tile.
  auto clean = [&](int kk) __attribute__((always_inline)) {
    const int tp = kk & (R::kTiles - 1);
#pragma clang loop unroll(disable)
    for (int c = lane; c < kAlloc; c += 64) {
      u32x4 w = s_tile[tp][c];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] &= ~(F8 ? nan_bytes(w[e]) : nonfinite_halves(w[e]));
      s_tile[tp][c] = w;
    }
    if constexpr (F8)
      if (s_scale[tp][n32] == 255) s_scale[tp][n32] = 0;
    wide_lds_wait();
  };

  // Step kk of the ring (ws_mla_wide.h): block kk + 1's scores with block kk's values'
  // product between their links, block kk + kAhead's loads over them, and the softmax of
  // block kk + 1 beside the last products.
  auto step = [&](int kk, float (&xa)[8], float (&xh)[8], bool& odd) __attribute__((always_inline)) {
    const int tp = kk & (R::kTiles - 1), tq = (kk + 1) & (R::kTiles - 1);
    wide_wait_barrier<(kAhead - 2) * R::kPer>();
    if (__builtin_expect(odd, 0)) clean(kk);
    const Dma d = issue_begin(kk + kAhead);
    f32x16 sc;
    VReg va[4];
    u32x4 pb[2];
    const uint32_t vt = vbase(tp);
    const int ts = token_scale(tq);
    if constexpr (F8) {
      KReg kr[2];
      u32x4 sa = p_scales(tp, 0, 0), sb = p_scales(tp, 0, 1);
      kr[0] = qk_read(tq, 0);
#pragma unroll
      for (int m = 0; m < 3; ++m) va[m] = vread(vt, m);
      int m = 0;
      auto pv = [&]() __attribute__((always_inline)) {
        va[(m + 3) & 3] = vread(vt, m + 3);
        pv_mfma(widened(va[m & 3]), pb[m >> 4], m);
        if (m == 0) sa = p_scales(tp, 1, 0);
        if (m == 6) sb = p_scales(tp, 1, 1);
        if (m < 16 && (m & 3) == 1) soft_p(xh, m < 8 ? sa : sb, pb[1], m >> 2);
        ++m;
      };
#pragma unroll
      for (int v = 0; v < 18; ++v) {
        if (!(v & 1) && v + 2 < 18) kr[((v >> 1) + 1) & 1] = qk_read(tq, (v >> 1) + 1);
        qk_link(sc, kr[(v >> 1) & 1], ts, v);
        if (v == 0) {
          soft_p(xa, sa, pb[0], 0);
          soft_p(xa, sa, pb[0], 1);
        } else if (v == 1) {
          soft_p(xa, sb, pb[0], 2);
          soft_p(xa, sb, pb[0], 3);
        } else {
          pv();
          if (!(v & 1)) pv();
        }
        if (v % 3 == 2 && v < 15) dma_one(d, v / 3);
      }
    } else {
      KReg kr[5];
#pragma unroll
      for (int u = 0; u < 4; ++u) kr[u] = qk_read(tq, u);
#pragma unroll
      for (int m = 0; m < 3; ++m) va[m] = vread(vt, m);
#pragma unroll
      for (int u = 0; u < 36; ++u) {
        if (u + 4 < 36) kr[(u + 4) % 5] = qk_read(tq, u + 4);
        qk_link(sc, kr[u % 5], ts, u);
        if (u < 4) {
          soft_p(xa, u32x4{}, pb[0], u);
        } else if ((u - 4) % 4 != 3) {
          const int m = 3 * ((u - 4) / 4) + (u - 4) % 4;
          va[(m + 3) & 3] = vread(vt, m + 3);
          pv_mfma(va[m & 3], pb[m >> 4], m);
          if (m < 16 && (m & 3) == 1) soft_p(xh, u32x4{}, pb[1], m >> 2);
        }
        if (u % 4 == 2) dma_one(d, u / 4);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // (MFMAs 24 and 25 behind the last link)
#pragma unroll
    for (int m = 24; m < 32; ++m) {
      if (m == 26) {
        __builtin_amdgcn_sched_barrier(0);
        qk_settle_short(sc);
        odd = soft_x(kk + 1, sc, xa, xh, false);
      }
      if (m + 3 < 32) va[(m + 3) & 3] = vread(vt, m + 3);
      pv_mfma(widened(va[m & 3]), pb[1], m);
      if (m == 24) {
        asm volatile("" : "+v"(s_run));  // not ahead of the MFMA
        soft_s(xa, xh);
      }
      if (!F8 && m == 27) dma_one(d, 9);
    }
  };
  for (int pass = 0;; ++pass) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[e][i] = 0.f;
    l_run = 0.f;
    s_run = 0.f;
    if (pid_base != 0) {
      pid_base = 0;
      fetch_pids();
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) issue(k);
    wide_wait_barrier<(kAhead - 1) * R::kPer>();
    if (rows > 0) {
      float xa[8], xh[8];
      bool odd;
      {
        f32x16 sc;
        scores(0, sc);
        odd = soft_x(0, sc, xa, xh, true);
      }
#pragma clang loop unroll(disable)
      for (int k = 0; k + 1 < nblk; ++k) {
        step(k, xa, xh, odd);
      }
      wide_lds_barrier();
      if (__builtin_expect(odd, 0)) clean(nblk - 1);
      values(nblk - 1, xa, xh);
    } else {  // the ring's waits, barriers and loads alone
#pragma clang loop unroll(disable)
      for (int k = 0; k + 1 < nblk; ++k) {
        wide_wait_barrier<(kAhead - 2) * R::kPer>();
        issue(k + kAhead);
      }
      wide_lds_barrier();
    }
    {  // the row's largest score (both its lanes)
      float lo, hi;
      pair_xor32(m_max, lo, hi);
      m_max = fmaxf(lo, hi);
    }
    const float top = m_max * sx;
    // every load of the pass has landed and every wave is done with the tiles
    const bool climbed = __builtin_amdgcn_ballot_w64(top > m_run + kWideHeadroomLog2) != 0;
    if (rows > 0 && climbed && lane == 0) s_redo = 1;
    wide_wait_barrier<0>();
    const bool redo = s_redo != 0;
    wide_wait_barrier<0>();  // every wave has read s_redo
    if (tid == 0) s_redo = 0;
    if (pass > 0 || !redo) break;
    // scores climbed out of the reference's headroom: again, from the rows' largest
    m_run = top == neg_inf() ? 0.f : top;
  }

  float lo, hi;
  pair_xor32(s_run, lo, hi);
  const float s_tot = lo + hi;
  pair_xor32(F8 ? s_run : l_run, lo, hi);
  const float l_tot = lo + hi;
  const float inv_l = s_tot == 0.f ? 0.f : 1.f / l_tot;
  const float lse_v = s_tot == 0.f ? neg_inf() : (m_run + __log2f(s_tot)) * kLn2;
  if (j2 == 0 && n32 < rows) {
    const size_t at = o_row0 + 32 * wave + n32;
    if (piece) p.part_lse[at] = lse_v;
    else if (p.lse) p.lse[at] = lse_v;
  }
  // The outputs leave through LDS, 1 KB a store instruction: accumulator ct value i is
  // column 32 ct + 8 (i / 4) + 4 j2 + i % 4.
  uint32_t* stage = (uint32_t*)&s_tile[0][0] + (size_t)(32 * wave) * 260;
  if (rows == 0) return;
  if (!piece && p.out_bf16) {
#pragma unroll
    for (int ct = 0; ct < 16; ++ct)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(uint2*)(stage + n32 * 260 + 16 * ct + 4 * q + 2 * j2) =
            make_uint2(pack_bf16x2(acc[ct][4 * q] * inv_l, acc[ct][4 * q + 1] * inv_l),
                       pack_bf16x2(acc[ct][4 * q + 2] * inv_l, acc[ct][4 * q + 3] * inv_l));
    wide_lds_wait();
    rows_store((char*)(p.out_bf16 + (o_row0 + 32 * wave) * kRowsC), kRowsC * 2, stage + 4 * lane,
               16 * lane, rows);
    wide_lds_wait();
  }
  float* to = piece ? p.part_out : p.out_f32;
  if (to) {
    char* dst = (char*)(to + (o_row0 + 32 * wave) * kRowsC);
#pragma unroll
    for (int hc = 0; hc < 2; ++hc) {
#pragma unroll
      for (int c8 = 0; c8 < 8; ++c8)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int ct = 8 * hc + c8;
          *(float4*)(stage + n32 * 260 + 32 * c8 + 8 * q + 4 * j2) =
              make_float4(acc[ct][4 * q] * inv_l, acc[ct][4 * q + 1] * inv_l,
                          acc[ct][4 * q + 2] * inv_l, acc[ct][4 * q + 3] * inv_l);
        }
      wide_lds_wait();
      rows_store(dst, kRowsC * 4, stage + 4 * lane, 1024 * hc + 16 * lane, rows);
      wide_lds_wait();  // the next half overwrites the rows
    }
  }
}

// Combines the pieces of the tiles that were split: two rows a workgroup, one thread per
// four columns.
constexpr int kRowsJoin = 2;
__global__ __launch_bounds__(256) void mla_rows_join_kernel(const RowsParams p) {
  const RowsPlace tl = rows_place<true>(p, blockIdx.x);
  if (tl.b < 0 || tl.splits == 1 || tl.piece < 0 || tl.piece + tl.splits > p.pieces) return;
  const int c = threadIdx.x & 127;
  const int tr = blockIdx.y * kRowsJoin + (threadIdx.x >> 7);  // row of the tile
  const int r = tl.tile * kRowsTile + tr;
  if (r >= tl.n * p.H || tr >= p.piece_rows) return;
  const size_t slot = (size_t)tl.piece * p.piece_rows + tr;
  const PieceAcc x = piece_stream<float4>((const char*)(p.part_out + slot * kRowsC + 4 * c),
                                          (size_t)p.piece_rows * kRowsC * 4, p.part_lse + slot,
                                          p.piece_rows, 0, 1, tl.splits);
  const float inv = x.sum == 0.f ? 0.f : 1.f / x.sum;
  const float4 o = make_float4(x.a.x * inv, x.a.y * inv, x.a.z * inv, x.a.w * inv);
  const size_t at = (size_t)tl.c0 * p.H + r;
  if (p.out_f32) ((float4*)p.out_f32)[at * (kRowsC / 4) + c] = o;
  if (p.out_bf16)
    ((uint2*)p.out_bf16)[at * (kRowsC / 4) + c] =
        make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
  if (p.lse && c == 0) p.lse[at] = x.sum == 0.f ? neg_inf() : x.m + __logf(x.sum);
}

// ---------------------------------------------------------------------------

struct RowsPlan {
  long long tiles, grid, pieces;
  int fill, piece_rows;
  bool fit;
};
// decode: one token a sequence
static RowsPlan rows_plan(int N, int B, int H, bool decode, int max_len, int n_splits) {
  RowsPlan r;
  const long long each = (H + kRowsTile - 1) / kRowsTile;
  r.tiles = decode ? B * each : std::min((long long)N * H / kRowsTile + B, (long long)N * each);
  r.fill = choose_workgroups(0, 1, 1LL << 30, 1);
  r.fit = r.tiles < r.fill && B <= 256;
  r.piece_rows = (int)std::min<long long>(kRowsTile, decode ? H : (long long)N * H);
  r.grid = r.tiles;
  r.pieces = 0;
  if (n_splits > 1) {
    r.pieces = r.grid = r.tiles * n_splits;
  } else if (n_splits == 0 && max_len > 32 * kRowsMinShare) {
    // Only a tile of more than M blocks is split.  All items fit `fill`, or M is the blocks
    // over `fill`, and then split tiles are fewer than `fill` and leave twice as many pieces
    // at the most.
    r.pieces = r.fit ? r.fill : 2LL * r.fill + 64;
    r.grid = r.fit ? r.fill : r.tiles + r.pieces;
  }
  return r;
}
static size_t rows_bytes(const RowsPlan& pl) {
  if (pl.pieces == 0) return 0;
  const size_t rows = (size_t)pl.pieces * pl.piece_rows;
  return align256(rows * 4) + rows * kRowsC * 4;
}

static int rows_sizes(const char* name, int N, int B, int H, bool decode, int max_len,
                      int n_splits) {
  if (N < 0 || B < 0 || B > kMaxSeqs || H <= 0 || H > 1024 || max_len < 0 || n_splits < 0 ||
      n_splits > kRowsMaxSplits)
    return set_error(WS_EINVAL,
                     "%s: bad sizes N=%d B=%d H=%d max_len=%d n_splits=%d (B <= %d, H <= 1024, "
                     "n_splits <= %d)",
                     name, N, B, H, max_len, n_splits, kMaxSeqs, kRowsMaxSplits);
  if ((long long)N * H + 256LL * B >= (1LL << 31) || max_len > (1 << 30))
    return set_error(WS_EINVAL, "%s: %d tokens of %d heads exceed the row index range", name, N, H);
  if (rows_plan(N, B, H, decode, max_len, n_splits).grid * 256 >= (1LL << 32))
    return set_error(WS_EINVAL, "%s: %d tokens of %d heads exceed the launch grid", name, N, H);
  return WS_OK;
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

static int rows_run(const char* name, const uint16_t* q_nope, const uint16_t* q_pe,
                    const void* latent_pages, const uint8_t* latent_scale, int scale_block,
                    const int32_t* page_table, const int32_t* kv_len, const int32_t* cu_new, int N,
                    int B, int H, int page_size, int max_pages, int num_pages, int max_len,
                    int n_splits, float scale, uint16_t* out_bf16, float* out_f32, float* lse,
                    void* workspace, size_t workspace_bytes, void* stream) {
  if (!q_nope || !q_pe || !latent_pages || !page_table || !kv_len || (!out_bf16 && !out_f32))
    return set_error(WS_EINVAL, "%s: null pointer", name);
  const bool decode = !cu_new;
  if (int rc = rows_sizes(name, N, B, H, decode, max_len, n_splits)) return rc;
  if (page_size <= 0 || page_size % 32 || max_pages <= 0 || num_pages <= 0 ||
      (long long)max_len > (long long)page_size * max_pages)
    return set_error(WS_EINVAL,
                     "%s: bad paging page_size=%d max_pages=%d num_pages=%d max_len=%d (page_size "
                     "must be a multiple of 32)",
                     name, page_size, max_pages, num_pages, max_len);
  if ((long long)num_pages * page_size >= (1LL << 31))  // bit 31 marks bad page ids
    return set_error(WS_EINVAL, "%s: pools of %lld tokens exceed the 31-bit token index", name,
                     (long long)num_pages * page_size);
  if (latent_scale && (scale_block <= 0 || (scale_block & (scale_block - 1)) || page_size % scale_block))
    return set_error(WS_EINVAL, "%s: scale_block %d must be a power of two that divides page_size %d",
                     name, scale_block, page_size);
  if (!aligned16(q_nope) || !aligned16(q_pe) || !aligned16(latent_pages) || !aligned16(out_bf16) ||
      !aligned16(out_f32))
    return set_error(WS_EINVAL, "%s: buffers must be 16-byte aligned", name);
  if (!(scale - scale == 0.f)) return set_error(WS_EINVAL, "%s: scale must be finite", name);
  if (N == 0 || B == 0) return WS_OK;
  const RowsPlan pl = rows_plan(N, B, H, decode, max_len, n_splits);
  const size_t need = rows_bytes(pl);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(WS_EWORKSPACE, "%s: workspace %zu < %zu bytes", name, workspace_bytes, need);
  if (need > 0 && ((uintptr_t)workspace & 255u) != 0)
    return set_error(WS_EINVAL, "%s: workspace must be 256-byte aligned", name);
  RowsParams p;
  p.q_nope = q_nope;
  p.q_pe = q_pe;
  p.latent = latent_pages;
  p.scale = latent_scale;
  p.page_table = page_table;
  p.kv_len = kv_len;
  p.cu_new = cu_new;
  p.out_bf16 = out_bf16;
  p.out_f32 = out_f32;
  p.lse = lse;
  p.part_lse = (float*)workspace;
  p.part_out = (float*)((char*)workspace + align256((size_t)pl.pieces * pl.piece_rows * 4));
  p.N = N;
  p.B = B;
  p.H = H;
  p.page_size = page_size;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.cap = (int)std::min<long long>((long long)page_size * max_pages, 1LL << 30);
  p.block_log2 = 0;
  while (latent_scale && (1 << p.block_log2) < scale_block) ++p.block_log2;
  p.n_splits = n_splits == 0 && pl.pieces == 0 ? 1 : n_splits;
  p.fill = pl.fill;
  p.fit = pl.fit;
  p.pieces = (int)pl.pieces;
  p.piece_rows = pl.piece_rows;
  // the smallest normal float for 0: every finite score then rounds to the same
  // probability, and masked tokens stay -inf
  p.scale_log2 = std::max((scale < 0.f ? -scale : scale) * kLog2e, 1.17549435e-38f);
  p.q_sign = scale < 0.f ? 0x80008000u : 0u;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)pl.grid), block(256);
  if (latent_scale)
    hipLaunchKernelGGL(mla_rows_kernel<true>, grid, block, 0, s, p);
  else
    hipLaunchKernelGGL(mla_rows_kernel<false>, grid, block, 0, s, p);
  int rc = check_launch(name);
  if (rc != WS_OK || pl.pieces == 0) return rc;
  hipLaunchKernelGGL(mla_rows_join_kernel,
                     dim3((unsigned)pl.tiles, (pl.piece_rows + kRowsJoin - 1) / kRowsJoin), block, 0,
                     s, p);
  return check_launch(name);
}

static int rows_plan_out(const char* name, int N, int B, int H, bool decode, int max_len,
                         int n_splits, int* pieces_out, size_t* bytes_out) {
  if (int rc = rows_sizes(name, N, B, H, decode, max_len, n_splits)) return rc;
  const RowsPlan pl = rows_plan(N, B, H, decode, max_len, n_splits);
  if (pieces_out) *pieces_out = (int)pl.pieces;
  if (bytes_out) *bytes_out = rows_bytes(pl);
  return WS_OK;
}

}  // namespace ws

using namespace ws;

extern "C" int ws_mla_prompt_plan(int N, int B, int H, int max_len, int n_splits, int* pieces_out,
                                  size_t* workspace_bytes_out) {
  return rows_plan_out("ws_mla_prompt_plan", N, B, H, false, max_len, n_splits, pieces_out,
                       workspace_bytes_out);
}

extern "C" int ws_mla_prompt(const uint16_t* q_nope, const uint16_t* q_pe, const void* latent_pages,
                             const uint8_t* latent_scale, const int32_t* page_table,
                             const int32_t* kv_len, const int32_t* cu_new, int N, int B, int H,
                             int page_size, int max_pages, int num_pages, int scale_block,
                             int max_len, int n_splits, float scale, uint16_t* out_bf16,
                             float* out_f32, float* lse, void* workspace, size_t workspace_bytes,
                             void* stream) {
  if (!cu_new) return set_error(WS_EINVAL, "ws_mla_prompt: null pointer");
  return rows_run("ws_mla_prompt", q_nope, q_pe, latent_pages, latent_scale, scale_block, page_table,
                  kv_len, cu_new, N, B, H, page_size, max_pages, num_pages, max_len, n_splits, scale,
                  out_bf16, out_f32, lse, workspace, workspace_bytes, stream);
}

extern "C" int ws_mla8_decode_plan(int B, int H, int max_len, int n_splits, int* pieces_out,
                                   size_t* workspace_bytes_out) {
  return rows_plan_out("ws_mla8_decode_plan", B, B, H, true, max_len, n_splits, pieces_out,
                       workspace_bytes_out);
}

extern "C" int ws_mla8_decode_partial(const uint16_t* q_nope, const uint16_t* q_pe,
                                      const uint8_t* latent_pages, const uint8_t* latent_scale,
                                      const int32_t* page_table, const int32_t* gpu_len, int B,
                                      int H, int page_size, int max_pages, int num_pages,
                                      int scale_block, int max_len, int n_splits, float scale,
                                      float* out, float* lse, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  if (!latent_scale || !out || !lse)
    return set_error(WS_EINVAL, "ws_mla8_decode_partial: null pointer");
  return rows_run("ws_mla8_decode_partial", q_nope, q_pe, latent_pages, latent_scale, scale_block,
                  page_table, gpu_len, nullptr, B, B, H, page_size, max_pages, num_pages, max_len,
                  n_splits, scale, nullptr, out, lse, workspace, workspace_bytes, stream);
}

extern "C" int ws_mla8_decode_full(const uint16_t* q_nope, const uint16_t* q_pe,
                                   const uint8_t* latent_pages, const uint8_t* latent_scale,
                                   const int32_t* page_table, const int32_t* gpu_len, int B, int H,
                                   int page_size, int max_pages, int num_pages, int scale_block,
                                   int max_len, int n_splits, float scale, uint16_t* out_bf16,
                                   float* lse, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  if (!latent_scale || !out_bf16 || !lse)
    return set_error(WS_EINVAL, "ws_mla8_decode_full: null pointer");
  return rows_run("ws_mla8_decode_full", q_nope, q_pe, latent_pages, latent_scale, scale_block,
                  page_table, gpu_len, nullptr, B, B, H, page_size, max_pages, num_pages, max_len,
                  n_splits, scale, out_bf16, nullptr, lse, workspace, workspace_bytes, stream);
}
