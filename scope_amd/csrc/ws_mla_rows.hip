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
// 8-bit pages (e4m3, a power of two per `block` tokens) are widened once for the four waves:
// a wave's part of a block comes to LDS as it is, is read back, multiplied by its tokens'
// scales (exact in bf16) and written into the block's bf16 tile, two steps ahead.
//
// Prompts of many tiles a sequence have the latents widened once for all tiles, in a pass of
// its own, and run over that copy (kWidenTiles).
//
// The scores stay with bf16 products.  gfx950's scaled 8-bit products take e4m3 latents and
// a query split into two e4m3 halves without any widening, at the same rate, but add up
// their 64 terms in some 17 bits below the largest one, not in fp32: an lse off by 4e-5
// instead of 3e-6 (4000 new tokens of 4 sequences, 16 heads, behind 500 to 8000 8-bit
// tokens: 614 us; 667 with the widening in the steps, 554 + 10 over a widened copy).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "ws_attn.h"
#include "ws_mla_ring.h"
#include "ws_plan.h"
#include "ws_reduce.h"

namespace ws {

constexpr int kRowsC = 512;
constexpr int kRowsPe = 64;
constexpr int kRowsTile = 128;       // rows of a tile, 32 a wave (mla_few_kernel: 32)
constexpr int kRowsMaxSplits = 256;  // of a tile
// Blocks of a split, at the least (2, 4 and 8, us: decode of one sequence of 2048 tokens 15.9, 15.7
// and 17.7, of 8 of 1000 16.3, 16.0 and 17.5, a prompt of 128 tokens 27.9, 16.5 and 16.5; 16 tokens
// behind 1000 21.5, 23.0 and 27.1).
constexpr int kRowsMinShare = 4;

// Division by a number that the host knows: n / d = n m >> s for 0 <= n < 2^31, with 2^k the
// least power of two >= d, m = floor(2^(31 + k) / d) + 1 (2^31 for d = 1) and s = 31 + k: m d
// exceeds 2^s by at most d <= 2^k, which n < 2^31 keeps below a unit of the quotient.  A
// division by a variable takes some 40 instructions, a quarter of a workgroup's start.
struct Divisor {
  uint32_t m, s;
};
static Divisor divisor(uint32_t d) {
  uint32_t k = 0;
  while ((1ull << k) < d) ++k;
  return Divisor{d == 1 ? 1u << 31 : (uint32_t)((1ull << (31 + k)) / d + 1), 31 + k};
}
__device__ __forceinline__ int quotient(int n, const Divisor& d) {
  return (int)(((unsigned long long)(unsigned)n * d.m) >> d.s);
}

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
  uint16_t* part_out;  // [pieces][piece_rows][512], with part_lse [pieces][piece_rows]
  float* part_lse;
  int N, B, H, page_size, max_pages, num_pages, cap, block_log2;
  int n_splits;  // of every tile; 0: by the lengths, about `fill` workgroups in all
  int fill;
  bool fit;       // the tiles are fewer than `fill`: all items are to fit
  bool join_shared;
  int pieces;     // room for them
  int piece_rows;
  int tile;       // rows of a tile (a power of two)
  int tile_log2;
  Divisor by_H, by_page;
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
  s.tiles = (int)((unsigned)(s.n * p.H + p.tile - 1) >> p.tile_log2);
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

// Wave sums and maxima of the ROCm device library (DPP sequences; every lane active).
extern "C" __device__ float __ockl_wfred_add_f32(float);

// Item `at` of the list of all tiles' splits (TILES: of the split tiles): where the items do
// not fit the chip at once, longest sequences first (up to 64 of them), their last tile
// first.  A tile has one split for every M of its sequence's blocks, M the batch's blocks
// over `fill` workgroups; where the tiles alone are fewer than those, M is the least of four
// between that and the blocks over `fill` less the tiles at which all items fit (the last
// one fits for sure: a split more than M's quotient for every tile).  Every kernel of a call finds the same.  Every lane must call
// it; the result is uniform.  PER: sequences of a lane (0: any number, in a loop that reads
// them again; they are not split to fit).
template <bool TILES, int PER>
__device__ __forceinline__ RowsPlace rows_place_n(const RowsParams& p, int at) {
  const int lane = threadIdx.x & 63;
  const int per = PER > 0 ? PER : (p.B + 63) >> 6;
  const int b0 = lane * per;
  RowsSeq held[PER > 0 ? PER : 1];
  auto seq = [&](int k) __attribute__((always_inline)) {
    if constexpr (PER > 0) return held[k];
    else return rows_seq(p, b0 + k);
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      held[k] = rows_seq(p, min(b0 + k, p.B - 1));
      if (b0 + k >= p.B) held[k].tiles = held[k].blocks = 0;
    }
  }
  const int mine = PER > 0 ? PER : max(min(per, p.B - b0), 0);
  float rM = 0.f;
  if (p.n_splits == 0) {
    float sum = 0.f;
    int tiles = 0;
#pragma unroll 4
    for (int k = 0; k < mine; ++k) {
      const RowsSeq s = seq(k);
      sum = fmaf((float)s.tiles, (float)s.blocks, sum);  // (the same in every kernel)
      tiles += s.tiles;
    }
    const float total = __ockl_wfred_add_f32(sum);
    auto blocks_at = [&](int places) {
      return (int)fminf(ceilf(fmaxf(total * __builtin_amdgcn_rcpf((float)max(places, 1)), (float)kRowsMinShare)),
                        1e9f);
    };
    int M = uniform(blocks_at(p.fill));
    if (PER > 0 && p.fit) {
      const int room = p.fill - uniform((int)__ockl_wfred_add_u32((unsigned)tiles));
      const int gap = uniform(blocks_at(room)) + 1 - M;
      uint32_t cnt[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float r = __builtin_amdgcn_rcpf((float)(M + (gap * c + 2) / 3));
        uint32_t n = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k)
          n += held[k].tiles * min(max(plan_nsplits(held[k].blocks, r), 1), kRowsMaxSplits);
        cnt[c >> 1] += min(n, 1023u) << (16 * (c & 1));  // (sums of 64 lanes stay below 2^16)
      }
      cnt[0] = uniform((int)__ockl_wfred_add_u32(cnt[0]));
      cnt[1] = uniform((int)__ockl_wfred_add_u32(cnt[1]));
      int best = M + gap;
#pragma unroll
      for (int c = 2; c >= 0; --c)
        if ((int)((cnt[c >> 1] >> (16 * (c & 1))) & 0xffffu) <= p.fill) best = M + (gap * c + 2) / 3;
      M = best;
    }
    rM = __builtin_amdgcn_rcpf((float)M);
  }
  auto splits_of = [&](const RowsSeq& s) {
    if (p.n_splits > 0) return p.n_splits;
    return min(max(plan_nsplits(s.blocks, rM), 1), kRowsMaxSplits);
  };
  // a lane's items, and the pieces before its first sequence in the batch's order
  int items = 0, units = 0, key = -1;
#pragma unroll 4
  for (int k = 0; k < mine; ++k) {
    const RowsSeq s = seq(k);
    const int splits = splits_of(s);
    units += splits > 1 ? s.tiles * splits : 0;
    items += !TILES ? s.tiles * splits : splits > 1 ? s.tiles : 0;
    key = s.blocks;
  }
  const int before = __ockl_wfscan_add_i32(units, true) - units;
  int from = lane;  // the lane whose sequences stand at this lane's place in the list
  if (!TILES && PER == 1 && !p.fit && p.B > 1) {  // (splits that fit once are alike)
    int rank = 0;
    const int mark = lane < p.B ? key : -1;  // (no sequence: behind the others)
    for (int j0 = 0; j0 < p.B; j0 += 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int other = __builtin_amdgcn_readlane(mark, j0 + j);
        rank += other > mark || (other == mark && j0 + j < lane) ? 1 : 0;
      }
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
  auto take = [&](int k) __attribute__((always_inline)) {  // whether the item is sequence k's
    const int b = uniform(owner * per + k);
    if (b >= p.B || left < 0) return true;  // (left < 0: sums past 2^31, cu_new not non-decreasing)
    RowsSeq s;
    if constexpr (PER > 0) {
      s.c0 = __builtin_amdgcn_readlane(held[k].c0, owner);
      s.n = __builtin_amdgcn_readlane(held[k].n, owner);
      s.len = __builtin_amdgcn_readlane(held[k].len, owner);
      s.tiles = __builtin_amdgcn_readlane(held[k].tiles, owner);
      s.blocks = __builtin_amdgcn_readlane(held[k].blocks, owner);
    } else {
      s = rows_seq(p, b);
    }
    const int splits = uniform(splits_of(s));
    const int tiles = uniform(s.tiles);
    const int here = !TILES ? tiles * splits : splits > 1 ? tiles : 0;
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
      return true;
    }
    left -= here;
    piece += splits > 1 ? tiles * splits : 0;
    return false;
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (r.b < 0 && left >= 0 && take(k)) break;
  } else {
    for (int k = 0; k < per; ++k)
      if (take(k)) break;
  }
  return r;
}
template <bool TILES>
__device__ __forceinline__ RowsPlace rows_place(const RowsParams& p, int at) {
  if (p.B <= 64) return rows_place_n<TILES, 1>(p, at);
  if (p.B <= 256) return rows_place_n<TILES, 4>(p, at);
  return rows_place_n<TILES, 0>(p, at);
}

// ---------------------------------------------------------------------------
// the LDS ring

// Both kinds of pages have ws_mla_ring.h's bf16 tiles.  bf16: four, loaded three blocks ahead.
// 8 bits: three, and per wave two slots for its eight rows of a block as they are in the
// pages, 36 chunks of 16 bytes each, and the rows' scales, loaded four blocks ahead.  Lane l has
// chunks l / 8 + 8 i (i < 5; past the 36th the last one) of row l % 8: one scale a lane, one
// address and constant steps on either side.  (8 lanes' writes into the tile meet 4 chunk
// slots mod 8, twice each, a fifth of the LDS cycles; chunks (l / 8) ^ (l % 2) + 8 i meet 8
// and took as many cycles.)
constexpr int kRowsTileBytes = 16 * kWideTileAlloc;
constexpr int kRawRows = 8;             // of a wave
constexpr int kRawDma = 5;              // load instructions, and one for the scales
constexpr int kRawBytes = 1024 * kRawDma;
template <bool F8>
struct RowsRing {
  static constexpr int kTiles = F8 ? 3 : kWideTiles;
  static constexpr int kRowBytes = F8 ? 576 : 1152;
  // LDS: tiles, then the bf16 sink or the waves' raw slots, then the raw slots' scales
  static constexpr int kRaw = kTiles * kRowsTileBytes;
  static constexpr int kScales = kRaw + (F8 ? 4 * 2 * kRawBytes : 1024);
  // and, for 8 bits, the last k-step of the queries (a lane's own 16 bytes), whose registers
  // the widening takes: what the compiler spilled instead came back behind the loads under
  // way, which memory answers in order
  static constexpr int kQuery = kScales + (F8 ? 4 * 2 * 256 : 0);
  static constexpr int kLds = kQuery + (F8 ? 256 * 16 : 0);
};
static_assert(kRowsTile == 1 << 7, "tile_log2");
static_assert(RowsRing<true>::kLds <= 160 * 1024 - 64 && RowsRing<false>::kLds <= 160 * 1024 - 64, "LDS");
static_assert(RowsRing<true>::kScales >= kRowsTile * 65 * 16, "the queries are staged in the tiles");

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

// The wait states that a VALU read of the last product's result asks for (16 passes and
// four).
__device__ __forceinline__ void qk_settle(f32x16& c) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(c) : : "memory");
}
// The same with two other MFMAs issued in between (each waits for the one before it).
__device__ __forceinline__ void qk_settle_short(f32x16& c) {
  asm volatile("s_nop 3" : "+v"(c) : : "memory");
}

template <bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
// Eight e4m3 values times a power of two as bf16 (exact).
__device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi, float scale) {
  return u32x4{widen2<false>(lo, scale), widen2<true>(lo, scale), widen2<false>(hi, scale),
               widen2<true>(hi, scale)};
}
__device__ __forceinline__ u32x4 rows_lds_b128(uint32_t addr) {
  return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)addr;
}
__device__ __forceinline__ uint32_t rows_lds_b32(uint32_t addr) {
  return *(const __attribute__((address_space(3))) uint32_t*)(uintptr_t)addr;
}
__device__ __forceinline__ void rows_lds_put(uint32_t addr, const u32x4& v) {
  *(__attribute__((address_space(3))) u32x4*)(uintptr_t)addr = v;
}
template <int N>
__device__ __forceinline__ void rows_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// Stores `rows` staged 1 KB rows (row h at src + 260 h dwords, lane part at src) to dst + h *
// row_bytes + col_byte.
__device__ __forceinline__ void rows_store(char* dst, int row_bytes, const uint32_t* src,
                                           int col_byte, int rows) {
  if (rows == 32) {
    wide_store_rows(dst, row_bytes, src, col_byte, 32);
    return;
  }
  for (int h = 0; h < rows; ++h)
    *(u32x4*)(dst + (size_t)h * row_bytes + col_byte) = *(const u32x4*)(src + h * 260);
}

// Whether a row's reference does not serve its largest score: that climbed out of the
// headroom, or lies far below, as it can where every score of the row's first block is -inf
// and the reference is 0 (a reference that is a score is no larger than the largest).
__device__ __forceinline__ bool reference_off(float top, float m_run) {
  return top > m_run + kWideHeadroomLog2 || (top < m_run - kWideHeadroomLog2 && top != neg_inf());
}

// What a bf16 pair holds of infinities and NaN: their halves' bits, all set.
__device__ __forceinline__ uint32_t nonfinite_halves(uint32_t w) {
  const uint32_t hit = (((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15;
  return hit * 0xffffu;
}
// A workgroup's rows and tokens, and where its outputs go.
struct RowsWork {
  RowsPlace pl;
  bool piece, len_good;
  int R_all, row0, here, first_pos, lim_lo, nblk, t_begin, t_end;
  size_t g_row0, o_row0;  // the tile's first row of q, and of the outputs (or its piece)
};
// False: the workgroup has nothing to do (it is past the list, or its rows see nothing and
// are written here: (0, -inf), NaN for an invalid length).
__device__ __forceinline__ bool rows_work(const RowsParams& p, RowsWork& w) {
  const int tid = threadIdx.x;
  w.pl = rows_place<false>(p, blockIdx.x);
  const RowsPlace& pl = w.pl;
  w.piece = pl.splits > 1;
  if (pl.b < 0 || (w.piece && (pl.piece < 0 || pl.piece >= p.pieces))) return false;
  w.R_all = pl.n * p.H;
  w.row0 = pl.tile * p.tile;
  w.here = min(p.tile, w.R_all - w.row0);
  w.len_good = len_ok(pl.len, 0, p.cap);
  w.first_pos = pl.len - pl.n;  // position of the sequence's first query
  // tokens that the tile's first row and its last one see
  w.lim_lo = w.first_pos + quotient(w.row0, p.by_H) + 1;
  const int lim_hi =
      w.len_good ? max(w.first_pos + quotient(w.row0 + w.here - 1, p.by_H) + 1, 0) : 0;
  const int nb = (lim_hi + 31) / 32;
  // (nb split / splits without 64 bits: splits is at most kRowsMaxSplits)
  const unsigned each = (unsigned)nb / (unsigned)pl.splits, rest = (unsigned)nb - each * (unsigned)pl.splits;
  const int blk0 = (int)(pl.split * each + pl.split * rest / (unsigned)pl.splits);
  const int blk1 = (int)((pl.split + 1) * each + (pl.split + 1) * rest / (unsigned)pl.splits);
  w.nblk = blk1 - blk0;
  w.t_begin = 32 * blk0;
  w.t_end = min(lim_hi, 32 * blk1);
  w.g_row0 = (size_t)pl.c0 * p.H + w.row0;
  w.o_row0 = w.piece ? (size_t)pl.piece * p.piece_rows : w.g_row0;
  if (w.nblk > 0) return true;
  const float fill = w.len_good ? 0.f : qnan();
  const uint32_t fill2 = pack_bf16x2(fill, fill);
  for (int x = tid; x < w.here * (kRowsC / 4); x += 256) {
    const size_t at = w.o_row0 * (kRowsC / 4) + x;
    if (w.piece) {
      ((uint2*)p.part_out)[at] = make_uint2(fill2, fill2);
    } else {
      if (p.out_f32) ((float4*)p.out_f32)[at] = make_float4(fill, fill, fill, fill);
      if (p.out_bf16) ((uint2*)p.out_bf16)[at] = make_uint2(fill2, fill2);
    }
  }
  if (tid < w.here) {
    const float l = w.len_good ? neg_inf() : qnan();
    if (w.piece) p.part_lse[w.o_row0 + tid] = l;
    else if (p.lse) p.lse[w.o_row0 + tid] = l;
  }
  return false;
}

// Bound by the matrix units with the power they may draw, and the instructions that feed them
// (a wave alone on its SIMD, 512 registers): a step of 32 tokens and 128 rows is 68 products of
// 32 x 32 x 16 a wave, 2176 cycles of the matrix unit, and takes 3100 over bf16 tiles, 4000 with
// 8-bit blocks widened in it (some 100 instructions more).  8192 tokens of a prompt, 16
// heads: 949 us, 1.23 PFLOP/s of the products the rows need (744 us on zeros, where power does
// not bind).  4000 tokens in 4 chunks over 8-bit pages: 558 us, 1.18 PFLOP/s.  4 tokens of 16
// heads each behind 4000 to 32000: 43 us, 3.7 TB/s; 24 prompts up to 600 tokens of 20 heads 78
// us; decode of 128 heads, 8 sequences of 16000 to 32768 8-bit tokens: 63 us, 0.8 PFLOP/s.
// Around its steps a workgroup spends 3 us before its first product and 4 us behind the last.
template <bool F8>
__global__ __launch_bounds__(256) void mla_rows_kernel(const RowsParams p) {
  using R = RowsRing<F8>;
  constexpr int kRow = R::kRowBytes;
  constexpr int kTileChunks = kWideTileAlloc;
  constexpr int kPer = F8 ? kRawDma + 1 : kWideDmaPerWave;  // a wave's load instructions of a block
  __shared__ __attribute__((aligned(1024))) char s_mem[R::kLds];
  __shared__ int s_redo;
  __shared__ int s_odd[2];  // by a block's parity: its tile is to be cleaned (soft_x)
  const int tid = threadIdx.x;
  const int wave = uniform(tid >> 6);
  const int lane = tid & 63;
  const int n32 = lane & 31;  // row of the wave (QK B, PV B, output) or token (A operands)
  const int j2 = lane >> 5;
  RowsWork w;
  if (!rows_work(p, w)) return;
  if (tid == 0) s_redo = s_odd[0] = s_odd[1] = 0;  // read after the ring's barriers
  const int nblk = w.nblk, t_begin = w.t_begin, t_end = w.t_end, here = w.here;
  const int rows = min(max(here - 32 * wave, 0), 32);  // this wave's
  // the tokens that the lane's row sees (past the rows: the last one again)
  const int lim_lane = w.first_pos + quotient(min(w.row0 + 32 * wave + n32, w.R_all - 1), p.by_H) + 1;

  const uint32_t lds0 =
      (uint32_t)uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_mem);
  u32x4* const s_tile = (u32x4*)s_mem;
  const uint32_t raw0 = lds0 + R::kRaw + 2 * kRawBytes * wave;       // this wave's (8 bits)
  const uint32_t scale0 = lds0 + R::kScales + 2 * 256 * wave;
  // bf16: byte offsets, within a block's rows in HBM, of the chunks this lane loads, two to a
  // register (the largest is 31 * 1152 + 1136).  8 bits: the lane's first chunk in a tile.
  constexpr int kOff = F8 ? 1 : kPer / 2;
  uint32_t offp[kOff];
  if constexpr (F8) {
    offp[0] = 16 * (uint32_t)(wide_row_off(lane & 7) + kWideRowsT * wave + 2 * (lane >> 3));
  } else {
#pragma unroll
    for (int j = 0; j < kOff; ++j) {
      uint32_t v = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = 64 * min(wave + 4 * (2 * j + h), kWideTileDma - 1) + lane;
        const int r = wide_row_of(c);
        const int x = min(c - wide_row_off(r), kWideRowData - 1);
        v |= (uint32_t)(r * kRow + 16 * x) << (16 * h);
      }
      offp[j] = v;
    }
  }
  // Per-lane part of the transposed reads: lane 4 e + r of a 16-lane group addresses token
  // row 4 j2 + e, columns 4 r .. 4 r + 3 of the group's 16.
  const uint32_t v_lane = [&] {
    const int ch = (lane >> 4) & 1, e = (lane >> 2) & 3, r = lane & 3;
    return (uint32_t)(16 * wide_row_off(4 * j2 + e) + 2 * (16 * ch + 4 * r));
  }();

  // Pool token index of the first row of each block, 64 at a time (lane l: block pid_base +
  // l); a page id outside the pool is clamped and marks the index with bit 31.
  const int32_t* pt = p.page_table + (size_t)w.pl.b * p.max_pages;
  int pid_base = 0;
  int m_tok = 0;
  uint32_t bad_bits = 0;  // of the blocks requested last: whether their page id was bad
  auto first_tok = [&]() __attribute__((always_inline)) {
    return t_begin + 32 * min(pid_base + lane, nblk - 1);
  };
  auto set_pids = [&](int raw) __attribute__((always_inline)) {
    const int t0 = first_tok();
    const int page = quotient(t0, p.by_page);
    const int pid = clamp_page(raw, p.num_pages);
    m_tok = (pid * p.page_size + (t0 - page * p.page_size)) | (raw == pid ? 0 : (int)0x80000000u);
  };
  auto fetch_pids = [&]() __attribute__((always_inline)) { set_pids(pt[quotient(first_tok(), p.by_page)]); };
  int raw_pid = pt[quotient(first_tok(), p.by_page)];

  // Q^T of this wave's rows, through LDS a 1 KB row an instruction (row slots of 65 chunks):
  // k-step u holds columns 16 u + 8 j2 .. + 8.
  u32x4 qb[36];
  {
    const uint16_t* qrow0 = p.q_nope + (w.g_row0 + 32 * wave) * kRowsC;
    const uint32_t qst = lds0 + (uint32_t)(32 * wave * 65 * 16);
#pragma clang loop unroll(disable)
    for (int h = 0; h < rows; ++h)
      rows_dma16(16 * lane, qrow0 + h * kRowsC, qst + (uint32_t)(h * 65 * 16), 0);
    const u32x4* pe =
        (const u32x4*)(p.q_pe + (w.g_row0 + min(32 * wave + n32, here - 1)) * kRowsPe);
#pragma unroll
    for (int u = 32; u < 36; ++u) qb[u] = pe[2 * (u - 32) + j2];
    asm volatile("s_waitcnt vmcnt(0)" : "+v"(raw_pid) : : "memory");
    set_pids(raw_pid);
    const u32x4* qs = s_tile + (32 * wave + min(n32, max(rows - 1, 0))) * 65 + j2;
#pragma unroll
    for (int u = 0; u < 32; ++u) qb[u] = qs[2 * u];
    if (p.q_sign) {
#pragma unroll
      for (int u = 0; u < 36; ++u) qb[u] ^= p.q_sign;
    }
  }
  if constexpr (F8) rows_lds_put(lds0 + R::kQuery + 16 * tid, qb[35]);
  // the queries in registers, and every wave done with its staged rows, before the loads
#pragma unroll
  for (int u = 0; u < 36; ++u) asm volatile("" : : "v"(qb[u]));
  wide_lds_barrier();

  // Block k's loads, this wave's kPer instructions: bf16 into tile k % 4, 8 bits into raw slot
  // k % 2.  Rows past t_end read the last row's last chunk; a block past the last is the last
  // one again, for a tile that nothing reads.
  const char* g0 = (const char*)p.latent;
  struct Dma {
    const char* sb;
    const uint8_t* ss;
    uint32_t wbase, last, lim;  // (8 bits, lim: the block's last row)
    uint32_t off;               // (8 bits: the lane's first chunk, from instruction 0 on)
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
    if constexpr (F8) {
      d.lim = (uint32_t)(nt - 1);
      d.wbase = raw0 + kRawBytes * (k & 1);
      d.last = scale0 + 256 * (k & 1);
      d.ss = p.scale + (tok >> p.block_log2);
    } else {
      d.lim = nt >= 32 ? 0xffffu : (uint32_t)((nt - 1) * kRow + kRow - 16);
      const uint32_t tb = lds0 + (uint32_t)(k & 3) * kRowsTileBytes;
      d.wbase = tb + 1024 * wave;
      d.last = wave == 0 ? tb + 1024 * (kWideTileDma - 1) : lds0 + R::kRaw;
    }
    // recomputed per block (not hoisted)
    asm volatile("" : "+s"(d.wbase), "+s"(d.last));
    return d;
  };
  auto dma_one = [&](Dma& d, int i) __attribute__((always_inline)) {
    if constexpr (F8) {
      int l = lane;
      asm volatile("" : "+v"(l));  // (recomputed at each use)
      const uint32_t row = min((uint32_t)(kRawRows * wave + (l & 7)), d.lim);
      if (i == 0) d.off = row * kRow + 16 * (l >> 3);
      if (i < kRawDma - 1)
        rows_dma16(d.off + 128 * i, d.sb, d.wbase, 1024 * i);
      else if (i < kRawDma)
        rows_dma16(d.off + 128 * i - 16 * max((l >> 3) - 3, 0), d.sb, d.wbase, 1024 * i);
      else
        rows_dma1(row >> p.block_log2, d.ss, d.last);
    } else {
      asm volatile("" : "+v"(offp[i >> 1]));  // unpacked at each use
      const uint32_t pr = offp[i >> 1];
      const uint32_t off = min((i & 1) ? pr >> 16 : pr & 0xffffu, d.lim);
      if (i < kPer - 1) rows_dma16(off, d.sb, d.wbase, 4 * 1024 * i);
      else rows_dma16(off, d.sb, d.last, 0);
    }
  };
  auto issue = [&](int k) __attribute__((always_inline)) {
    Dma d = issue_begin(k);
#pragma unroll
    for (int i = 0; i < kPer; ++i) dma_one(d, i);
  };
  // 8 bits: the lane's scale and chunk i of its row of block k, as they are in the raw slot (its
  // loads done), and the chunk into the tile (`to`: the lane's first place there)
  auto raw_scale = [&](int k) __attribute__((always_inline)) {
    return __builtin_bit_cast(float, rows_lds_b32(scale0 + 256 * (k & 1) + 4 * lane) << 23);
  };
  auto raw_read = [&](int k, int i) __attribute__((always_inline)) {
    return rows_lds_b128(raw0 + kRawBytes * (k & 1) + 16 * lane + 1024 * i);
  };
  auto raw_put = [&](const u32x4& x, float sc, uint32_t to, int i) __attribute__((always_inline)) {
    if (i == kRawDma - 1) {  // (lanes from 32 on: chunk 35 once more)
      int l = lane;
      asm volatile("" : "+v"(l));
      to -= 32 * max((l >> 3) - 3, 0);
    }
    rows_lds_put(to + 256 * i, widen8(x[0], x[1], sc));
    rows_lds_put(to + 256 * i + 16, widen8(x[2], x[3], sc));
  };
  auto tile_of = [&](int k) __attribute__((always_inline)) {
    return F8 ? (int)((unsigned)k % 3u) : k & 3;
  };
  auto widen_block = [&](int k) __attribute__((always_inline)) {
    const uint32_t to = lds0 + (uint32_t)tile_of(k) * kRowsTileBytes + offp[0];
    const float sc = raw_scale(k);
#pragma unroll
    for (int i = 0; i < kRawDma; ++i) raw_put(raw_read(k, i), sc, to, i);
  };
  f32x16 acc[16];
  float m_run = neg_inf();  // reference of the lane's row: its largest score in the first block
  float m_max = neg_inf();  // the lane's largest raw score so far
  float l_run = 0.f;  // the lane's sum of probabilities as rounded
  float s_run = 0.f;  // and in fp32

  const u32x4* arow0 = s_tile + wide_row_off(n32) + j2;
  auto qk_read = [&](int tile, int u) __attribute__((always_inline)) {
    return arow0[tile * kTileChunks + 2 * u];
  };
  auto last_query = [&]() __attribute__((always_inline)) {
    if constexpr (F8) return rows_lds_b128(lds0 + R::kQuery + 16 * tid);
    else return qb[35];
  };
  auto qk_link = [&](f32x16& sc, const u32x4& kr, int u, const u32x4& last) __attribute__((always_inline)) {
    if (u == 0) qk_first(sc, kr, qb[0]);
    else qk_next(sc, kr, u == 35 ? last : qb[u]);
  };
  auto vbase = [&](int tile) __attribute__((always_inline)) {
    uint32_t vl = v_lane;
    asm volatile("" : "+v"(vl));  // (one register, the rest in the instruction's offset)
    return lds0 + (uint32_t)tile * kRowsTileBytes + vl;
  };
  // V^T operand of MFMA m: tokens 16 (m / 16) .., columns 32 (m % 16) ..
  auto vread = [&](uint32_t vt, int m) __attribute__((always_inline)) {
    const uint32_t a = vt + 16 * kWideRowsS * (m >> 4) + 64 * (m & 15);
    const uint2 lo = lds_read_tr_b64(a);
    const uint2 hi = lds_read_tr_b64(a + 16 * kWideRowsT);
    return u32x4{lo.x, lo.y, hi.x, hi.y};
  };
  // the memory clobber keeps the operand reads where the source puts them
  auto pv_mfma = [&](const u32x4& va, const u32x4& pbs, int m) __attribute__((always_inline)) {
    f32x16& a = acc[m & 15];
    a = mfma32x32x16(va, pbs, a);
    asm volatile("" : "+a"(a));
    asm volatile("" : : : "memory");
  };
  const float sx = p.scale_log2;
  // Whether the tile's first row does not see all of block kb, or its page id is bad (alike in
  // the four waves).
  auto masked = [&](int kb) __attribute__((always_inline)) {
    return t_begin + 32 * kb + 32 > w.lim_lo || ((bad_bits >> (kb & 31)) & 1) != 0;
  };
  // The scores of block kb in the log2 domain less the reference (xa: the first 16 tokens',
  // xh: the others').  In a masked block a score that a row does not see is -inf, and an
  // infinity or a NaN in a token shows in its score: where a row of the wave does not see
  // it, the tile is cleaned before its values are taken.  Returns whether the block is masked.
  auto soft_x = [&](int kb, const f32x16& sc, float (&xa)[8], float (&xh)[8], bool first)
      __attribute__((always_inline)) {
    const int t0 = t_begin + 32 * kb;
    f32x16 v = sc;
    const bool look = masked(kb);
    if (look) {
      const bool bad_page = (bad_bits >> (kb & 31)) & 1;
      int l = lane;  // recomputed here rather than kept live
      asm volatile("" : "+v"(l));
      const int lim = lim_lane - t0 - 4 * (l >> 5);
      const float bad = bad_page ? qnan() : 0.f;
      float hidden = 0.f;  // NaN: a score that is not seen is not finite
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool seen = 8 * (i >> 2) + (i & 3) < lim;
        hidden = __builtin_fmaf(seen ? 0.f : v[i], 0.f, hidden);
        v[i] = seen ? v[i] + bad : neg_inf();
      }
      if (__builtin_amdgcn_ballot_w64(hidden != hidden) != 0) s_odd[kb & 1] = 1;
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
    return look;
  };
  // One dword of a k-step's P^T (two exp2), its probabilities added to the row sum as rounded
  auto soft_p = [&](float (&xs)[8], u32x4& pbs, int dd) __attribute__((always_inline)) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    xs[2 * dd] = __builtin_amdgcn_exp2f(xs[2 * dd]);
    xs[2 * dd + 1] = __builtin_amdgcn_exp2f(xs[2 * dd + 1]);
    const uint32_t pk = pack_bf16x2(xs[2 * dd], xs[2 * dd + 1]);
    pbs[dd] = pk;
    l_run = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pk),
                                            __builtin_bit_cast(bf16x2_t, 0x3f803f80u), l_run, false);
  };
  auto soft_s = [&](const float (&xa)[8], const float (&xh)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s_run += xa[i] + xh[i];
  };
  // The last block's values' product by itself (its tile is in and synchronised)
  auto values = [&](int kk, float (&xa)[8], float (&xh)[8]) __attribute__((always_inline)) {
    const uint32_t vt = vbase(tile_of(kk));
    u32x4 va[4], pb[2];
#pragma unroll
    for (int dd = 0; dd < 4; ++dd) soft_p(xa, pb[0], dd);
#pragma unroll
    for (int m = 0; m < 3; ++m) va[m] = vread(vt, m);
#pragma unroll
    for (int m = 0; m < 32; ++m) {
      if (m + 3 < 32) va[(m + 3) & 3] = vread(vt, m + 3);
      pv_mfma(va[m & 3], pb[m >> 4], m);
      if (m < 16 && (m & 3) == 1) soft_p(xh, pb[1], m >> 2);
    }
    soft_s(xa, xh);
  };
  // NaN into the columns of a row's sums in which block kk's tile has an infinity or a NaN of
  // a token that the row sees: what the values' product would add (its score is not finite,
  // so its weight is 0 or NaN).  A product of 2^127 there and 2^127 where a token is seen goes
  // past fp32's range, and its opposite after it leaves NaN.  (8-bit pages hold NaN besides
  // numbers, which a row that sees it has from its score.)
  auto mark = [&](int kk) __attribute__((always_inline)) {
    const uint32_t vt = vbase(tile_of(kk));
    const int lim = lim_lane - (t_begin + 32 * kk) - 4 * j2;
#pragma clang loop unroll(disable)
    for (int s = 0; s < 2; ++s) {
      u32x4 vis;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int t = 16 * s + 8 * (d >> 1) + 2 * (d & 1);  // soft_x's tokens 8 s + 2 d and the next
        vis[d] = (t < lim ? 0x7f00u : 0u) | (t + 1 < lim ? 0x7f000000u : 0u);
      }
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        u32x4 x = vread(vt + 16 * kWideRowsS * s, c), y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t at = nonfinite_halves(x[e]);
          x[e] = at & 0x7f007f00u;
          y[e] = at & 0xff00ff00u;
        }
        pv_mfma(x, vis, c);
        pv_mfma(y, vis, c);
      }
    }
  };
  // Takes the infinities and NaN out of block kk's tile, where a token that some row of the
  // workgroup does not see holds one (0 * inf would bring it into that row); rows that see it
  // have it from mark.  (look: the block is masked.)  All waves call it behind the barrier at which each has its scores of
  // the tile; a wave that is ahead notes the other parity.
  auto clean = [&](int kk, bool look) __attribute__((always_inline)) {
    if (!look || __builtin_expect(uniform(s_odd[kk & 1]) == 0, 1)) return;
    int k = kk, first = tid;
    asm volatile("" : "+s"(k), "+v"(first));  // (nothing of this is kept from step to step)
    if (!F8 && rows > 0) mark(k);
    wide_lds_barrier();  // every wave has read the note and the tile
    if (first == 0) s_odd[k & 1] = 0;
    const uint32_t tile = lds0 + (uint32_t)tile_of(k) * kRowsTileBytes;
#pragma clang loop unroll(disable)
    for (int c = first; c < kTileChunks; c += 256) {
      u32x4 x = rows_lds_b128(tile + 16 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] &= ~nonfinite_halves(x[e]);
      rows_lds_put(tile + 16 * c, x);
    }
    wide_lds_barrier();
  };

  // Step kk of the ring (ws_mla_wide.h): block kk + 1's scores with block kk's values'
  // product between their links, the loads over them (bf16: block kk + 3's; 8 bits: block kk
  // + 4's, behind the widening of this wave's part of block kk + 2), and the softmax of
  // block kk + 1 beside the last products.
  auto step = [&](int kk, float (&xa)[8], float (&xh)[8], bool& look) __attribute__((always_inline)) {
    const int tp = tile_of(kk), tq = tile_of(kk + 1);
    if constexpr (F8) wide_lds_barrier();
    else wide_wait_barrier<kPer>();
    clean(kk, look);
    if constexpr (F8) rows_wait<kPer>();  // block kk + 2's loads
    Dma d = issue_begin(kk + (F8 ? 4 : 3));
    const uint32_t to = lds0 + (uint32_t)tile_of(kk + 2) * kRowsTileBytes + offp[0];
    f32x16 sc;
    constexpr int kLead = F8 ? 3 : 4;  // links that an operand is read ahead
    u32x4 kr[kLead + 1], va[4], pb[2], raw, last;
    float rs = 1.f;
    if constexpr (F8) rs = raw_scale(kk + 2);
    const uint32_t vt = vbase(tp);
#pragma unroll
    for (int u = 0; u < kLead; ++u) kr[u] = qk_read(tq, u);
#pragma unroll
    for (int m = 0; m < 3; ++m) va[m] = vread(vt, m);
#pragma unroll
    for (int u = 0; u < 36; ++u) {
      if (u + kLead < 36) kr[(u + kLead) % (kLead + 1)] = qk_read(tq, u + kLead);
      if (u == 32) last = last_query();
      qk_link(sc, kr[u % (kLead + 1)], u, last);
      if (u < 4) {
        soft_p(xa, pb[0], u);
      } else if ((u - 4) % 4 != 3) {
        const int m = 3 * ((u - 4) / 4) + (u - 4) % 4;
        va[(m + 3) & 3] = vread(vt, m + 3);
        pv_mfma(va[m & 3], pb[m >> 4], m);
        if (m < 16 && (m & 3) == 1) soft_p(xh, pb[1], m >> 2);
      }
      if constexpr (F8) {
        if (u % 5 == 0 && u / 5 < kRawDma) raw = raw_read(kk + 2, u / 5);
        if (u % 5 == 3 && u / 5 < kRawDma) raw_put(raw, rs, to, u / 5);
        if (u >= 5 * kRawDma && u < 5 * kRawDma + kPer) dma_one(d, u - 5 * kRawDma);
      } else {
        if (u % 4 == 2) dma_one(d, u / 4);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // (MFMAs 24 and 25 behind the last link)
#pragma unroll
    for (int m = 24; m < 32; ++m) {
      if (m == 26) {
        __builtin_amdgcn_sched_barrier(0);
        qk_settle_short(sc);
        look = soft_x(kk + 1, sc, xa, xh, false);
      }
      if (m + 3 < 32) va[(m + 3) & 3] = vread(vt, m + 3);
      pv_mfma(va[m & 3], pb[1], m);
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
    if constexpr (F8) {
      issue(0);
      issue(1);
      rows_wait<kPer>();
      widen_block(0);
      wide_lds_wait();  // the raw slot is read
      issue(2);
      rows_wait<kPer>();
      widen_block(1);
      wide_lds_wait();
      issue(3);
      wide_lds_barrier();
    } else {
      issue(0);
      issue(1);
      issue(2);
      wide_wait_barrier<2 * kPer>();
    }
    if (rows > 0) {
      float xa[8], xh[8];
      bool look;
      {
        f32x16 sc;
        u32x4 kr[5];
        const u32x4 last = last_query();
#pragma unroll
        for (int u = 0; u < 4; ++u) kr[u] = qk_read(0, u);
#pragma unroll
        for (int u = 0; u < 36; ++u) {
          if (u + 4 < 36) kr[(u + 4) % 5] = qk_read(0, u + 4);
          qk_link(sc, kr[u % 5], u, last);
        }
        qk_settle(sc);
        look = soft_x(0, sc, xa, xh, true);
      }
#pragma clang loop unroll(disable)
      for (int k = 0; k + 1 < nblk; ++k) step(k, xa, xh, look);
      wide_lds_barrier();  // every wave has its scores of the last tile
      clean(nblk - 1, look);
      values(nblk - 1, xa, xh);
    } else {  // the ring's waits, barriers and loads alone
#pragma clang loop unroll(disable)
      for (int k = 0; k + 1 < nblk; ++k) {
        if constexpr (F8) {
          wide_lds_barrier();
          clean(k, masked(k));
          rows_wait<kPer>();
          widen_block(k + 2);
          wide_lds_wait();
          issue(k + 4);
        } else {
          wide_wait_barrier<kPer>();
          clean(k, masked(k));
          issue(k + 3);
        }
      }
      wide_lds_barrier();
      clean(nblk - 1, masked(nblk - 1));
    }
    {  // the row's largest score (both its lanes)
      float lo, hi;
      pair_xor32(m_max, lo, hi);
      m_max = fmaxf(lo, hi);
    }
    const float top = m_max * sx;
    // every load of the pass has landed and every wave is done with the tiles
    const bool off = __builtin_amdgcn_ballot_w64(reference_off(top, m_run)) != 0;
    if (rows > 0 && off && lane == 0) s_redo = 1;
    wide_wait_barrier<0>();
    const bool redo = s_redo != 0;
    wide_wait_barrier<0>();  // every wave has read s_redo
    if (tid == 0) s_redo = 0;
    if (pass > 0 || !redo) break;
    // scores out of the reference's reach: again, from the rows' largest
    m_run = top == neg_inf() ? 0.f : top;
  }

  float lo, hi;
  pair_xor32(s_run, lo, hi);
  const float s_tot = lo + hi;
  pair_xor32(l_run, lo, hi);
  const float l_tot = lo + hi;
  const float inv_l = s_tot == 0.f ? 0.f : 1.f / l_tot;
  const float lse_v = s_tot == 0.f ? neg_inf() : (m_run + __log2f(s_tot)) * kLn2;
  int el = lane;  // (what the end takes of the lane is spilled around the loop otherwise)
  asm volatile("" : "+v"(el));
  const int en = el & 31, ej = el >> 5;
  if (ej == 0 && en < rows) {
    const size_t at = w.o_row0 + 32 * wave + en;
    if (w.piece) p.part_lse[at] = lse_v;
    else if (p.lse) p.lse[at] = lse_v;
  }
  // The outputs leave through LDS, 1 KB a store instruction: accumulator ct value i is
  // column 32 ct + 8 (i / 4) + 4 ej + i % 4.
  uint32_t* stage = (uint32_t*)s_mem + (size_t)(32 * wave) * 260;
  if (rows == 0) return;
  uint16_t* to16 = w.piece ? p.part_out : p.out_bf16;
  if (to16) {
#pragma unroll
    for (int ct = 0; ct < 16; ++ct)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(uint2*)(stage + en * 260 + 16 * ct + 4 * q + 2 * ej) =
            make_uint2(pack_bf16x2(acc[ct][4 * q] * inv_l, acc[ct][4 * q + 1] * inv_l),
                       pack_bf16x2(acc[ct][4 * q + 2] * inv_l, acc[ct][4 * q + 3] * inv_l));
    wide_lds_wait();
    rows_store((char*)(to16 + (w.o_row0 + 32 * wave) * kRowsC), kRowsC * 2, stage + 4 * el,
               16 * el, rows);
    wide_lds_wait();
  }
  if (!w.piece && p.out_f32) {
    char* dst = (char*)(p.out_f32 + (w.o_row0 + 32 * wave) * kRowsC);
#pragma unroll
    for (int hc = 0; hc < 2; ++hc) {
#pragma unroll
      for (int c8 = 0; c8 < 8; ++c8)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int ct = 8 * hc + c8;
          *(float4*)(stage + en * 260 + 32 * c8 + 8 * q + 4 * ej) =
              make_float4(acc[ct][4 * q] * inv_l, acc[ct][4 * q + 1] * inv_l,
                          acc[ct][4 * q + 2] * inv_l, acc[ct][4 * q + 3] * inv_l);
        }
      wide_lds_wait();
      rows_store(dst, kRowsC * 4, stage + 4 * el, 1024 * hc + 16 * el, rows);
      wide_lds_wait();  // the next half overwrites the rows
    }
  }
}

// 8-bit pages under few rows (kFewRows): a tile is one wave's 32 rows, the four waves take
// every fourth block of its tokens each, and their sums meet in LDS at the end.  With 16 rows
// the products are small beside the loads, so what counts is that each wave keeps a block on
// its way while it works on another, without a barrier: a block takes a wave 5200 cycles,
// 1300 of the CU, the HBM some 2000 of its share.  The latents are widened where they are
// read: the scores' operand by its token's scale, the values' operand as it is, with the
// scale on the token's probability.  Bound by HBM in long batches (16 sequences of 3000 to
// 32768 tokens, 16 heads: 193 MB in 46 us, 4.2 TB/s), by one chain of loads, a block and the
// merge in short ones (one of 8192: 11.8 us).
constexpr int kFewTile = 32;
constexpr int kFewDma = 19;  // 1 KB load instructions of a block, and one for the scales
constexpr int kFewSlot = 1024 * kFewDma;
constexpr int kFewWave = 2 * (kFewSlot + 256);
// Rows of 36 chunks of 16 bytes and one chunk of padding every four rows: the score reads (16
// rows, one chunk each) meet 16 chunk slots mod 16, and the transposed reads (rows 4 j .. 4 j
// + 3 and those 8 further on, 32 bytes of each) 8 different pairs of them.
__host__ __device__ constexpr int few_row_off(int r) { return 36 * r + (r >> 2); }
static_assert(few_row_off(31) + 36 <= 64 * kFewDma, "a block fills its load instructions");
static_assert(few_row_off(16 + 8 + 4 + 3) == 580 + 290 + 145 + 108, "row offsets add up");
static_assert(32 * 260 * 4 <= kFewWave && 32 * 65 * 16 <= 2 * kFewSlot, "outputs and queries are staged there");

// ds_read_b64_tr_b8: in each 16-lane group lanes 2 e and 2 e + 1 address the halves of
// row e's 16 bytes; result lane i holds byte i of rows 0 .. 7 (measured in bounds).
__device__ __forceinline__ uint2 lds_read_tr8_b64(uint32_t addr) {
  typedef int i32x2_t __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) i32x2_t lds_i32x2_t;
  const i32x2_t v = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_t*)(uintptr_t)addr);
  return make_uint2((uint32_t)v[0], (uint32_t)v[1]);
}
// qk_first and qk_next with an operand that has just been computed (two wait states).
__device__ __forceinline__ void qk_first_new(f32x16& c, const u32x4& a, const u32x4& b) {
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b) : "memory");
}
__device__ __forceinline__ void qk_next_new(f32x16& c, const u32x4& a, const u32x4& b) {
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b) : "memory");
}
// The bytes of four e4m3 values that are NaN, all set.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t hit = (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
  return hit * 0xffu;
}

__global__ __launch_bounds__(256) void mla_few_kernel(const RowsParams p) {
  constexpr int kRow = 576;
  __shared__ __attribute__((aligned(1024))) char s_mem[4 * kFewWave];
  __shared__ float2 s_ml[4][32];
  const int tid = threadIdx.x;
  const int wave = uniform(tid >> 6);
  const int lane = tid & 63;
  const int n32 = lane & 31;
  const int j2 = lane >> 5;
  RowsWork w;
  if (!rows_work(p, w)) return;
  const int t_begin = w.t_begin, t_end = w.t_end, here = w.here;
  const int nblk = max((w.nblk - wave + 3) >> 2, 0);  // this wave's
  const int lim_lane = w.first_pos + quotient(min(w.row0 + n32, w.R_all - 1), p.by_H) + 1;
  const uint32_t lds0 = (uint32_t)uniform(
      (int)((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_mem + kFewWave * wave));
  char* const mem = s_mem + kFewWave * wave;
  // offsets, within a block's rows in HBM, of the chunks this lane loads, two to a register
  constexpr int kOff = (kFewDma + 1) / 2;
  uint32_t offp[kOff];
#pragma unroll
  for (int j = 0; j < kOff; ++j) {
    uint32_t v = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 64 * min(2 * j + h, kFewDma - 1) + lane;
      const int g = min(c / 145, 7);
      const int r = 4 * g + min((c - 145 * g) / 36, 3);
      v |= (uint32_t)(r * kRow + 16 * min(c - few_row_off(r), 35)) << (16 * h);
    }
    offp[j] = v;
  }
  const uint32_t v_lane = [&] {
    const int ch = (lane >> 4) & 1, e = (lane & 15) >> 1;
    return (uint32_t)(16 * few_row_off(8 * (e >> 2) + 4 * j2 + (e & 3)) + 16 * ch + 8 * (lane & 1));
  }();

  // Pool token index of the wave's blocks, 64 at a time (ws_mla_wide.h), bit 31: a bad page.
  const int32_t* pt = p.page_table + (size_t)w.pl.b * p.max_pages;
  int pid_base = 0, m_tok = 0;
  auto first_tok = [&]() __attribute__((always_inline)) {
    return t_begin + 32 * (wave + 4 * min(pid_base + lane, nblk - 1));
  };
  auto set_pids = [&](int raw) __attribute__((always_inline)) {
    const int t0 = first_tok();
    const int page = quotient(t0, p.by_page);
    const int pid = clamp_page(raw, p.num_pages);
    m_tok = (pid * p.page_size + (t0 - page * p.page_size)) | (raw == pid ? 0 : (int)0x80000000u);
  };
  uint32_t bad_bits = 0;
  // Block i's loads into slot i % 2
  auto issue = [&](int i) __attribute__((always_inline)) {
    if (i - pid_base >= 64) {
      pid_base += 64;
      set_pids(pt[quotient(first_tok(), p.by_page)]);
    }
    const int tok_raw = __builtin_amdgcn_readlane(m_tok, i - pid_base);
    const uint32_t bit = 1u << (i & 1);
    bad_bits = tok_raw < 0 ? bad_bits | bit : bad_bits & ~bit;
    const uint32_t tok = (uint32_t)tok_raw & 0x7fffffffu;
    const int nt = min(t_end - (t_begin + 32 * (wave + 4 * i)), 32);
    const char* sb = (const char*)p.latent + (size_t)tok * kRow;
    const uint32_t lim = nt >= 32 ? 0xffffu : (uint32_t)((nt - 1) * kRow + kRow - 16);
    const uint32_t base = lds0 + kFewSlot * (i & 1);
#pragma unroll
    for (int j = 0; j < kFewDma; ++j) {
      asm volatile("" : "+v"(offp[j >> 1]));
      const uint32_t pr = offp[j >> 1];
      rows_dma16(min((j & 1) ? pr >> 16 : pr & 0xffffu, lim), sb, base, 1024 * j);
    }
    rows_dma1(min((uint32_t)n32 >> p.block_log2, (uint32_t)(nt - 1) >> p.block_log2),
              p.scale + (tok >> p.block_log2), lds0 + 2 * kFewSlot + 256 * (i & 1));
  };

  // Q^T of the tile's rows: k-steps 2 u and 2 u + 1 hold columns 32 u + 16 j2 .. + 8 and the
  // eight behind them, as a 16-byte read of the latents delivers them.
  u32x4 qb[36];
  if (nblk > 0) {
    int raw_pid = pt[quotient(first_tok(), p.by_page)];
    const uint16_t* qrow0 = p.q_nope + w.g_row0 * kRowsC;
#pragma clang loop unroll(disable)
    for (int h = 0; h < here; ++h)
      rows_dma16(16 * lane, qrow0 + h * kRowsC, lds0 + (uint32_t)(h * 65 * 16), 0);
    const u32x4* pe = (const u32x4*)(p.q_pe + (w.g_row0 + min(n32, here - 1)) * kRowsPe);
#pragma unroll
    for (int u = 32; u < 36; ++u) qb[u] = pe[4 * ((u - 32) >> 1) + 2 * j2 + (u & 1)];
    asm volatile("s_waitcnt vmcnt(0)" : "+v"(raw_pid) : : "memory");
    set_pids(raw_pid);
    const u32x4* qs = (const u32x4*)mem + min(n32, here - 1) * 65;
#pragma unroll
    for (int u = 0; u < 32; ++u) qb[u] = qs[4 * (u >> 1) + 2 * j2 + (u & 1)];
    if (p.q_sign) {
#pragma unroll
      for (int u = 0; u < 36; ++u) qb[u] ^= p.q_sign;
    }
#pragma unroll
    for (int u = 0; u < 36; ++u) asm volatile("" : : "v"(qb[u]));
    wide_lds_wait();  // the staged rows are read
  }

  f32x16 acc[16];
  float m_run = neg_inf(), m_max = neg_inf(), s_run = 0.f;
  const float sx = p.scale_log2;
  auto pv_mfma = [&](const u32x4& va, const u32x4& pbs, int m) __attribute__((always_inline)) {
    f32x16& a = acc[m & 15];
    a = mfma32x32x16(va, pbs, a);
    asm volatile("" : "+a"(a));
    asm volatile("" : : : "memory");
  };
  auto block = [&](int i) __attribute__((always_inline)) {
    const uint32_t tile = lds0 + kFewSlot * (i & 1);
    const uint32_t scales = lds0 + 2 * kFewSlot + 256 * (i & 1);
    const int t0 = t_begin + 32 * (wave + 4 * i);
    f32x16 v;
    {
      const float ts = __builtin_bit_cast(float, rows_lds_b32(scales + 4 * n32) << 23);
      uint32_t row = 16 * (uint32_t)few_row_off(n32) + 16 * j2;
      asm volatile("" : "+v"(row));
      u32x4 kr[4];
#pragma unroll
      for (int u = 0; u < 3; ++u) kr[u] = rows_lds_b128(tile + row + 32 * u);
#pragma unroll
      for (int u = 0; u < 18; ++u) {
        if (u + 3 < 18) kr[(u + 3) & 3] = rows_lds_b128(tile + row + 32 * (u + 3));
        const u32x4& k = kr[u & 3];
        if (u == 0) qk_first_new(v, widen8(k[0], k[1], ts), qb[0]);
        else qk_next_new(v, widen8(k[0], k[1], ts), qb[2 * u]);
        qk_next_new(v, widen8(k[2], k[3], ts), qb[2 * u + 1]);
      }
      qk_settle(v);
    }
    // (mla_rows_kernel's soft_x)
    bool odd = false;
    const bool bad_page = (bad_bits >> (i & 1)) & 1;
    const int lim = lim_lane - t0 - 4 * j2;
    if (t0 + 32 > w.lim_lo || bad_page) {
      bool hidden = false;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool seen = 8 * (e >> 2) + (e & 3) < lim;
        hidden |= !seen && !(__builtin_fabsf(v[e]) < __builtin_inff());
        v[e] = !seen ? neg_inf() : bad_page ? qnan() : v[e];
      }
      odd = __builtin_amdgcn_ballot_w64(hidden) != 0;
    }
    float r = max3(v[0], v[1], v[2]);
#pragma unroll
    for (int e = 3; e < 15; e += 2) r = max3(r, v[e], v[e + 1]);
    m_max = max3(r, v[15], m_max);
    if (i == 0) {
      float lo, hi;
      pair_xor32(m_max * sx, lo, hi);
      m_run = m_run == neg_inf() ? fmaxf(lo, hi) : m_run;
      m_run = m_run == neg_inf() ? 0.f : m_run;
    }
    if (__builtin_expect(odd, 0)) {  // (mla_rows_kernel's clean: the slot is the wave's own)
#pragma clang loop unroll(disable)
      for (int c = lane; c < kFewSlot / 16; c += 64) {
        u32x4 x = rows_lds_b128(tile + 16 * c);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] &= ~nan_bytes(x[e]);
        rows_lds_put(tile + 16 * c, x);
      }
      uint32_t* sp = (uint32_t*)(mem + 2 * kFewSlot + 256 * (i & 1)) + lane;
      if (*sp == 255) *sp = 0;
      wide_lds_wait();
    }
    u32x4 pb[2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const u32x4 ts = rows_lds_b128(scales + 4 * (16 * s + 8 * g + 4 * j2));
        float e[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          e[c] = __builtin_amdgcn_exp2f(__builtin_fmaf(v[8 * s + 4 * g + c], sx, -m_run));
          s_run += e[c];
          e[c] *= __builtin_bit_cast(float, ts[c] << 23);
        }
        pb[s][2 * g] = pack_bf16x2(e[0], e[1]);
        pb[s][2 * g + 1] = pack_bf16x2(e[2], e[3]);
      }
    uint32_t vt = v_lane;
    asm volatile("" : "+v"(vt));
    vt += tile;
    auto vread = [&](int m) __attribute__((always_inline)) {
      return lds_read_tr8_b64(vt + 16 * 580 * (m >> 4) + 32 * (m & 15));
    };
    uint2 va[4];
#pragma unroll
    for (int m = 0; m < 3; ++m) va[m] = vread(m);
    u32x4 cur = widen8(va[0].x, va[0].y, 1.f);
#pragma unroll
    for (int m = 0; m < 32; ++m) {
      if (m + 3 < 32) va[(m + 3) & 3] = vread(m + 3);
      const u32x4 now = cur;
      if (m + 1 < 32) cur = widen8(va[(m + 1) & 3].x, va[(m + 1) & 3].y, 1.f);
      pv_mfma(now, pb[m >> 4], m);
    }
  };

  for (int pass = 0;; ++pass) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[e][i] = 0.f;
    s_run = 0.f;
    if (nblk == 0) break;
    if (pid_base != 0) {
      pid_base = 0;
      set_pids(pt[quotient(first_tok(), p.by_page)]);
    }
    issue(0);
    if (nblk > 1) issue(1);
#pragma clang loop unroll(disable)
    for (int i = 0; i < nblk; ++i) {
      if (i + 1 < nblk) rows_wait<kFewDma + 1>();
      else rows_wait<0>();
      block(i);
      wide_lds_wait();  // the slot is read
      if (i + 2 < nblk) issue(i + 2);
    }
    float lo, hi;
    pair_xor32(m_max, lo, hi);
    m_max = fmaxf(lo, hi);
    const float top = m_max * sx;
    if (pass > 0 || __builtin_amdgcn_ballot_w64(reference_off(top, m_run)) == 0) break;
    m_run = top == neg_inf() ? 0.f : top;
  }

  // The waves' sums at the largest of their references
  float lo, hi;
  pair_xor32(s_run, lo, hi);
  const float l_w = lo + hi;
  if (j2 == 0) s_ml[wave][n32] = make_float2(l_w == 0.f ? neg_inf() : m_run, l_w);
  __syncthreads();
  float M = neg_inf(), total = 0.f;
#pragma unroll
  for (int o = 0; o < 4; ++o) M = fmaxf(M, s_ml[o][n32].x);
#pragma unroll
  for (int o = 0; o < 4; ++o) {
    const float2 ml = s_ml[o][n32];
    total += ml.x == neg_inf() ? 0.f : __builtin_amdgcn_exp2f(ml.x - M) * ml.y;
  }
  const float f = l_w == 0.f ? 0.f : __builtin_amdgcn_exp2f(m_run - M) / total;
  if (wave == 0 && j2 == 0 && n32 < here) {
    const float lse_v = total == 0.f ? neg_inf() : (M + __log2f(total)) * kLn2;
    const size_t at = w.o_row0 + n32;
    if (w.piece) p.part_lse[at] = lse_v;
    else if (p.lse) p.lse[at] = lse_v;
  }
  uint16_t* to16 = w.piece ? p.part_out : p.out_bf16;
  float* to32 = w.piece ? nullptr : p.out_f32;
  float* stage = (float*)mem;
#pragma unroll
  for (int hc = 0; hc < 2; ++hc) {  // 256 columns at a time
    if (hc > 0) __syncthreads();
    if (n32 < here)
#pragma unroll
    for (int c8 = 0; c8 < 8; ++c8)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int ct = 8 * hc + c8;
        *(float4*)(stage + n32 * 260 + 32 * c8 + 8 * q + 4 * j2) =
            make_float4(acc[ct][4 * q] * f, acc[ct][4 * q + 1] * f, acc[ct][4 * q + 2] * f,
                        acc[ct][4 * q + 3] * f);
      }
    __syncthreads();
    for (int row = wave; row < here; row += 4) {
      float4 x = *(const float4*)((const float*)s_mem + row * 260 + 4 * lane);
#pragma unroll
      for (int o = 1; o < 4; ++o) {
        const float4 y = *(const float4*)((const float*)(s_mem + kFewWave * o) + row * 260 + 4 * lane);
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
      }
      const size_t at = (w.o_row0 + row) * (kRowsC / 4) + 64 * hc + lane;
      if (to16) ((uint2*)to16)[at] = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
      if (to32) ((float4*)to32)[at] = x;
    }
  }
}

// Combines the pieces of the tiles that were split: a wave a row, or (p.join_shared: many
// pieces a tile, on average) a workgroup a row, each wave a quarter of the pieces.  A lane has
// eight columns.  (Without shared rows a workgroup takes kJoinRows: in a call whose tiles
// fill the chip hardly any is split, and every workgroup looks for its tile first.)  A launch,
// the look for the tile and one chain of loads, 5 us; 8 tiles of 128 rows in 32 pieces each, 34 MB,
// 9.7 us.  Shared rows for kJoinShared pieces a tile and more, over the fewest tiles that the
// call's rows can make: 16 tiles of 16 pieces 50 us with the attention and 64 with a wave a row, 24
// prompts of 2 or 3 pieces 88 and 69.  (Over the most tiles, a sequence more for each, 8 x 4
// drafted tokens of 16 heads over 4000 to 32000 8-bit tokens took 54 us instead of 40.5, 20 x 7 of
// 4 heads over bf16 54 instead of 45; 12 x 10 of 16 heads, 24 tiles for 15, 56 instead of 58.)
constexpr int kJoinRows = 16;
constexpr int kJoinShared = 12;
struct JoinAcc {
  float m, sum;
  float a[8];
};
__device__ __forceinline__ void join_pieces(JoinAcc& x, const uint16_t* out, const float* lse,
                                            int rows, int first, int step, int n) {
  const int lane = threadIdx.x & 63;
  constexpr int U = 16;  // pieces under way
  for (int s = first; s < n; s += U * step) {
    float l[U];
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) l[u] = lse[(size_t)min(s + u * step, n - 1) * rows];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = ((const u32x4*)(out + (size_t)min(s + u * step, n - 1) * rows * kRowsC))[lane];
    float m = x.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u * step >= n) l[u] = neg_inf();
      m = fmaxf(m, l[u]);
    }
    const float f = acc_factor(x.m, m);
    x.m = m;
    x.sum *= f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x.a[i] *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u * step >= n) continue;
      const float wt = piece_weight(l[u], m);
      x.sum += wt;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x.a[2 * i] += wt * __builtin_bit_cast(float, v[u][i] << 16);
        x.a[2 * i + 1] += wt * __builtin_bit_cast(float, v[u][i] & 0xffff0000u);
      }
    }
  }
}
__device__ __forceinline__ void join_row(const RowsParams& p, const RowsPlace& tl, int tr, bool shared,
                                         JoinAcc (*s_acc)[64]) {
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  JoinAcc x;
  x.m = neg_inf();
  x.sum = 0.f;
#pragma unroll
  for (int c = 0; c < 8; ++c) x.a[c] = 0.f;
  const size_t slot = (size_t)tl.piece * p.piece_rows + tr;
  join_pieces(x, p.part_out + slot * kRowsC, p.part_lse + slot, p.piece_rows, shared ? wave : 0,
              shared ? 4 : 1, tl.splits);
  if (shared) {
    if (wave > 0) s_acc[wave - 1][lane] = x;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int o = 0; o < 3; ++o) {
      const JoinAcc y = s_acc[o][lane];
      const float m = fmaxf(x.m, y.m);
      const float fx = acc_factor(x.m, m), fy = acc_factor(y.m, m);
      x.m = m;
      x.sum = x.sum * fx + y.sum * fy;
#pragma unroll
      for (int c = 0; c < 8; ++c) x.a[c] = x.a[c] * fx + y.a[c] * fy;
    }
  }
  const float inv = x.sum == 0.f ? 0.f : 1.f / x.sum;
#pragma unroll
  for (int c = 0; c < 8; ++c) x.a[c] *= inv;
  const size_t at = (size_t)tl.c0 * p.H + tl.tile * p.tile + tr;
  if (p.out_f32) {
    float4* dst = (float4*)(p.out_f32 + at * kRowsC) + 2 * lane;
    dst[0] = make_float4(x.a[0], x.a[1], x.a[2], x.a[3]);
    dst[1] = make_float4(x.a[4], x.a[5], x.a[6], x.a[7]);
  }
  if (p.out_bf16) {
    u32x4 o;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = pack_bf16x2(x.a[2 * c], x.a[2 * c + 1]);
    ((u32x4*)(p.out_bf16 + at * kRowsC))[lane] = o;
  }
  if (p.lse && lane == 0) p.lse[at] = x.sum == 0.f ? neg_inf() : x.m + __logf(x.sum);
}
__global__ __launch_bounds__(256) void mla_rows_join_kernel(const RowsParams p) {
  __shared__ JoinAcc s_acc[3][64];
  const RowsPlace tl = rows_place<true>(p, blockIdx.x);
  if (tl.b < 0 || tl.splits == 1 || tl.piece < 0 || tl.piece + tl.splits > p.pieces) return;
  const int wave = uniform(threadIdx.x >> 6);
  const int here = min(p.tile, tl.n * p.H - tl.tile * p.tile);
  const bool shared = p.join_shared;
  // row of the tile (with `shared` the whole workgroup's)
  int tr = shared ? blockIdx.y : blockIdx.y * kJoinRows + wave;
  for (int more = shared ? 1 : kJoinRows / 4; more > 0 && tr < here; --more, tr += 4)
    join_row(p, tl, tr, shared, s_acc);
}

// The tokens of every sequence that has rows, from 8-bit pages, as bf16 rows [b][pad], one page a
// sequence (table: its id), for prompts whose tiles read them many times.  Tokens in a bad page
// are NaN.  Bound by HBM: 20500 tokens, 35 MB, 13.8 us (9.8 where the last cache holds the pages).
// (A chunk of 2400 tokens of 16 heads beside 23 idle sequences, 8000 tokens each: 609 us, and 669
// with the idle ones' tokens too.)
constexpr int kWidenTokens = 32;  // of a workgroup
__global__ __launch_bounds__(256) void latent_widen_kernel(const RowsParams p, uint16_t* copy,
                                                           int32_t* table, int pad) {
  const int b = blockIdx.y, t0 = blockIdx.x * kWidenTokens;
  if (blockIdx.x == 0 && threadIdx.x == 0) table[b] = b;
  const RowsSeq seq = rows_seq(p, b);
  const int len = seq.len;
  if (seq.n == 0 || !len_ok(len, 0, min(p.cap, pad)) || t0 >= len) return;
  const int page = t0 / p.page_size;  // (32 tokens lie in one page)
  const int raw = p.page_table[(size_t)b * p.max_pages + page];
  const int pid = clamp_page(raw, p.num_pages);
  const size_t tok = (size_t)pid * p.page_size + (t0 - page * p.page_size);
  const u32x4* src = (const u32x4*)((const uint8_t*)p.latent + tok * 576);
  u32x4* dst = (u32x4*)(copy + ((size_t)b * pad + t0) * 576);
  const int n = min(kWidenTokens, len - t0) * 36;
#pragma unroll
  for (int j = 0; j < (kWidenTokens * 36 + 255) / 256; ++j) {
    const int i = threadIdx.x + 256 * j;
    if (i >= n) break;
    const u32x4 w = src[i];
    const float s =
        raw == pid ? __builtin_bit_cast(float, (uint32_t)p.scale[(tok + i / 36) >> p.block_log2] << 23) : qnan();
    dst[2 * i] = widen8(w[0], w[1], s);
    dst[2 * i + 1] = widen8(w[2], w[3], s);
  }
}

// ---------------------------------------------------------------------------

// Tiles of a sequence, on average, from which its latents are widened in a pass of their own,
// and the largest copy.  Widening in the steps costs every tile again, the copy once (4
// prompts of 16 heads behind 500 to 8000 tokens, in the steps and by the copy: 64 new tokens,
// 8 tiles each, 55 and 59 us, 96 66 and 67, 128 78 and 77, 256 139 and 129).
constexpr int kWidenTiles = 12;
constexpr size_t kWidenBytes = 256u << 20;

// Rows of a sequence, on average, up to which 8-bit pages are read by mla_few_kernel, and
// with few tokens up to a whole tile of the other kernel's, for the shorter start and end
// (mla_rows_kernel and mla_few_kernel, with the join, us: 8 x 4 drafted tokens of 16 heads over
// 4000 to 32000 49 and 40.5, 16 x 4 92 and 75.5; decode of 16 sequences of 3000 to 32768 tokens, 16
// heads 83 and 50, 40 heads 88 and 79, 32 of 64 heads 183 and 134, 128 heads 202 and 273; one of
// 4000 tokens, 16 heads 21 and 16, 128 heads 24.6 and 19.3; 4 of 8000, 128 heads 34 and 28.6; 60
// of 500 to 2000 54.5 and 48.2, 140 of 500 to 4000 137 and 160).
constexpr int kFewRows = 64;
constexpr long long kFewTokens = 1 << 17;

struct RowsPlan {
  long long tiles, grid, pieces, joins;
  size_t copy;  // bytes of the widened latents (0: none)
  int pad;      // tokens of a sequence there
  int fill, piece_rows, tile;
  bool fit, few, join_shared;
};
// decode: one token a sequence
static RowsPlan rows_plan(int N, int B, int H, bool decode, bool fp8, int max_len, int n_splits) {
  RowsPlan r;
  const long long rows = (long long)N * H;
  r.few = fp8 && (rows <= (long long)kFewRows * B ||
                  (rows <= (long long)kRowsTile * B && (long long)B * max_len <= kFewTokens));
  r.tile = r.few ? kFewTile : kRowsTile;
  const long long each = (H + r.tile - 1) / r.tile;
  r.tiles = decode ? B * each : std::min((long long)N * H / r.tile + B, (long long)N * each);
  r.pad = std::max((max_len + 31) & ~31, 32);
  r.copy = fp8 && !decode && (long long)N * H >= (long long)kWidenTiles * r.tile * B
               ? (size_t)B * r.pad * 1152
               : 0;
  if (r.copy > kWidenBytes) r.copy = 0;
  r.fill = choose_workgroups(0, 1, 1LL << 30, 1);
  r.fit = r.tiles < r.fill && B <= 256;
  r.piece_rows = (int)std::min<long long>(r.tile, decode ? H : (long long)N * H);
  r.grid = r.tiles;
  r.pieces = r.joins = 0;
  if (n_splits > 1) {
    r.pieces = r.grid = r.tiles * n_splits;
    r.joins = r.tiles;
  } else if (n_splits == 0 && max_len > 32 * kRowsMinShare) {
    // Only a tile of more than M blocks is split.  All items fit `fill`, or M is the blocks
    // over `fill`, and then split tiles are fewer than `fill` and leave twice as many pieces
    // at the most.
    r.pieces = r.fit ? r.fill : 2LL * r.fill + 64;
    r.grid = r.fit ? r.fill : r.tiles + r.pieces;
    r.joins = std::min<long long>(r.tiles, r.fill);
  }
  // pieces a tile: of the tiles that there are at the least (r.tiles is the most)
  const long long least = std::max(((long long)N * H + r.tile - 1) / r.tile, (long long)std::min(N, B));
  r.join_shared = n_splits > 1 ? n_splits >= kJoinShared : r.pieces >= kJoinShared * (decode ? r.tiles : least);
  return r;
}
// The workspace: the pieces' lse and outputs, the copy's table and rows.
static size_t rows_piece_bytes(const RowsPlan& pl) {
  const size_t rows = (size_t)pl.pieces * pl.piece_rows;
  return align256(rows * 4) + align256(rows * kRowsC * 2);
}
static size_t rows_bytes(const RowsPlan& pl, int B) {
  return rows_piece_bytes(pl) + (pl.copy ? align256((size_t)B * 4) + pl.copy : 0);
}

static int rows_sizes(const char* name, int N, int B, int H, bool decode, bool fp8, int max_len,
                      int n_splits) {
  if (N < 0 || B < 0 || B > kMaxSeqs || H <= 0 || H > 1024 || max_len < 0 || n_splits < 0 ||
      n_splits > kRowsMaxSplits)
    return set_error(WS_EINVAL,
                     "%s: bad sizes N=%d B=%d H=%d max_len=%d n_splits=%d (B <= %d, H <= 1024, "
                     "n_splits <= %d)",
                     name, N, B, H, max_len, n_splits, kMaxSeqs, kRowsMaxSplits);
  if ((long long)N * H + 256LL * B >= (1LL << 31) || max_len > (1 << 30))
    return set_error(WS_EINVAL, "%s: %d tokens of %d heads exceed the row index range", name, N, H);
  if (rows_plan(N, B, H, decode, fp8, max_len, n_splits).grid * 256 >= (1LL << 32))
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
  if (int rc = rows_sizes(name, N, B, H, decode, latent_scale != nullptr, max_len, n_splits)) return rc;
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
  const RowsPlan pl = rows_plan(N, B, H, decode, latent_scale != nullptr, max_len, n_splits);
  const size_t need = rows_bytes(pl, B);
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
  p.part_out = (uint16_t*)((char*)workspace + align256((size_t)pl.pieces * pl.piece_rows * 4));
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
  p.tile = pl.tile;
  p.tile_log2 = pl.few ? 5 : 7;
  p.by_H = divisor((uint32_t)H);
  p.by_page = divisor((uint32_t)page_size);
  p.join_shared = pl.join_shared;
  // the smallest normal float for 0: every finite score then rounds to the same
  // probability, and masked tokens stay -inf
  p.scale_log2 = std::max((scale < 0.f ? -scale : scale) * kLog2e, 1.17549435e-38f);
  p.q_sign = scale < 0.f ? 0x80008000u : 0u;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)pl.grid), block(256);
  if (pl.copy) {
    int32_t* table = (int32_t*)((char*)workspace + rows_piece_bytes(pl));
    uint16_t* copy = (uint16_t*)((char*)table + align256((size_t)B * 4));
    hipLaunchKernelGGL(latent_widen_kernel, dim3((unsigned)(pl.pad / kWidenTokens), (unsigned)B), block, 0, s,
                       p, copy, table, pl.pad);
    if (int rc = check_launch(name)) return rc;
    p.latent = copy;
    p.page_table = table;
    p.page_size = p.cap = pl.pad;  // (a length past max_len, which the call rules out, is NaN)
    p.by_page = divisor((uint32_t)pl.pad);
    p.max_pages = 1;
    p.num_pages = B;
  }
  if (pl.few)
    hipLaunchKernelGGL(mla_few_kernel, grid, block, 0, s, p);
  else if (latent_scale && !pl.copy)
    hipLaunchKernelGGL(mla_rows_kernel<true>, grid, block, 0, s, p);
  else
    hipLaunchKernelGGL(mla_rows_kernel<false>, grid, block, 0, s, p);
  int rc = check_launch(name);
  if (rc != WS_OK || pl.pieces == 0) return rc;
  hipLaunchKernelGGL(mla_rows_join_kernel,
                     dim3((unsigned)pl.joins, p.join_shared ? pl.piece_rows : (pl.piece_rows + kJoinRows - 1) / kJoinRows),
                     block, 0, s, p);
  return check_launch(name);
}

static int rows_plan_out(const char* name, int N, int B, int H, bool decode, bool fp8, int max_len,
                         int n_splits, int* pieces_out, size_t* bytes_out) {
  if (int rc = rows_sizes(name, N, B, H, decode, fp8, max_len, n_splits)) return rc;
  const RowsPlan pl = rows_plan(N, B, H, decode, fp8, max_len, n_splits);
  if (pieces_out) *pieces_out = (int)pl.pieces;
  if (bytes_out) *bytes_out = rows_bytes(pl, B);
  return WS_OK;
}

}  // namespace ws

using namespace ws;

extern "C" int ws_mla_prompt_plan(int N, int B, int H, int fp8, int max_len, int n_splits,
                                  int* pieces_out, size_t* workspace_bytes_out) {
  return rows_plan_out("ws_mla_prompt_plan", N, B, H, false, fp8 != 0, max_len, n_splits, pieces_out,
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
  return rows_plan_out("ws_mla8_decode_plan", B, B, H, true, true, max_len, n_splits, pieces_out,
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
