// Prompt attention over the pages (gfx950): the new tokens of every sequence,
// ragged and causal, over everything of the sequence that the partition holds,
// bf16 pages or 8-bit ones (e4m3 with an e8m0 scale per token and KV head).
//
// Query i of a sequence's n (tokens cu[b] .. cu[b + 1] of q) stands at position
// len - n + i of the len tokens in the pages and sees positions 0 .. its own.
// The query rows of a KV head are (token, head of the group) pairs, row = i G + g,
// so the G heads that share K and V share their loads: a workgroup takes a tile of
// 32 NW consecutive rows, a wave 32 of them, and walks the tokens in tiles
// of 32 through LDS with a running maximum and sum (one pass over K and V).
//
//   S^T[token, row] = K Q^T   A = K from LDS (16 bytes a lane), B = Q in registers
//   O^T[col, row] += V^T P^T  A = V^T read transposed from LDS, B = P as it comes out
//                             of S^T: the 32x32 product's output rows 8 a + 4 h + b of
//                             lane half h are taken as k slots in that order, in P and
//                             V alike
// A row is one lane column: its maximum takes one exchange between the lane halves,
// its rescaling no exchange at all.
//
// P is rounded to bf16 for the values' product, the matrix cores' operand type (as the
// decode kernels round theirs); its row sum takes the values before, in fp32 as the maximum,
// the output's sums and the pieces.  Error against 64 bits: 2.0e-3 to 2.3e-3 of the
// output, where fp32 work rounded to bf16 at the end has 1.5e-3 to 1.7e-3.
//
// A row sees nothing of the tokens past its position: their scores are masked, and
// so are their values, which P = 0 alone would not do for an infinity or a NaN
// (0 * inf): where a tile that some row masks holds one, values_masked adds it to the rows
// that see it.
//
// With few rows the tokens are split over several workgroups of a tile, so that all
// take about as many, whatever the sequences' lengths; prompt_join_kernel combines
// their pieces (fp32, with their lse).
//
// Long prompts are bound by the power of the products and by the vector work beside them:
// 8192 tokens of 8 x 4 heads of 128 take 525 to 550 us (1.00 to 1.05 PFLOP/s; 392 on
// zeros, at a higher clock).  Few rows are bound by HBM: 567 MB in 93.7 us (6.1 TB/s) and
// the join 5.0.
#include <algorithm>
#include <type_traits>

#include "ws_attn.h"
#include "ws_plan.h"
#include "ws_reduce.h"

namespace ws {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kPromptMaxD = 256;
constexpr int kPromptTile = 32;    // tokens of a tile
constexpr int kPromptSlots = 4;    // LDS slots of K and of V
// 16-byte chunks of a tile's row lie in LDS in an order of their own, chunk ^ f(row), so
// that no two of a read meet in a bank (256 bytes of banks): 16 rows' 16-byte loads of
// one K chunk, 4 rows' transposed reads of 64 bytes of V.  f keeps a chunk in its group
// of the row's largest power of two of chunks, p; 16 / p rows apart lies the next row
// that begins at the same bank.
__host__ __device__ constexpr int prompt_pow2(int D) {
  const int ch = D / 8, p = ch & -ch;
  return p < 16 ? p : 16;
}
__host__ __device__ constexpr int prompt_k_swap(int D, int row) {
  return (row / (16 / prompt_pow2(D))) & (prompt_pow2(D) - 1);
}
__host__ __device__ constexpr int prompt_v_swap(int D, int row) {
  return prompt_pow2(D) == 16  ? (row & 3) << 2
         : prompt_pow2(D) == 8 ? (row >> 1 & 1) << 2
                               : 0;
}
constexpr int kPromptMaxSplits = 64;

struct PromptParams {
  const uint16_t* q;
  const void* k_pages;
  const void* v_pages;
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  const int32_t* page_table;
  const int32_t* kv_len;
  const int32_t* cu_new;
  uint16_t* out_bf16;
  float* out_f32;
  float* lse;
  float* part_out;  // [pieces][rows of a tile][D], with part_lse [pieces][rows] (split tiles')
  float* part_lse;
  int N, B, Hq, Hkv, G, page_size, max_pages, num_pages, cap;
  int n_splits;  // of every tile; 0: by the lengths, `share` workgroups in all (0: one a tile)
  int share;
  long long pieces;  // room for them
  float scale_log2;  // >= 0
  uint32_t q_sign;   // 0x80008000 where the caller's scale is negative
};

// Holds a value's computation between the sched_barriers around it: values that no
// memory access needs are otherwise placed by the compiler.
template <class T>
__device__ __forceinline__ void pin(T& x) {
  asm volatile("" : "+v"(x));
}
// The same of an output's sums, which lie in the accumulation registers in the kernels
// that take more than 256 registers.
template <bool ACC>
__device__ __forceinline__ void pin_sum(f32x16& x) {
  if constexpr (ACC)
    asm volatile("" : "+a"(x));
  else
    asm volatile("" : "+v"(x));
}
__device__ __forceinline__ u32x4 lds_read_b128(uint32_t addr) {
  return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)addr;
}
__device__ __forceinline__ f32x16 mfma32x32x16(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool HI>
__device__ __forceinline__ uint32_t cvt2_fp8(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
__device__ __forceinline__ u32x4 cvt8_fp8(uint32_t lo, uint32_t hi, float scale) {
  return u32x4{cvt2_fp8<false>(lo, scale), cvt2_fp8<true>(lo, scale), cvt2_fp8<false>(hi, scale),
               cvt2_fp8<true>(hi, scale)};
}

// Whether one of eight bf16 values is an infinity or a NaN.
__device__ __forceinline__ bool any_nonfinite(const u32x4& w) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    bad |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// Two bf16 values without their infinities and NaN (0 there), and 1 where they are
// +inf or NaN (pos), -inf or NaN (neg).
__device__ __forceinline__ void split_nonfinite(uint32_t& w, uint32_t& pos, uint32_t& neg) {
  // the exponent bits of each half all set: a carry out of them into the sign's place
  const uint32_t lo = (((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15;  // 1 per half
  const uint32_t man = (((w & 0x007f007fu) + 0x007f007fu) & 0x00800080u) >> 7;  // a NaN's
  const uint32_t sign = (w >> 15) & 0x00010001u;
  pos = (lo & (man | ~sign)) * 0x3f80u;
  neg = (lo & (man | sign)) * 0x3f80u;
  w &= ~(lo * 0xffffu);
}

// A workgroup's place in the list of all sequences' tiles of `rows` rows (of the tiles
// alone, or of every tile's splits).
struct PromptPlace {
  int b;              // the sequence (< 0: past the list's end)
  int tile;           // tile of its rows
  int split, splits;  // and which of the tile's splits
  int piece;          // a split tile's piece, less the KV head: (piece * Hkv + kvh)
  int c0, n;          // the sequence's first row of q and its tokens
  int len;
};
// What the list needs of a sequence.
struct PromptSeq {
  int c0, n, len, tiles, blocks;
};
__device__ __forceinline__ PromptSeq prompt_seq(const PromptParams& p, int b, int rows) {
  PromptSeq s;
  s.c0 = min(max(p.cu_new[b], 0), p.N);
  s.n = min(max(p.cu_new[b + 1], s.c0), p.N) - s.c0;
  s.len = p.kv_len[b];
  s.tiles = (s.n * p.G + rows - 1) / rows;
  s.blocks = len_ok(s.len, 0, p.cap) ? (s.len + kPromptTile - 1) / kPromptTile : 0;
  return s;
}
constexpr int kPromptMinShare = 8;  // tiles of tokens of a split, at the least

// Item `at` of the list: longest sequences first (up to 64 of them), their last tile
// first, since it walks the most tokens: the short ones fill the chip's end.  The splits
// of a sequence's tiles: as many as give each `per_split` tiles of tokens, the batch's
// total over `share` workgroups (computed alike by every caller).  Every lane must call
// it; the result is uniform.
template <bool TILES>
__device__ __forceinline__ PromptPlace prompt_place(const PromptParams& p, int at, int rows) {
  const int lane = threadIdx.x & 63;
  const int per = (p.B + 63) >> 6;
  const int b0 = lane * per;
  int per_split = 0;
  if (p.share > 0) {
    float total = 0.f;
    for (int k = 0; k < per && b0 + k < p.B; ++k) {
      const PromptSeq s = prompt_seq(p, b0 + k, rows);
      total = fmaf((float)s.tiles, (float)s.blocks, total);  // (the same in both kernels)
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o);
    per_split = max((int)min(total * (float)p.Hkv / (float)p.share, 1e9f) + 1, kPromptMinShare);
  }
  auto splits_of = [&](const PromptSeq& s) {
    if (p.share == 0) return max(p.n_splits, 1);
    return max(min((s.blocks + per_split - 1) / per_split, kPromptMaxSplits), 1);
  };
  // a lane's items, and the pieces before its first sequence in the batch's order
  int items = 0, units = 0, key = -1;
  for (int k = 0; k < per && b0 + k < p.B; ++k) {
    const PromptSeq s = prompt_seq(p, b0 + k, rows);
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
  PromptPlace r{-1, 0, 0, 1, 0, 0, 0, 0};
  if (past == 0) return r;
  const int slot = __builtin_ctzll(past);
  int left = at - __builtin_amdgcn_readlane(incl - items, slot);
  const int owner = __builtin_amdgcn_readlane(from, slot);
  int piece = __builtin_amdgcn_readlane(before, owner);
  for (int k = 0; k < per; ++k) {
    const int b = uniform(owner * per + k);
    if (b >= p.B) break;
    const PromptSeq s = prompt_seq(p, b, rows);
    const int splits = uniform(splits_of(s));
    const int here = uniform(TILES ? s.tiles : s.tiles * splits);
    if (left < 0) break;  // (sums past 2^31: cu_new is not non-decreasing)
    if (left < here) {
      const int t = TILES ? left : left / splits;
      r.b = b;
      r.tile = TILES ? t : uniform(s.tiles) - 1 - t;
      r.split = TILES ? 0 : left - t * splits;
      r.splits = splits;
      r.piece = piece + r.tile * splits + r.split;
      r.c0 = uniform(s.c0);
      r.n = uniform(s.n);
      r.len = uniform(s.len);
      break;
    }
    left -= here;
    piece += splits > 1 ? uniform(s.tiles) * splits : 0;
  }
  return r;
}

constexpr int kPromptWaves = 4;  // of a workgroup (one in some calls, prompt_plan)
template <int D, bool F8, int NW>
struct PromptShape {
  static constexpr int kRow = 2 * D;               // bytes of a row in LDS
  static constexpr int kTile = kPromptTile * kRow;  // and of a slot
  // 16-byte pieces (bf16: 8 columns; 8-bit: 16) of a tile's K or V, and of a thread's
  static constexpr int kRowPieces = F8 ? D / 16 : D / 8;
  static constexpr int kPieces = kPromptTile * kRowPieces;
  static constexpr int kThreads = 64 * NW;
  static constexpr int kLoads = (kPieces + kThreads - 1) / kThreads;
};

template <int I, int N, class F>
__device__ __forceinline__ void static_for_prompt(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for_prompt<I + 1, N>(f);
  }
}

// 16 bytes a lane from `base` + off to LDS at `lds` + AT + 16 * lane, with no register
// between (counted by vmcnt; the caller waits, then passes a barrier).  In assembly because
// the compiler would wait for every one of them ahead of any LDS read.
// ONCE: the tile is read once (the calls of few rows), so it need not stay in the caches
// (the non-temporal hint: 140 -> 129 us for 8 x 5 tokens over 4000 to 32000).
// m0 is named as written, though the compiler says that it need not keep a reserved
// register across the block: what counts is that it expects no old value there.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int AT, bool ONCE>
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t off, uint32_t lds) {
  if constexpr (ONCE)
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                 :
                 : "v"(off), "s"(base), "s"(lds), "n"(AT)
                 : "memory", "scc", "m0");
  else
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(off), "s"(base), "s"(lds), "n"(AT)
                 : "memory", "scc", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N < 63 ? N : 63) : "memory");
}

// The loop is a pipeline over 32-token tiles: step t takes the softmax of tile t,
// whose scores the step before computed, the scores of tile t + 1 and the values'
// product of tile t - 1, three independent strands, so that the matrix cores run
// under the softmax's vector work (which costs about as many cycles: 32 rows x 32
// tokens take 512 cycles of products at D = 128, and 16 exponentials of 16 cycles and
// some 50 other instructions of 4).  A row whose maximum moved rescales its sums after
// the step's products, which still are relative to the old one.
//
// K and V go through LDS in four slots each: step t reads K of tile t + 1 and V of
// tile t - 1.  bf16 tiles are loaded straight to LDS, three steps ahead (K of tile t + 4
// and V of t + 2 in step t, to the slots the step before has left); 8-bit ones through
// registers, requested two steps before they are converted and written.  One barrier a
// step.
//
// FEW: calls of few rows.  A tile of tokens is read by one workgroup only, so it need not
// stay in the caches, and waves without rows only load.
template <int D, bool F8, int NW, bool FEW>
__global__ __launch_bounds__(64 * NW, D <= 128 ? 2 : 1) void prompt_kernel(const PromptParams p) {
  static_assert(D % 32 == 0 && D <= kPromptMaxD, "head width: a multiple of 32 up to 256");
  using Sh = PromptShape<D, F8, NW>;
  constexpr int KS = D / 16;  // k-steps of the scores
  constexpr int DT = D / 32;  // 32-column tiles of the output
  constexpr int CH = Sh::kRowPieces;
  constexpr int LD = Sh::kLoads;
  constexpr int kRows = 32 * NW;
  // k-steps whose q lies in LDS, for the registers that 8-bit tiles take on their way: what
  // the compiler spilled instead came back behind the loads under way, which memory answers
  // in order (8 x 12 tokens over 16000: 114 -> 88 us, 8-bit chunks 381 -> 362).  The loop of
  // the calls of few rows spills nothing since; the other one still reloads six registers
  // in four steps.  Narrower heads need fewer registers, wider ones have twice as many.
  constexpr int kQl = F8 && D == 128 ? 2 : 0;
  constexpr bool kAcc = D > 128 || NW == 1;  // more than 256 registers
  __shared__ __attribute__((aligned(256))) char s_k[kPromptSlots * Sh::kTile];
  __shared__ __attribute__((aligned(256))) char s_v[kPromptSlots * Sh::kTile];
  __shared__ u32x4 s_q[kQl > 0 ? kQl * Sh::kThreads : 1];
  __shared__ int s_bad[2];  // a slot's values held an infinity or a NaN (masked tiles only)

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int n32 = lane & 31;
  const int h = lane >> 5;
  const int id = blockIdx.x;
  const int kvh = id % p.Hkv;
  const PromptPlace tl = prompt_place<false>(p, id / p.Hkv, kRows);
  const bool piece = tl.splits > 1;
  const long long piece_at = (long long)tl.piece * p.Hkv + kvh;
  if (tl.b < 0 || (piece && (piece_at < 0 || piece_at >= p.pieces))) return;
  const int G = p.G;
  const int R = tl.n * G;  // rows of the sequence and KV head
  const int len = tl.len;
  const bool len_good = len_ok(len, 0, p.cap);
  const int first_pos = len - tl.n;  // position of the sequence's first query
  const int row0 = tl.tile * kRows;
  const int rows_here = min(kRows, R - row0);
  // visible tokens of the workgroup's first and last row
  const int lim_lo = first_pos + row0 / G + 1;
  const int lim_hi = len_good ? max(first_pos + (row0 + rows_here - 1) / G + 1, 0) : 0;
  const int nb = (lim_hi + kPromptTile - 1) / kPromptTile;
  const int blk0 = (int)((long long)tl.split * nb / tl.splits);
  const int blk1 = (int)((long long)(tl.split + 1) * nb / tl.splits);

  // the lane's row, the tokens it sees, and its row of out / lse
  const int tile_row = wave * 32 + n32;
  const bool live = row0 + tile_row < R;
  const bool idle = FEW && row0 + wave * 32 >= R;  // none of the wave's rows is
  const int r = min(row0 + tile_row, R - 1);
  const int i = r / G;
  const int lim = first_pos + i + 1;
  const size_t out_row = (size_t)(tl.c0 + i) * p.Hq + kvh * G + (r - i * G);
  u32x4 qb[KS];
  const u32x4* qp = (const u32x4*)(p.q + out_row * D);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    qb[s] = qp[2 * s + h];
#pragma unroll
    for (int e = 0; e < 4; ++e) qb[s][e] ^= p.q_sign;
    if constexpr (D > 192) asm volatile("" : "+a"(qb[s]));  // (there is room beside the sums)
  }

#pragma unroll
  for (int j = 0; j < kQl; ++j) s_q[j * Sh::kThreads + tid] = qb[KS - kQl + j];  // (the lane's own)
  auto q_operand = [&](int ks) __attribute__((always_inline)) {
    return ks < KS - kQl ? qb[ks] : s_q[(ks - (KS - kQl)) * Sh::kThreads + tid];
  };

  f32x16 acc[DT];
  float m_run, l_run;
  m_run = neg_inf();
  l_run = 0.f;
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    acc[d] = f32x16{};
    pin_sum<kAcc>(acc[d]);
  }

  // Tiles that every row sees whole: [blk0, blkm), in the pipeline; the others up to blk1.
  const int blkm = max(blk0, min(blk1, max(lim_lo, 0) / kPromptTile));
  // The pool token index of a tile's first token, for 64 tiles at a time, one a lane (a
  // load a step would be waited for together with the tiles under way), and the tiles
  // whose page id is bad.  Tiles past the last are the last one again.
  int win = 0;
  uint32_t win_tok = 0;
  uint64_t win_bad = 0;
  bool bad_page = false;  // of a tile that every row sees: every row is NaN
  auto fetch_window = [&](int blk) __attribute__((always_inline)) {
    win = blk;
    const int x = min(blk + lane, blk1 - 1);
    const int t = x * kPromptTile;  // (< len)
    const int page = t / p.page_size;
    const int raw = p.page_table[(size_t)tl.b * p.max_pages + page];
    const int pid = clamp_page(raw, p.num_pages);
    win_tok = ((uint32_t)pid * (uint32_t)p.Hkv + (uint32_t)kvh) * (uint32_t)p.page_size +
              (uint32_t)(t - page * p.page_size);
    win_bad = __builtin_amdgcn_ballot_w64(raw != pid);
    bad_page |= __builtin_amdgcn_ballot_w64(raw != pid && x < blkm) != 0;
  };
  // asked for in the tiles' order
  auto tile_tok = [&](int blk) __attribute__((always_inline)) {
    if (blk - win >= 64) fetch_window(blk);
    return (uint32_t)__builtin_amdgcn_readlane((int)win_tok, blk - win);
  };
  const uint32_t lds_k = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_k;
  const uint32_t lds_v = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_v;
  // Straight to LDS: chunks of 1 KB, NW of them at a time, one a wave (a wave past the
  // tile's end its first one again).  A lane's 16 bytes of the row are those that belong at
  // its place; the offsets are the same for every tile.
  constexpr int kDma = Sh::kTile / 1024;
  constexpr int LQ = (kDma + NW - 1) / NW;
  uint32_t dma_k[LQ], dma_v[LQ];
#pragma unroll
  for (int u = 0; u < LQ; ++u) {
    const int q = wave + u * NW < kDma ? wave + u * NW : min(wave, kDma - 1);
    const int at = 64 * q + lane;
    const int row = at / (D / 8);
    const int c = at - row * (D / 8);
    dma_k[u] = row * Sh::kRow + 16 * (c ^ prompt_k_swap(D, row));
    dma_v[u] = row * Sh::kRow + 16 * (c ^ prompt_v_swap(D, row));
  }
  const uint32_t lds_kw = lds_k + 1024 * min(wave, kDma - 1);
  const uint32_t lds_vw = lds_v + 1024 * min(wave, kDma - 1);
  auto dma_tile = [&](const void* pages, uint32_t tok, const uint32_t (&off)[LQ], uint32_t lds,
                      auto slot) __attribute__((always_inline)) {
    constexpr int kSlot = decltype(slot)::value * Sh::kTile;
    const char* base = (const char*)pages + (size_t)tok * Sh::kRow;
    static_for_prompt<0, LQ>([&](auto i) __attribute__((always_inline)) {
      constexpr int u = decltype(i)::value;
      if constexpr ((u + 1) * NW <= kDma)
        load_to_lds<kSlot + 1024 * NW * u, FEW>(base, off[u], lds);
      else
        load_to_lds<kSlot, FEW>(base, off[u], wave + u * NW < kDma ? lds + 1024 * NW * u : lds);
    });
  };
  // Through registers: pieces tid, tid + threads, ... of a tile.
  struct Regs {
    u32x4 w[LD];
    uint32_t s[F8 ? LD : 1];
  };
  auto load_tile = [&](const void* pages, const uint8_t* scale, uint32_t tok, Regs& g)
                       __attribute__((always_inline)) {
    const char* base = (const char*)pages + (size_t)tok * (16 * CH);
#pragma unroll
    for (int u = 0; u < LD; ++u) {
      const uint32_t piece = min(tid + u * Sh::kThreads, Sh::kPieces - 1);
      g.w[u] = *(const u32x4*)(base + 16 * piece);
      if (F8) g.s[u] = *(scale + tok + piece / CH);
    }
  };
  // The same of a tile that may hold fewer tokens: rows past the last repeat it.
  auto load_last = [&](const void* pages, const uint8_t* scale, uint32_t tok, int last, Regs& g)
                       __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < LD; ++u) {
      const int piece = min(tid + u * Sh::kThreads, Sh::kPieces - 1);
      const int t = piece / CH;
      const size_t row = (size_t)tok + min(t, last);
      g.w[u] = ((const u32x4*)pages)[row * CH + (piece - t * CH)];
      if (F8) g.s[u] = scale[row];
    }
  };
  // Writes them to an LDS slot of K or V; with `bad`, notes an infinity or a NaN there.
  auto store_tile = [&](bool is_v, int slot, const Regs& g, int* bad)
                        __attribute__((always_inline)) {
    char* to = (is_v ? s_v : s_k) + slot * Sh::kTile;
#pragma unroll
    for (int u = 0; u < LD; ++u) {
      const int piece = tid + u * Sh::kThreads;
      if (Sh::kPieces % Sh::kThreads != 0 && piece >= Sh::kPieces) continue;
      const int t = piece / CH;
      const int c = piece - t * CH;
      const int sw = is_v ? prompt_v_swap(D, t) : prompt_k_swap(D, t);
      if constexpr (F8) {
        const float sc = __builtin_bit_cast(float, g.s[u] << 23);
        const u32x4 a = cvt8_fp8(g.w[u][0], g.w[u][1], sc);
        const u32x4 b = cvt8_fp8(g.w[u][2], g.w[u][3], sc);
        *(u32x4*)(to + t * Sh::kRow + 16 * ((2 * c) ^ sw)) = a;
        *(u32x4*)(to + t * Sh::kRow + 16 * ((2 * c + 1) ^ sw)) = b;
        if (bad && (any_nonfinite(a) || any_nonfinite(b))) *bad = 1;
      } else {
        *(u32x4*)(to + t * Sh::kRow + 16 * (c ^ sw)) = g.w[u];
        if (bad && any_nonfinite(g.w[u])) *bad = 1;
      }
    }
  };

  // the exponents' reference of a running maximum (none yet, or a scale of 0: 0)
  auto ref = [&](float m) __attribute__((always_inline)) {
    return m == neg_inf() ? 0.f : m * p.scale_log2;
  };
  // S^T of a K slot
  // (the order within a group of chunks is every group's, so are the addresses)
  constexpr int kGroup = prompt_pow2(D);
  uint32_t ka[kGroup / 2];
#pragma unroll
  for (int ks = 0; ks < kGroup / 2; ++ks)
    ka[ks] = lds_k + n32 * Sh::kRow + 16 * ((2 * ks + h) ^ prompt_k_swap(D, n32));
  auto keys_operand = [&](int slot, int ks) __attribute__((always_inline)) {
    return lds_read_b128(ka[ks % (kGroup / 2)] + slot * Sh::kTile +
                         16 * kGroup * (ks / (kGroup / 2)));
  };
  auto scores = [&](int slot, f32x16& s) __attribute__((always_inline)) {
    s = f32x16{};
    u32x4 a[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) a[ks] = keys_operand(slot, ks);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      s = mfma32x32x16(a[ks], q_operand(ks), s);
  };
  // a lane's largest score of a tile
  auto row_max = [&](const f32x16& s) __attribute__((always_inline)) {
    float bm = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) bm = fmaxf(bm, s[i]);
    return bm;
  };
  // moves the row's running maximum; the factor of the sums so far (1: it stays)
  auto new_max = [&](float bm) __attribute__((always_inline)) {
    float lo, hi;
    pair_xor32(bm, lo, hi);
    bm = fmaxf(lo, hi);
    // (-inf - -inf is NaN, and no reason to move)
    const bool move = (bm - m_run) * p.scale_log2 > kLazyRescaleLog2;
    const float m_new = move ? bm : m_run;
    const float f = move ? __builtin_amdgcn_exp2f((m_run - m_new) * p.scale_log2) : 1.f;
    m_run = m_new;
    return f;
  };
  // P of the masked tile blk from its scores; alpha: the factor of the sums so far
  auto softmax_masked = [&](int blk, bool bad, f32x16& s, u32x4 (&pb)[2],
                     float& alpha) __attribute__((always_inline)) {
    const int seen = lim - blk * kPromptTile;  // tokens of the tile that the row sees
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = bad ? qnan() : s[i];
      s[i] = 8 * (i >> 2) + 4 * h + (i & 3) < seen ? x : neg_inf();
    }
    alpha = new_max(row_max(s));
    const float mc = ref(m_run);
    float ps = 0.f, e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      e[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.scale_log2, -mc));
      e[i] = 8 * (i >> 2) + 4 * h + (i & 3) < seen ? e[i] : 0.f;
      ps += e[i];
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) pb[i >> 3][(i >> 1) & 3] = pack_bf16x2(e[i], e[i + 1]);
    l_run = l_run * alpha + ps;
  };
  // O^T += V^T P^T of a V slot: lane group g4 of 16 lanes reads 4 tokens x 16 columns
  // transposed
  const int g4 = lane >> 4;
  const int l16 = lane & 15;
  constexpr int kVa = kGroup / 4;
  uint32_t va[kVa];
#pragma unroll
  for (int d = 0; d < kVa; ++d) {
    const int row = 4 * (g4 >> 1) + (l16 >> 2);  // (its swap is that of rows 8 k away)
    va[d] = lds_v + row * Sh::kRow + 8 * (l16 & 1) +
            16 * ((4 * d + 2 * (g4 & 1) + ((l16 & 3) >> 1)) ^ prompt_v_swap(D, row));
  }
  auto values_operand = [&](int slot, int ks, int d) __attribute__((always_inline)) {
    const uint32_t at =
        va[d % kVa] + slot * Sh::kTile + 16 * ks * Sh::kRow + 16 * kGroup * (d / kVa);
    const uint2 x = lds_read_tr_b64(at);
    const uint2 y = lds_read_tr_b64(at + 8 * Sh::kRow);
    return u32x4{x.x, x.y, y.x, y.y};
  };
  auto values = [&](int slot, const u32x4 (&pb)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const u32x4 a = values_operand(slot, ks, d);
        acc[d] = mfma32x32x16(a, pb[ks], acc[d]);
        if (kAcc) pin_sum<kAcc>(acc[d]);
      }
  };
  // The same where the slot holds an infinity or a NaN that some rows do not see: the
  // finite values' product, and from two products of 0 and 1 whether a row sees an
  // infinity of either sign (a NaN counts as both) in a column.
  auto values_masked = [&](int slot, int blk, const u32x4 (&pb)[2])
                           __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      f32x16 pos{}, neg{};
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        u32x4 fin = values_operand(slot, ks, d), ap, an, vis;
        // vis: 1 for the k slots (tokens 0 .. 3 and 8 .. 11 past 16 ks + 4 h) that are seen
        const int seen = lim - blk * kPromptTile - 16 * ks - 4 * h;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t f = fin[e], u, w;
          split_nonfinite(f, u, w);
          fin[e] = f;
          ap[e] = u;
          an[e] = w;
          const int t = 8 * (e >> 1) + 2 * (e & 1);
          vis[e] = (t < seen ? 0x3f80u : 0u) | (t + 1 < seen ? 0x3f800000u : 0u);
        }
        acc[d] = mfma32x32x16(fin, pb[ks], acc[d]);
        pos = mfma32x32x16(ap, vis, pos);
        neg = mfma32x32x16(an, vis, neg);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (pos[i] > 0.f) acc[d][i] -= neg_inf();
        if (neg[i] > 0.f) acc[d][i] += neg_inf();
      }
      if (kAcc) pin_sum<kAcc>(acc[d]);
    }
  };
  // acc times alpha, where some row's maximum moved
  auto rescale = [&](const float& alpha) __attribute__((always_inline)) {
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(alpha != 1.f) == 0, 1)) return;
    float f = alpha;
    asm("" : "+v"(f));  // (else the products are taken every step, ahead of the test)
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      acc[d] = acc[d] * f;
      pin_sum<kAcc>(acc[d]);
    }
  };

  if (blk0 < blkm) {
    const int T = blkm - blk0;
    f32x16 s[2];
    u32x4 pb[2][2];
    Regs kg[2], vg[2];  // (8-bit)
    fetch_window(blk0);
    uint32_t tok[5];  // of tiles t .. t + 4
#pragma unroll
    for (int i = 0; i < 5; ++i) tok[i] = tile_tok(blk0 + i);
    // tile t of K (V) into slot t & 3, in the order of the steps that read them
    if constexpr (F8) {
      load_tile(p.k_pages, p.k_scale, tok[0], kg[0]);
      load_tile(p.k_pages, p.k_scale, tok[1], kg[1]);
      store_tile(false, 0, kg[0], nullptr);
      store_tile(false, 1, kg[1], nullptr);
      load_tile(p.k_pages, p.k_scale, tok[2], kg[0]);
      load_tile(p.v_pages, p.v_scale, tok[0], vg[0]);
      load_tile(p.k_pages, p.k_scale, tok[3], kg[1]);
      load_tile(p.v_pages, p.v_scale, tok[1], vg[1]);
    } else {
      using std::integral_constant;
      dma_tile(p.k_pages, tok[0], dma_k, lds_kw, integral_constant<int, 0>{});
      dma_tile(p.k_pages, tok[1], dma_k, lds_kw, integral_constant<int, 1>{});
      dma_tile(p.k_pages, tok[2], dma_k, lds_kw, integral_constant<int, 2>{});
      dma_tile(p.v_pages, tok[0], dma_v, lds_vw, integral_constant<int, 0>{});
      dma_tile(p.k_pages, tok[3], dma_k, lds_kw, integral_constant<int, 3>{});
      dma_tile(p.v_pages, tok[1], dma_v, lds_vw, integral_constant<int, 1>{});
    }
    // the values of "tile -1", which step 0 adds with weights of 0
    for (int i = tid; i < Sh::kTile / 16; i += Sh::kThreads)
      ((u32x4*)(s_v + 3 * Sh::kTile))[i] = u32x4{0, 0, 0, 0};
    pb[1][0] = pb[1][1] = u32x4{0, 0, 0, 0};
    if (!F8) wait_loads<4 * LQ>();
    __syncthreads();
    if (!idle) scores(0, s[0]);
    float alpha = 1.f;  // of the tile whose softmax is next
    float m_kept = m_run;  // the maximum without that tile's
    if (!idle) alpha = new_max(row_max(s[0]));
    __syncthreads();
    auto step = [&](auto slot, int t) __attribute__((always_inline)) {
      constexpr int c = decltype(slot)::value;  // t & 3
      constexpr int u = c & 1;
      if constexpr (F8) {  // K of tile t + 2 and V of t; K of t + 4 and V of t + 2 requested
        store_tile(false, c ^ 2, kg[u], nullptr);
        store_tile(true, c, vg[u], nullptr);
        load_tile(p.k_pages, p.k_scale, tok[4], kg[u]);
        load_tile(p.v_pages, p.v_scale, tok[2], vg[u]);
      } else {
        dma_tile(p.k_pages, tok[4], dma_k, lds_kw, slot);
        dma_tile(p.v_pages, tok[2], dma_v, lds_vw, std::integral_constant<int, (c ^ 2)>{});
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) tok[i] = tok[i + 1];
      tok[4] = tile_tok(blk0 + t + 5);
      if (!idle) {
        // The scores of tile t + 1 under the exponentials of tile t, then the values of
        // tile t - 1 under its sums and the next tile's maximum: one product and its share
        // of the vector work at a time (sched_barrier keeps the order; the compiler's own
        // runs the exponentials after the products).
        constexpr int kExp = 16 / KS > 0 ? (16 + KS - 1) / KS : 1;
        constexpr int kAhead = DT > 1 ? 3 : 2;  // V operands under way
        constexpr int kKeys = 8;                // and K operands
        u32x4 a[KS], av[2 * DT], ql[kQl > 0 ? kQl : 1];
#pragma unroll
        for (int ks = 0; ks < KS && ks < kKeys; ++ks) a[ks] = keys_operand((c + 1) & 3, ks);
        float mc, ps, bm;
        mc = ref(m_run);
        ps = 0.f;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          s[u ^ 1] = mfma32x32x16(a[ks], ks < KS - kQl ? qb[ks] : ql[ks - (KS - kQl)],
                                  ks == 0 ? f32x16{} : s[u ^ 1]);
          pin_sum<kAcc>(s[u ^ 1]);
#pragma unroll
          for (int j = 0; j < kQl; ++j)
            if (ks == KS - kQl + j - 3) ql[j] = q_operand(KS - kQl + j);
          if (ks + kKeys < KS) a[ks + kKeys] = keys_operand((c + 1) & 3, ks + kKeys);
#pragma unroll
          for (int e = ks * kExp; e < (ks + 1) * kExp && e < 16; ++e) {
            float x = s[u][e];
            pin(x);
            x = __builtin_amdgcn_exp2f(fmaf(x, p.scale_log2, -mc));
            pin(x);
            s[u][e] = x;
          }
#pragma unroll
          for (int j = 0; j < kAhead; ++j)
            if (ks == (KS > kAhead ? KS - kAhead + j : 0))
              av[j] = values_operand((c + 3) & 3, j / DT, j % DT);
          __builtin_amdgcn_sched_barrier(0);
        }
        constexpr int kSum = 8 / (2 * DT) > 0 ? (8 + 2 * DT - 1) / (2 * DT) : 1;
        float next_alpha;
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) {
          const int f = j + kAhead;
          if (f < 2 * DT) av[f] = values_operand((c + 3) & 3, f / DT, f % DT);
          acc[j % DT] = mfma32x32x16(av[j], pb[u ^ 1][j / DT], acc[j % DT]);
          pin_sum<kAcc>(acc[j % DT]);
#pragma unroll
          for (int e = j * kSum; e < (j + 1) * kSum && e < 8; ++e) {
            const int i = 2 * e;
            const float x = s[u][i], y = s[u][i + 1];
            pin(ps);
            ps += x + y;
            pin(ps);
            uint32_t w = pack_bf16x2(x, y);
            pin(w);
            pb[u][i >> 3][(i >> 1) & 3] = w;
          }
          if (j == DT) {
            bm = row_max(s[u ^ 1]);
          }
          if (j == 2 * DT - 1) {
            l_run = l_run * alpha + ps;
            m_kept = m_run;
            next_alpha = new_max(bm);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        rescale(alpha);
        alpha = next_alpha;
      }
      if (!F8) wait_loads<4 * LQ>();  // those of this step and the one before may go on
      __syncthreads();
    };
    int t = 0;
#pragma unroll 1
    for (; t + 4 <= T; t += 4) {
      step(std::integral_constant<int, 0>{}, t);
      step(std::integral_constant<int, 1>{}, t + 1);
      step(std::integral_constant<int, 2>{}, t + 2);
      step(std::integral_constant<int, 3>{}, t + 3);
    }
    if (t < T) step(std::integral_constant<int, 0>{}, t);
    if (t + 1 < T) step(std::integral_constant<int, 1>{}, t + 1);
    if (t + 2 < T) step(std::integral_constant<int, 2>{}, t + 2);
    const int last = (T - 1) & 3;
    if (!idle) {
      if (last & 1)
        values(last, pb[1]);
      else
        values(last, pb[0]);
    }
    m_run = m_kept;  // (tile T may hold tokens not seen)
    if (!F8) wait_loads<0>();  // the tiles past the last, which nothing reads
  }
  // The others, masked, one after the other.
  if (blkm < blk1) {
    if (tid < 2) s_bad[tid] = 0;
    Regs kg, vg;
    fetch_window(blkm);
    uint32_t tok = tile_tok(blkm);
    bool next_bad = win_bad & 1;
    auto last_of = [&](int blk) { return min(kPromptTile, len - blk * kPromptTile) - 1; };
    load_last(p.k_pages, p.k_scale, tok, last_of(blkm), kg);
    load_last(p.v_pages, p.v_scale, tok, last_of(blkm), vg);
    __syncthreads();
    int c = 0;
#pragma unroll 1
    for (int blk = blkm; blk < blk1; ++blk) {
      const bool bad = next_bad;
      store_tile(false, c, kg, nullptr);
      // (s_bad stays set: the slow sum is right for any tile)
      store_tile(true, c, vg, &s_bad[c]);
      const int next = min(blk + 1, blk1 - 1);
      tok = tile_tok(next);
      next_bad = (win_bad >> (next - win)) & 1;
      load_last(p.k_pages, p.k_scale, tok, last_of(next), kg);
      load_last(p.v_pages, p.v_scale, tok, last_of(next), vg);
      __syncthreads();
      if (!idle) {
        f32x16 s;
        u32x4 pb[2];
        float alpha;
        scores(c, s);
        softmax_masked(blk, bad, s, pb, alpha);
        rescale(alpha);
        if (uniform(s_bad[c]))
          values_masked(c, blk, pb);
        else
          values(c, pb);
      }
      c ^= 1;
    }
  }

  // Outputs: lane half h of a row holds columns 32 d + 8 a + 4 h + b.
  float l_lo, l_hi;
  pair_xor32(l_run, l_lo, l_hi);
  const float l = l_lo + l_hi;
  if (!live) return;
  const bool none = l == 0.f;
  const bool gone = !len_good || bad_page;
  const float inv = gone ? qnan() : none ? 0.f : 1.f / l;
  const float lse_v = gone ? qnan() : none ? neg_inf() : (ref(m_run) + __log2f(l)) * kLn2;
  const size_t at = piece ? (size_t)piece_at * kRows + tile_row : out_row;
  if (h == 0) {
    if (piece) p.part_lse[at] = lse_v;
    else if (p.lse) p.lse[at] = lse_v;
  }
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int col = 32 * d + 8 * a + 4 * h;
      const float4 o = make_float4(acc[d][4 * a] * inv, acc[d][4 * a + 1] * inv,
                                   acc[d][4 * a + 2] * inv, acc[d][4 * a + 3] * inv);
      if (piece) {
        *(float4*)(p.part_out + at * D + col) = o;
      } else {
        if (p.out_f32) *(float4*)(p.out_f32 + at * D + col) = o;
        if (p.out_bf16)
          *(uint2*)(p.out_bf16 + at * D + col) =
              make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
      }
    }
}

// Combines the pieces of the tiles that were split: a workgroup for kJoinRows rows of a
// tile and KV head, one thread per four columns.
constexpr int kJoinRows = 8;
__global__ __launch_bounds__(256) void prompt_join_kernel(const PromptParams p, int D, int rows) {
  const int id = blockIdx.x;
  const int kvh = id % p.Hkv;
  const PromptPlace tl = prompt_place<true>(p, id / p.Hkv, rows);
  const long long piece_at = (long long)tl.piece * p.Hkv + kvh;
  if (tl.b < 0 || tl.splits == 1 || piece_at < 0 ||
      piece_at + (long long)(tl.splits - 1) * p.Hkv >= p.pieces)
    return;
  const int R = tl.n * p.G;
  const int c4 = D >> 2;
  for (int t = threadIdx.x; t < kJoinRows * c4; t += 256) {
    const int tr = blockIdx.y * kJoinRows + t / c4;  // row of the tile
    const int c = t % c4;
    const int r = tl.tile * rows + tr;
    if (r >= R) return;  // (so has every later row)
    const int i = r / p.G;
    const size_t out_row = (size_t)(tl.c0 + i) * p.Hq + kvh * p.G + (r - i * p.G);
    const size_t slot = (size_t)piece_at * rows + tr;
    const size_t step = (size_t)p.Hkv * rows;  // to the row's next piece
    const PieceAcc x =
        piece_stream<float4>((const char*)(p.part_out + slot * D + 4 * c), step * D * 4,
                             p.part_lse + slot, (int)step, 0, 1, tl.splits);
    const float inv = x.sum == 0.f ? 0.f : 1.f / x.sum;
    const float4 o = make_float4(x.a.x * inv, x.a.y * inv, x.a.z * inv, x.a.w * inv);
    if (p.out_f32) ((float4*)p.out_f32)[out_row * c4 + c] = o;
    if (p.out_bf16)
      ((uint2*)p.out_bf16)[out_row * c4 + c] =
          make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
    if (p.lse && c == 0) p.lse[out_row] = x.sum == 0.f ? neg_inf() : x.m + __logf(x.sum);
  }
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
static bool prompt_width_ok(int D) { return D >= 32 && D <= kPromptMaxD && D % 32 == 0; }

// How a call runs.
//
// Calls of few rows: a sequence's rows of a KV head fill half a tile on average, at the
// most, and K and V are read about once, so the reads are the bound.  bf16 up to 128
// columns, rows that one wave holds: a wave by itself needs no barrier, and several on a CU
// keep as much under way (8 x 5 tokens of 8 x 4 heads over 4000 to 32000: 97 us against 111
// with four waves that share the loads; 16 x 8 over 2000: 34 against 42).  Twice the rows
// would read K and V twice (12 tokens over 16000: 130 us with one wave, 110 with four; 16
// over 8000 81 and 68, the other way in a small batch, 4 x 8 of 4 x 8 heads, 29 and 31).
// 8-bit pages take four waves' conversions (8 x 16 over 8000: 107 us with one wave, 57 with
// four), and wider heads four waves' registers (256 columns, 8 x 5 over 16000, at the time
// 262 and 211).
struct PromptPlan {
  bool few;
  int waves;         // of a workgroup
  int rows;          // of a tile: 32 a wave
  long long tiles;   // of all sequences and KV heads, at the most
  int share;         // workgroups the tokens are shared by, where they are split by the lengths
  long long pieces;  // at the most; 0: no tile is split
  long long grid;
};
static PromptPlan prompt_plan(int N, int B, int Hq, int Hkv, int D, bool fp8, int max_len,
                              int n_splits) {
  const int G = Hq / Hkv;
  PromptPlan r;
  r.few = (long long)N * G <= 64LL * B;
  r.waves = (long long)N * G <= 32LL * B && !fp8 && D <= 128 ? 1 : kPromptWaves;
  r.rows = 32 * r.waves;
  const long long full = ((long long)N * G + r.rows - 1) / r.rows;
  r.tiles = (full + B) * Hkv;
  r.share = 0;
  r.pieces = 0;
  r.grid = r.tiles;
  if (n_splits > 1) {
    r.pieces = r.grid = r.tiles * n_splits;
  } else if (n_splits == 0) {
    // Where the tiles are fewer than the workgroups that fit the chip: shares that make,
    // with every tile's last one, as many pieces as fit it once.  (8 x 5 tokens of 4 x 8
    // heads over 4000 to 32000, us with the join: once 97, twice 108, three times 118.)
    const int lds = 160 * 1024 / (kPromptSlots * 2 * kPromptTile * 2 * D + 256);
    const int per_cu = r.waves == 1 ? std::min(lds, 8) : D <= 128 ? 2 : 1;
    const long long fill = choose_workgroups(0, per_cu, 1LL << 30, 1);
    if (full * Hkv < fill && max_len > kPromptMinShare * kPromptTile) {
      r.share = (int)std::max(fill - r.tiles, fill / 2);
      // every split but a tile's last is a whole share (and the shares' total, a sum in
      // fp32, is off by less than 64 of them); only tiles longer than a share are split,
      // and only split ones leave pieces
      r.grid = r.tiles + r.share + 64;
      r.pieces = std::min<long long>(r.tiles, r.share) + r.share + 64;
    }
  }
  return r;
}
static size_t prompt_bytes(const PromptPlan& pl, int D) {
  if (pl.pieces == 0) return 0;
  const size_t rows = (size_t)pl.pieces * pl.rows;
  return align256(rows * 4) + rows * D * 4;
}

template <int D, bool F8>
static void prompt_launch(const PromptParams& p, const PromptPlan& pl, hipStream_t s) {
  const dim3 grid((unsigned)pl.grid), block(64 * pl.waves);
  if constexpr (!F8 && D <= 128) {
    if (pl.waves == 1) {
      hipLaunchKernelGGL((prompt_kernel<D, F8, 1, true>), grid, block, 0, s, p);
      return;
    }
  }
  if (pl.few)
    hipLaunchKernelGGL((prompt_kernel<D, F8, kPromptWaves, true>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((prompt_kernel<D, F8, kPromptWaves, false>), grid, block, 0, s, p);
}
template <bool F8>
static void prompt_launch_width(const PromptParams& p, const PromptPlan& pl, int D,
                                hipStream_t s) {
  switch (D) {
    case 32: prompt_launch<32, F8>(p, pl, s); break;
    case 64: prompt_launch<64, F8>(p, pl, s); break;
    case 96: prompt_launch<96, F8>(p, pl, s); break;
    case 128: prompt_launch<128, F8>(p, pl, s); break;
    case 160: prompt_launch<160, F8>(p, pl, s); break;
    case 192: prompt_launch<192, F8>(p, pl, s); break;
    case 224: prompt_launch<224, F8>(p, pl, s); break;
    default: prompt_launch<256, F8>(p, pl, s); break;
  }
}

static int prompt_sizes(const char* name, int N, int B, int Hq, int Hkv, int D, bool fp8,
                        int max_len, int n_splits) {
  if (N < 0 || B < 0 || B > kMaxSeqs || Hkv <= 0 || Hq <= 0 || Hq % Hkv || max_len < 0 ||
      n_splits < 0 || n_splits > kPromptMaxSplits)
    return set_error(WS_EINVAL,
                     "%s: bad sizes N=%d B=%d Hq=%d Hkv=%d max_len=%d n_splits=%d (B <= %d, "
                     "n_splits <= %d)",
                     name, N, B, Hq, Hkv, max_len, n_splits, kMaxSeqs, kPromptMaxSplits);
  if (!prompt_width_ok(D))
    return set_error(WS_EINVAL, "%s: head_dim %d unsupported (multiples of 32 up to 256)", name, D);
  if ((long long)N * (Hq / Hkv) + 256LL * B >= (1LL << 31) || max_len > (1 << 30))
    return set_error(WS_EINVAL, "%s: %d tokens of %d heads exceed the row index range", name, N, Hq);
  const PromptPlan pl = prompt_plan(N, B, Hq, Hkv, D, fp8, max_len, n_splits);
  if (pl.grid * 64 * pl.waves >= (1LL << 32))
    return set_error(WS_EINVAL, "%s: %d tokens of %d heads exceed the launch grid", name, N, Hq);
  return WS_OK;
}

}  // namespace ws

using namespace ws;

extern "C" int ws_gqa_prompt_plan(int N, int B, int Hq, int Hkv, int D, int fp8, int max_len,
                                  int n_splits, int* pieces_out, size_t* workspace_bytes_out) {
  if (int rc = prompt_sizes("ws_gqa_prompt_plan", N, B, Hq, Hkv, D, fp8 != 0, max_len, n_splits)) return rc;
  const PromptPlan pl = prompt_plan(N, B, Hq, Hkv, D, fp8 != 0, max_len, n_splits);
  if (pieces_out) *pieces_out = (int)pl.pieces;
  if (workspace_bytes_out) *workspace_bytes_out = prompt_bytes(pl, D);
  return WS_OK;
}

extern "C" int ws_gqa_prompt(const uint16_t* q, const void* k_pages, const void* v_pages,
                             const uint8_t* k_scale, const uint8_t* v_scale,
                             const int32_t* page_table, const int32_t* kv_len,
                             const int32_t* cu_new, int N, int B, int Hq, int Hkv, int D,
                             int page_size, int max_pages, int num_pages, int max_len,
                             int n_splits, float scale, uint16_t* out_bf16, float* out_f32,
                             float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  static const char* name = "ws_gqa_prompt";
  if (!q || !k_pages || !v_pages || !page_table || !kv_len || !cu_new || (!out_bf16 && !out_f32) ||
      (k_scale == nullptr) != (v_scale == nullptr))
    return set_error(WS_EINVAL, "%s: null pointer", name);
  if (int rc = prompt_sizes(name, N, B, Hq, Hkv, D, k_scale != nullptr, max_len, n_splits)) return rc;
  if (page_size <= 0 || page_size % 32 || max_pages <= 0 || num_pages <= 0 ||
      (long long)max_len > (long long)page_size * max_pages)
    return set_error(WS_EINVAL,
                     "%s: bad paging page_size=%d max_pages=%d num_pages=%d max_len=%d "
                     "(page_size must be a multiple of 32)",
                     name, page_size, max_pages, num_pages, max_len);
  if ((long long)num_pages * Hkv * page_size > 0xffffffffLL)
    return set_error(WS_EINVAL, "%s: pools of %lld tokens exceed the 32-bit token index", name,
                     (long long)num_pages * Hkv * page_size);
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out_bf16) ||
      !aligned16(out_f32))
    return set_error(WS_EINVAL, "%s: buffers must be 16-byte aligned", name);
  if (!(scale - scale == 0.f)) return set_error(WS_EINVAL, "%s: scale must be finite", name);
  if (N == 0 || B == 0) return WS_OK;
  const PromptPlan pl = prompt_plan(N, B, Hq, Hkv, D, k_scale != nullptr, max_len, n_splits);
  const size_t need = prompt_bytes(pl, D);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(WS_EWORKSPACE, "%s: workspace %zu < %zu bytes", name, workspace_bytes, need);
  if (need > 0 && ((uintptr_t)workspace & 255u) != 0)
    return set_error(WS_EINVAL, "%s: workspace must be 256-byte aligned", name);
  PromptParams p;
  p.q = q;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.page_table = page_table;
  p.kv_len = kv_len;
  p.cu_new = cu_new;
  p.out_bf16 = out_bf16;
  p.out_f32 = out_f32;
  p.lse = lse;
  p.part_lse = (float*)workspace;
  p.part_out = (float*)((char*)workspace + align256((size_t)pl.pieces * pl.rows * 4));
  p.N = N;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.page_size = page_size;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.cap = (int)std::min<long long>((long long)page_size * max_pages, 1LL << 30);
  p.n_splits = n_splits;
  p.share = pl.share;
  p.pieces = pl.pieces;
  p.scale_log2 = (scale < 0.f ? -scale : scale) * kLog2e;
  p.q_sign = scale < 0.f ? 0x80008000u : 0u;
  hipStream_t s = (hipStream_t)stream;
  if (k_scale)
    prompt_launch_width<true>(p, pl, D, s);
  else
    prompt_launch_width<false>(p, pl, D, s);
  int rc = check_launch(name);
  if (rc != WS_OK || pl.pieces == 0) return rc;
  hipLaunchKernelGGL(prompt_join_kernel, dim3((unsigned)pl.tiles, pl.rows / kJoinRows), dim3(256), 0,
                     s, p, D, pl.rows);
  return check_launch(name);
}
