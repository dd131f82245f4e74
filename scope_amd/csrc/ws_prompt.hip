// Prompt attention over the pages (gfx950): the new tokens of every sequence,
// ragged and causal, over everything of the sequence that the partition holds,
// bf16 pages or 8-bit ones (e4m3 with an e8m0 scale per token and KV head).
//
// Query i of a sequence's n (tokens cu[b] .. cu[b + 1] of q) stands at position
// len - n + i of the len tokens in the pages and sees positions 0 .. its own.
// The query rows of a KV head are (token, head of the group) pairs, row = i G + g,
// so the G heads that share K and V share their loads: a workgroup takes a tile of
// 32 RB NW consecutive rows, a wave 32 RB of them, and walks the tokens in blocks
// of 64 through LDS with a running maximum and sum (one pass over K and V).
//
//   S^T[token, row] = K Q^T   A = K from LDS (16 bytes a lane), B = Q in registers
//   O^T[col, row] += V^T P^T  A = V^T read transposed from LDS, B = P as it comes out
//                             of S^T: the 32x32 product's output rows 8 a + 4 h + b of
//                             lane half h are taken as k slots in that order, in P and
//                             V alike
// A row is one lane column: its maximum takes one exchange between the lane halves,
// its rescaling no exchange at all.
//
// A row sees nothing of the tokens past its position: their scores are masked, and
// so are their values, which P = 0 alone would not do for an infinity or a NaN
// (0 * inf): where a block that some row masks holds one, its products are added
// token by token (pv_masked).
//
// With few rows the tokens are split over n_splits workgroups per tile, whose pieces
// (fp32, with their lse) prompt_join_kernel combines.
#include <algorithm>

#include "ws_attn.h"
#include "ws_plan.h"
#include "ws_reduce.h"

namespace ws {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kPromptMaxD = 256;
constexpr int kPromptBlock = 64;   // tokens of a block
constexpr int kPromptPad = 32;     // bytes of padding of an LDS row: an odd multiple of 32
                                   // bytes from row to row, so that 8 rows' 16-byte loads
                                   // and 4 rows' transposed 32-byte reads meet no bank twice
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
  float* part_out;  // [n_splits][N * Hq][D], with part_lse when n_splits > 1
  float* part_lse;
  int N, B, Hq, Hkv, G, page_size, max_pages, num_pages, cap, n_splits, tiles;
  float scale_log2;  // >= 0
  uint32_t q_sign;   // 0x80008000 where the caller's scale is negative
};

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

struct PromptTile {
  int b, tile;  // sequence and tile of its rows (b < 0: none)
  int c0, n;    // the sequence's first row of q and its tokens
};

// Tile `t` of the list of all sequences' tiles of `rows` rows.  Every lane must
// call it; the result is uniform.
__device__ __forceinline__ int prompt_tokens(const PromptParams& p, int b, int& c0) {
  c0 = min(max(p.cu_new[b], 0), p.N);
  return min(max(p.cu_new[b + 1], c0), p.N) - c0;
}
__device__ __forceinline__ PromptTile prompt_tile(const PromptParams& p, int t, int rows) {
  const int lane = threadIdx.x & 63;
  const int per = (p.B + 63) >> 6;
  const int b0 = lane * per;
  int sum = 0, c0;
  for (int k = 0; k < per; ++k)
    if (b0 + k < p.B) sum += (prompt_tokens(p, b0 + k, c0) * p.G + rows - 1) / rows;
  const int incl = __ockl_wfscan_add_i32(sum, true);
  const uint64_t past = __builtin_amdgcn_ballot_w64(incl > t);
  PromptTile r{-1, 0, 0, 0};
  if (past == 0) return r;
  const int at = __builtin_ctzll(past);
  int left = t - __builtin_amdgcn_readlane(incl - sum, at);
  for (int k = 0; k < per; ++k) {
    const int b = uniform(at * per + k);
    if (b >= p.B) break;
    const int n = uniform(prompt_tokens(p, b, c0));
    const int tiles = (n * p.G + rows - 1) / rows;
    if (left < tiles) {
      // the last tile first: it walks the most tokens
      r = PromptTile{b, tiles - 1 - left, uniform(c0), n};
      break;
    }
    left -= tiles;
  }
  return r;
}

template <int D, bool F8, int RB, int NW>
struct PromptShape {
  static constexpr int kRows = 32 * RB * NW;
  static constexpr int kStride = 2 * D + kPromptPad;  // bytes of an LDS row
  static constexpr int kTile = kPromptBlock * kStride;
  static constexpr int kBufs = NW > 1 ? 2 : 1;
  static constexpr int kLds = kBufs * 2 * kTile;
  // 16-byte pieces (bf16 columns: 8; 8-bit: 16) of a block's K or V, and of a thread's
  static constexpr int kPieces = kPromptBlock * D / (F8 ? 16 : 8);
  static constexpr int kThreads = 64 * NW;
  static constexpr int kLoads = (kPieces + kThreads - 1) / kThreads;
};

template <int D, bool F8, int RB, int NW>
__global__ __launch_bounds__(64 * NW, 1) void prompt_kernel(const PromptParams p) {
  static_assert(D % 32 == 0 && D <= kPromptMaxD, "head width: a multiple of 32 up to 256");
  using Sh = PromptShape<D, F8, RB, NW>;
  constexpr int KS = D / 16;           // k-steps of the scores
  constexpr int DT = D / 32;           // 32-column tiles of the output
  constexpr int CH = F8 ? D / 16 : D / 8;  // 16-byte pieces of a token's row
  constexpr int LD = Sh::kLoads;
  __shared__ __attribute__((aligned(256))) char s_kv[Sh::kLds];
  __shared__ int s_bad[2];  // a block's values hold an infinity or a NaN (masked blocks only)

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int n32 = lane & 31;
  const int h = lane >> 5;
  const int id = blockIdx.x;
  const int kvh = id % p.Hkv;
  const int rest = id / p.Hkv;
  const int split = rest % p.n_splits;
  const PromptTile tl = prompt_tile(p, rest / p.n_splits, Sh::kRows);
  if (tl.b < 0) return;
  const int G = p.G;
  const int R = tl.n * G;  // rows of the sequence and KV head
  const int len = uniform(p.kv_len[tl.b]);
  const bool len_good = len_ok(len, 0, p.cap);
  const int first_pos = len - tl.n;  // position of the sequence's first query
  const int row0 = tl.tile * Sh::kRows;
  const int rows_here = min(Sh::kRows, R - row0);
  // visible tokens of the tile's first and last row
  const int lim_lo = first_pos + row0 / G + 1;
  const int lim_hi = len_good ? max(first_pos + (row0 + rows_here - 1) / G + 1, 0) : 0;
  const int nb = (lim_hi + kPromptBlock - 1) / kPromptBlock;
  const int blk0 = (int)((long long)split * nb / p.n_splits);
  const int blk1 = (int)((long long)(split + 1) * nb / p.n_splits);

  // the wave's rows
  int lim[RB];        // visible tokens of the lane's row
  size_t out_row[RB]; // its row of out / lse
  bool live[RB];
  u32x4 qb[RB][KS];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = row0 + (wave * RB + rb) * 32 + n32;
    live[rb] = r < R;
    const int rr = min(r, R - 1);
    const int i = rr / G;
    lim[rb] = first_pos + i + 1;
    out_row[rb] = (size_t)(tl.c0 + i) * p.Hq + kvh * G + (rr - i * G);
    const u32x4* qp = (const u32x4*)(p.q + out_row[rb] * D);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qb[rb][s] = qp[2 * s + h];
#pragma unroll
      for (int e = 0; e < 4; ++e) qb[rb][s][e] ^= p.q_sign;
    }
  }

  f32x16 acc[RB][DT];
  float m_run[RB], l_run[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    m_run[rb] = neg_inf();
    l_run[rb] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[rb][d] = f32x16{};
  }

  // A block's two 32-token halves: pool token index of the half's first token, its last
  // row that holds a token (later rows repeat it), and whether the page id was bad.
  struct Half {
    uint32_t tok;
    int last;
    bool bad;
  };
  auto half_of = [&](int blk, int hf) __attribute__((always_inline)) {
    const int t = min(blk * kPromptBlock + 32 * hf, len - 1) & ~31;
    const int page = t / p.page_size;
    const int raw = p.page_table[(size_t)tl.b * p.max_pages + page];
    const int pid = clamp_page(raw, p.num_pages);
    Half x;
    x.tok = ((uint32_t)pid * (uint32_t)p.Hkv + (uint32_t)kvh) * (uint32_t)p.page_size +
            (uint32_t)(t - page * p.page_size);
    x.last = min(31, len - 1 - t);
    x.bad = raw != pid;
    return x;
  };
  // Registers of the block under way: pieces tid, tid + threads, ... of K and V.
  u32x4 kr[LD], vr[LD];
  uint32_t ksr[F8 ? LD : 1], vsr[F8 ? LD : 1];
  auto load_block = [&](const Half (&hv)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < LD; ++u) {
      const int piece = tid + u * Sh::kThreads;
      if (Sh::kPieces % Sh::kThreads != 0 && piece >= Sh::kPieces) continue;
      const int t = piece / CH;
      const int c = piece - t * CH;
      const Half& x = t < 32 ? hv[0] : hv[1];
      const size_t row = (size_t)x.tok + min(t & 31, x.last);
      kr[u] = ((const u32x4*)p.k_pages)[row * CH + c];
      vr[u] = ((const u32x4*)p.v_pages)[row * CH + c];
      if (F8) {
        ksr[u] = p.k_scale[row];
        vsr[u] = p.v_scale[row];
      }
    }
  };
  // Writes them to LDS buffer `buf`; with `check`, notes an infinity or a NaN in V.
  auto store_block = [&](int buf, bool check) __attribute__((always_inline)) {
    char* kb = s_kv + buf * 2 * Sh::kTile;
    char* vb = kb + Sh::kTile;
#pragma unroll
    for (int u = 0; u < LD; ++u) {
      const int piece = tid + u * Sh::kThreads;
      if (Sh::kPieces % Sh::kThreads != 0 && piece >= Sh::kPieces) continue;
      const int t = piece / CH;
      const int c = piece - t * CH;
      if (F8) {
        const int at = t * Sh::kStride + 32 * c;
        const float ks = __builtin_bit_cast(float, ksr[u] << 23);
        const float vs = __builtin_bit_cast(float, vsr[u] << 23);
        *(u32x4*)(kb + at) = cvt8_fp8(kr[u][0], kr[u][1], ks);
        *(u32x4*)(kb + at + 16) = cvt8_fp8(kr[u][2], kr[u][3], ks);
        const u32x4 v0 = cvt8_fp8(vr[u][0], vr[u][1], vs);
        const u32x4 v1 = cvt8_fp8(vr[u][2], vr[u][3], vs);
        *(u32x4*)(vb + at) = v0;
        *(u32x4*)(vb + at + 16) = v1;
        if (check && (any_nonfinite(v0) || any_nonfinite(v1))) s_bad[buf] = 1;
      } else {
        const int at = t * Sh::kStride + 16 * c;
        *(u32x4*)(kb + at) = kr[u];
        *(u32x4*)(vb + at) = vr[u];
        if (check && any_nonfinite(vr[u])) s_bad[buf] = 1;
      }
    }
  };

  // the exponents' reference of a running maximum (none yet, or a scale of 0: 0)
  auto ref = [&](float m) __attribute__((always_inline)) {
    return m == neg_inf() ? 0.f : m * p.scale_log2;
  };
  auto compute = [&](int blk, int buf, bool masked, bool bad0, bool bad1)
                     __attribute__((always_inline)) {
    const char* kb = s_kv + buf * 2 * Sh::kTile;
    const uint32_t vb = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)(
        s_kv + buf * 2 * Sh::kTile + Sh::kTile);
    f32x16 s[RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) s[rb][0] = s[rb][1] = f32x16{};
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 a = *(const u32x4*)(kb + (32 * tt + n32) * Sh::kStride + 32 * ks + 16 * h);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) s[rb][tt] = mfma32x32x16(a, qb[rb][ks], s[rb][tt]);
      }
    const int t0 = blk * kPromptBlock;
    u32x4 pb[RB][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int seen = lim[rb] - t0;  // tokens of the block that the row sees
      if (masked) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int t = 32 * tt + 8 * (i >> 2) + 4 * h + (i & 3);
            float x = s[rb][tt][i];
            if (tt ? bad1 : bad0) x = qnan();
            s[rb][tt][i] = t < seen ? x : neg_inf();
          }
      }
      float bm = s[rb][0][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) bm = fmaxf(bm, s[rb][0][i]);
#pragma unroll
      for (int i = 0; i < 16; ++i) bm = fmaxf(bm, s[rb][1][i]);
      float lo, hi;
      pair_xor32(bm, lo, hi);
      bm = fmaxf(lo, hi);
      // (-inf - -inf is NaN, and no reason to move)
      const bool move = (bm - m_run[rb]) * p.scale_log2 > kLazyRescaleLog2;
      if (__builtin_amdgcn_ballot_w64(move) != 0) {
        const float m_new = fmaxf(m_run[rb], bm);
        const float alpha =
            m_new == neg_inf() ? 1.f
                               : __builtin_amdgcn_exp2f((m_run[rb] - m_new) * p.scale_log2);
        m_run[rb] = m_new;
        l_run[rb] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[rb][d] = acc[rb][d] * alpha;
      }
      const float mc = ref(m_run[rb]);
      float ps = 0.f;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        float e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          e[i] = __builtin_amdgcn_exp2f(fmaf(s[rb][tt][i], p.scale_log2, -mc));
          if (masked) {
            const int t = 32 * tt + 8 * (i >> 2) + 4 * h + (i & 3);
            e[i] = t < seen ? e[i] : 0.f;
          }
          ps += e[i];
        }
#pragma unroll
        for (int i = 0; i < 16; i += 2) pb[rb][2 * tt + (i >> 3)][(i >> 1) & 3] = pack_bf16x2(e[i], e[i + 1]);
      }
      l_run[rb] += ps;
    }
    if (masked && uniform(s_bad[buf])) {
      // pv_masked: token by token, only where the row sees the token
#pragma unroll 1
      for (int t = 0; t < kPromptBlock; ++t) {
        const int idx = 16 * (t >> 5) + 4 * ((t >> 3) & 3) + (t & 3);  // register of the owner half
        const char* vrow = s_kv + buf * 2 * Sh::kTile + Sh::kTile + t * Sh::kStride;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          uint32_t w = 0;
#pragma unroll
          for (int k = 0; k < 16; ++k) w = k == (idx >> 1) ? pb[rb][k >> 2][k & 3] : w;
          w = (uint32_t)__shfl((int)w, n32 + 32 * ((t >> 2) & 1));
          const float pt = __builtin_bit_cast(float, (idx & 1) ? w & 0xffff0000u : w << 16);
          const bool vis = t0 + t < lim[rb];
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int col = 32 * d + 8 * (i >> 2) + 4 * h + (i & 3);
              const float v = bf16_to_f32(*(const uint16_t*)(vrow + 2 * col));
              if (vis) acc[rb][d][i] += pt * v;
            }
        }
      }
      return;
    }
    // V^T: lane group g4 of 16 lanes reads 4 tokens x 16 columns transposed
    const int g4 = lane >> 4;
    const int l16 = lane & 15;
    const uint32_t va = vb + (4 * (g4 >> 1) + (l16 >> 2)) * Sh::kStride + 32 * (g4 & 1) +
                        8 * (l16 & 3);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const uint2 x = lds_read_tr_b64(va + 16 * ks * Sh::kStride + 64 * d);
        const uint2 y = lds_read_tr_b64(va + (16 * ks + 8) * Sh::kStride + 64 * d);
        const u32x4 a = {x.x, x.y, y.x, y.y};
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) acc[rb][d] = mfma32x32x16(a, pb[rb][ks], acc[rb][d]);
      }
  };

  if (blk0 < blk1) {
    // a block some row of the tile masks a token of
    auto is_masked = [&](int blk) { return (blk + 1) * kPromptBlock > lim_lo; };
    Half cur[2] = {half_of(blk0, 0), half_of(blk0, 1)};
    load_block(cur);
    if (tid < 2) s_bad[tid] = 0;
    __syncthreads();
    store_block(0, is_masked(blk0));
    Half nxt[2] = {half_of(min(blk0 + 1, blk1 - 1), 0), half_of(min(blk0 + 1, blk1 - 1), 1)};
    load_block(nxt);
    __syncthreads();
#pragma unroll 1
    for (int blk = blk0; blk < blk1; ++blk) {
      const int buf = Sh::kBufs == 2 ? (blk - blk0) & 1 : 0;
      const bool bad0 = cur[0].bad, bad1 = cur[1].bad;
      if (is_masked(blk) || bad0 || bad1)
        compute(blk, buf, true, bad0, bad1);
      else
        compute(blk, buf, false, false, false);
      if (blk + 1 == blk1) break;
      if (Sh::kBufs == 1) __syncthreads();
      // (s_bad stays set once a masked block held a bad value: the blocks after it take
      // the slow sum too, which is right for any block)
      store_block(Sh::kBufs == 2 ? buf ^ 1 : 0, is_masked(blk + 1));
      cur[0] = nxt[0];
      cur[1] = nxt[1];
      const int want = min(blk + 2, blk1 - 1);
      nxt[0] = half_of(want, 0);
      nxt[1] = half_of(want, 1);
      load_block(nxt);
      __syncthreads();
    }
  }

  // Outputs: lane half h of a row holds columns 32 d + 8 a + 4 h + b.
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    float lo, hi;
    pair_xor32(l_run[rb], lo, hi);
    const float l = lo + hi;
    if (!live[rb]) continue;
    const bool none = l == 0.f;
    const float inv = !len_good ? qnan() : none ? 0.f : 1.f / l;
    const float lse_v = !len_good ? qnan()
                        : none    ? neg_inf()
                                  : (ref(m_run[rb]) + __log2f(l)) * kLn2;
    const size_t rows = (size_t)p.N * p.Hq;
    const bool piece = p.n_splits > 1;
    const size_t at = piece ? split * rows + out_row[rb] : out_row[rb];
    if (h == 0) {
      if (piece) p.part_lse[at] = lse_v;
      else if (p.lse) p.lse[at] = lse_v;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int col = 32 * d + 8 * a + 4 * h;
        const float4 o = make_float4(acc[rb][d][4 * a] * inv, acc[rb][d][4 * a + 1] * inv,
                                     acc[rb][d][4 * a + 2] * inv, acc[rb][d][4 * a + 3] * inv);
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
}

// Combines the splits' pieces of a row: D / 4 threads a row.
__global__ __launch_bounds__(256) void prompt_join_kernel(const PromptParams p, int D) {
  const int c4 = D >> 2;
  const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
  const size_t rows = (size_t)p.N * p.Hq;
  const size_t row = (size_t)(t / c4);
  const int c = (int)(t - (long long)row * c4);
  if (row >= rows) return;
  // rows before the first sequence and behind the last are nobody's
  const int tok = (int)(row / p.Hq);
  if (tok < p.cu_new[0] || tok >= p.cu_new[p.B]) return;
  float M = neg_inf();
  for (int s = 0; s < p.n_splits; ++s) M = max_nan(M, p.part_lse[s * rows + row]);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float L = 0.f;
  if (M != neg_inf())
    for (int s = 0; s < p.n_splits; ++s) {
      const float l = p.part_lse[s * rows + row];
      if (l == neg_inf()) continue;
      const float w = __expf(l - M);
      const float4 o = ((const float4*)p.part_out)[(s * rows + row) * c4 + c];
      L += w;
      a.x += w * o.x; a.y += w * o.y; a.z += w * o.z; a.w += w * o.w;
    }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const float4 o = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
  if (p.out_f32) ((float4*)p.out_f32)[row * c4 + c] = o;
  if (p.out_bf16)
    ((uint2*)p.out_bf16)[row * c4 + c] =
        make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
  if (p.lse && c == 0) p.lse[row] = L == 0.f ? neg_inf() : M + __logf(L);
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
static bool prompt_width_ok(int D) { return D >= 32 && D <= kPromptMaxD && D % 32 == 0; }

// How a call runs: rows of a tile and splits of its tokens.
struct PromptPlan {
  bool wide;  // four waves a workgroup
  int rows, tiles, splits;
};
static PromptPlan prompt_plan(int N, int B, int Hq, int Hkv, int max_len, int n_splits) {
  const int G = Hq / Hkv;
  PromptPlan r;
  r.wide = (long long)N * G > 64LL * B;
  r.rows = r.wide ? 128 : 32;
  r.tiles = (int)(((long long)N * G + r.rows - 1) / r.rows) + B;
  r.splits = n_splits;
  if (n_splits == 0) {
    // enough workgroups for the chip, of at least 4 blocks each
    const int most = std::max(1, max_len / (4 * kPromptBlock));
    const long long wgs = (long long)((N * (long long)G + r.rows - 1) / r.rows) * Hkv;
    const int want = choose_workgroups(0, r.wide ? 2 : 4, 1LL << 30, 1);
    r.splits = (int)std::min<long long>(std::max<long long>(want / std::max(wgs, 1LL), 1),
                                        std::min(most, kPromptMaxSplits));
  }
  return r;
}
static size_t prompt_bytes(int N, int Hq, int D, int splits) {
  if (splits <= 1) return 0;
  const size_t rows = (size_t)N * Hq * splits;
  return align256(rows * 4) + rows * D * 4;
}

template <bool F8>
static void prompt_launch(const PromptParams& p, const PromptPlan& pl, int D, hipStream_t s) {
  const dim3 grid((unsigned)pl.tiles * p.Hkv * p.n_splits);
#define WS_PROMPT_CASE(DD)                                                              \
  case DD:                                                                              \
    if (pl.wide)                                                                        \
      hipLaunchKernelGGL((prompt_kernel<DD, F8, 1, 4>), grid, dim3(256), 0, s, p);      \
    else                                                                                \
      hipLaunchKernelGGL((prompt_kernel<DD, F8, 1, 1>), grid, dim3(64), 0, s, p);       \
    break;
  switch (D) {
    WS_PROMPT_CASE(32) WS_PROMPT_CASE(64) WS_PROMPT_CASE(96) WS_PROMPT_CASE(128)
    WS_PROMPT_CASE(160) WS_PROMPT_CASE(192) WS_PROMPT_CASE(224) WS_PROMPT_CASE(256)
  }
#undef WS_PROMPT_CASE
}

static int prompt_sizes(const char* name, int N, int B, int Hq, int Hkv, int D, int max_len,
                        int n_splits) {
  if (N < 0 || B < 0 || B > kMaxSeqs || Hkv <= 0 || Hq <= 0 || Hq % Hkv || max_len < 0 ||
      n_splits < 0 || n_splits > kPromptMaxSplits)
    return set_error(WS_EINVAL,
                     "%s: bad sizes N=%d B=%d Hq=%d Hkv=%d max_len=%d n_splits=%d (B <= %d, "
                     "n_splits <= %d)",
                     name, N, B, Hq, Hkv, max_len, n_splits, kMaxSeqs, kPromptMaxSplits);
  if (!prompt_width_ok(D))
    return set_error(WS_EINVAL, "%s: head_dim %d unsupported (multiples of 32 up to 256)", name, D);
  if ((long long)N * (Hq / Hkv) + 128LL * B >= (1LL << 31) || max_len > (1 << 30))
    return set_error(WS_EINVAL, "%s: %d tokens of %d heads exceed the row index range", name, N, Hq);
  const PromptPlan pl = prompt_plan(N, B, Hq, Hkv, max_len, n_splits);
  if ((long long)pl.tiles * Hkv * pl.splits * 256 >= (1LL << 32))
    return set_error(WS_EINVAL, "%s: %d tokens of %d heads exceed the launch grid", name, N, Hq);
  return WS_OK;
}

}  // namespace ws

using namespace ws;

extern "C" int ws_gqa_prompt_plan(int N, int B, int Hq, int Hkv, int D, int max_len, int n_splits,
                                  int* n_splits_out, size_t* workspace_bytes_out) {
  if (int rc = prompt_sizes("ws_gqa_prompt_plan", N, B, Hq, Hkv, D, max_len, n_splits)) return rc;
  const PromptPlan pl = prompt_plan(N, B, Hq, Hkv, max_len, n_splits);
  if (n_splits_out) *n_splits_out = pl.splits;
  if (workspace_bytes_out) *workspace_bytes_out = prompt_bytes(N, Hq, D, pl.splits);
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
  if (int rc = prompt_sizes(name, N, B, Hq, Hkv, D, max_len, n_splits)) return rc;
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
  const PromptPlan pl = prompt_plan(N, B, Hq, Hkv, max_len, n_splits);
  const size_t need = prompt_bytes(N, Hq, D, pl.splits);
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
  p.part_out = (float*)((char*)workspace + align256((size_t)N * Hq * pl.splits * 4));
  p.N = N;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.page_size = page_size;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.cap = (int)std::min<long long>((long long)page_size * max_pages, 1LL << 30);
  p.n_splits = pl.splits;
  p.tiles = pl.tiles;
  p.scale_log2 = (scale < 0.f ? -scale : scale) * kLog2e;
  p.q_sign = scale < 0.f ? 0x80008000u : 0u;
  hipStream_t s = (hipStream_t)stream;
  if (k_scale)
    prompt_launch<true>(p, pl, D, s);
  else
    prompt_launch<false>(p, pl, D, s);
  int rc = check_launch(name);
  if (rc != WS_OK || pl.splits == 1) return rc;
  const long long threads = (long long)N * Hq * (D / 4);
  hipLaunchKernelGGL(prompt_join_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s,
                     p, D);
  return check_launch(name);
}
