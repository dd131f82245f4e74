// Split-KV GQA decode attention over 8-bit pages (gfx950): e4m3 keys and values
// with one power-of-two scale (e8m0 byte) per token and KV head.
//
// The work decomposition is the bf16 kernel's (ws_plan.h): every wave is one
// split of the list of all 32-token blocks, streams its range through a register
// ring that runs across row boundaries, and leaves whole rows in out / lse and
// pieces of rows in the workspace.  What differs:
//
//  - A token of a head is D + 1 bytes for K and for V each, half the bf16 pool's,
//    so a wave's block is half as large: keeping the same bytes in flight takes
//    twice the waves or stages (gqa8_stages, gqa8_splits).
//  - The value times its scale is a bf16 number (an e4m3 value has 4 significant
//    bits, and a power of two moves the exponent only), so converting with the
//    scale is exact and the matrix products are the bf16 pool's:
//    v_cvt_scalef32_pk_bf16_fp8 takes two values and the token's scale.
//  - The key columns are permuted, in K and q alike, so that a lane's 16-byte load
//    feeds two k-steps: lane group j's eight columns of k-step 2 i and 2 i + 1
//    are columns 64 i + 16 j .. + 7 and + 8 .. + 15.
//  - Pieces are fp32: a bf16 piece would round the outputs once more, which shows
//    beside the rounding of the probabilities to bf16 for the values' product
//    (softmax_block; their sums are fp32): error against 64 bits 1.4 of the plain
//    form's with fp32 pieces, 1.6 with bf16 ones.
//
// Bound by HBM: 621 MB (16 sequences of 1000 to 32000 tokens, 8 x 4 heads of 128) take
// 102.6 to 103.9 us, 6.0 TB/s, and their merge 4.9; 8192 tokens of 4 x 8 heads 5.6 and 5.9 (the
// start chain: lengths, page ids, blocks).
#include <algorithm>
#include <type_traits>

#include "ws_attn.h"
#include "ws_plan.h"
#include "ws_reduce.h"

namespace ws {

constexpr int kGqa8MaxD = 256;
constexpr int kGqa8Waves = 2;  // waves per workgroup, each its own split

// Value columns of a lane: 4, 8 or 16 bytes, the least that D / 16 lanes hold
// and that divides D.
__host__ __device__ constexpr int gqa8_lane_cols(int D) { return D <= 64 ? 4 : D <= 128 ? 8 : 16; }
// Stages of the register ring.
__host__ __device__ constexpr int gqa8_stages(int D) { return D <= 128 ? 3 : 2; }
__host__ __device__ constexpr int gqa8_waves_per_simd(int D) { return D <= 128 ? 2 : 1; }

template <int N> struct Bytes { typedef uint32_t type; };
template <> struct Bytes<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <> struct Bytes<16> { typedef u32x4 type; };

template <int I, int N, class F>
__device__ __forceinline__ void static_for8(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for8<I + 1, N>(f);
  }
}

// Two e4m3 values (low or high half of w) times a power of two, as bf16.
template <bool HI>
__device__ __forceinline__ uint32_t cvt2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
// Eight values as a matrix operand.
__device__ __forceinline__ u32x4 cvt8(uint32_t lo, uint32_t hi, float scale) {
  return u32x4{cvt2<false>(lo, scale), cvt2<true>(lo, scale), cvt2<false>(hi, scale),
               cvt2<true>(hi, scale)};
}
// An e8m0 byte as the float the conversion takes (its exponent field).
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __builtin_bit_cast(float, byte << 23);
}

struct Gqa8Params {
  const uint16_t* q;
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  const int32_t* page_table;
  const int32_t* len;
  float* out;
  float* lse;
  float* part_out;
  float* part_lse;
  int B, Hkv, G, page_size, max_pages, num_pages, cap, n_splits;
  float scale_log2;
};

// A block's metadata, uniform across the wave (as the bf16 kernel's).
struct Gqa8Block {
  int row;       // kv row
  uint32_t tok;  // pool index of the block's first token
  int nt;        // valid tokens | k8First | k8Last | k8BadPage
};
constexpr int k8NtMask = 63;
constexpr int k8First = 64;
constexpr int k8Last = 128;
constexpr int k8BadPage = 256;

template <int D>
__global__ __launch_bounds__(64 * kGqa8Waves, gqa8_waves_per_simd(D)) void gqa8_decode_kernel(
    const Gqa8Params p) {
  static_assert(D % 32 == 0 && D <= kGqa8MaxD, "head width: a multiple of 32 up to 256");
  constexpr int C = gqa8_lane_cols(D);
  constexpr int LV = D / C;  // lanes n16 that hold value columns
  static_assert(D % C == 0 && LV <= 16, "value columns of a lane");
  using VT = typename Bytes<C>::type;
  constexpr int P64 = D / 64;  // pairs of k-steps
  constexpr bool TAIL = D % 64 != 0;
  constexpr int KS = D / 32;
  constexpr int S = gqa8_stages(D);
  constexpr int W = kGqa8Waves;
  __shared__ int s_pref[kMaxSeqs + 1];
  __shared__ int s_len[kMaxSeqs];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int n16 = lane & 15;
  const int j = lane >> 4;
  const int G = p.G;
  const int split = uniform(blockIdx.x * W + (tid >> 6));
  const Plan plan = plan_build(p.len, 0, p.cap, p.B, p.Hkv, p.n_splits, s_pref, s_len, split, 1,
                               kAlignStep);
  // Sequences without tokens: (0, -inf), or NaN for an invalid length.
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (s_pref[b + 1] != s_pref[b]) continue;
    const bool ok = len_ok(p.len[b], 0, p.cap);
    const size_t q0 = (size_t)b * p.Hkv * G;
    for (int i = tid; i < p.Hkv * G * D; i += 64 * W) p.out[q0 * D + i] = ok ? 0.f : qnan();
    for (int i = tid; i < p.Hkv * G; i += 64 * W) p.lse[q0 + i] = ok ? neg_inf() : qnan();
  }
  if (!plan.has_work) return;  // no barrier below: waves run independently
  const int x_begin = uniform(plan.begin);
  const int x_end = uniform(plan.end);
  const int nblk = x_end - x_begin;

  // Metadata window: lane l describes block xb + l (the last block past the end).
  int m_row, m_nt;
  uint32_t m_tok;
  auto fetch_meta = [&](int xb) __attribute__((always_inline)) {
    const int x = min(xb + lane, x_end - 1);
    int lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_pref[mid] <= x) lo = mid;
      else hi = mid - 1;
    }
    const int len = s_len[lo];
    const int nbb = (len + 31) >> 5;
    const int rel = x - s_pref[lo];
    const int kvh = rel / nbb;
    const int t0 = (rel - kvh * nbb) * 32;
    const int page = t0 / p.page_size;
    const int raw = p.page_table[(size_t)lo * p.max_pages + page];
    const int pid = clamp_page(raw, p.num_pages);
    m_row = lo * p.Hkv + kvh;
    m_tok = ((uint32_t)pid * (uint32_t)p.Hkv + (uint32_t)kvh) * (uint32_t)p.page_size +
            (uint32_t)(t0 - page * p.page_size);
    m_nt = min(32, len - t0) | (t0 == 0 ? k8First : 0) | (t0 + 32 >= len ? k8Last : 0) |
           (raw == pid ? 0 : k8BadPage);
  };
  auto read_meta = [&](int l) __attribute__((always_inline)) {
    Gqa8Block m;
    m.row = __builtin_amdgcn_readlane(m_row, l);
    m.tok = (uint32_t)__builtin_amdgcn_readlane((int)m_tok, l);
    m.nt = __builtin_amdgcn_readlane(m_nt, l);
    return m;
  };

  // One stage of the ring.  Rows past the valid tokens repeat the last valid one.
  // The scales of a lane's value tokens are two dwords, which may hold bytes past
  // the valid tokens (compute_block takes 1 for those).
  struct Stage {
    u32x4 k[2][P64 > 0 ? P64 : 1];
    uint2 kt[2];
    uint32_t ks[2];
    VT v[8];
    uint32_t vs[2];
  };
  auto load = [&](const Gqa8Block& m, bool valid, Stage& st) __attribute__((always_inline)) {
    // past the range's end every lane reads the pool's first row: the same
    // instructions and registers, a cache hit, no HBM traffic
    const size_t tok = valid ? m.tok : 0;
    const int last = valid ? (m.nt & k8NtMask) - 1 : 0;
    // the block's addresses are uniform, a lane's offsets in it 32-bit
    const uint8_t* kb = p.k_pages + tok * D;
    const uint8_t* vb = p.v_pages + tok * D;
    const uint8_t* ksb = p.k_scale + tok;
    const uint8_t* vsb = p.v_scale + tok;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const uint32_t r = min(16 * tt + n16, last);
#pragma unroll
      for (int i = 0; i < P64; ++i) st.k[tt][i] = ld_stream(kb + (r * D + 16 * j) + 64 * i);
      if (TAIL) st.kt[tt] = *(const uint2*)(kb + (r * D + 8 * j) + 64 * P64);
      st.ks[tt] = ksb[r];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t r = min(pv_token(i, j), last);
      st.v[i] = __builtin_nontemporal_load(
          (const VT*)(vb + (r * D + ((LV == 16 || n16 < LV) ? C * n16 : 0))));
    }
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) st.vs[tt] = *(const uint32_t*)(vsb + (16 * tt + 4 * j));
  };
  // q of a kv row as the QK B operand, in the keys' column order.
  u32x4 qb[KS];
  auto load_q = [&](int row) __attribute__((always_inline)) {
    const u32x4* qp = (const u32x4*)(p.q + (size_t)(row * G + min(n16, G - 1)) * D);
#pragma unroll
    for (int s = 0; s < 2 * P64; ++s) qb[s] = qp[8 * (s >> 1) + 2 * j + (s & 1)];
    if (TAIL) qb[KS - 1] = qp[8 * P64 + j];
  };

  f32x4 acc[C];
#pragma unroll
  for (int e = 0; e < C; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = neg_inf();
  float l_run = 0.f;

  auto compute_block = [&](const Gqa8Block& m, const Stage& st) __attribute__((always_inline)) {
    f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
    const float k0 = scale_of(st.ks[0]), k1 = scale_of(st.ks[1]);
#pragma unroll
    for (int i = 0; i < P64; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s0 = mfma16x16x32(cvt8(st.k[0][i][2 * u], st.k[0][i][2 * u + 1], k0), qb[2 * i + u], s0);
        s1 = mfma16x16x32(cvt8(st.k[1][i][2 * u], st.k[1][i][2 * u + 1], k1), qb[2 * i + u], s1);
      }
    if (TAIL) {
      s0 = mfma16x16x32(cvt8(st.kt[0].x, st.kt[0].y, k0), qb[KS - 1], s0);
      s1 = mfma16x16x32(cvt8(st.kt[1].x, st.kt[1].y, k1), qb[KS - 1], s1);
    }
    const int nt = m.nt & k8NtMask;
    float alpha;
    bool rescale;
    const u32x4 pb = softmax_block(s0, s1, j, nt, p.scale_log2, m_run, l_run, alpha, rescale);
    uint32_t vs[2] = {st.vs[0], st.vs[1]};
    if (nt < 32) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (pv_token(i, j) >= nt) {
          const int sh = 8 * (i & 3);
          vs[i >> 2] = (vs[i >> 2] & ~(0xffu << sh)) | (127u << sh);
        }
    }
    struct {
      uint32_t w[C / 2];
      __device__ __forceinline__ uint32_t operator[](int i) const { return w[i]; }
    } vr[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float sc = scale_of((vs[i >> 2] >> (8 * (i & 3))) & 0xffu);
      uint32_t raw[C / 4];
      __builtin_memcpy(raw, &st.v[i], C);
#pragma unroll
      for (int d = 0; d < C / 4; ++d) {
        vr[i].w[2 * d] = cvt2<false>(raw[d], sc);
        vr[i].w[2 * d + 1] = cvt2<true>(raw[d], sc);
      }
    }
    pv_block(acc, vr, pb, alpha, rescale);
  };

  // The piece of kv row `row` in (m_run, l_run, acc): final when this wave held the
  // whole row, else a workspace slot; NaN if one of its page ids was bad.
  auto flush = [&](int row, bool whole, bool bad) __attribute__((always_inline)) {
    const float l_tot = wave_sum_xor16_32(l_run);
    if (n16 >= G) return;
    const float inv = bad ? qnan() : 1.f / l_tot;
    const float lse_v = bad ? qnan() : (m_run + __log2f(l_tot)) * kLn2;
    const size_t at = (size_t)(whole ? row : split + row) * G + n16;
    float* o = (whole ? p.out : p.part_out) + at * D + 4 * C * j;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (LV < 16 && 4 * j + i >= LV) continue;
#pragma unroll
      for (int e = 0; e < C; e += 4)
        ((float4*)(o + C * i + e))[0] = make_float4(acc[e][i] * inv, acc[e + 1][i] * inv,
                                                    acc[e + 2][i] * inv, acc[e + 3][i] * inv);
    }
    if (j == 0) (whole ? p.lse : p.part_lse)[at] = lse_v;
  };

  // Ring of S stages: step k requests block k + S - 1 (past the range's end the last
  // block again), then runs block k's math.  The loop body is a whole turn of the
  // ring with no early exit.
  int xb = x_begin;
  fetch_meta(xb);
  Gqa8Block mq[S];
  Stage st[S];
  mq[0] = read_meta(0);
  int run_row = mq[0].row;
  bool run_first = (mq[0].nt & k8First) != 0;
  bool run_last = false;
  bool run_bad = false;
  load_q(mq[0].row);
  static_for8<0, S - 1>([&](auto i) __attribute__((always_inline)) {
    constexpr int s = decltype(i)::value;
    if (s > 0) mq[s] = read_meta(min(s, nblk - 1));
    load(mq[s], s < nblk, st[s]);
  });
  auto step = [&](auto stage, int k) __attribute__((always_inline)) {
    constexpr int s = decltype(stage)::value;
    constexpr int ld = (s + S - 1) % S;
    constexpr int nx = (s + 1) % S;
    const int want = min(k + S - 1, nblk - 1);
    if (x_begin + want - xb == 64) {
      xb += 64;
      fetch_meta(xb);
    }
    mq[ld] = read_meta(x_begin + want - xb);
    load(mq[ld], k + S - 1 < nblk, st[ld]);
    __builtin_amdgcn_sched_barrier(0);
    const Gqa8Block& cur = mq[s];
    if (cur.row != run_row) {
      flush(run_row, run_first && run_last, run_bad);
      run_row = cur.row;
      run_first = (cur.nt & k8First) != 0;
      run_bad = false;
      m_run = neg_inf();
      l_run = 0.f;
#pragma unroll
      for (int e = 0; e < C; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    run_last = (cur.nt & k8Last) != 0;
    run_bad |= (cur.nt & k8BadPage) != 0;
    compute_block(cur, st[s]);
    __builtin_amdgcn_sched_barrier(0);
    if (mq[nx].row != cur.row) load_q(mq[nx].row);
  };
  int base = 0;
  for (; base + S <= nblk; base += S)
    static_for8<0, S>([&](auto i) __attribute__((always_inline)) {
      step(i, base + decltype(i)::value);
    });
  static_for8<0, S - 1>([&](auto i) __attribute__((always_inline)) {
    if (base + decltype(i)::value < nblk) step(i, base + decltype(i)::value);
  });
  flush(run_row, run_first && run_last, run_bad);
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

static bool gqa8_width_ok(int D) { return D >= 32 && D <= kGqa8MaxD && D % 32 == 0; }

// Splits (waves) of a call: n_splits when given, else per CU what keeps the HBM
// busy, at most what the blocks of the longest possible batch feed with 2 each.  Steps
// with their merge, us, at 2 / 4 / 6 / 8 / 12 waves per CU (a workgroup holds two, so odd
// counts leave CUs with one more than others and lose):
//   128 columns, 621 MB   123  110  104  105  111     64 columns, 204 MB  70  50  43  42  44
//   128 columns, 135 MB    32   32   33   35   42    256 columns, 159 MB  33  33  42  38  45
static int gqa8_splits(int n_splits, int rows_kv, int max_len, int D) {
  if (n_splits > 0) return n_splits;
  const long long max_blocks = (long long)rows_kv * ((max_len + 31) / 32);
  return choose_workgroups(0, D <= 64 ? 8 : D <= 128 ? 6 : 4, max_blocks, 2);
}

static int gqa8_launch(const uint16_t* q, const uint8_t* k_pages, const uint8_t* v_pages,
                       const uint8_t* k_scale, const uint8_t* v_scale, const int32_t* page_table,
                       const int32_t* gpu_len, int B, int Hq, int Hkv, int D, int page_size,
                       int max_pages, int num_pages, int max_len, int n_splits, float scale,
                       uint16_t* out_bf16, float* out, float* lse, void* workspace,
                       size_t workspace_bytes, void* stream, const char* name) {
  if (!q || !k_pages || !v_pages || !k_scale || !v_scale || !page_table || !gpu_len || !out ||
      !lse)
    return set_error(WS_EINVAL, "%s: null pointer", name);
  if (B < 0 || B > kMaxSeqs || Hkv <= 0 || Hq <= 0 || Hq % Hkv)
    return set_error(WS_EINVAL, "%s: bad batch/heads B=%d Hq=%d Hkv=%d (B <= %d)", name, B, Hq,
                     Hkv, kMaxSeqs);
  const int G = Hq / Hkv;
  if (G > 16) return set_error(WS_EINVAL, "%s: group size %d unsupported (1 to 16)", name, G);
  if (!gqa8_width_ok(D))
    return set_error(WS_EINVAL, "%s: head_dim %d unsupported (multiples of 32 up to 256)", name, D);
  if (page_size <= 0 || page_size % 32 || max_pages <= 0 || num_pages <= 0 || max_len < 0 ||
      (long long)max_len > (long long)page_size * max_pages)
    return set_error(WS_EINVAL,
                     "%s: bad paging page_size=%d max_pages=%d num_pages=%d max_len=%d "
                     "(page_size must be a multiple of 32)",
                     name, page_size, max_pages, num_pages, max_len);
  if ((long long)num_pages * Hkv * page_size > 0xffffffffLL)
    return set_error(WS_EINVAL, "%s: pools of %lld tokens exceed the 32-bit token index", name,
                     (long long)num_pages * Hkv * page_size);
  if (n_splits < 0) return set_error(WS_EINVAL, "%s: n_splits %d < 0", name, n_splits);
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) ||
      !aligned16(out_bf16) || ((uintptr_t)v_scale & 3u))
    return set_error(WS_EINVAL, "%s: buffers must be 16-byte aligned (scales: 4)", name);
  if (B == 0) return WS_OK;
  if (!plan_fits(B, Hkv, max_len))
    return set_error(WS_EINVAL, "%s: %lld kv rows of %d tokens exceed the block index range", name,
                     (long long)B * Hkv, max_len);
  const int rows_kv = B * Hkv;
  const int n = gqa8_splits(n_splits, rows_kv, max_len, D);
  if (n > kMaxSplits)
    return set_error(WS_EINVAL, "%s: %d splits exceed the merge's %d", name, n, kMaxSplits);
  const size_t need = ws::workspace_bytes(rows_kv, G, D, n, true);
  if (!workspace || workspace_bytes < need)
    return set_error(WS_EWORKSPACE, "%s: workspace %zu < %zu bytes", name, workspace_bytes, need);
  if (((uintptr_t)workspace & 255u) != 0)
    return set_error(WS_EINVAL, "%s: workspace must be 256-byte aligned", name);
  const SplitWorkspace w = carve_workspace(workspace, rows_kv, G, n);
  Gqa8Params prm;
  prm.q = q;
  prm.k_pages = k_pages;
  prm.v_pages = v_pages;
  prm.k_scale = k_scale;
  prm.v_scale = v_scale;
  prm.page_table = page_table;
  prm.len = gpu_len;
  prm.out = out;
  prm.lse = lse;
  prm.part_out = (float*)w.part_out;
  prm.part_lse = w.part_lse;
  prm.B = B;
  prm.Hkv = Hkv;
  prm.G = G;
  prm.page_size = page_size;
  prm.max_pages = max_pages;
  prm.num_pages = num_pages;
  prm.cap = (int)std::min<long long>((long long)page_size * max_pages, 1LL << 30);
  prm.scale_log2 = scale * kLog2e;
  prm.n_splits = n;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((n + kGqa8Waves - 1) / kGqa8Waves), block(64 * kGqa8Waves);
#define WS_GQA8_CASE(DD)                                                    \
  case DD:                                                                  \
    hipLaunchKernelGGL((gqa8_decode_kernel<DD>), grid, block, 0, s, prm);   \
    break;
  switch (D) {
    WS_GQA8_CASE(32) WS_GQA8_CASE(64) WS_GQA8_CASE(96) WS_GQA8_CASE(128)
    WS_GQA8_CASE(160) WS_GQA8_CASE(192) WS_GQA8_CASE(224) WS_GQA8_CASE(256)
  }
#undef WS_GQA8_CASE
  int rc = check_launch(name);
  if (rc != WS_OK) return rc;
  const MlaLayout lay = {false, 1, G, B, kAlignStep, true};
  rc = merge_split_pieces(gpu_len, 0, lay, Hkv, G, D, prm.cap, n, out, lse, w, out_bf16, s);
  return rc != WS_OK ? rc : check_launch(name);
}

}  // namespace ws

using namespace ws;

extern "C" int ws_gqa8_decode_plan(int rows_kv, int heads, int D, int max_len, int n_splits,
                                   int* n_splits_out, size_t* workspace_bytes_out) {
  if (!gqa8_width_ok(D))
    return set_error(WS_EINVAL, "ws_gqa8_decode_plan: head_dim %d unsupported (multiples of 32 "
                                "up to 256)", D);
  if (rows_kv < 0 || max_len < 0 || n_splits < 0 || heads <= 0 || heads > 16)
    return set_error(WS_EINVAL, "ws_gqa8_decode_plan: bad arguments");
  const int n = gqa8_splits(n_splits, rows_kv, max_len, D);
  if (n_splits_out) *n_splits_out = n;
  if (workspace_bytes_out) *workspace_bytes_out = ws::workspace_bytes(rows_kv, heads, D, n, true);
  return WS_OK;
}

extern "C" int ws_gqa8_decode_partial(const uint16_t* q, const uint8_t* k_pages,
                                      const uint8_t* v_pages, const uint8_t* k_scale,
                                      const uint8_t* v_scale, const int32_t* page_table,
                                      const int32_t* gpu_len, int B, int Hq, int Hkv, int D,
                                      int page_size, int max_pages, int num_pages, int max_len,
                                      int n_splits, float scale, float* out, float* lse,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  return gqa8_launch(q, k_pages, v_pages, k_scale, v_scale, page_table, gpu_len, B, Hq, Hkv, D,
                     page_size, max_pages, num_pages, max_len, n_splits, scale, nullptr, out, lse,
                     workspace, workspace_bytes, stream, "ws_gqa8_decode_partial");
}

extern "C" int ws_gqa8_decode_full(const uint16_t* q, const uint8_t* k_pages,
                                   const uint8_t* v_pages, const uint8_t* k_scale,
                                   const uint8_t* v_scale, const int32_t* page_table,
                                   const int32_t* gpu_len, int B, int Hq, int Hkv, int D,
                                   int page_size, int max_pages, int num_pages, int max_len,
                                   int n_splits, float scale, uint16_t* out_bf16, float* out,
                                   float* lse, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  if (!out_bf16) return set_error(WS_EINVAL, "ws_gqa8_decode_full: out_bf16 is null");
  return gqa8_launch(q, k_pages, v_pages, k_scale, v_scale, page_table, gpu_len, B, Hq, Hkv, D,
                     page_size, max_pages, num_pages, max_len, n_splits, scale, out_bf16, out, lse,
                     workspace, workspace_bytes, stream, "ws_gqa8_decode_full");
}
