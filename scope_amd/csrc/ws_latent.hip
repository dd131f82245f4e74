// The latent cache of absorbed MLA as it is written and read back (gfx950).
//
// ws_latent_rope_append: a token's latent is
//   [ c rsqrt(mean(c^2) + eps) w , R(position) pe ]         512 + 64 columns
// (the norm with a weight only) and goes to its slot of the pages, beside the rotary
// positions of the heads' q_pe.  R turns 32 pairs, columns (i, i + 32) or (2 i, 2 i + 1), as
// ws_rope does, its angle in 64 bits.
//
// 8-bit pages hold e4m3 values and an e8m0 scale for every block of `block` slots: 2^e, e
// the least >= -126 with max|x| <= 448 2^e over the block's tokens.  A block that already
// holds tokens keeps at least its scale; where a new token raises it, the older tokens'
// values are rounded again at the new scale (a power of two apart, so only what falls below
// e4m3's normal range changes).  An infinity or a NaN becomes e4m3's NaN in its place and
// takes no part in the scale.
//
// ws_latent_gather reads ranges of tokens back as bf16 rows (e4m3 times a power of two is a
// bf16 number: exact).
//
// With a scale for one token, in bf16 and back, all of it is bound by HBM or, for a decode step's
// few tokens, by the launch and one chain of loads: 32 tokens into 8-bit pages 3.9 us; 16100 tokens
// of 16 heads into bf16 pages 21.8 us (103 MB: 4.7 TB/s, where a copy of 1 GiB has 5.1; 17.4 over
// pages that the last cache holds); 29700 tokens read back from 8 bits 11.4 us (51 MB), 7700 in 150
// ranges from bf16 5.9 us (18 MB).  With a scale for several tokens the runs bound it, two of them
// one after the other in some workgroup, each a chain of loads: 4651 tokens to blocks of 32 12.6 us
// (32 MB, 2.5 TB/s), 16000 29.7 (3.1 TB/s).
#include <math.h>

#include <algorithm>

#include "ws_attn.h"
#include "ws_plan.h"

namespace ws {

constexpr int kLatC = 512;
constexpr int kLatPe = 64;
constexpr int kLatW = kLatC + kLatPe;
constexpr int kLatPairs = kLatPe / 2;
constexpr int kLatTokens = 4;  // most tokens of a workgroup, one a wave
// With a scale for several tokens: waves of a workgroup, tokens a wave takes at a time (in
// registers between the two looks at them), and the tokens whose runs a workgroup looks for: as
// many as leave kRunGroups workgroups (one for each token: 780 tokens 10.7 us instead of 8.1,
// 1200 15.5 instead of 10.3; 384 to 1024 workgroups are alike on average), up to kRunWindow or, with scales of 32 tokens and more, twice
// that (16000 tokens of 4 sequences: 29.7 us instead of 34; with scales of 2 tokens 132 instead
// of 116).
constexpr int kRunWaves = 8;
constexpr int kRunTokens = 4;
constexpr int kRunChunk = kRunWaves * kRunTokens;
constexpr int kRunWindow = 16;
constexpr int kRunGroups = 768;
constexpr int kRunTurns = 8;  // tokens whose q_pe a workgroup turns there

// Wave sums and maxima of the ROCm device library (DPP sequences; every lane active).
extern "C" __device__ float __ockl_wfred_add_f32(float);
extern "C" __device__ uint32_t __ockl_wfred_max_u32(uint32_t);
extern "C" __device__ int __ockl_wfred_min_i32(int);

struct LatentParams {
  const uint16_t* c;
  const uint16_t* pe;
  const uint16_t* q;
  int64_t c_stride, pe_stride, q_stride, q_head;  // elements
  const int32_t* positions;
  const float* inv_freq;
  const void* weight;
  const int32_t* slots;
  uint16_t* q_out;
  void* pages;
  uint8_t* scale;
  int N, H, num_slots, block_log2, tokens, window;
  int run_groups;  // workgroups that write runs, ahead of those that turn q_pe (and write the rest)
  bool weight_f32;
  float eps, factor;
};

__device__ __forceinline__ void lat_unpack8(const u32x4& w, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __builtin_bit_cast(float, w[i] << 16);
    x[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ u32x4 lat_pack8(const float* x) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  return w;
}
// Four values times s as e4m3, rounded to nearest even (finite ones: |x s| <= 448).
__device__ __forceinline__ uint32_t lat_pack4(const float* x, float s) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_fabsf(x[i]) < __builtin_inff() ? x[i] * s : qnan();
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}
// The bits of the largest finite magnitude of n values, at least `top`.
template <int N>
__device__ __forceinline__ uint32_t lat_top(const float* x, uint32_t top) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu;
    top = max(top, b < 0x7f800000u ? b : 0u);
  }
  return top;
}
// The e8m0 byte 127 + e of a largest magnitude: e the least >= -126 with top <= 1.75 *
// 2^(8 + e).
__device__ __forceinline__ int lat_byte(uint32_t top) {
  return max((int)((top + 0x1fffffu) >> 23) - 8, 1);
}
// 2^(127 - byte), byte from 1 to 254
__device__ __forceinline__ float lat_inverse(int byte) { return ldexpf(1.f, 127 - byte); }

// (cos, sin) of pair pr of token tok, scaled.
__device__ __forceinline__ float2 lat_angle(const LatentParams& p, int tok, int pr) {
  const double turns =
      (double)p.positions[tok] * ((double)p.inv_freq[pr] * 0.15915494309189535);
  const float f = (float)(2.0 * (turns - rint(turns)));
  float sn, cs;
  sincospif(f, &sn, &cs);
  return make_float2(cs * p.factor, sn * p.factor);
}

// A token's latent across a wave: lane l holds columns 8 l .. 8 l + 7 of c, and lanes 0 to
// 3 a quarter of pe turned: two times eight columns from pc0 and pc1.
struct Latent {
  float c[8];
  float pe[16];
};
template <bool ADJACENT>
struct PeCols {
  __device__ static int first(int l) { return ADJACENT ? 16 * l : 8 * l; }
  __device__ static int second(int l) { return ADJACENT ? 16 * l + 8 : kLatPairs + 8 * l; }
};
template <bool ADJACENT>
__device__ __forceinline__ void lat_turn(float* x, const float2* cs) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 w = cs[i];
    const int a = ADJACENT ? 2 * i : i;
    const int b = ADJACENT ? 2 * i + 1 : i + 8;
    const float u = x[a], v = x[b];
    x[a] = u * w.x - v * w.y;
    x[b] = v * w.x + u * w.y;
  }
}
// cs: the token's 32 (cos, sin).  Every lane of the wave must call it.
template <bool ADJACENT>
__device__ __forceinline__ void lat_load(const LatentParams& p, int tok, const float* weight,
                                         const float2* cs, Latent& x) {
  const int lane = threadIdx.x & 63;
  const u32x4 wc = *(const u32x4*)(p.c + (size_t)tok * p.c_stride + 8 * lane);
  u32x4 wa = {0, 0, 0, 0}, wb = {0, 0, 0, 0};
  if (lane < 4) {
    const uint16_t* pe = p.pe + (size_t)tok * p.pe_stride;
    wa = *(const u32x4*)(pe + PeCols<ADJACENT>::first(lane));
    wb = *(const u32x4*)(pe + PeCols<ADJACENT>::second(lane));
  }
  lat_unpack8(wc, x.c);
  if (p.weight) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x.c[i], x.c[i], sum);
    const float r = 1.f / sqrtf(__ockl_wfred_add_f32(sum) * (1.f / kLatC) + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x.c[i] = x.c[i] * r * weight[i];
  }
  lat_unpack8(wa, x.pe);
  lat_unpack8(wb, x.pe + 8);
  if (lane < 4) lat_turn<ADJACENT>(x.pe, cs + 8 * lane);
}
template <bool ADJACENT>
__device__ __forceinline__ void lat_put8(const LatentParams& p, int slot, const Latent& x, float s) {
  const int lane = threadIdx.x & 63;
  uint8_t* row = (uint8_t*)p.pages + (size_t)slot * kLatW;
  *(uint2*)(row + 8 * lane) = make_uint2(lat_pack4(x.c, s), lat_pack4(x.c + 4, s));
  if (lane < 4) {
    *(uint2*)(row + kLatC + PeCols<ADJACENT>::first(lane)) =
        make_uint2(lat_pack4(x.pe, s), lat_pack4(x.pe + 4, s));
    *(uint2*)(row + kLatC + PeCols<ADJACENT>::second(lane)) =
        make_uint2(lat_pack4(x.pe + 8, s), lat_pack4(x.pe + 12, s));
  }
}
__device__ __forceinline__ uint32_t lat_wave_top(const Latent& x) {
  return __ockl_wfred_max_u32(lat_top<16>(x.pe, lat_top<8>(x.c, 0u)));  // (lanes past 3 hold zeros of pe)
}
__device__ __forceinline__ void lat_weight(const LatentParams& p, float* w) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (!p.weight) return;
  if (p.weight_f32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = ((const float*)p.weight)[8 * lane + i];
  } else {
    lat_unpack8(*(const u32x4*)((const uint16_t*)p.weight + 8 * lane), w);
  }
}
__device__ __forceinline__ bool lat_slot_ok(const LatentParams& p, int slot) {
  return slot >= 0 && slot < p.num_slots;
}

// kRunTokens tokens across a wave, as they are: lane l holds columns 8 l .. 8 l + 7 of each
// one's c and its norm's factor, and lane 4 t + q (t < kRunTokens) quarter q of token t's pe.
struct Run {
  u32x4 c[kRunTokens];
  u32x4 pe[2];
  float r[kRunTokens];
};
// Tokens tok .. tok + n - 1 (the last one again past those), and their angles to s_cs, the
// wave's part of LDS.
template <bool ADJACENT>
__device__ __forceinline__ void run_load(const LatentParams& p, int tok, int n, float2* s_cs, Run& x) {
  const int lane = threadIdx.x & 63, q = lane & 3;
#pragma unroll
  for (int t = 0; t < kRunTokens; ++t)
    x.c[t] = *(const u32x4*)(p.c + (size_t)(tok + min(t, n - 1)) * p.c_stride + 8 * lane);
  x.pe[0] = x.pe[1] = u32x4{0, 0, 0, 0};
  if (lane < 4 * kRunTokens) {
    const uint16_t* pe = p.pe + (size_t)(tok + min(lane >> 2, n - 1)) * p.pe_stride;
    x.pe[0] = *(const u32x4*)(pe + PeCols<ADJACENT>::first(q));
    x.pe[1] = *(const u32x4*)(pe + PeCols<ADJACENT>::second(q));
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the angles before are read)
#pragma unroll 1
  for (int i = lane; i < kRunTokens * kLatPairs; i += 64)
    s_cs[i] = lat_angle(p, tok + min(i / kLatPairs, n - 1), i % kLatPairs);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int t = 0; t < kRunTokens; ++t) x.r[t] = 1.f;
  if (!p.weight) return;
#pragma unroll
  for (int t = 0; t < kRunTokens; ++t) {
    float v[8];
    lat_unpack8(x.c[t], v);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
    x.r[t] = sum;
  }
#pragma unroll
  for (int t = 0; t < kRunTokens; ++t)
    x.r[t] = 1.f / sqrtf(__ockl_wfred_add_f32(x.r[t]) * (1.f / kLatC) + p.eps);
}
// Eight columns of token t's c, normalised; the lane's sixteen columns of pe, turned.
__device__ __forceinline__ void run_c(const Run& x, int t, const float* weight, float* v) {
  lat_unpack8(x.c[t], v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = v[i] * x.r[t] * weight[i];
}
template <bool ADJACENT>
__device__ __forceinline__ void run_pe(const Run& x, const float2* s_cs, float* v) {
  const int lane = threadIdx.x & 63;
  lat_unpack8(x.pe[0], v);
  lat_unpack8(x.pe[1], v + 8);
  if (lane < 4 * kRunTokens) lat_turn<ADJACENT>(v, s_cs + (lane >> 2) * kLatPairs + 8 * (lane & 3));
}
template <bool ADJACENT>
__device__ __forceinline__ uint32_t run_top(const Run& x, const float* weight, const float2* s_cs) {
  float v[16];
  run_pe<ADJACENT>(x, s_cs, v);
  uint32_t top = lat_top<16>(v, 0u);  // (lanes past the tokens hold zeros)
#pragma unroll
  for (int t = 0; t < kRunTokens; ++t) {
    run_c(x, t, weight, v);
    top = lat_top<8>(v, top);
  }
  return top;
}
template <bool ADJACENT>
__device__ __forceinline__ void run_put(const LatentParams& p, int tok, int n, const Run& x, const float* weight,
                                        const float2* s_cs, float s) {
  const int lane = threadIdx.x & 63;
  float v[16];
#pragma unroll
  for (int t = 0; t < kRunTokens; ++t) {
    if (t >= n) break;
    run_c(x, t, weight, v);
    uint8_t* row = (uint8_t*)p.pages + (size_t)p.slots[tok + t] * kLatW;
    *(uint2*)(row + 8 * lane) = make_uint2(lat_pack4(v, s), lat_pack4(v + 4, s));
  }
  run_pe<ADJACENT>(x, s_cs, v);
  if (lane < 4 * n) {
    const int q = lane & 3;
    uint8_t* row = (uint8_t*)p.pages + (size_t)p.slots[tok + (lane >> 2)] * kLatW + kLatC;
    *(uint2*)(row + PeCols<ADJACENT>::first(q)) = make_uint2(lat_pack4(v, s), lat_pack4(v + 4, s));
    *(uint2*)(row + PeCols<ADJACENT>::second(q)) = make_uint2(lat_pack4(v + 8, s), lat_pack4(v + 12, s));
  }
}

// With a scale for several tokens, a workgroup takes the run of tokens from tok on whose
// slots lie in one block, if tok is the run's first: the block's tokens follow one another in
// a call, so nobody else writes the block.  Two looks at the tokens: their largest magnitude,
// then their values (up to kRunChunk tokens from the registers, more from the cache again).  (A
// wave for every fourth token, one at a time, and read again: 4651 tokens to blocks of 32 53.7
// us.)
//
// at: the lane of the run's first token in `slots`, which holds the slots of tokens base +
// lane (-1 outside the call).
template <bool ADJACENT>
__device__ void lat_block(const LatentParams& p, int base, int at, int slots, float2* s_all, int* s_top) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tok = base + at;
  const int block = __builtin_amdgcn_readlane(slots, at) >> p.block_log2;
  // the run's tokens and its lowest slot, alike in every wave
  int low = 0x7fffffff, end = at;
  for (;;) {
    const bool in = lat_slot_ok(p, slots) && slots >> p.block_log2 == block;
    const uint64_t out = __builtin_amdgcn_ballot_w64(!in) & (~0ull << end);
    const int stop = out ? __builtin_ctzll(out) : 64;
    low = min(low, __ockl_wfred_min_i32(lane >= end && lane < stop ? slots : 0x7fffffff));
    end = stop;
    if (stop < 64) break;
    base += 64;
    slots = base + lane < p.N ? p.slots[base + lane] : -1;
    end = 0;
  }
  const int count = uniform(base + end - tok);
  low = uniform(low);
  const int first = low - (block << p.block_log2);  // tokens that the block held before
  const int had = first > 0 ? p.scale[block] : 0;
  float w[8];
  lat_weight(p, w);
  float2* s_cs = s_all + wave * (kRunTokens * kLatPairs);
  __syncthreads();  // (the run before is done with s_top and the scale)
  if (tid == 0) *s_top = 0;
  __syncthreads();
  Run x;
  const int own = kRunTokens * wave;  // the wave's first token of a chunk
  const bool once = count <= kRunChunk;
  uint32_t top = 0;
  for (int i = own; i < count; i += kRunChunk) {
    run_load<ADJACENT>(p, tok + i, min(count - i, kRunTokens), s_cs, x);
    top = max(top, run_top<ADJACENT>(x, w, s_cs));
  }
  top = __ockl_wfred_max_u32(top);
  if (lane == 0) atomicMax(s_top, (int)top);
  __syncthreads();
  const int byte = max(lat_byte((uint32_t)*s_top), had);
  const float s = lat_inverse(byte);
  for (int i = own; i < count; i += kRunChunk) {
    const int n = min(count - i, kRunTokens);
    if (!once) run_load<ADJACENT>(p, tok + i, n, s_cs, x);
    run_put<ADJACENT>(p, tok + i, n, x, w, s_cs, s);
  }
  if (byte > had && first > 0) {  // the older tokens at the new scale
    const float f = ldexpf(1.f, had - byte);
    uint32_t* old = (uint32_t*)((uint8_t*)p.pages + ((size_t)block << p.block_log2) * kLatW);
    for (int i = tid; i < first * (kLatW / 4); i += 64 * kRunWaves) {
      typedef float f32x2_t __attribute__((ext_vector_type(2)));
      const uint32_t v = old[i];
      const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(v, false);
      const f32x2_t b = __builtin_amdgcn_cvt_pk_f32_fp8(v, true);
      const float y[4] = {a[0], a[1], b[0], b[1]};
      old[i] = lat_pack4(y, f);
    }
  }
  if (tid == 0) p.scale[block] = (uint8_t)byte;
}

// RUNS: 8-bit pages with a scale for several tokens.
template <bool ADJACENT, bool RUNS>
__global__ __launch_bounds__(RUNS ? 64 * kRunWaves : 256, RUNS ? 4 : 1) void latent_append_kernel(const LatentParams p) {
  constexpr int kThreads = RUNS ? 64 * kRunWaves : 256;
  __shared__ float2 s_cs[(RUNS ? kRunChunk : kLatTokens) * kLatPairs];
  __shared__ int s_top;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (RUNS && (int)blockIdx.x < p.run_groups) {
    const int base = (int)blockIdx.x * p.window - 1;
    const int t = base + lane;
    const int slots = t >= 0 && t < p.N ? p.slots[t] : -1;
    const int prev = __shfl_up(slots, 1);
    // tokens of the window that begin a run
    uint64_t begins = __builtin_amdgcn_ballot_w64(
        lane >= 1 && lane <= p.window && lat_slot_ok(p, slots) &&
        !(lat_slot_ok(p, prev) && prev >> p.block_log2 == slots >> p.block_log2));
    for (; begins; begins &= begins - 1)
      lat_block<ADJACENT>(p, base, __builtin_ctzll(begins), slots, s_cs, &s_top);
    return;
  }
  const int t0 = ((int)blockIdx.x - (RUNS ? p.run_groups : 0)) * p.tokens;
  const int nt = min(p.tokens, p.N - t0);
  if (tid < nt * kLatPairs)
    s_cs[tid] = lat_angle(p, t0 + tid / kLatPairs, tid % kLatPairs);
  __syncthreads();
  if (!RUNS && wave < nt) {
    const int tok = t0 + wave;
    const int slot = p.slots[tok];
    float w[8];
    lat_weight(p, w);
    Latent x;
    lat_load<ADJACENT>(p, tok, w, s_cs + wave * kLatPairs, x);
    if (lat_slot_ok(p, slot)) {  // (the same in every lane)
      if (p.scale) {
        const int byte = lat_byte(lat_wave_top(x));
        lat_put8<ADJACENT>(p, slot, x, lat_inverse(byte));
        if (lane == 0) p.scale[slot] = (uint8_t)byte;
      } else {
        uint16_t* row = (uint16_t*)p.pages + (size_t)slot * kLatW;
        *(u32x4*)(row + 8 * lane) = lat_pack8(x.c);
        if (lane < 4) {
          *(u32x4*)(row + kLatC + PeCols<ADJACENT>::first(lane)) = lat_pack8(x.pe);
          *(u32x4*)(row + kLatC + PeCols<ADJACENT>::second(lane)) = lat_pack8(x.pe + 8);
        }
      }
    }
  }
  // q_pe: four lanes a head
  const int l = tid & 3;
  for (int r = tid >> 2; r < nt * p.H; r += kThreads / 4) {
    const int t = r / p.H;
    const int h = r - t * p.H;
    const size_t tok = (size_t)(t0 + t);
    const uint16_t* src = p.q + tok * p.q_stride + h * p.q_head;
    uint16_t* dst = p.q_out + (tok * p.H + h) * kLatPe;
    float x[16];
    lat_unpack8(*(const u32x4*)(src + PeCols<ADJACENT>::first(l)), x);
    lat_unpack8(*(const u32x4*)(src + PeCols<ADJACENT>::second(l)), x + 8);
    lat_turn<ADJACENT>(x, s_cs + t * kLatPairs + 8 * l);
    *(u32x4*)(dst + PeCols<ADJACENT>::first(l)) = lat_pack8(x);
    *(u32x4*)(dst + PeCols<ADJACENT>::second(l)) = lat_pack8(x + 8);
  }
}

// ---------------------------------------------------------------------------
// rows read back

struct GatherParams {
  const void* pages;
  const uint8_t* scale;
  const int32_t* page_table;
  const int32_t* start;  // nullptr: 0
  const int32_t* cu;
  uint16_t* c_out;
  uint16_t* pe_out;
  int64_t c_stride, pe_stride;
  int N, B, page_size, max_pages, num_pages, cap, block_log2, rows;
};

constexpr int kGatherRows = 32;   // most rows of a workgroup
constexpr int kGatherParts = 36;  // 16-column parts of a row

// A workgroup takes p.rows rows (8, or 32 once those fill the chip: 4000 rows of 8 bits 4.6 and
// 5.5 us, 36000 16.5 and 14.4; 16000 of bf16 9.6 and 8.6): their places first (a thread a row, the sequence by bisection
// over cu in LDS), then 16 columns a thread.
template <bool F8>
__global__ __launch_bounds__(256) void latent_gather_kernel(const GatherParams p) {
  __shared__ int s_cu[kMaxSeqs + 1];
  __shared__ int s_slot[kGatherRows];
  __shared__ float s_scale[kGatherRows];
  const int tid = threadIdx.x;
  const int r0 = (int)blockIdx.x * p.rows;
  const int nr = min(p.rows, p.N - r0);
  for (int b = tid; b <= p.B; b += 256) s_cu[b] = p.cu[b];
  __syncthreads();
  if (tid < nr) {
    const int r = r0 + tid;
    int slot = -1;  // outside every sequence: not written
    if (r >= s_cu[0] && r < s_cu[p.B]) {
      int lo = 0, hi = p.B - 1;  // the last b with cu[b] <= r
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_cu[mid] <= r) lo = mid;
        else hi = mid - 1;
      }
      const long long t = (long long)(p.start ? p.start[lo] : 0) + (r - s_cu[lo]);
      slot = -2;  // no such token: NaN
      if (t >= 0 && t < p.cap) {
        const int page = (int)t / p.page_size;
        const int pid = p.page_table[(size_t)lo * p.max_pages + page];
        if (pid >= 0 && pid < p.num_pages) {
          slot = pid * p.page_size + ((int)t - page * p.page_size);
          if (F8) {
            const uint32_t byte = p.scale[slot >> p.block_log2];
            s_scale[tid] = byte == 255 ? qnan() : ldexpf(1.f, (int)byte - 127);
          }
        }
      }
    }
    s_slot[tid] = slot;
  }
  __syncthreads();
  for (int i = tid; i < nr * kGatherParts; i += 256) {
    const int r = i / kGatherParts;
    const int part = i - r * kGatherParts;
    const int slot = s_slot[r];
    if (slot == -1) continue;
    u32x4 a, b;
    if (slot < 0) {
      a = b = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
    } else if constexpr (F8) {
      const u32x4 w = ((const u32x4*)((const uint8_t*)p.pages + (size_t)slot * kLatW))[part];
      const float s = s_scale[r];
      float x[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        const f32x2_t u = __builtin_amdgcn_cvt_pk_f32_fp8(w[e], false);
        const f32x2_t v = __builtin_amdgcn_cvt_pk_f32_fp8(w[e], true);
        x[4 * e] = u[0] * s;
        x[4 * e + 1] = u[1] * s;
        x[4 * e + 2] = v[0] * s;
        x[4 * e + 3] = v[1] * s;
      }
      a = lat_pack8(x);
      b = lat_pack8(x + 8);
    } else {
      const u32x4* src = (const u32x4*)((const uint16_t*)p.pages + (size_t)slot * kLatW);
      a = src[2 * part];
      b = src[2 * part + 1];
    }
    const size_t row = (size_t)(r0 + r);
    uint16_t* dst = part < 32 ? p.c_out + row * p.c_stride + 16 * part
                              : p.pe_out + row * p.pe_stride + 16 * (part - 32);
    *(u32x4*)dst = a;
    *(u32x4*)(dst + 8) = b;
  }
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

static int latent_pool(const char* name, const void* pages, const uint8_t* scale, int scale_block,
                       int page_size, int num_pages, int* block_log2) {
  if (!pages) return set_error(WS_EINVAL, "%s: null pointer", name);
  if (page_size <= 0 || num_pages <= 0 || (long long)num_pages * page_size > 0x7fffffffLL)
    return set_error(WS_EINVAL, "%s: bad paging page_size=%d num_pages=%d (slots are 32-bit)", name,
                     page_size, num_pages);
  if (!aligned16(pages))
    return set_error(WS_EINVAL, "%s: buffers must be 16-byte aligned", name);
  *block_log2 = 0;
  if (scale) {
    if (scale_block <= 0 || (scale_block & (scale_block - 1)) || page_size % scale_block)
      return set_error(WS_EINVAL,
                       "%s: scale_block %d must be a power of two that divides page_size %d", name,
                       scale_block, page_size);
    while ((1 << *block_log2) < scale_block) ++*block_log2;
  }
  return WS_OK;
}

}  // namespace ws

using namespace ws;

extern "C" int ws_latent_rope_append(const uint16_t* c, int64_t c_stride, const uint16_t* pe,
                                     int64_t pe_stride, const uint16_t* q_pe, int64_t q_stride,
                                     int64_t q_head_stride, const int32_t* positions,
                                     const float* inv_freq, int adjacent, float factor,
                                     const void* norm_weight, int weight_f32, float eps,
                                     const int32_t* slots, uint16_t* q_out, void* latent_pages,
                                     uint8_t* latent_scale, int scale_block, int N, int H,
                                     int page_size, int num_pages, void* stream) {
  static const char* name = "ws_latent_rope_append";
  if (!c || !pe || !q_pe || !positions || !inv_freq || !slots || !q_out)
    return set_error(WS_EINVAL, "%s: null pointer", name);
  LatentParams p{};
  if (int rc = latent_pool(name, latent_pages, latent_scale, scale_block, page_size, num_pages,
                           &p.block_log2))
    return rc;
  if (N < 0 || H <= 0 || H > 1024)
    return set_error(WS_EINVAL, "%s: bad sizes N=%d H=%d (H <= 1024)", name, N, H);
  if (c_stride < kLatC || pe_stride < kLatPe || q_head_stride < kLatPe ||
      q_stride < (H - 1) * q_head_stride + kLatPe || c_stride % 8 || pe_stride % 8 || q_stride % 8 ||
      q_head_stride % 8)
    return set_error(WS_EINVAL, "%s: bad strides c=%lld pe=%lld q=%lld head=%lld", name,
                     (long long)c_stride, (long long)pe_stride, (long long)q_stride,
                     (long long)q_head_stride);
  if (!aligned16(c) || !aligned16(pe) || !aligned16(q_pe) || !aligned16(q_out) ||
      !aligned16(norm_weight))
    return set_error(WS_EINVAL, "%s: buffers must be 16-byte aligned", name);
  if (!(eps >= 0.f && eps < __builtin_inff()))
    return set_error(WS_EINVAL, "%s: eps must be finite and >= 0", name);
  if (N == 0) return WS_OK;
  p.c = c;
  p.c_stride = c_stride;
  p.pe = pe;
  p.pe_stride = pe_stride;
  p.q = q_pe;
  p.q_stride = q_stride;
  p.q_head = q_head_stride;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.weight = norm_weight;
  p.weight_f32 = weight_f32 != 0;
  p.eps = eps;
  p.factor = factor;
  p.slots = slots;
  p.q_out = q_out;
  p.pages = latent_pages;
  p.scale = latent_scale;
  p.N = N;
  p.H = H;
  p.num_slots = num_pages * page_size;
  // A token a workgroup while there are few, four (with runs: eight) once those fill the chip
  // (1024 tokens, 16 heads: 4.1 and 4.2 us, 4096: 8.0 and 7.4, with runs 18.6 and 12.9; 1024
  // tokens of 128 heads: 8.6 and 10.5).
  const bool runs = latent_scale && p.block_log2 > 0;
  p.tokens = N < 2048 ? 1 : runs ? kRunTurns : kLatTokens;
  const long long n = N;  // (sums past 32 bits)
  p.window = (int)std::min<long long>((n + kRunGroups - 1) / kRunGroups,
                                      p.block_log2 >= 5 ? 2 * kRunWindow : kRunWindow);
  p.run_groups = runs ? (int)((n + p.window - 1) / p.window) : 0;
  const long long grid = (n + p.tokens - 1) / p.tokens + p.run_groups;
  const int threads = runs ? 64 * kRunWaves : 256;
  if (grid * threads >= (1LL << 32))
    return set_error(WS_EINVAL, "%s: %d tokens exceed the launch grid", name, N);
  const auto kernel = runs ? (adjacent ? latent_append_kernel<true, true> : latent_append_kernel<false, true>)
                           : (adjacent ? latent_append_kernel<true, false> : latent_append_kernel<false, false>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3((unsigned)threads), 0, (hipStream_t)stream, p);
  return check_launch(name);
}

extern "C" int ws_latent_gather(const void* latent_pages, const uint8_t* latent_scale,
                                int scale_block, const int32_t* page_table, const int32_t* start,
                                const int32_t* cu_rows, uint16_t* c_out, int64_t c_stride,
                                uint16_t* pe_out, int64_t pe_stride, int N, int B, int page_size,
                                int max_pages, int num_pages, void* stream) {
  static const char* name = "ws_latent_gather";
  if (!page_table || !cu_rows || !c_out || !pe_out)
    return set_error(WS_EINVAL, "%s: null pointer", name);
  GatherParams p{};
  if (int rc = latent_pool(name, latent_pages, latent_scale, scale_block, page_size, num_pages,
                           &p.block_log2))
    return rc;
  if (N < 0 || B < 0 || B > kMaxSeqs || max_pages <= 0)
    return set_error(WS_EINVAL, "%s: bad sizes N=%d B=%d max_pages=%d (B <= %d)", name, N, B,
                     max_pages, kMaxSeqs);
  if (c_stride < kLatC || pe_stride < kLatPe || c_stride % 8 || pe_stride % 8 || !aligned16(c_out) ||
      !aligned16(pe_out))
    return set_error(WS_EINVAL, "%s: rows must be 16-byte aligned (strides c=%lld pe=%lld)", name,
                     (long long)c_stride, (long long)pe_stride);
  if (N == 0 || B == 0) return WS_OK;
  p.pages = latent_pages;
  p.scale = latent_scale;
  p.page_table = page_table;
  p.start = start;
  p.cu = cu_rows;
  p.c_out = c_out;
  p.pe_out = pe_out;
  p.c_stride = c_stride;
  p.pe_stride = pe_stride;
  p.N = N;
  p.B = B;
  p.page_size = page_size;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.cap = (int)std::min<long long>((long long)page_size * max_pages, 0x7fffffffLL);
  p.rows = N >= 8192 ? kGatherRows : 8;
  const long long groups = ((long long)N + p.rows - 1) / p.rows;
  if (groups * 256 >= (1LL << 32))
    return set_error(WS_EINVAL, "%s: %d rows exceed the launch grid", name, N);
  const dim3 g((unsigned)groups), b(256);
  hipStream_t s = (hipStream_t)stream;
  if (latent_scale)
    hipLaunchKernelGGL(latent_gather_kernel<true>, g, b, 0, s, p);
  else
    hipLaunchKernelGGL(latent_gather_kernel<false>, g, b, 0, s, p);
  return check_launch(name);
}
