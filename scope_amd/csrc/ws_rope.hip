// Rotary positions with several axes, and the write of the rotated keys and the
// values into the pages (gfx950).
//
// Pair i of a head's R / 2 rotary pairs turns by the angle
//   a = position[axis(i)][token] * inv_freq[i]
//   (x, y) -> f (x cos a - y sin a, y cos a + x sin a)
// where (x, y) are columns (i, i + R / 2), or (2 i, 2 i + 1) with adjacent pairs;
// columns >= R pass.  Text has one axis; images and video give time, height and
// width a share of the pairs each.
//
// The angle is reduced in 64 bits: position * inv_freq reaches 1e5 radians,
// where 32 bits are off by 4e-3, half a step of the bf16 result.  One value per
// (token, pair), shared by all heads through LDS, so it costs nothing beside the
// heads' traffic.
//
// The bound is HBM (q, k, v read once, q and the pages written once).  A lane
// holds 16 columns of a head row, the pairs' both halves among them, as two
// 16-byte loads; a row takes D / 16 lanes (rounded up to a power of two, so that
// the 8-bit write finds the row's maximum with lane exchanges).  16637 tokens of
// 32 + 4 + 4 heads of 128 columns (341 MB) take 66.6 to 67.1 us, 5.1 TB/s, as a large
// copy does; 3765 tokens of 24 + 8 + 8 heads of 96 into 8-bit pages 12.2 to 12.5 us (4.3
// TB/s); a step of 32 tokens 4.4 us.
//
// 8-bit pages hold e4m3 values with one power-of-two scale (e8m0 byte) per
// token and KV head: 2^e, e the least with max|x| <= 448 * 2^e.  A power of
// two costs no precision in a floating format (only range below 2^-9 of the
// row's maximum), the product is exact both ways, and the value times its scale
// is a bf16 number.
#include <math.h>

#include "ws_common.h"

namespace ws {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxPairs = 128;
constexpr int kRopeTokens = 4;  // most tokens of a workgroup

struct RopeParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_stride, k_stride, v_stride;  // elements from token to token
  const int32_t* positions;              // [axes][N]
  const float* inv_freq;
  uint32_t axis[kRopeMaxPairs / 16];  // two bits a pair
  uint16_t* q_out;                    // [N][Hq][D]
  uint16_t* k_out;                    // [N][Hkv][D] (no pages)
  const int32_t* slots;
  void* k_pages;
  void* v_pages;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int N, Hq, Hkv, D, rot, page_size, num_slots;
  int lanes_log2;  // lanes of a head row
  float factor;
};

enum RopeTo { kToRows, kToBf16Pages, kToFp8Pages };

__device__ __forceinline__ void unpack8(const u32x4& w, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __builtin_bit_cast(float, w[i] << 16);
    x[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ u32x4 pack8(const float* x) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  return w;
}
// Eight values times s as e4m3, rounded to nearest even (|x s| <= 448).
__device__ __forceinline__ uint2 pack8_e4m3(const float* x, float s) {
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * s, x[1] * s, 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * s, x[3] * s, lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * s, x[5] * s, 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] * s, x[7] * s, hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// The e8m0 byte of a row whose largest magnitude has the bits `top`: 127 + e, e
// the least with top <= 1.75 * 2^(8 + e); 127 for a row of zeros, 255 (NaN) for
// one with an infinity or a NaN.
__device__ __forceinline__ int e8m0_of(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  if (top == 0) return 127;
  return max((int)((top + 0x1fffffu) >> 23) - 8, 1);
}

template <bool ADJACENT, RopeTo TO>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const RopeParams p, int tokens) {
  __shared__ float2 s_cs[kRopeTokens * kRopeMaxPairs];
  const int tid = threadIdx.x;
  const int half = p.rot >> 1;
  const long long t0 = (long long)blockIdx.x * tokens;
  const int nt = (int)min((long long)tokens, p.N - t0);
  for (int i = tid; i < nt * half; i += kRopeThreads) {
    const int t = i / half;
    const int pr = i - t * half;
    const int ax = (p.axis[pr >> 4] >> (2 * (pr & 15))) & 3;
    const double turns = (double)p.positions[(size_t)ax * p.N + t0 + t] *
                         ((double)p.inv_freq[pr] * 0.15915494309189535);
    const float f = (float)(2.0 * (turns - rint(turns)));
    float sn, cs;
    sincospif(f, &sn, &cs);
    s_cs[t * half + pr] = make_float2(cs * p.factor, sn * p.factor);
  }
  __syncthreads();
  const int j = tid & ((1 << p.lanes_log2) - 1);  // 16 columns of the row
  const int per = kRopeThreads >> p.lanes_log2;   // rows at a time
  const bool on = 16 * j < p.D;
  const int heads = p.Hq + p.Hkv + (TO == kToRows ? 0 : p.Hkv);
  const bool turn = 16 * j < p.rot;
  // first columns of the lane's two 8-column halves
  const int c0 = turn && !ADJACENT ? 8 * j : 16 * j;
  const int c1 = turn && !ADJACENT ? half + 8 * j : 16 * j + 8;
  for (int r = tid >> p.lanes_log2; r < nt * heads; r += per) {
    const int t = r / heads;
    int h = r - t * heads;
    const size_t tok = (size_t)(t0 + t);
    const bool is_q = h < p.Hq;
    const bool is_v = h >= p.Hq + p.Hkv;
    if (!is_q) h -= is_v ? p.Hq + p.Hkv : p.Hq;
    const uint16_t* src =
        (is_q ? p.q + tok * p.q_stride : is_v ? p.v + tok * p.v_stride : p.k + tok * p.k_stride) +
        (size_t)h * p.D;
    u32x4 wa = {0, 0, 0, 0}, wb = {0, 0, 0, 0};
    if (on) {
      wa = *(const u32x4*)(src + c0);
      wb = *(const u32x4*)(src + c1);
    }
    float x[16];
    unpack8(wa, x);
    unpack8(wb, x + 8);
    if (turn && !is_v) {
      const float2* cs = s_cs + t * half + 8 * j;
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
    if (is_q || TO == kToRows) {
      uint16_t* dst = is_q ? p.q_out + (tok * p.Hq + h) * p.D : p.k_out + (tok * p.Hkv + h) * p.D;
      if (on) {
        *(u32x4*)(dst + c0) = pack8(x);
        *(u32x4*)(dst + c1) = pack8(x + 8);
      }
      continue;
    }
    const int slot = p.slots[tok];
    const bool put = slot >= 0 && slot < p.num_slots;
    const int page = put ? slot / p.page_size : 0;
    const size_t row = ((size_t)page * p.Hkv + h) * p.page_size + (put ? slot - page * p.page_size : 0);
    if (TO == kToBf16Pages) {
      uint16_t* dst = (uint16_t*)(is_v ? p.v_pages : p.k_pages) + row * p.D;
      if (on && put) {
        *(u32x4*)(dst + c0) = pack8(x);
        *(u32x4*)(dst + c1) = pack8(x + 8);
      }
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        top = max(top, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
      for (int o = 1; o < (1 << p.lanes_log2); o <<= 1)
        top = max(top, (uint32_t)__shfl_xor((int)top, o));
      const int byte = e8m0_of(top);
      // 2^(127 - byte) (bytes 1 to 247)
      const float s = byte == 255 ? qnan() : ldexpf(1.f, 127 - byte);
      uint8_t* dst = (uint8_t*)(is_v ? p.v_pages : p.k_pages) + row * p.D;
      if (on && put) {
        *(uint2*)(dst + c0) = pack8_e4m3(x, s);
        *(uint2*)(dst + c1) = pack8_e4m3(x + 8, s);
        if (j == 0) (is_v ? p.v_scale : p.k_scale)[row] = (uint8_t)byte;
      }
    }
  }
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Tokens of a workgroup: one while there are few (a decode step's tokens spread
// over the chip), four once those fill it (one angle per thread at 64 pairs).
static int rope_tokens(int N) { return N >= 2048 ? kRopeTokens : 1; }

template <RopeTo TO>
static void rope_launch(const RopeParams& p, bool adjacent, hipStream_t s) {
  const int tokens = rope_tokens(p.N);
  const dim3 grid((unsigned)((p.N + tokens - 1) / tokens)), block(kRopeThreads);
  if (adjacent)
    hipLaunchKernelGGL((rope_kernel<true, TO>), grid, block, 0, s, p, tokens);
  else
    hipLaunchKernelGGL((rope_kernel<false, TO>), grid, block, 0, s, p, tokens);
}

static int rope_fill(RopeParams& p, const char* name, const uint16_t* q, int64_t q_stride,
                     const uint16_t* k, int64_t k_stride, const int32_t* positions, int axes,
                     const float* inv_freq, const uint8_t* pair_axis, float factor,
                     uint16_t* q_out, int N, int Hq, int Hkv, int D, int rot) {
  if (!q || !k || !positions || !inv_freq || !q_out)
    return set_error(WS_EINVAL, "%s: null pointer", name);
  if (N < 0 || Hq <= 0 || Hkv <= 0 || D < 16 || D > 256 || D % 16 || rot < 16 || rot > D ||
      rot % 16 || axes < 1 || axes > 4)
    return set_error(WS_EINVAL,
                     "%s: bad sizes N=%d Hq=%d Hkv=%d D=%d rot=%d axes=%d (D and rot multiples "
                     "of 16, rot <= D <= 256, up to 4 axes)",
                     name, N, Hq, Hkv, D, rot, axes);
  if (q_stride < (int64_t)Hq * D || k_stride < (int64_t)Hkv * D || q_stride % 8 || k_stride % 8)
    return set_error(WS_EINVAL, "%s: bad token strides q=%lld k=%lld", name, (long long)q_stride,
                     (long long)k_stride);
  if (!aligned16(q) || !aligned16(k) || !aligned16(q_out))
    return set_error(WS_EINVAL, "%s: bf16 buffers must be 16-byte aligned", name);
  p = RopeParams{};
  for (int i = 0; i < rot / 2; ++i) {
    const int a = pair_axis ? pair_axis[i] : 0;
    if (a >= axes) return set_error(WS_EINVAL, "%s: pair %d on axis %d of %d", name, i, a, axes);
    p.axis[i >> 4] |= (uint32_t)a << (2 * (i & 15));
  }
  p.q = q;
  p.k = k;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.q_out = q_out;
  p.N = N;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.D = D;
  p.rot = rot;
  p.factor = factor;
  while ((16 << p.lanes_log2) < D) ++p.lanes_log2;
  return WS_OK;
}

}  // namespace ws

using namespace ws;

extern "C" int ws_rope(const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride,
                       const int32_t* positions, int axes, const float* inv_freq,
                       const uint8_t* pair_axis, int adjacent, float factor, uint16_t* q_out,
                       uint16_t* k_out, int N, int Hq, int Hkv, int D, int rot, void* stream) {
  static const char* name = "ws_rope";
  RopeParams p;
  if (int rc = rope_fill(p, name, q, q_stride, k, k_stride, positions, axes, inv_freq, pair_axis,
                         factor, q_out, N, Hq, Hkv, D, rot))
    return rc;
  if (!k_out) return set_error(WS_EINVAL, "%s: null pointer", name);
  if (!aligned16(k_out))
    return set_error(WS_EINVAL, "%s: bf16 buffers must be 16-byte aligned", name);
  if (N == 0) return WS_OK;
  p.k_out = k_out;
  rope_launch<kToRows>(p, adjacent != 0, (hipStream_t)stream);
  return check_launch(name);
}

extern "C" int ws_rope_append(const uint16_t* q, int64_t q_stride, const uint16_t* k,
                              int64_t k_stride, const uint16_t* v, int64_t v_stride,
                              const int32_t* positions, int axes, const float* inv_freq,
                              const uint8_t* pair_axis, int adjacent, float factor,
                              const int32_t* slots, uint16_t* q_out, void* k_pages, void* v_pages,
                              uint8_t* k_scale, uint8_t* v_scale, int N, int Hq, int Hkv, int D,
                              int rot, int page_size, int num_pages, void* stream) {
  static const char* name = "ws_rope_append";
  RopeParams p;
  if (int rc = rope_fill(p, name, q, q_stride, k, k_stride, positions, axes, inv_freq, pair_axis,
                         factor, q_out, N, Hq, Hkv, D, rot))
    return rc;
  if (!v || !slots || !k_pages || !v_pages || (k_scale == nullptr) != (v_scale == nullptr))
    return set_error(WS_EINVAL, "%s: null pointer", name);
  if (v_stride < (int64_t)Hkv * D || v_stride % 8)
    return set_error(WS_EINVAL, "%s: bad token stride v=%lld", name, (long long)v_stride);
  if (page_size <= 0 || num_pages <= 0 || (long long)num_pages * page_size > 0x7fffffffLL)
    return set_error(WS_EINVAL, "%s: bad paging page_size=%d num_pages=%d (slots are 32-bit)",
                     name, page_size, num_pages);
  if (!aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages))
    return set_error(WS_EINVAL, "%s: buffers must be 16-byte aligned", name);
  if (N == 0) return WS_OK;
  p.v = v;
  p.v_stride = v_stride;
  p.slots = slots;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.page_size = page_size;
  p.num_slots = num_pages * page_size;
  if (k_scale)
    rope_launch<kToFp8Pages>(p, adjacent != 0, (hipStream_t)stream);
  else
    rope_launch<kToBf16Pages>(p, adjacent != 0, (hipStream_t)stream);
  return check_launch(name);
}
