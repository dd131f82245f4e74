// Pages and slots of a ragged batch, handed out on the GPU from the request
// lengths: no host round trip between the lengths of a step and its launches.
//
// The free pages are a stack: stack[0 .. free_in[0]) are free, the top first.
// pages_extend gives every sequence the pages its n_new tokens need beyond
// those its len_in tokens hold, in the order of the sequences (an exclusive
// prefix sum over the needs), so the result depends on the inputs alone.
// pages_release pushes the pages of ended sequences back.
//
// The work is a few integers per sequence and per token: a launch costs more
// than the data.  So each is one launch: every workgroup scans the whole batch
// by itself (at most 2048 sequences, eight a thread, 64-bit sums: no order of
// workgroups, no second pass), keeps the prefix in LDS and then writes its share
// of the tokens, one thread a token, which finds its sequence by bisection.  A
// token that opens a page also writes the page's table entry: no other thread
// reads it, the others take the id from the stack as well.  16 sequences of one token
// take 3.0 to 3.2 us, 512 with 113981 tokens 9.6, the release of 37 sequences 3.5 to 3.7.
#include "ws_common.h"
#include "ws_plan.h"

namespace ws {

constexpr int kPagesThreads = 256;
constexpr int kPagesSeqs = kMaxSeqs / kPagesThreads;  // sequences of a thread
constexpr int kPagesTokens = 4;                       // tokens of a thread
constexpr long long kMaxTokens = 1LL << 30;

// Wave-wide and workgroup-wide inclusive sums of two 64-bit values.
struct Pair64 {
  long long a, b;
};
__device__ __forceinline__ Pair64 wave_scan(Pair64 v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long a = __shfl_up(v.a, o);
    const long long b = __shfl_up(v.b, o);
    if (lane >= o) {
      v.a += a;
      v.b += b;
    }
  }
  return v;
}
// Exclusive sums of v over the workgroup's threads; `total` over all of them.
__device__ __forceinline__ Pair64 block_scan(Pair64 v, Pair64& total) {
  constexpr int W = kPagesThreads / 64;
  __shared__ Pair64 s_wave[W];
  const int w = threadIdx.x >> 6;
  const Pair64 in = wave_scan(v);
  if ((threadIdx.x & 63) == 63) s_wave[w] = in;
  __syncthreads();
  Pair64 x{in.a - v.a, in.b - v.b};
  total = Pair64{0, 0};
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const Pair64 t = s_wave[i];
    if (i < w) {
      x.a += t.a;
      x.b += t.b;
    }
    total.a += t.a;
    total.b += t.b;
  }
  return x;
}

// Pages of `tokens` tokens (both at most 2^30).
__device__ __forceinline__ int pages_of(int tokens, int page_size) {
  return (int)(((unsigned)tokens + (unsigned)page_size - 1) / (unsigned)page_size);
}

struct ExtendParams {
  int32_t* page_table;
  const int32_t* len_in;
  const int32_t* n_new;
  const int32_t* stack;
  const int32_t* free_in;
  const int32_t* pos_base;  // or null
  int32_t* len_out;
  int32_t* cu_new;
  int32_t* positions;
  int32_t* slots;
  int32_t* free_out;
  int B, max_pages, num_pages, stack_size, page_size, n_tokens;
};

__global__ __launch_bounds__(kPagesThreads) void pages_extend_kernel(const ExtendParams p) {
  // sequence b: first token, length before, and the stack place of its first new
  // page (kNone: the sequence gets nothing)
  constexpr int kNone = -2;
  __shared__ int s_cu[kMaxSeqs + 1];
  __shared__ int s_len[kMaxSeqs];
  __shared__ int s_top[kMaxSeqs];
  __shared__ int s_used;
  const int tid = threadIdx.x;
  const bool lead = blockIdx.x == 0;
  const long long cap = (long long)p.page_size * p.max_pages;
  const int free_n = min(max(p.free_in[0], 0), p.stack_size);
  if (tid == 0) s_used = 0;
  int len[kPagesSeqs], n[kPagesSeqs], need[kPagesSeqs];
  Pair64 sum{0, 0};
  const int per = (p.B + kPagesThreads - 1) / kPagesThreads;
  const int b0 = tid * per;
#pragma unroll
  for (int k = 0; k < kPagesSeqs; ++k) {
    const int b = b0 + k;
    len[k] = n[k] = need[k] = 0;
    if (k >= per || b >= p.B) continue;
    len[k] = p.len_in[b];
    n[k] = p.n_new[b];
    if (len[k] >= 0 && n[k] >= 0 && (long long)len[k] + n[k] <= cap)  // (cap <= 2^30)
      need[k] = pages_of(len[k] + n[k], p.page_size) - pages_of(len[k], p.page_size);
    sum.a += max(n[k], 0);
    sum.b += need[k];
  }
  Pair64 total;
  Pair64 at = block_scan(sum, total);  // (its barrier also orders s_used = 0)
#pragma unroll
  for (int k = 0; k < kPagesSeqs; ++k) {
    const int b = b0 + k;
    if (k >= per || b >= p.B) continue;
    const long long end = at.a + max(n[k], 0);
    const bool ok = len[k] >= 0 && n[k] >= 0 && (long long)len[k] + n[k] <= cap &&
                    end <= p.n_tokens && (need[k] == 0 || at.b + need[k] <= free_n);
    s_cu[b] = (int)min(at.a, (long long)p.n_tokens);
    s_len[b] = len[k];
    s_top[b] = ok ? free_n - 1 - (int)min(at.b, (long long)free_n) : kNone;
    if (lead) {
      p.cu_new[b] = (int)min(at.a, (long long)p.n_tokens);
      p.len_out[b] = ok ? len[k] + n[k] : -1;
      // the needs' sums grow with b, so what is taken is the last success's
      if (ok && need[k] > 0) atomicMax(&s_used, (int)(at.b + need[k]));
    }
    at.a = end;
    at.b += need[k];
  }
  if (tid == 0) {
    const int all = (int)min(total.a, (long long)p.n_tokens);
    s_cu[p.B] = all;
    if (lead) p.cu_new[p.B] = all;
  }
  __syncthreads();
  if (lead && tid == 0) p.free_out[0] = free_n - s_used;

  const long long t0 = (long long)blockIdx.x * (kPagesThreads * kPagesTokens) + tid;
#pragma unroll
  for (int u = 0; u < kPagesTokens; ++u) {
    const long long t = t0 + u * kPagesThreads;
    if (t >= p.n_tokens) break;
    int lo = 0, hi = p.B;  // the last b with s_cu[b] <= t (B: past every token)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_cu[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    int position = 0, slot = -1;
    if (lo < p.B && s_top[lo] != kNone) {
      const int len0 = s_len[lo];
      const int pos = len0 + (int)(t - s_cu[lo]);
      const int page = (int)((unsigned)pos / (unsigned)p.page_size);
      const int off = pos - page * p.page_size;
      const int have = pages_of(len0, p.page_size);
      int32_t* entry = p.page_table + (size_t)lo * p.max_pages + page;
      int pid;
      if (page >= have) {
        pid = p.stack[s_top[lo] - (page - have)];
        if (off == 0) *entry = pid;
      } else {
        pid = *entry;
      }
      if (pid >= 0 && pid < p.num_pages) slot = pid * p.page_size + off;
      position = pos + (p.pos_base ? p.pos_base[lo] : 0);
    }
    p.positions[t] = position;
    p.slots[t] = slot;
  }
}

__global__ __launch_bounds__(kPagesThreads) void pages_release_kernel(
    const int32_t* __restrict__ page_table, const int32_t* __restrict__ len_in,
    const uint8_t* __restrict__ done, int32_t* __restrict__ stack,
    const int32_t* __restrict__ free_in, int32_t* __restrict__ len_out,
    int32_t* __restrict__ free_out, int B, int max_pages, int stack_size, int page_size) {
  __shared__ int s_at[kMaxSeqs];    // stack place of the sequence's first page
  __shared__ int s_held[kMaxSeqs];  // and how many it gives back
  const int tid = threadIdx.x;
  const int free_n = min(max(free_in[0], 0), stack_size);
  int held[kPagesSeqs];
  Pair64 sum{0, 0};
  const int per = (B + kPagesThreads - 1) / kPagesThreads;
  const int b0 = tid * per;
#pragma unroll
  for (int k = 0; k < kPagesSeqs; ++k) {
    const int b = b0 + k;
    held[k] = 0;
    if (k >= per || b >= B) continue;
    const int len = len_in[b];
    const bool end = done[b] != 0;
    if (end && len > 0)
      held[k] = min((int)(((unsigned)len - 1) / (unsigned)page_size) + 1, max_pages);
    if (blockIdx.x == 0) len_out[b] = end ? 0 : len;
    sum.a += held[k];
  }
  Pair64 total;
  Pair64 at = block_scan(sum, total);
#pragma unroll
  for (int k = 0; k < kPagesSeqs; ++k) {
    const int b = b0 + k;
    if (k >= per || b >= B) continue;
    s_at[b] = (int)min(free_n + at.a, (long long)stack_size);
    s_held[b] = held[k];
    at.a += held[k];
  }
  if (blockIdx.x == 0 && tid == 0)
    free_out[0] = (int)min(free_n + total.a, (long long)stack_size);
  __syncthreads();
  for (int b = blockIdx.x; b < B; b += gridDim.x) {
    const int n = min(s_held[b], stack_size - s_at[b]);
    for (int i = tid; i < n; i += kPagesThreads)
      stack[s_at[b] + i] = page_table[(size_t)b * max_pages + i];
  }
}

static int pages_sizes(const char* name, int B, int max_pages, int stack_size, int page_size) {
  if (B < 0 || B > kMaxSeqs || max_pages <= 0 || stack_size < 0 || page_size <= 0 ||
      (long long)page_size * max_pages > kMaxTokens)
    return set_error(WS_EINVAL,
                     "%s: bad sizes B=%d max_pages=%d stack_size=%d page_size=%d (B <= %d, "
                     "page_size * max_pages <= 2^30)",
                     name, B, max_pages, stack_size, page_size, kMaxSeqs);
  return WS_OK;
}

}  // namespace ws

using namespace ws;

extern "C" int ws_pages_extend(int32_t* page_table, const int32_t* len_in, const int32_t* n_new,
                               const int32_t* stack, const int32_t* free_in,
                               const int32_t* pos_base, int32_t* len_out, int32_t* cu_new,
                               int32_t* positions, int32_t* slots, int32_t* free_out, int B,
                               int max_pages, int num_pages, int stack_size, int page_size,
                               int n_tokens, void* stream) {
  static const char* name = "ws_pages_extend";
  if ((B > 0 && (!page_table || !len_in || !n_new || !len_out)) || !free_in || !free_out ||
      !cu_new || (stack_size > 0 && !stack) || (n_tokens > 0 && (!positions || !slots)))
    return set_error(WS_EINVAL, "%s: null pointer", name);
  if (int rc = pages_sizes(name, B, max_pages, stack_size, page_size)) return rc;
  if (num_pages < 0 || (long long)num_pages * page_size > 0x7fffffffLL || n_tokens < 0 ||
      n_tokens > kMaxTokens)
    return set_error(WS_EINVAL,
                     "%s: bad sizes num_pages=%d page_size=%d n_tokens=%d (slots are 32-bit)",
                     name, num_pages, page_size, n_tokens);
  if (free_out == free_in || (B > 0 && (len_out == len_in || len_out == n_new)))
    return set_error(WS_EINVAL, "%s: len_out / free_out must not alias their inputs", name);
  const ExtendParams prm = {page_table, len_in, n_new, stack, free_in, pos_base, len_out, cu_new,
                            positions, slots, free_out, B, max_pages, num_pages, stack_size,
                            page_size, n_tokens};
  const int per = kPagesThreads * kPagesTokens;
  const int grid = n_tokens > 0 ? (n_tokens + per - 1) / per : 1;
  hipLaunchKernelGGL(pages_extend_kernel, dim3(grid), dim3(kPagesThreads), 0, (hipStream_t)stream,
                     prm);
  return check_launch(name);
}

extern "C" int ws_pages_release(const int32_t* page_table, const int32_t* len_in,
                                const uint8_t* done, int32_t* stack, const int32_t* free_in,
                                int32_t* len_out, int32_t* free_out, int B, int max_pages,
                                int stack_size, int page_size, void* stream) {
  static const char* name = "ws_pages_release";
  if ((B > 0 && (!page_table || !len_in || !done || !len_out)) || !free_in || !free_out ||
      (stack_size > 0 && !stack))
    return set_error(WS_EINVAL, "%s: null pointer", name);
  if (int rc = pages_sizes(name, B, max_pages, stack_size, page_size)) return rc;
  if (free_out == free_in || (B > 0 && len_out == len_in))
    return set_error(WS_EINVAL, "%s: len_out / free_out must not alias their inputs", name);
  hipLaunchKernelGGL(pages_release_kernel, dim3(B < 1 ? 1 : (B < 256 ? B : 256)),
                     dim3(kPagesThreads), 0, (hipStream_t)stream, page_table, len_in, done, stack,
                     free_in, len_out, free_out, B, max_pages, stack_size, page_size);
  return check_launch(name);
}
