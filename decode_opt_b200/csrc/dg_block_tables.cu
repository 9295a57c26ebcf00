// SPDX-License-Identifier: MIT
//
// dg_block_tables.cu -- the paged cache's bookkeeping of one step, built on
// the GPU from the requests' lengths (include/decode_attention_b200.h gives
// the definition).
//
// Two exclusive sums over the requests (new tokens, new pages) and then one
// independent answer per token and per new page.  One launch: every CTA makes
// the sums for itself in shared memory (two loads per request from L2, one
// block scan) instead of waiting for another kernel or CTA, and then answers
// for its share of the tokens and pages.  A token finds its request by
// bisection in shared memory; a thread answers for four consecutive tokens,
// so that the 16 bytes a token costs leave in 16-byte stores.  A slot never
// waits for the table entry that the same launch writes: a page below
// ceil(c / P) is read from the table, a later one from the free list itself.
//
// Bound: a handful of dependent loads for a decode step (latency), the 16
// bytes a token at the other end.

#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "decode_attention_b200.h"
#include "decode_gemm_b200.h"
#include "sm100.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBatch = 16384;
constexpr int kTokensPerThread = 4;

struct Sums {
  long long tokens, pages;
};

__device__ __forceinline__ void report(int* status, int code) {
  if (status != nullptr) atomicCAS(status, 0, code);
}

// The request's lengths and pages, made safe: negative lengths count as 0,
// c + n stays within an int, pages stay within the table row.
struct Request {
  int c, n, held, need;   // cached, new; pages owned and pages owned after the step
  int code;               // status code, 0 if nothing had to be changed
};

__device__ __forceinline__ Request request_of(const dg_block_tables& a, int b) {
  Request r;
  r.code = 0;
  r.c = a.context_lens[b];
  r.n = a.new_lens[b];
  if (r.c < 0 || r.n < 0 || r.n > INT_MAX - max(r.c, 0)) {
    r.code = DG_ERR_LENGTH;
    r.c = max(r.c, 0);
    r.n = min(max(r.n, 0), INT_MAX - r.c);
  }
  const unsigned p = static_cast<unsigned>(a.page_size);
  r.held = static_cast<int>((static_cast<unsigned>(r.c) + p - 1u) / p);
  r.need = static_cast<int>((static_cast<unsigned>(r.c) + static_cast<unsigned>(r.n) + p - 1u) / p);
  if (r.need > a.table_width) {
    r.code = DG_ERR_TABLE_WIDTH;
    r.need = a.table_width;
    r.held = min(r.held, r.need);
  }
  return r;
}

__device__ __forceinline__ int clamp_int(long long v) {
  return v > INT_MAX ? INT_MAX : static_cast<int>(v);
}

// The last index i of starts[0 .. n) with starts[i] <= v (starts[0] = 0 <= v).
// Requests without tokens (or pages) share a start with the next; the last of
// them is the one that holds v.
__device__ __forceinline__ int owner_of(const int* starts, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) block_tables_kernel(const __grid_constant__ dg_block_tables a) {
  extern __shared__ int smem[];
  int* token_start = smem;                 // [batch + 1]
  int* page_start = smem + a.batch + 1;    // [batch + 1]
  __shared__ Sums warp_sum[kWarps];

  dg::sm100::griddep_launch_dependents();
  dg::sm100::griddep_wait();

  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const bool first_cta = blockIdx.x == 0;

  // Exclusive sums: each thread takes `per` consecutive requests.
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  Sums mine{0, 0};
  for (int b = b0; b < b1; ++b) {
    const Request r = request_of(a, b);
    mine.tokens += r.n;
    mine.pages += r.need - r.held;
    if (first_cta) {
      a.seq_lens[b] = r.c + r.n;
      if (r.code != 0) report(a.status, r.code);
    }
  }
  Sums scan = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, scan.tokens, off);
    const long long p = __shfl_up_sync(0xffffffffu, scan.pages, off);
    if (lane >= off) {
      scan.tokens += t;
      scan.pages += p;
    }
  }
  if (lane == 31) warp_sum[warp] = scan;
  __syncthreads();
  Sums before{scan.tokens - mine.tokens, scan.pages - mine.pages};
  for (int w = 0; w < warp; ++w) {
    before.tokens += warp_sum[w].tokens;
    before.pages += warp_sum[w].pages;
  }
  for (int b = b0; b < b1; ++b) {
    const Request r = request_of(a, b);
    token_start[b] = clamp_int(before.tokens);
    page_start[b] = clamp_int(before.pages);
    if (first_cta) a.query_start[b] = clamp_int(before.tokens);
    before.tokens += r.n;
    before.pages += r.need - r.held;
  }
  if (tid == kThreads - 1) {               // its `before` is now the total
    token_start[a.batch] = clamp_int(before.tokens);
    page_start[a.batch] = clamp_int(before.pages);
    if (first_cta) {
      a.query_start[a.batch] = clamp_int(before.tokens);
      if (before.tokens > INT_MAX || before.pages > INT_MAX) report(a.status, DG_ERR_LENGTH);
      if (before.tokens > a.num_tokens) report(a.status, DG_ERR_TOKENS);
    }
  }
  __syncthreads();

  const int cursor = a.cursor_in != nullptr ? min(max(a.cursor_in[0], 0), a.free_count) : 0;
  const int pages = page_start[a.batch];
  const int available = a.free_count - cursor;
  if (first_cta && tid == 0) {
    a.cursor_out[0] = cursor + min(pages, available);
    if (pages > available) report(a.status, DG_ERR_POOL);
  }

  const long long stride = static_cast<long long>(gridDim.x) * kThreads;
  const long long me = static_cast<long long>(blockIdx.x) * kThreads + tid;

  // New table entries.
  for (long long g = me; g < pages; g += stride) {
    const int page = static_cast<int>(g);
    const int b = owner_of(page_start, a.batch, page);
    const Request r = request_of(a, b);
    a.block_table[static_cast<long long>(b) * a.table_stride + r.held + (page - page_start[b])] =
        page < available ? a.free_pages[cursor + page] : -1;
  }

  // Tokens.
  const int total = token_start[a.batch];
  for (long long g = me * kTokensPerThread; g < a.num_tokens; g += stride * kTokensPerThread) {
    long long slot[kTokensPerThread];
    int position[kTokensPerThread], request[kTokensPerThread];
    int b = -1, next = -1;                 // the request of the token before, and where the next one begins
    Request r{};
#pragma unroll
    for (int i = 0; i < kTokensPerThread; ++i) {
      const long long t64 = g + i;
      slot[i] = -1;
      position[i] = 0;
      request[i] = -1;
      if (t64 >= total) continue;
      const int t = static_cast<int>(t64);
      if (t >= next) {
        b = owner_of(token_start, a.batch, t);
        next = token_start[b + 1];
        r = request_of(a, b);
      }
      const int p = r.c + (t - token_start[b]);
      const int column = static_cast<int>(static_cast<unsigned>(p) / static_cast<unsigned>(a.page_size));
      int entry = -1;
      if (column < r.held) {
        entry = a.block_table[static_cast<long long>(b) * a.table_stride + column];
      } else if (column < r.need) {
        const long long from = static_cast<long long>(page_start[b]) + (column - r.held);
        if (from < available) entry = a.free_pages[cursor + from];
      }
      if (entry >= 0)
        slot[i] = static_cast<long long>(entry) * a.page_size +
                  (p - static_cast<long long>(column) * a.page_size);
      position[i] = p;
      request[i] = b;
    }
    if (g + kTokensPerThread <= a.num_tokens) {
      longlong2* s = reinterpret_cast<longlong2*>(a.slots + g);
      s[0] = make_longlong2(slot[0], slot[1]);
      s[1] = make_longlong2(slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.positions + g) = make_int4(position[0], position[1], position[2], position[3]);
      *reinterpret_cast<int4*>(a.requests + g) = make_int4(request[0], request[1], request[2], request[3]);
    } else {
      for (int i = 0; i < kTokensPerThread && g + i < a.num_tokens; ++i) {
        a.slots[g + i] = slot[i];
        a.positions[g + i] = position[i];
        a.requests[g + i] = request[i];
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

extern "C" int dg_build_block_tables(const dg_block_tables* args, void* stream, int pdl_attr) {
  if (args == nullptr) return cudaErrorInvalidValue;
  const dg_block_tables& a = *args;
  if (a.batch < 1 || a.batch > kMaxBatch || a.page_size < 1 || a.table_width < 1 || a.num_tokens < 0 ||
      a.free_count < 0 || a.table_stride < a.table_width)
    return cudaErrorInvalidValue;
  if (a.context_lens == nullptr || a.new_lens == nullptr || a.block_table == nullptr || a.seq_lens == nullptr ||
      a.query_start == nullptr || a.cursor_out == nullptr || (a.free_count > 0 && a.free_pages == nullptr) ||
      (a.num_tokens > 0 && (a.slots == nullptr || a.positions == nullptr || a.requests == nullptr)))
    return cudaErrorInvalidValue;
  if (!aligned16(a.slots) || !aligned16(a.positions) || !aligned16(a.requests)) return cudaErrorInvalidValue;
  // Other CTAs read these while CTA 0 writes.
  if (a.seq_lens == a.context_lens || a.seq_lens == a.new_lens || a.cursor_out == a.cursor_in)
    return cudaErrorInvalidValue;

  // One CTA answers for 2048 tokens in one round; past one CTA an SM a CTA
  // takes several rounds rather than the sums being made once more.
  const int sms = dg_num_sms();
  const long long rounds = (static_cast<long long>(a.num_tokens) + kThreads * kTokensPerThread - 1) /
                           (kThreads * kTokensPerThread);
  long long ctas = rounds < 1 ? 1 : rounds;
  if (ctas > (sms > 0 ? sms : 148)) ctas = sms > 0 ? sms : 148;
  const size_t smem = static_cast<size_t>(a.batch + 1) * 2 * sizeof(int);
  if (smem > 48 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(block_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(smem));
    if (err != cudaSuccess) return err;
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1]{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (pdl_attr) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, block_tables_kernel, a);
}
