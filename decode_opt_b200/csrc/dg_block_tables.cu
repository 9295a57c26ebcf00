// SPDX-License-Identifier: MIT
//
// dg_block_tables.cu -- the paged cache's bookkeeping of one step, built on
// the GPU from the requests' lengths (include/decode_attention_b200.h gives
// the definition).
//
// Two exclusive sums over the requests (new tokens, new pages) and then one
// independent answer per token, the first token of a new page entering it into
// the table.  One launch: every CTA makes the sums for itself in shared memory
// (two loads per request from L2, one block scan) instead of waiting for
// another kernel or CTA, and then answers for its share of the tokens.  A warp
// takes 32 tokens at a time, a lane each: it finds the requests of the first
// and the last and a lane searches between those two only (in a prompt: not at
// all).  The loop is kept short and rolled: a decode step runs through it once,
// and much of what that costs is the fetching of its instructions (four tokens
// a lane, unrolled: 5.9 us for 16 requests instead of 4.4).  A slot never waits
// for the table entry that the same launch writes: a page below ceil(c / P) is
// read from the table, a later one from the free list itself.
//
// Bound: the launch, three dependent loads and the scan for a decode step
// (B200, in a graph: 4.5 us for 16 requests, 5.9 for 512); the searches'
// instructions at the other end (4096 prompts, 1.4 million tokens, 23 MB:
// 16 us, where the bytes alone would take 3.6).

#include <cuda_runtime.h>

#include <atomic>
#include <climits>
#include <cstdint>

#include "decode_attention_b200.h"
#include "decode_gemm_b200.h"
#include "sm100.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBatch = 16384;
constexpr int kTile = kThreads * 4;      // requests of one scan

struct Sums {
  long long tokens, pages;
};

__device__ __forceinline__ void report(int* status, int code) {
  if (status != nullptr) atomicCAS(status, 0, code);
}

// Pages of `tokens` tokens.
__device__ __forceinline__ int pages_of(const dg_block_tables& a, int shift, unsigned tokens) {
  const unsigned up = tokens + static_cast<unsigned>(a.page_size) - 1u;     // < 2^32
  return static_cast<int>(shift >= 0 ? up >> shift : up / static_cast<unsigned>(a.page_size));
}

__device__ __forceinline__ int clamp_int(long long v) {
  return v > INT_MAX ? INT_MAX : static_cast<int>(v);
}

// The last index i of [lo, hi) with starts[i] <= v; starts[lo] <= v.  Requests
// without tokens (or pages) share a start with the next; the last of them is
// the one that holds v.
__device__ __forceinline__ int owner_of(const int* starts, int lo, int hi, int v) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads, 2)
    block_tables_kernel(const __grid_constant__ dg_block_tables a, int shift) {
  extern __shared__ __align__(16) int smem[];
  const int room = (a.batch + 4) & ~3;           // each array begins on 16 bytes
  int* token_start = smem;                       // [batch + 1]
  int* page_start = smem + room;                 // [batch + 1]
  int* context = smem + 2 * room;                // [batch]
  __shared__ Sums warp_sum[2][kWarps];

  dg::sm100::griddep_launch_dependents();
  dg::sm100::griddep_wait();

  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const bool first_cta = blockIdx.x == 0;
  const int cursor = a.cursor_in != nullptr ? min(max(a.cursor_in[0], 0), a.free_count) : 0;
  const int available = a.free_count - cursor;

  // Exclusive sums, kTile requests at a time, four consecutive ones a thread;
  // the next tile's lengths are on their way during this one's scan.
  const bool wide = ((reinterpret_cast<uintptr_t>(a.context_lens) | reinterpret_cast<uintptr_t>(a.new_lens)) & 15u) == 0;
  auto fetch = [&](int tile, int (&c)[4], int (&n)[4]) {
    const int b = tile * kTile + tid * 4;
    if (wide && b + 4 <= a.batch) {
      const int4 x = *reinterpret_cast<const int4*>(a.context_lens + b);
      const int4 y = *reinterpret_cast<const int4*>(a.new_lens + b);
      c[0] = x.x; c[1] = x.y; c[2] = x.z; c[3] = x.w;
      n[0] = y.x; n[1] = y.y; n[2] = y.z; n[3] = y.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = b + i < a.batch ? a.context_lens[b + i] : 0;
        n[i] = b + i < a.batch ? a.new_lens[b + i] : 0;
      }
    }
  };
  int c[4], n[4];
  fetch(0, c, n);
  Sums carry{0, 0};                              // of the tiles before
  for (int tile = 0; tile * kTile < a.batch; ++tile) {
    const int b = tile * kTile + tid * 4;
    int need[4];
    int next_c[4], next_n[4];
    if ((tile + 1) * kTile < a.batch) fetch(tile + 1, next_c, next_n);
    Sums mine{0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // Made safe: below zero counts as 0, c + n stays within an int.
      if (c[i] < 0 || n[i] < 0 || n[i] > INT_MAX - max(c[i], 0)) {
        if (first_cta) report(a.status, DG_ERR_LENGTH);
        c[i] = max(c[i], 0);
        n[i] = min(max(n[i], 0), INT_MAX - c[i]);
      }
      const int all = pages_of(a, shift, static_cast<unsigned>(c[i]) + static_cast<unsigned>(n[i]));
      if (first_cta && all > a.table_width) report(a.status, DG_ERR_TABLE_WIDTH);
      need[i] = min(all, a.table_width) - min(pages_of(a, shift, static_cast<unsigned>(c[i])), a.table_width);
      mine.tokens += n[i];
      mine.pages += need[i];
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
    if (lane == 31) warp_sum[tile & 1][warp] = scan;
    __syncthreads();                             // (a sum is overwritten two barriers after it was read)
    Sums before{carry.tokens + scan.tokens - mine.tokens, carry.pages + scan.pages - mine.pages};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const Sums v = warp_sum[tile & 1][w];
      if (w < warp) {
        before.tokens += v.tokens;
        before.pages += v.pages;
      }
      carry.tokens += v.tokens;
      carry.pages += v.pages;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (b + i < a.batch) {
        token_start[b + i] = clamp_int(before.tokens);
        page_start[b + i] = clamp_int(before.pages);
        context[b + i] = c[i];
      }
      before.tokens += n[i];
      before.pages += need[i];
      c[i] = next_c[i];
      n[i] = next_n[i];
    }
  }
  if (tid == 0) {
    token_start[a.batch] = clamp_int(carry.tokens);
    page_start[a.batch] = clamp_int(carry.pages);
    if (first_cta) {
      if (carry.tokens > INT_MAX || carry.pages > INT_MAX) report(a.status, DG_ERR_LENGTH);
      if (carry.tokens > a.num_tokens) report(a.status, DG_ERR_TOKENS);
      if (carry.pages > available) report(a.status, DG_ERR_POOL);
      a.cursor_out[0] = cursor + static_cast<int>(min(carry.pages, static_cast<long long>(available)));
    }
  }
  __syncthreads();

  const int total = token_start[a.batch];
  const long long stride = static_cast<long long>(gridDim.x) * kThreads;
  const long long me = static_cast<long long>(blockIdx.x) * kThreads + tid;

  // Starts and lengths after the step, spread over the CTAs.
  for (long long b = me; b <= a.batch; b += stride) {
    const int start = token_start[b];
    a.query_start[b] = start;
    if (b < a.batch) {
      const int old = context[b];
      a.seq_lens[b] = old + min(max(a.new_lens[b], 0), INT_MAX - old);
    }
  }

  // More tokens than the outputs hold: the new pages that begin past them are
  // entered here.
  if (total > a.num_tokens) {
    for (long long g = me; g < page_start[a.batch]; g += stride) {
      const int page = static_cast<int>(g);
      const int b = owner_of(page_start, 0, a.batch, page);
      const int held = min(pages_of(a, shift, static_cast<unsigned>(context[b])), a.table_width);
      const int column = held + (page - page_start[b]);
      const long long token = token_start[b] + (static_cast<long long>(column) * a.page_size - context[b]);
      if (token >= a.num_tokens)
        a.block_table[b * a.table_stride + column] = page < available ? a.free_pages[cursor + page] : -1;
    }
  }

  // Tokens, 32 at a time: a warp takes a run of them.  A new page is entered
  // into the table by its first token.
  const int chunks = static_cast<int>((static_cast<long long>(a.num_tokens) + 31) / 32);
  const int warps = static_cast<int>(gridDim.x) * kWarps, me_warp = static_cast<int>(blockIdx.x) * kWarps + warp;
  const int chunk0 = static_cast<int>(static_cast<long long>(chunks) * me_warp / warps);
  const int chunk1 = static_cast<int>(static_cast<long long>(chunks) * (me_warp + 1) / warps);
  int last = -1;                                 // the request of the last token so far
#pragma unroll 1
  for (int chunk = chunk0; chunk < chunk1; ++chunk) {
    const long long t64 = static_cast<long long>(chunk) * 32 + lane;
    long long slot = -1;
    int position = 0, request = -1;
    if (t64 - lane < total) {
      const int begin = chunk * 32, t = begin + lane;
      const int end = min(begin + 31, total - 1);
      if (last < 0) last = owner_of(token_start, 0, a.batch, begin);
      const int first = last;
      // The request of the last token: onwards by doubled steps, then by bisection.
      int hop = 1;
      while (last + hop < a.batch && token_start[last + hop] <= end) {
        last += hop;
        hop <<= 1;
      }
      last = owner_of(token_start, last, min(last + hop, a.batch), end);
      if (t64 < total) {
        request = owner_of(token_start, first, last + 1, t);
        const int cached = context[request], page0 = page_start[request];
        const int held = min(pages_of(a, shift, static_cast<unsigned>(cached)), a.table_width);
        const int need = held + (page_start[request + 1] - page0);
        position = cached + (t - token_start[request]);
        const unsigned p = static_cast<unsigned>(position);
        const unsigned col = shift >= 0 ? p >> shift : p / static_cast<unsigned>(a.page_size);
        const unsigned inside = p - col * static_cast<unsigned>(a.page_size);
        const int column = static_cast<int>(col);
        int* place = a.block_table + request * a.table_stride + column;
        int entry = -1;
        if (column < held) {
          entry = *place;
        } else if (column < need) {
          const int taken = page0 + (column - held);
          if (taken < available) entry = a.free_pages[cursor + taken];
          if (inside == 0 && t64 < a.num_tokens) *place = entry;
        }
        if (entry >= 0) slot = static_cast<long long>(entry) * a.page_size + inside;
      }
    }
    if (t64 < a.num_tokens) {
      a.slots[t64] = slot;
      a.positions[t64] = position;
      a.requests[t64] = request;
    }
  }
}

// The kernel's three arrays.
constexpr size_t smem_of(int batch) { return static_cast<size_t>((batch + 4) & ~3) * 3 * sizeof(int); }
constexpr size_t kStaticSmem = sizeof(Sums) * 2 * kWarps;          // of the kernel's own, beside them
constexpr size_t kPlainSmem = 48 * 1024 - kStaticSmem;             // what it may take without asking
static_assert(smem_of(kMaxBatch) + kStaticSmem <= 227 * 1024 - 1024, "shared memory");

// Whether the free list lies in a row of the table: a launch reads the one and
// writes the other in no order.
bool free_list_in_table(const dg_block_tables& a) {
  const uintptr_t from = reinterpret_cast<uintptr_t>(a.free_pages), to = from + 4ull * a.free_count;
  const uintptr_t table = reinterpret_cast<uintptr_t>(a.block_table);
  const unsigned long long row = 4ull * a.table_width, step = 4ull * a.table_stride;
  // The first row that ends past the list's beginning.
  const unsigned long long b = from < table + row ? 0 : (from - table - row) / step + 1;
  return a.free_count > 0 && b < static_cast<unsigned long long>(a.batch) && table + b * step < to;
}

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
  const void* ints[] = {a.context_lens, a.new_lens, a.free_pages, a.cursor_in, a.block_table, a.seq_lens,
                        a.query_start, a.positions, a.requests, a.cursor_out, a.status};
  for (const void* p : ints)
    if ((reinterpret_cast<uintptr_t>(p) & 3u) != 0) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a.slots) & 7u) != 0) return cudaErrorInvalidValue;
  // Other CTAs read these while CTA 0 writes.
  if (a.seq_lens == a.context_lens || a.seq_lens == a.new_lens || a.cursor_out == a.cursor_in)
    return cudaErrorInvalidValue;
  if (free_list_in_table(a)) return cudaErrorInvalidValue;

  const size_t smem = smem_of(a.batch);
  // A token a thread; past the CTAs that fit at once a CTA takes several
  // rounds rather than the sums being made again.
  const int sms = dg_num_sms() > 0 ? dg_num_sms() : 148;
  const long long rounds = (static_cast<long long>(a.num_tokens) + kThreads - 1) / kThreads;
  const long long most = static_cast<long long>(sms) * (smem <= 100 * 1024 ? 2 : 1);
  const long long ctas = rounds < 1 ? 1 : rounds < most ? rounds : most;
  int shift = -1;
  if ((a.page_size & (a.page_size - 1)) == 0)
    for (shift = 0; (1 << shift) < a.page_size; ++shift) {}
  if (smem > kPlainSmem) {
    // Raised once per device, to what the largest batch takes: it is the
    // kernel's, not the call's, and another thread may be about to launch.
    static std::atomic<unsigned long long> ready{0};
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    const unsigned long long bit = 1ull << (dev & 63);
    if ((ready.load(std::memory_order_acquire) & bit) == 0) {
      err = cudaFuncSetAttribute(block_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(smem_of(kMaxBatch)));
      if (err != cudaSuccess) return err;
      ready.fetch_or(bit, std::memory_order_release);
    }
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
  return cudaLaunchKernelEx(&cfg, block_tables_kernel, a, shift);
}
