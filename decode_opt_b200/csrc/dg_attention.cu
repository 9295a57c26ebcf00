// SPDX-License-Identifier: MIT
//
// dg_attention.cu -- attention of one new token per request over a paged
// key-value cache (include/decode_attention_b200.h gives the definition).
//
// Bound: the live tokens' keys and values are read once per kv head (for up to
// 16 query heads a kv head; more read them once per 16), 2 * D values a token,
// against 4 * D operations a token and query head: HBM traffic by its numbers.
// What a kernel meets before that is the rate at which 8 warps an SM (their
// rings and accumulators fill shared memory and registers) get through the
// instructions of a tile: 16 tokens of 16-bit keys and 8 heads keep up with
// HBM, 32 tokens of e4m3 and 16 heads do not, nor do heads of 256 (spills).
// B200, calls one after another (in a graph): 1.08M tokens of 4 heads of 128,
// bf16, 8 query heads each (2.21 GB) 333 us (330), 6.6 TB/s, 104% of a copy's
// rate; a ragged batch of 61 requests on 8 heads (0.70 GB) 124 us (123), 5.7
// TB/s; 64 requests in e4m3 under 16 query heads a kv head (1.0 GB) 233 us
// (221), 4.4 TB/s; 64 heads on 4 of 256 on the ragged lengths 220 us (218), 3.2
// TB/s; one request of 2049 tokens 10.9 us (9.8).
//
// Split.  The work is cut into tiles of TOK tokens of one (request, kv head,
// group of ROWS query heads) "item"; all tiles of all items stand in one
// line, each item preceded by the units that its beginning and end cost, and
// CTA c of G takes units [U c / G, U (c+1) / G) of it -- equal shares whatever the
// lengths are, one CTA an SM.  The line is laid out on the device from
// seq_lens (one scan of the batch per CTA), so that the host needs no
// lengths.  A CTA therefore works on a run of items: the first and the last
// may be shared with its neighbours, those between are its own.  Within an
// item's share the CTA's warps take tiles in turn; items of a few tiles are
// done by one warp each, without the join.  Every warp has its own ring of
// TOK-token stages filled by its own cp.async copies: no barrier in the loop,
// and the ring runs on across items, so that the end of one does not drain
// it.  16-byte copies with the row's address from the page table (one table
// entry per token and lane, fetched a tile ahead) take any page size and
// strides; tokens that are not live are zero-filled and masked.
//
// Products: mma.sync m16n8k16, the query heads as its 16 rows.  The tensor
// pipe is 16 to 19% busy with 16-bit caches, 42% with e4m3 and 16 heads an item
// (of active cycles).  tcgen05's 64 or 128 rows would multiply zeros with
// the heads as rows; with keys, then values, as rows and the heads as columns
// they would be full, and e4m3 would need no widening.  16-bit caches of heads
// up to 128 under up to 16 heads have little to gain from that (80 to 104% of a
// copy's rate); wider heads, larger groups and e4m3 with more than 8 heads
// would, and it is not built.
//
// Scores stay in registers: the accumulator
// layout of S = Q K^T is the operand layout of P V.  P enters as two terms,
// hi = p cut to 16 bits and lo = round(p - hi): 16 to 17 bits of p with bf16
// caches, 22 with fp16 and e4m3, so that its rounding (2^-8 in bf16) does not
// show in the result.  (Ragged batch, against the value in 64 bits rounded
// once: 3.6 of 1000 bf16 outputs round the other way, 0.7 in 32 bits; the
// error of either is 1.66e-3.)  With up to 8 query heads a kv head
// (ROWS = 8) the lo terms fill the 8 rows that would be empty, at no cost;
// with more (ROWS = 16) they are a second product.  Cut towards zero and with
// lo kept above 0, both terms have the sign of p, so that an infinite value
// stays infinite (0 times it would be NaN) where p itself is not 0.
//
// e4m3 caches are widened to fp16 (exact) on the way into the product.  Both
// products are indifferent to the order of their inner index, and the columns
// of the second to a permutation, so that fragments are read as 16 and 8
// consecutive bytes a lane: no 8-bit transposition.  q is scaled by a power
// of two per head to fit fp16's range, exactly undone in fp32.
//
// Join.  The warps' (m, l, o) are joined in shared memory, in warp order.  A
// share of an item goes to the workspace; the last of the item's CTAs to
// arrive (a ticket) joins the shares in CTA order.  No CTA waits for another.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "decode_attention_b200.h"
#include "decode_gemm_b200.h"
#include "sm100.cuh"
#include "warp_mma.cuh"

namespace {

using dg::warp::Bf16;
using dg::warp::Fp16;

constexpr int kMaxCtas = 160;            // CTAs of a launch: one an SM (148)
constexpr int kMaxRows = 16;             // query heads an item
constexpr int kMaxDim = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFp8Max = 448.0f;        // of the output's quantisation, as dg_quantize_act
constexpr float kQuantEps = 1.0e-4f;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLowest = -3.402823466e38f;

// Workspace: tickets, then (m, l) per share and row, then the shares.
constexpr size_t kTicketBytes = 1024;    // kMaxCtas ints
constexpr size_t kShares = 2 * kMaxCtas; // a CTA's first and last item
constexpr size_t kWorkspaceBytes =
    kTicketBytes + kShares * kMaxRows * sizeof(float2) + kShares * kMaxRows * kMaxDim * sizeof(float);
static_assert(kMaxCtas * sizeof(int) <= kTicketBytes, "tickets");

struct Params {
  dg_attention_args a;
  int group;               // query heads a kv head
  int groups;              // items a kv head: ceil(group / ROWS)
  int page_shift;          // log2(page_size), -1 if it is no power of two
  int aligned;             // page_size is a multiple of TOK
  int* tickets;
  float2* share_ml;        // [share][kMaxRows]
  float* share_o;          // [share][kMaxRows][kMaxDim]
};

// Compile-time shape: MM the 16-bit type of the products, E4M3 the cache, DP
// the head dimension padded to 64 / 128 / 256, ROWS the query heads an item.
template <typename MM_, bool E4M3_, int DP_, int ROWS_>
struct Shape {
  using MM = MM_;
  static constexpr bool kE4m3 = E4M3_;
  static constexpr int DP = DP_, ROWS = ROWS_;
  static constexpr int ES = E4M3_ ? 1 : 2;
  // A stage holds a tile's keys and values.  With heads of 256 there is room
  // for 4 warps' rings then, and for 8 if keys and values are stages of their
  // own, half as much of them on its way: worth it where the products weigh
  // more (ragged batch of 64 heads on 4, bf16: 281 -> 219 us; e4m3, 8 heads an
  // item: 230 -> 202; but bf16, 4 heads an item: 144 -> 158).
  static constexpr bool HALVES = DP_ == 256 && (E4M3_ || ROWS_ == 16);
  static constexpr int NW = DP_ == 64 ? 12 : DP_ == 128 || HALVES ? 8 : 4;   // warps
  static constexpr int TOK = E4M3_ || DP_ == 64 ? 32 : 16;       // tokens a tile
  static constexpr int STAGES = DP_ == 64 ? 2 : 3;
  static constexpr int PITCH = DP_ * ES;                         // bytes a row
  static constexpr int KV_BYTES = TOK * PITCH;                   // a tile's keys, and its values
  static constexpr int STAGE = HALVES ? KV_BYTES : 2 * KV_BYTES;
  static constexpr int RING = NW * STAGES * STAGE;
  static constexpr int JOIN = 8192;                              // floats of the join's buffer (32 KiB)
  static constexpr int JOIN_COLS =                               // columns a round: a power of two from 32
      NW * ROWS_ * DP_ <= JOIN ? DP_ : NW * ROWS_ * 128 <= JOIN ? 128 : NW * ROWS_ * 64 <= JOIN ? 64 : 32;
  static constexpr int SOLO = 8;                                 // tiles of an item that one warp does alone
  // What an item costs beyond its tiles (join, uneven warps), in tiles: CTAs
  // with 3 and with 15 items of the same units differed by 1.7 to 4.5 us an
  // item.  One figure for tiles of all head dimensions, whose times differ;
  // measured with heads of 128.  Ragged batch, 8 heads an item: 129.8 us at 4,
  // 123.7 at 8, 123.0 at 14, 122.7 at 20; 16 heads: 161.7, 149.9, 142.1, 135.4
  // (still falling at 20, and not tried beyond).
  static constexpr int EXTRA_SOLO = 1, EXTRA = ROWS_ == 8 ? 14 : 20;
  static constexpr int MIN_RUN = 8;                              // units a CTA takes at least
  static constexpr int NT = TOK / 8;                             // score tiles of 8 tokens
  static constexpr int KS = DP_ / 16;                            // inner steps of Q K^T
  static constexpr int OT = DP_ / 8;                             // output tiles of 8 columns
  static constexpr int CHUNKS = DP_ / 32;                        // of the joins
  static constexpr int PACK = CHUNKS < 4 ? CHUNKS : 4;           // floats of a share's access
  static constexpr int RPT = (ROWS_ + NW - 1) / NW;              // rows a warp finishes: warp, warp + NW, ...
  // 2^kBias is the probability of the maximum: fp16's subnormals start at
  // 2^-14, so its probabilities are lifted out of them.
  static constexpr float kBias = sizeof(MM_) != 0 && __is_same(MM_, Fp16) ? 10.0f : 0.0f;
  // How far a score may pass the reference exponent: 2^(kLag + kBias) stays
  // well inside fp16.
  static constexpr float kLag = 5.0f;
  static constexpr size_t SMEM = RING + sizeof(float) * (JOIN + 2 * NW * ROWS_) +
                                 sizeof(uint32_t) * NW * STAGES;
  static_assert(NW * ROWS_ * JOIN_COLS <= JOIN && SMEM <= 227 * 1024 - 1024, "shared memory");
  static_assert(kMaxCtas * ROWS_ <= JOIN, "join factors fit the join buffers");

  // Output column of position `n` of output tile `t` (see the e4m3 fragments).
  static __device__ __forceinline__ int column(int t, int n) {
    return E4M3_ ? (t >> 3) * 64 + n * 8 + (t & 7) : t * 8 + n;
  }
  // Where row `r` keeps its 16-byte chunk `c`: the eight chunks that one phase
  // of the fragment loads reads fall into different banks.  16-bit: one chunk
  // of 8 consecutive rows.  e4m3: 4 chunks of rows (2i, 2i + 1) for keys, 2
  // chunks of rows 0, 2, 4, 6 (or 1, 3, 5, 7) for values.
  static __device__ __forceinline__ int swizzled(int r, int c) {
    return E4M3_ ? c ^ ((r & 6) ^ ((r & 1) << 2)) : c ^ (r & 7);
  }
};

__device__ __forceinline__ void report(int* status, int code) {
  if (status != nullptr) atomicCAS(status, 0, code);
}

// a / b for a line that may be longer than 32 bits; it rarely is, and the
// 32-bit division is a quarter of the instructions.
__device__ __forceinline__ unsigned long long divided(unsigned long long a, unsigned long long b) {
  if (((a | b) >> 32) == 0) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}

// The live tokens [first_live, len) of a request as tiles.
__device__ __forceinline__ int first_live(const dg_attention_args& a, int len) {
  return a.window > 0 && len > a.window ? len - a.window : 0;
}
template <typename S>
__device__ __forceinline__ int tiles_of(const dg_attention_args& a, int len) {
  return len > 0 ? (len - 1) / S::TOK + 1 - first_live(a, len) / S::TOK : 0;
}
// Units of the line before an item's first tile: what the item costs beyond
// its tiles.
template <typename S>
__device__ __forceinline__ int extra_of(int tiles) {
  return tiles <= S::SOLO ? S::EXTRA_SOLO : S::EXTRA;
}
__device__ __forceinline__ int length_of(const dg_attention_args& a, int b, bool tell) {
  const int len = a.seq_lens[b];
  const long long most = static_cast<long long>(a.table_width) * a.page_size;
  if (len >= 0 && len <= most) return len;
  if (tell) report(a.status, DG_ERR_SEQ_LEN);
  return len < 0 ? 0 : static_cast<int>(most);
}
// The units of all of a request's items.
template <typename S>
__device__ __forceinline__ long long units_of(const dg_attention_args& a, int b, int items) {
  const int tiles = tiles_of<S>(a, length_of(a, b, false));
  return tiles != 0 ? static_cast<long long>(tiles + extra_of<S>(tiles)) * items : 0;
}

// A place in a CTA's run of the line, in units from the run's beginning (a
// run of 2^31 units would be 10^13 bytes): one item's share.
template <typename S>
struct Cursor {
  int run;               // the run's units
  int x;                 // the item's first unit (below 0: in an earlier CTA's run)
  int b, item;           // request, item of the request
  int len, tiles;        // the request's length, an item's tiles
  int t0, count;         // the share: tiles [t0, t0 + count) of the item
  int turn;              // solo shares before this one
  bool solo;             // one warp's work (turn % NW) instead of the CTA's

  // The share [t0, ...) of the item; false if the run ends before it.
  __device__ __forceinline__ bool settle() {
    const int extra = extra_of<S>(tiles);
    count = min(tiles, run - x - extra) - t0;
    // One warp takes as many steps as the item has tiles, but several items go
    // side by side: worth it where the run holds more than the one.
    solo = tiles <= S::SOLO && count == tiles && run >= 2 * (tiles + extra);
    return count > 0;
  }
  // At the unit `from` of the line; request `request` begins at unit `base`.
  __device__ __forceinline__ bool start(const dg_attention_args& a, int request, long long base, long long from,
                                        long long to) {
    b = request;
    run = static_cast<int>(to - from);
    turn = 0;
    len = length_of(a, b, false);
    tiles = tiles_of<S>(a, len);
    const int units = tiles + extra_of<S>(tiles);
    const unsigned long long off = static_cast<unsigned long long>(from - base);
    item = static_cast<int>(divided(off, static_cast<unsigned long long>(units)));
    x = -static_cast<int>(off - static_cast<unsigned long long>(item) * units);
    t0 = max(0, -x - extra_of<S>(tiles));
    return settle();
  }
  // To the next share; false at the end of the run.
  __device__ __forceinline__ bool advance(const dg_attention_args& a, int items) {
    x += tiles + extra_of<S>(tiles);
    if (x >= run) return false;
    if (solo) ++turn;
    if (++item == items) {
      item = 0;
      do {
        ++b;             // x < run: a later request has tiles
        len = length_of(a, b, false);
        tiles = tiles_of<S>(a, len);
      } while (tiles == 0);
    }
    t0 = 0;
    return settle();
  }
  // This warp's tiles of the share: first, first + step, ...
  __device__ __forceinline__ int first_tile(int warp) const {
    return !solo ? warp : (turn % S::NW == warp ? 0 : count);
  }
  __device__ __forceinline__ int step() const { return solo ? 1 : S::NW; }
};

// One warp's copies: tile after tile of the CTA's run, ahead of the products.
// Where page_size is a multiple of TOK (`p.aligned`) a tile lies in one page:
// one table entry a tile, and a lane's addresses are a line.  Otherwise every
// lane looks up one token, and its row's address goes round by shuffles.
template <typename S>
struct Loader {
  static constexpr int CH = S::DP * S::ES / 16;     // chunks a row
  static constexpr int RPI = 32 / CH;               // rows an instruction
  static constexpr uint32_t kWhole = S::TOK == 32 ? 0xffffffffu : (1u << (S::TOK & 31)) - 1u;
  Cursor<S> at;
  int tile;              // of the share
  bool more;             // a tile is pending
  // The pending tile: its live tokens; page and offset in it of its first
  // token, or of this lane's.
  uint32_t bits;
  int page, offset;
  // The share's head in the caches; aligned: this lane's row and chunk of it.
  const char *keys, *values;

  __device__ __forceinline__ void open(const Params& p, int lane) {
    const dg_attention_args& a = p.a;
    const int head = p.groups == 1 ? at.item : at.item / p.groups;
    const int row = p.aligned ? lane / CH : 0, chunk = p.aligned ? lane % CH : 0;
    keys = static_cast<const char*>(a.k_cache) + (head * a.k_cache_stride[2] + row * a.k_cache_stride[1]) * S::ES +
           chunk * 16;
    values = static_cast<const char*>(a.v_cache) + (head * a.v_cache_stride[2] + row * a.v_cache_stride[1]) * S::ES +
             chunk * 16;
  }
  __device__ __forceinline__ void look_up(const Params& p, int lane) {
    const int lo = first_live(p.a, at.len);
    const int tok = (lo / S::TOK + at.t0 + tile) * S::TOK;
    const int from = lo - tok, to = at.len - tok;      // to > 0, from < TOK
    bits = kWhole;
    if (to < S::TOK) bits &= (1u << to) - 1u;
    if (from > 0) bits &= ~((1u << from) - 1u);
    const unsigned t = static_cast<unsigned>(tok) + (p.aligned ? 0u : static_cast<unsigned>(lane));
    unsigned column;
    if (p.page_shift >= 0) {
      column = t >> p.page_shift;
      offset = static_cast<int>(t & ((1u << p.page_shift) - 1u));
    } else {
      column = t / static_cast<unsigned>(p.a.page_size);
      offset = static_cast<int>(t - column * static_cast<unsigned>(p.a.page_size));
    }
    page = -1;
    if (p.aligned || ((bits >> (lane % S::TOK)) & 1u & (lane < S::TOK)) != 0u)
      page = p.a.block_table[at.b * p.a.table_stride + column];
  }
  // Moves to the warp's next tile, through the shares that have none for it.
  __device__ __forceinline__ void prepare(const Params& p, int warp, int lane, int items) {
    if (!more) return;
    if (tile >= at.count) {
      do {
        if (!at.advance(p.a, items)) {
          more = false;
          return;
        }
        tile = at.first_tile(warp);
      } while (tile >= at.count);
      open(p, lane);
    }
    look_up(p, lane);
    tile += at.step();
  }
  // Copies the pending tile's keys, values or both into a stage.
  template <bool KEYS, bool VALUES>
  __device__ __forceinline__ void issue(const Params& p, uint32_t stage, uint32_t* mask, int lane) const {
    constexpr int kValuesAt = KEYS ? S::KV_BYTES : 0;
    if (!more) return;
    const dg_attention_args& a = p.a;
    const int chunk = lane % CH;
    const bool wanted = chunk * 16 < a.head_dim * S::ES;
    // Row i * RPI + lane / CH: its swizzle is the lane's and the row step's.
    const uint32_t dst = stage + (lane / CH) * S::PITCH + S::swizzled(lane / CH, chunk) * 16;
    const bool good = page >= 0 && page < a.num_pages;
    if (p.aligned) {
      if (KEYS && !good && lane == 0) report(a.status, DG_ERR_PAGE);
      const uint32_t live = good ? bits : 0u;
      if (KEYS && lane == 0) *mask = live;
      const char* k = keys + (page * a.k_cache_stride[0] + offset * a.k_cache_stride[1]) * S::ES;
      const char* v = values + (page * a.v_cache_stride[0] + offset * a.v_cache_stride[1]) * S::ES;
      const long long k_step = a.k_cache_stride[1] * (RPI * S::ES), v_step = a.v_cache_stride[1] * (RPI * S::ES);
      if (live == kWhole) {
#pragma unroll
        for (int i = 0; i < S::TOK / RPI; ++i, k += k_step, v += v_step) {
          const uint32_t to = (dst ^ (S::swizzled(i * RPI, 0) * 16)) + i * RPI * S::PITCH;
          if (wanted) {
            if (KEYS) dg::warp::cp_async16(to, k);
            if (VALUES) dg::warp::cp_async16(to + kValuesAt, v);
          }
        }
      } else {
        if (!good) {         // nothing is read, but the addresses are still some
          k = static_cast<const char*>(a.k_cache);
          v = static_cast<const char*>(a.v_cache);
        }
        const long long ks = good ? k_step : 0, vs = good ? v_step : 0;
#pragma unroll
        for (int i = 0; i < S::TOK / RPI; ++i, k += ks, v += vs) {
          const uint32_t to = (dst ^ (S::swizzled(i * RPI, 0) * 16)) + i * RPI * S::PITCH;
          const uint32_t bytes = (live >> (i * RPI + lane / CH)) & 1u ? 16u : 0u;
          if (wanted) {
            if (KEYS) dg::warp::cp_async16(to, k, bytes);
            if (VALUES) dg::warp::cp_async16(to + kValuesAt, v, bytes);
          }
        }
      }
      return;
    }
    const bool seen = lane < S::TOK && ((bits >> (lane % S::TOK)) & 1u) != 0u;
    if (KEYS && seen && !good) report(a.status, DG_ERR_PAGE);
    const uint32_t live = __ballot_sync(0xffffffffu, seen && good);
    if (KEYS && lane == 0) *mask = live;
    long long k_at = 0, v_at = 0;
    if (seen && good) {
      k_at = (page * a.k_cache_stride[0] + offset * a.k_cache_stride[1]) * S::ES;
      v_at = (page * a.v_cache_stride[0] + offset * a.v_cache_stride[1]) * S::ES;
    }
#pragma unroll
    for (int i = 0; i < S::TOK / RPI; ++i) {
      const int r = i * RPI + lane / CH;
      const long long kr = __shfl_sync(0xffffffffu, k_at, r);
      const long long vr = __shfl_sync(0xffffffffu, v_at, r);
      const uint32_t bytes = (live >> r) & 1u ? 16u : 0u;
      const uint32_t to = (dst ^ (S::swizzled(i * RPI, 0) * 16)) + i * RPI * S::PITCH;
      if (wanted) {
        if (KEYS) dg::warp::cp_async16(to, keys + kr + (bytes ? chunk * 16 : 0), bytes);
        if (VALUES) dg::warp::cp_async16(to + kValuesAt, values + vr + (bytes ? chunk * 16 : 0), bytes);
      }
    }
  }
};

// A pair of q's values as floats.
__device__ __forceinline__ float2 unpack_q(uint32_t v, int type) {
  return type == DG_TYPE_BF16 ? Bf16::unpack(v) : Fp16::unpack(v);
}

// cap * tanh(x).  Up to kNearCap: x + x^3 p(x^2), p of the least relative error
// that its degree allows there (found by Remez exchange: 2^-26; with its
// roundings 2^-23).  Beyond, 1 - 2 / (e^(2x) + 1) no longer cancels: 2^-21.
// The second alone, for all, is off by 2^-23 of the cap, not of the score.  Most
// heads' scores stay below half the cap, and their warps take the first alone.
// (33 requests of 24 fp16 heads 63.5 -> 64.3 us, e4m3 with 16 heads an item
// 237 -> 246; tanhf() in place of both 64.8 and 264.)
constexpr float kNearCap = 0.5f;
__device__ __forceinline__ float capped_near(float x, float cap) {
  const float t = x * x;
  const float p = fmaf(fmaf(fmaf(0.0172414915f, t, -0.0530454943f), t, 0.133258790f), t, -0.333331439f);
  const float u = cap * x;
  return fmaf(u * t, p, u);
}
__device__ __forceinline__ float capped_far(float x, float cap) {
  return cap - 2.0f * cap * dg::warp::rcp_approx(dg::warp::exp2_approx(x * (2.0f * kLog2e)) + 1.0f);
}

// One warp's state for one item.
template <typename S>
struct Warp {
  static constexpr int R = S::ROWS == 8 ? 1 : 2;     // rows a lane: lane / 4 (and + 8)
  uint32_t q[S::KS][2 * R];                          // [step][first half's rows, second half's rows]
  float o[S::OT][4];
  float m[R], l[R];
  float factor[R];                                   // score -> exponent of 2 (capped: -> score over the cap)

  // Loads an item's q as it lies in memory; nothing waits for it before
  // begin().
  __device__ __forceinline__ void fetch(const Params& p, int b, int item, int lane) {
    const dg_attention_args& a = p.a;
    const int head = p.groups == 1 ? item : item / p.groups;
    const int quad = lane & 3;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = (item - head * p.groups) * S::ROWS + (lane >> 2) + 8 * r;
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] +
                            (static_cast<long long>(head) * p.group + row) * a.q_stride[1];
      const bool real = row < p.group;
#pragma unroll
      for (int ks = 0; ks < S::KS; ++ks) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // Inner index of the two values: as ldmatrix deals 16-bit keys, or
          // 4 consecutive ones of the lane's 16 bytes of e4m3 keys.
          const int d = S::kE4m3 ? (ks >> 2) * 64 + quad * 16 + (ks & 3) * 4 + h * 2 : ks * 16 + quad * 2 + h * 8;
          q[ks][h * R + r] = real && d < a.head_dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
        }
      }
    }
  }

  __device__ __forceinline__ void begin(const Params& p, int item) {
    const dg_attention_args& a = p.a;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float f = a.scale;
      if constexpr (S::kE4m3) {
        float top = 0.0f;
#pragma unroll
        for (int ks = 0; ks < S::KS; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 v = unpack_q(q[ks][h * R + r], a.type);
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^-e and 2^e of top's exponent e; none for 0, subnormals, infinity.
        const uint32_t e = __float_as_uint(top) >> 23;
        const bool scaled = e > 0 && e < 254;
        const float down = scaled ? __uint_as_float((254u - e) << 23) : 1.0f;
        const float up = scaled ? __uint_as_float(e << 23) : 1.0f;
#pragma unroll
        for (int ks = 0; ks < S::KS; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 v = unpack_q(q[ks][h * R + r], a.type);
            q[ks][h * R + r] = Fp16::pack(v.x * down, v.y * down);
          }
        f *= up;
        if (a.k_scale != nullptr) f *= a.k_scale[p.groups == 1 ? item : item / p.groups];
      }
      factor[r] = a.softcap > 0.0f ? f / a.softcap : f * kLog2e;
      m[r] = kNegInf;
      l[r] = 0.0f;
    }
#pragma unroll
    for (int t = 0; t < S::OT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[t][i] = 0.0f;
  }

  __device__ __forceinline__ void a_of(int ks, uint32_t (&x)[4]) const {
    if constexpr (R == 1) {
      x[0] = q[ks][0];
      x[1] = 0u;
      x[2] = q[ks][1];
      x[3] = 0u;
    } else {
      x[0] = q[ks][0];
      x[1] = q[ks][1];
      x[2] = q[ks][2];
      x[3] = q[ks][3];
    }
  }

  // One tile, of whose TOK tokens `live` are to be seen: its probabilities s
  // (to the reference exponent m, which may move), then their part of o.
  __device__ __forceinline__ void scores(const Params& p, uint32_t keys, uint32_t live, int lane,
                                         float (&s)[S::NT][4]) {
    const int g = lane >> 2, quad = lane & 3;
#pragma unroll
    for (int t = 0; t < S::NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][i] = 0.0f;

    if constexpr (!S::kE4m3) {
      // Matrices: tokens 0-7 x (values 0-7, 8-15), tokens 8-15 x the same.
      // Chunk 2 ks + side of the row; stages are aligned to 128 bytes, so that
      // the step's part of the chunk goes in by exclusive or and offset.
      const uint32_t at = keys + ((lane & 7) + (lane >> 4) * 8) * S::PITCH + S::swizzled(lane, (lane >> 3) & 1) * 16;
#pragma unroll
      for (int ks = 0; ks < S::KS; ++ks) {
        uint32_t x[4];
        a_of(ks, x);
#pragma unroll
        for (int t = 0; t < S::NT; t += 2) {
          uint32_t k[4];
          dg::warp::ldmatrix_x4(k, (at ^ (ks * 32 & 127)) + (ks * 32 & ~127) + t * 8 * S::PITCH);
          S::MM::mma(s[t], x, k[0], k[1]);
          S::MM::mma(s[t + 1], x, k[2], k[3]);
        }
      }
    } else {
      const uint32_t at = keys + g * S::PITCH + S::swizzled(g, quad) * 16;    // chunk 4 blk + quad, as above
#pragma unroll
      for (int blk = 0; blk < S::KS / 4; ++blk) {
#pragma unroll
        for (int t = 0; t < S::NT; ++t) {
          const uint4 k =
              dg::warp::ld_shared_v4((at ^ (blk * 64 & 127)) + (blk * 64 & ~127) + t * 8 * S::PITCH);
          const uint32_t w[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t x[4];
            a_of(blk * 4 + i, x);
            S::MM::mma(s[t], x, dg::warp::e4m3_low(w[i]), dg::warp::e4m3_high(w[i]));
          }
        }
      }
    }

    // Exponents, masked; the running maximum and sum.
    const bool capped = p.a.softcap > 0.0f;
    const float cap = p.a.softcap * kLog2e;
#pragma unroll
    for (int t = 0; t < S::NT; ++t)
#pragma unroll
      for (int i = 0; i < 2 * R; ++i) s[t][i] *= factor[i >> 1];
    if (capped) {
      // Here s is the score over the cap.
      float top = 0.0f;
#pragma unroll
      for (int t = 0; t < S::NT; ++t)
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) top = fmaxf(top, fabsf(s[t][i]));
      if (__any_sync(0xffffffffu, top > kNearCap)) {
#pragma unroll
        for (int t = 0; t < S::NT; ++t)
#pragma unroll
          for (int i = 0; i < 2 * R; ++i)
            s[t][i] = fabsf(s[t][i]) > kNearCap ? capped_far(s[t][i], cap) : capped_near(s[t][i], cap);
      } else {
#pragma unroll
        for (int t = 0; t < S::NT; ++t)
#pragma unroll
          for (int i = 0; i < 2 * R; ++i) s[t][i] = capped_near(s[t][i], cap);
      }
    }
    if (live != Loader<S>::kWhole) {
#pragma unroll
      for (int t = 0; t < S::NT; ++t)
#pragma unroll
        for (int i = 0; i < 2 * R; ++i)
          if (((live >> (t * 8 + quad * 2 + (i & 1))) & 1u) == 0u) s[t][i] = kNegInf;
    }
    // The reference exponent m follows the maximum only when it falls kLag
    // behind (probabilities up to 2^(kLag + kBias) are as exact as others), so
    // that the sums so far are seldom scaled; the first tile has none.
    float alpha[R];
    bool moved = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = s[0][2 * r];
#pragma unroll
      for (int t = 0; t < S::NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) top = fmaxf(top, s[t][2 * r + i]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // -inf stands for "no token so far" alone: a row whose scores are -inf
      // or NaN has seen some.
      top = live != 0u ? fmaxf(top, kLowest) : kNegInf;
      alpha[r] = 1.0f;
      if (top > m[r] + S::kLag || m[r] == kNegInf) {
        moved = moved || m[r] != kNegInf;
        alpha[r] = m[r] == kNegInf ? 0.0f : dg::warp::exp2_approx(m[r] - top);
        m[r] = top;
      }
      const float from = (m[r] == kNegInf ? 0.0f : m[r]) - S::kBias;
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < S::NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float e = dg::warp::exp2_approx(s[t][2 * r + i] - from);
          s[t][2 * r + i] = e;
          sum += e;
        }
      l[r] = l[r] * alpha[r] + sum;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int t = 0; t < S::OT; ++t) {
        o[t][0] *= alpha[0];
        o[t][1] *= alpha[0];
        o[t][2] *= alpha[R - 1];
        o[t][3] *= alpha[R - 1];
      }
    }
  }

  __device__ __forceinline__ void weigh(uint32_t values, int lane, const float (&s)[S::NT][4]) {
    const int g = lane >> 2, quad = lane & 3;
#pragma unroll
    for (int kk = 0; kk < S::NT / 2; ++kk) {
      // hi and lo of the probabilities of 16 tokens as the first operand.
      uint32_t hi[2 * R], lo[2 * R];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float u = s[kk * 2 + h][2 * r], v = s[kk * 2 + h][2 * r + 1];
          const uint32_t top = S::MM::cut(u, v);
          const float2 back = S::MM::unpack(top);
          hi[h * R + r] = top;
          // (e4m3 has no infinity to keep; a probability below kTiny is itself:
          // with kTiny, 2^-34 of the largest in fp16, 100,000 tokens of no
          // weight added 2^-17 of their values)
          lo[h * R + r] = S::kE4m3 ? S::MM::pack(u - back.x, v - back.y)
                                   : S::MM::pack(fmaxf(u - back.x, fminf(u, S::MM::kTiny)),
                                                 fmaxf(v - back.y, fminf(v, S::MM::kTiny)));
        }
      uint32_t x[4], y[4];
      if constexpr (R == 1) {
        x[0] = hi[0];
        x[1] = lo[0];          // rows 8-15: the low terms of rows 0-7
        x[2] = hi[1];
        x[3] = lo[1];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = hi[i];
          y[i] = lo[i];
        }
      }
      if constexpr (!S::kE4m3) {
        const uint32_t at = values + (lane & 15) * S::PITCH + S::swizzled(lane, lane >> 4) * 16;
#pragma unroll
        for (int t = 0; t < S::OT; t += 2) {
          uint32_t v[4];
          dg::warp::ldmatrix_x4_trans(v, (at ^ (t * 16 & 127)) + (t * 16 & ~127) + kk * 16 * S::PITCH);
          S::MM::mma(o[t], x, v[0], v[1]);
          S::MM::mma(o[t + 1], x, v[2], v[3]);
          if constexpr (R == 2) {
            S::MM::mma(o[t], y, v[0], v[1]);
            S::MM::mma(o[t + 1], y, v[2], v[3]);
          }
        }
      } else {
        // A lane holds 8 consecutive columns 64 j + 8 g of its tokens 2 quad,
        // + 1, + 8, + 9: position g of the 8 output tiles of block j.
        const uint32_t at = values + quad * 2 * S::PITCH + S::swizzled(quad * 2, g >> 1) * 16 + (g & 1) * 8;
#pragma unroll
        for (int j = 0; j < S::DP / 64; ++j) {
          uint2 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = kk * 16 + (i & 1) + (i >> 1) * 8;        // beyond 2 quad
            const int flip = (S::swizzled(i & 1, j * 4) * 16) & 127;
            v[i] = dg::warp::ld_shared_v2((at ^ flip) + (j * 64 & ~127) + r * S::PITCH);
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            // Columns 2w and 2w + 1 of the 8, tokens paired.
            const uint32_t sel = w & 1 ? 0x7362u : 0x5140u;
            const uint32_t b0 = __byte_perm(w < 2 ? v[0].x : v[0].y, w < 2 ? v[1].x : v[1].y, sel);
            const uint32_t b1 = __byte_perm(w < 2 ? v[2].x : v[2].y, w < 2 ? v[3].x : v[3].y, sel);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t f0 = c ? dg::warp::e4m3_high(b0) : dg::warp::e4m3_low(b0);
              const uint32_t f1 = c ? dg::warp::e4m3_high(b1) : dg::warp::e4m3_low(b1);
              S::MM::mma(o[j * 8 + w * 2 + c], x, f0, f1);
              if constexpr (R == 2) S::MM::mma(o[j * 8 + w * 2 + c], y, f0, f1);
            }
          }
        }
      }
    }
  }
};

__device__ __forceinline__ float max_ref(float a, float b) { return a < b ? b : a; }
__device__ __forceinline__ float min_ref(float a, float b) { return b < a ? b : a; }

__device__ __forceinline__ void store_out(const dg_attention_args& a, long long at, float v) {
  if (a.type == DG_TYPE_BF16)
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(a.out)[at] = __float2half_rn(v);
}

// N floats of a share as one access; loads past L1, where another CTA's share
// of the launch before may lie.
template <int N>
__device__ __forceinline__ void store_pack(float* to, const float* x) {
  if constexpr (N == 4)
    *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
  else
    *reinterpret_cast<float2*>(to) = make_float2(x[0], x[1]);
}
template <int N>
__device__ __forceinline__ void load_pack(const float* from, float (&x)[N]) {
  if constexpr (N == 4) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(from));
    x[0] = v.x;
    x[1] = v.y;
    x[2] = v.z;
    x[3] = v.w;
  } else {
    const float2 v = __ldcg(reinterpret_cast<const float2*>(from));
    x[0] = v.x;
    x[1] = v.y;
  }
}

// What a finished row is multiplied with.  None of its tokens may have been
// seen (bad pages): it is 0 then, as where there are none.
__device__ __forceinline__ float inverse_sum(float m, float l) { return m == kNegInf ? 0.0f : 1.0f / l; }

// A finished row: this lane's column of each 32-column chunk, unnormalised.
template <typename S>
__device__ __forceinline__ void finish_row(const Params& p, int b, int item, int row, const float (&v)[S::CHUNKS],
                                           float m, float l, int lane) {
  const dg_attention_args& a = p.a;
  const int head = p.groups == 1 ? item : item / p.groups;
  const int in_group = (item - head * p.groups) * S::ROWS + row;
  if (in_group >= p.group) return;
  const int h = head * p.group + in_group;
  float norm = inverse_sum(m, l);
  if (S::kE4m3 && a.v_scale != nullptr) norm *= a.v_scale[head];
  const long long at = b * a.out_stride[0] + h * a.out_stride[1];
#pragma unroll
  for (int c = 0; c < S::CHUNKS; ++c) {
    const int d = S::column(c * 4 + (lane >> 3), lane & 7);
    if (d < a.head_dim) store_out(a, at + d, v[c] * norm);
  }
  if (a.lse != nullptr && lane == 0)
    a.lse[static_cast<long long>(b) * a.heads + h] = (m - S::kBias) * kLn2 + logf(l);
  if constexpr (S::DP >= 128) {
    if (a.q_out != nullptr) {
      // 128 columns are 4 chunks; quantised as the rounded bf16 values.
      const long long width = static_cast<long long>(a.heads) * a.head_dim;
#pragma unroll
      for (int blk = 0; blk < S::DP / 128; ++blk) {
        if (blk * 128 >= a.head_dim) break;
        float x[4], top = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x[c] = __bfloat162float(__float2bfloat16_rn(v[blk * 4 + c] * norm));
          top = max_ref(top, fabsf(x[c]));
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = max_ref(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float scale = max_ref(top, kQuantEps) / kFp8Max;
        uint8_t* q = static_cast<uint8_t*>(a.q_out) + b * width + static_cast<long long>(h) * a.head_dim;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float y = min_ref(max_ref(x[c] / scale, -kFp8Max), kFp8Max);
          q[S::column((blk * 4 + c) * 4 + (lane >> 3), lane & 7)] = __nv_fp8_e4m3(y).__x;
        }
        if (lane == 0) a.q_scales[(b * width + static_cast<long long>(h) * a.head_dim) / 128 + blk] = scale;
      }
    }
  }
}

// An item that this warp did alone, from its registers: 16 output tiles (128
// columns) at a time, two values of each a lane.
template <typename S>
__device__ __forceinline__ void finish_solo(const Params& p, int b, int item, const Warp<S>& w, int lane) {
  const dg_attention_args& a = p.a;
  const int head = p.groups == 1 ? item : item / p.groups;
  const int g = lane >> 2, quad = lane & 3;
  const long long width = static_cast<long long>(a.heads) * a.head_dim;
#pragma unroll
  for (int r = 0; r < Warp<S>::R; ++r) {
    float l = w.l[r];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int in_group = (item - head * p.groups) * S::ROWS + g + 8 * r;
    const bool real = in_group < p.group;
    const int h = head * p.group + in_group;
    float norm = inverse_sum(w.m[r], l);
    if (S::kE4m3 && a.v_scale != nullptr) norm *= a.v_scale[head];
    const long long at = b * a.out_stride[0] + h * a.out_stride[1];
    if (real && a.lse != nullptr && quad == 0)
      a.lse[static_cast<long long>(b) * a.heads + h] = (w.m[r] - S::kBias) * kLn2 + logf(l);
    constexpr int BLOCK = S::OT < 16 ? S::OT : 16;
#pragma unroll
    for (int t0 = 0; t0 < S::OT; t0 += BLOCK) {
      float top = 0.0f;
      float x[BLOCK][2];
#pragma unroll
      for (int t = 0; t < BLOCK; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float(&o)[4] = w.o[t0 + t];
          const float v = (Warp<S>::R == 1 ? o[i] + o[2 + i] : o[2 * r + i]) * norm;
          const int d = S::column(t0 + t, quad * 2 + i);
          if (real && d < a.head_dim) store_out(a, at + d, v);
          x[t][i] = __bfloat162float(__float2bfloat16_rn(v));
          top = max_ref(top, fabsf(x[t][i]));
        }
      if (S::DP >= 128 && a.q_out != nullptr && t0 * 8 < a.head_dim) {
        top = max_ref(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max_ref(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (!real) continue;
        const float scale = max_ref(top, kQuantEps) / kFp8Max;
        const long long q_at = b * width + static_cast<long long>(h) * a.head_dim;
#pragma unroll
        for (int t = 0; t < BLOCK; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            static_cast<uint8_t*>(a.q_out)[q_at + S::column(t0 + t, quad * 2 + i)] =
                __nv_fp8_e4m3(min_ref(max_ref(x[t][i] / scale, -kFp8Max), kFp8Max)).__x;
        if (quad == 0) a.q_scales[(q_at + t0 * 8) / 128] = scale;
      }
    }
  }
}

// Requests without live tokens, dealt over the CTAs.
template <typename S>
__device__ __forceinline__ void finish_empty(const dg_attention_args& a, int cta, int ctas, int tid) {
  const int lane = tid & 31, warp = tid >> 5;
  const long long width = static_cast<long long>(a.heads) * a.head_dim;
  for (int b = cta; b < a.batch; b += ctas) {
    if (length_of(a, b, tid == 0) != 0) continue;
    for (int h = warp; h < a.heads; h += S::NW)
      for (int d = lane; d < a.head_dim; d += 32) {
        store_out(a, b * a.out_stride[0] + h * a.out_stride[1] + d, 0.0f);
        if (a.q_out != nullptr) static_cast<uint8_t*>(a.q_out)[b * width + h * a.head_dim + d] = 0;
      }
    for (int h = tid; h < a.heads && a.lse != nullptr; h += S::NW * 32)
      a.lse[static_cast<long long>(b) * a.heads + h] = kNegInf;
    for (int i = tid; i < width / 128 && a.q_out != nullptr; i += S::NW * 32)
      a.q_scales[b * (width / 128) + i] = kQuantEps / kFp8Max;
  }
}

template <typename S>
__global__ void __launch_bounds__(S::NW * 32, 1) attention_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) unsigned char smem[];
  float* join = reinterpret_cast<float*>(smem + S::RING);               // [NW][ROWS][JOIN_COLS]
  float* warp_m = join + S::JOIN;                                       // [NW][ROWS]
  float* warp_l = warp_m + S::NW * S::ROWS;
  uint32_t* masks = reinterpret_cast<uint32_t*>(warp_l + S::NW * S::ROWS);   // [NW][STAGES]
  __shared__ long long scan_sum[S::NW];
  __shared__ long long found_base;
  __shared__ int found_request, is_last;

  dg::sm100::griddep_launch_dependents();
  dg::sm100::griddep_wait();

  const dg_attention_args& a = p.a;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  constexpr int kThreads = S::NW * 32;
  const int cta = static_cast<int>(blockIdx.x), ctas = static_cast<int>(gridDim.x);
  const int items = a.kv_heads * p.groups;

  // The line of tiles: its length, and the request where this CTA's run
  // begins.
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += units_of<S>(a, b, items);
  long long scan = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, scan, off);
    if (lane >= off) scan += v;
  }
  if (lane == 31) scan_sum[warp] = scan;
  // Columns past head_dim are never copied: zero in keys, values and q.
  if (a.head_dim < S::DP)
    for (int i = tid; i < S::RING / 16; i += kThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  long long total = 0, before = scan - mine;
#pragma unroll
  for (int w = 0; w < S::NW; ++w) {
    if (w < warp) before += scan_sum[w];
    total += scan_sum[w];
  }
  // CTAs in use, and this one's run [x0, x1) of the line.
  const int used = static_cast<int>(min(static_cast<long long>(ctas), (total + S::MIN_RUN - 1) / S::MIN_RUN));
  if (cta >= used) {
    finish_empty<S>(a, cta, ctas, tid);
    return;
  }
  const long long x0 = static_cast<long long>(divided(total * cta, used));
  const long long x1 = static_cast<long long>(divided(total * (cta + 1), used));
  if (before <= x0 && x0 < before + mine) {
    long long base = before;
    int b = b0;
    for (;; ++b) {
      const long long n = units_of<S>(a, b, items);
      if (x0 < base + n) break;
      base += n;
    }
    found_request = b;
    found_base = base;
  }
  __syncthreads();

  Cursor<S> at;
  bool run = at.start(a, found_request, found_base, x0, x1);
  Loader<S> loader;
  loader.at = at;
  loader.tile = at.first_tile(warp);
  loader.more = run;
  if (run) loader.open(p, lane);
  const uint32_t ring = dg::sm100::smem_addr(smem) + warp * (S::STAGES * S::STAGE);
  uint32_t* mask = masks + warp * S::STAGES;
  loader.prepare(p, warp, lane, items);
  if constexpr (S::HALVES) {
    loader.template issue<true, false>(p, ring, mask, lane);
    dg::warp::cp_async_commit();
    loader.template issue<false, true>(p, ring + S::STAGE, mask, lane);
    dg::warp::cp_async_commit();
    loader.prepare(p, warp, lane, items);
  } else {
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; ++i) {
      loader.template issue<true, true>(p, ring + i * S::STAGE, mask + i, lane);
      dg::warp::cp_async_commit();
      loader.prepare(p, warp, lane, items);
    }
  }

  Warp<S> w;
  int stage = 0;                            // of the tile (of its keys)
  int turn = 0;                             // tiles so far, modulo 2
  bool mine_too = run && (!at.solo || at.first_tile(warp) == 0);
  if (mine_too) w.fetch(p, at.b, at.item, lane);
  while (run) {
    const Cursor<S> share = at;
    const bool work = mine_too;
    if (work) {
      w.begin(p, share.item);
      const int step = share.step();
      for (int tile = share.first_tile(warp); tile < share.count; tile += step) {
        float s[S::NT][4];
        dg::warp::cp_async_wait<S::STAGES - 2>();
        __syncwarp();      // every lane's copies of this stage landed, every lane is done with the one before
        if constexpr (S::HALVES) {
          // Stages in turn: keys, values, the next tile's keys.
          const int values = stage == 2 ? 0 : stage + 1, next = values == 2 ? 0 : values + 1;
          loader.template issue<true, false>(p, ring + next * S::STAGE, mask + (turn ^ 1), lane);
          dg::warp::cp_async_commit();
          w.scores(p, ring + stage * S::STAGE, mask[turn], lane, s);
          dg::warp::cp_async_wait<S::STAGES - 2>();
          __syncwarp();
          loader.template issue<false, true>(p, ring + stage * S::STAGE, mask, lane);
          dg::warp::cp_async_commit();
          loader.prepare(p, warp, lane, items);
          w.weigh(ring + values * S::STAGE, lane, s);
          stage = next;
          turn ^= 1;
        } else {
          const int ahead = stage == 0 ? S::STAGES - 1 : stage - 1;
          const uint32_t from = ring + stage * S::STAGE;
          loader.template issue<true, true>(p, ring + ahead * S::STAGE, mask + ahead, lane);
          dg::warp::cp_async_commit();
          loader.prepare(p, warp, lane, items);
          w.scores(p, from, mask[stage], lane, s);
          w.weigh(from + S::KV_BYTES, lane, s);
          stage = stage == S::STAGES - 1 ? 0 : stage + 1;
        }
      }
    }
    // The next share's q is on its way during the join.
    run = at.advance(a, items);
    mine_too = run && (!at.solo || at.first_tile(warp) == 0);
    if (mine_too) w.fetch(p, at.b, at.item, lane);
    if (share.solo) {
      if (work) finish_solo<S>(p, share.b, share.item, w, lane);
      continue;
    }

    // Join the warps.
    const int g = lane >> 2, quad = lane & 3;
#pragma unroll
    for (int r = 0; r < Warp<S>::R; ++r) {
      float l = w.l[r];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (quad == 0) {
        warp_m[warp * S::ROWS + g + 8 * r] = w.m[r];
        warp_l[warp * S::ROWS + g + 8 * r] = l;
      }
    }
    __syncthreads();
    float mine_by[Warp<S>::R];              // this warp's weight in the joined rows
#pragma unroll
    for (int r = 0; r < Warp<S>::R; ++r) {
      float top = kNegInf;
#pragma unroll
      for (int v = 0; v < S::NW; ++v) top = fmaxf(top, warp_m[v * S::ROWS + g + 8 * r]);
      mine_by[r] = w.m[r] == kNegInf ? 0.0f : dg::warp::exp2_approx(w.m[r] - top);
    }
    float row_m[S::RPT], row_l[S::RPT], sum[S::RPT][S::CHUNKS];
#pragma unroll
    for (int i = 0; i < S::RPT; ++i) {
      const int row = warp + i * S::NW;
      if (row >= S::ROWS) break;
      float top = kNegInf, l = 0.0f;
#pragma unroll
      for (int v = 0; v < S::NW; ++v) top = fmaxf(top, warp_m[v * S::ROWS + row]);
#pragma unroll
      for (int v = 0; v < S::NW; ++v) {
        const float mv = warp_m[v * S::ROWS + row];
        if (mv != kNegInf) l += warp_l[v * S::ROWS + row] * dg::warp::exp2_approx(mv - top);
      }
      row_m[i] = top;
      row_l[i] = l;
    }
    // Column x of row r stands at x ^ 8 (r % 4): neither the writes (4 rows, 8
    // columns each) nor the reads (32 columns of a row) meet in a bank.
    constexpr int ROUND_CHUNKS = S::JOIN_COLS / 32;
#pragma unroll
    for (int c0 = 0; c0 < S::CHUNKS; c0 += ROUND_CHUNKS) {
      if (c0 != 0) __syncthreads();
#pragma unroll
      for (int t = 0; t < ROUND_CHUNKS * 4; ++t) {
        const float(&o)[4] = w.o[c0 * 4 + t];
        float* dst = join + (warp * S::ROWS + g) * S::JOIN_COLS + ((t * 8 + quad * 2) ^ ((g & 3) * 8));
        if constexpr (S::ROWS == 8) {
          *reinterpret_cast<float2*>(dst) = make_float2((o[0] + o[2]) * mine_by[0], (o[1] + o[3]) * mine_by[0]);
        } else {
          *reinterpret_cast<float2*>(dst) = make_float2(o[0] * mine_by[0], o[1] * mine_by[0]);
          *reinterpret_cast<float2*>(dst + 8 * S::JOIN_COLS) =
              make_float2(o[2] * mine_by[Warp<S>::R - 1], o[3] * mine_by[Warp<S>::R - 1]);
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < S::RPT; ++i) {
        const int row = warp + i * S::NW;
        if (row >= S::ROWS) break;
#pragma unroll
        for (int c = 0; c < ROUND_CHUNKS; ++c) {
          float v = 0.0f;
#pragma unroll
          for (int u = 0; u < S::NW; ++u)
            v += join[(u * S::ROWS + row) * S::JOIN_COLS + ((c * 32 + lane) ^ ((row & 3) * 8))];
          sum[i][c0 + c] = v;
        }
      }
    }

    const int n_tiles = share.tiles;
    if (share.count == n_tiles) {              // the whole item
#pragma unroll
      for (int i = 0; i < S::RPT; ++i)
        if (warp + i * S::NW < S::ROWS)
          finish_row<S>(p, share.b, share.item, warp + i * S::NW, sum[i], row_m[i], row_l[i], lane);
      continue;
    }

    // A share: to the workspace, slot 2c for an item that began in an earlier
    // CTA, 2c + 1 for one that begins here.
    const size_t slot = 2 * static_cast<size_t>(cta) + (share.t0 == 0 ? 1 : 0);
#pragma unroll
    for (int i = 0; i < S::RPT; ++i) {
      const int row = warp + i * S::NW;
      if (row >= S::ROWS) break;
      // A lane's columns side by side.
      float* dst = p.share_o + (slot * kMaxRows + row) * kMaxDim + lane * S::CHUNKS;
#pragma unroll
      for (int c = 0; c < S::CHUNKS; c += S::PACK) store_pack<S::PACK>(dst + c, &sum[i][c]);
      if (lane == 0) p.share_ml[slot * kMaxRows + row] = make_float2(row_m[i], row_l[i]);
    }
    // The CTAs of the item: those that own its first and its last tile.
    const long long first_unit = x0 + share.x + extra_of<S>(n_tiles);
    const int c0 = static_cast<int>(divided((first_unit + 1) * used - 1, total));
    const int c1 = static_cast<int>(divided((first_unit + n_tiles) * used - 1, total));
    const int n = c1 - c0 + 1;
    __syncthreads();
    if (tid == 0) {                         // releases the CTA's share, acquires the others'
      const int seen = dg::sm100::atomic_add_acq_rel_gpu(p.tickets + c0, 1);
      is_last = seen == n - 1;
      if (seen == n - 1) dg::sm100::store_relaxed_gpu(p.tickets + c0, 0);   // ready for the next launch
    }
    __syncthreads();
    if (is_last == 0) continue;

    // Join the shares, in CTA order.
    float* by = join;                       // [ROWS][kMaxCtas] weights
#pragma unroll
    for (int i = 0; i < S::RPT; ++i) {
      const int row = warp + i * S::NW;
      if (row >= S::ROWS) break;
      constexpr int PER_LANE = (kMaxCtas + 31) / 32;
      float2 ml[PER_LANE];
      float top = kNegInf;
#pragma unroll
      for (int k = 0; k < PER_LANE; ++k) {
        const int c = lane + k * 32;
        const size_t from = 2 * static_cast<size_t>(c0 + c) + (c == 0 ? 1 : 0);
        ml[k] = c < n ? __ldcg(p.share_ml + from * kMaxRows + row) : make_float2(kNegInf, 0.0f);
      }
#pragma unroll
      for (int k = 0; k < PER_LANE; ++k) top = fmaxf(top, ml[k].x);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      float l = 0.0f;
#pragma unroll
      for (int k = 0; k < PER_LANE; ++k) {
        const float f = ml[k].x == kNegInf ? 0.0f : dg::warp::exp2_approx(ml[k].x - top);
        if (lane + k * 32 < n) by[row * kMaxCtas + lane + k * 32] = f;
        l += f * ml[k].y;
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
      __syncwarp();
      float v[S::CHUNKS];
#pragma unroll
      for (int c = 0; c < S::CHUNKS; ++c) v[c] = 0.0f;
#pragma unroll 8
      for (int c = 0; c < n; ++c) {
        const size_t from = 2 * static_cast<size_t>(c0 + c) + (c == 0 ? 1 : 0);
        const float* src = p.share_o + (from * kMaxRows + row) * kMaxDim + lane * S::CHUNKS;
        const float f = by[row * kMaxCtas + c];
#pragma unroll
        for (int k = 0; k < S::CHUNKS; k += S::PACK) {
          float x[S::PACK];
          load_pack<S::PACK>(src + k, x);
#pragma unroll
          for (int j = 0; j < S::PACK; ++j) v[k + j] += f * x[j];
        }
      }
      finish_row<S>(p, share.b, share.item, row, v, top, l, lane);
    }
    __syncthreads();                        // the join buffers and is_last are free again
  }
  dg::warp::cp_async_wait<0>();
  finish_empty<S>(a, cta, ctas, tid);
}

using Kernel = void (*)(const Params);

struct Entry {
  Kernel fn;
  size_t smem;
  int threads, rows, tok;
  std::atomic<unsigned long long> ready;    // per device: shared memory limit raised
};

template <typename S>
Entry& entry() {
  static Entry e{attention_kernel<S>, S::SMEM, S::NW * 32, S::ROWS, S::TOK, {0}};
  return e;
}

template <typename MM, bool E4M3, int DP>
Entry& pick_rows(bool few) {
  return few ? entry<Shape<MM, E4M3, DP, 8>>() : entry<Shape<MM, E4M3, DP, 16>>();
}

Entry& pick(const dg_attention_args& a, bool few) {
  const int d = a.head_dim;
  if (a.cache_type == DG_TYPE_E4M3) return d <= 128 ? pick_rows<Fp16, true, 128>(few) : pick_rows<Fp16, true, 256>(few);
  if (a.cache_type == DG_TYPE_FP16)
    return d <= 64 ? pick_rows<Fp16, false, 64>(few)
                   : d <= 128 ? pick_rows<Fp16, false, 128>(few) : pick_rows<Fp16, false, 256>(few);
  return d <= 64 ? pick_rows<Bf16, false, 64>(few)
                 : d <= 128 ? pick_rows<Bf16, false, 128>(few) : pick_rows<Bf16, false, 256>(few);
}

bool refused(const dg_attention_args& a) {
  if (a.batch < 1 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0 || a.page_size < 1 ||
      a.num_pages < 1 || a.table_width < 1 || a.table_stride < a.table_width || a.window < 0)
    return true;
  if (a.type != DG_TYPE_BF16 && a.type != DG_TYPE_FP16) return true;
  const bool e4m3 = a.cache_type == DG_TYPE_E4M3;
  if (!e4m3 && a.cache_type != a.type) return true;
  if (a.head_dim < 8 || a.head_dim > kMaxDim || a.head_dim % (e4m3 ? 16 : 8) != 0) return true;
  if (a.q == nullptr || a.k_cache == nullptr || a.v_cache == nullptr || a.block_table == nullptr ||
      a.seq_lens == nullptr || a.out == nullptr || a.workspace == nullptr)
    return true;
  if (!e4m3 && (a.k_scale != nullptr || a.v_scale != nullptr)) return true;
  if (!(a.softcap >= 0.0f) || !(a.scale == a.scale)) return true;
  if ((reinterpret_cast<uintptr_t>(a.q) & 3u) != 0 || a.q_stride[0] % 2 != 0 || a.q_stride[1] % 2 != 0) return true;
  if (((reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache)) & 15u) != 0) return true;
  if ((reinterpret_cast<uintptr_t>(a.out) & 1u) != 0) return true;
  const void* words[] = {a.block_table, a.seq_lens, a.k_scale, a.v_scale, a.lse, a.q_scales, a.status};
  for (const void* p : words)
    if ((reinterpret_cast<uintptr_t>(p) & 3u) != 0) return true;
  for (int i = 0; i < 3; ++i)
    if (a.k_cache_stride[i] % (e4m3 ? 16 : 8) != 0 || a.v_cache_stride[i] % (e4m3 ? 16 : 8) != 0) return true;
  if ((a.q_out != nullptr) != (a.q_scales != nullptr)) return true;
  if (a.q_out != nullptr && (a.head_dim % 128 != 0 || a.type != DG_TYPE_BF16)) return true;
  if (a.workspace_bytes < kWorkspaceBytes || (reinterpret_cast<uintptr_t>(a.workspace) & 15u) != 0) return true;
  // Items a request and tiles an item stay within ints.
  if (static_cast<long long>(a.heads) > (1 << 20)) return true;
  return false;
}

}  // namespace

extern "C" {

unsigned long long dg_attention_workspace_bytes(void) { return kWorkspaceBytes; }

int dg_paged_attention(const dg_attention_args* args, void* stream, int pdl_attr) {
  if (args == nullptr || refused(*args)) return cudaErrorInvalidValue;
  Params p{};
  p.a = *args;
  // Caps below 2^-100 leave nothing of a score and those above take nothing
  // from it; in between their quotients and products stay finite.
  if (p.a.softcap > 0.0f)
    p.a.softcap = p.a.softcap < 0x1p-100f ? 0x1p-100f : p.a.softcap > 0x1p100f ? 0x1p100f : p.a.softcap;
  p.group = p.a.heads / p.a.kv_heads;
  Entry& e = pick(p.a, p.group <= 8);
  p.groups = (p.group + e.rows - 1) / e.rows;
  p.page_shift = -1;
  if ((p.a.page_size & (p.a.page_size - 1)) == 0) {
    p.page_shift = 0;
    while ((1 << p.page_shift) < p.a.page_size) ++p.page_shift;
  }
  p.aligned = p.a.page_size % e.tok == 0 ? 1 : 0;
  unsigned char* ws = static_cast<unsigned char*>(p.a.workspace);
  p.tickets = reinterpret_cast<int*>(ws);
  p.share_ml = reinterpret_cast<float2*>(ws + kTicketBytes);
  p.share_o = reinterpret_cast<float*>(ws + kTicketBytes + kShares * kMaxRows * sizeof(float2));

  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const unsigned long long bit = 1ull << (dev & 63);
  if ((e.ready.load(std::memory_order_acquire) & bit) == 0) {
    err = cudaFuncSetAttribute(e.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(e.smem));
    if (err != cudaSuccess) return err;
    e.ready.fetch_or(bit, std::memory_order_release);
  }
  int ctas = dg_num_sms();
  if (ctas < 1) ctas = 148;
  if (ctas > kMaxCtas) ctas = kMaxCtas;

  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1]{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(e.threads), 1, 1);
  cfg.dynamicSmemBytes = e.smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (pdl_attr) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, e.fn, p);
}

}  // extern "C"
