// SPDX-License-Identifier: MIT
//
// dg_rotary.cu -- rotary positions with several axes (forward and inverse)
// and the write of keys and values into a paged cache
// (include/decode_attention_b200.h gives the definition).
//
// Pure traffic: every value is read once and written once, 3 multiply-adds a
// pair.  A "row" is one head of one token's q, k or v, a "unit" of it 2 * VE
// values: the two 16-byte vectors whose values pair up, so that a rotation
// never crosses threads and an output may be its input.  A thread keeps one
// unit and takes rows in steps, so that neighbouring lanes read neighbouring
// vectors whatever the head counts are, and has the next row's vectors on the
// way while it turns one.  cos and sin are fetched once per token and pair
// into shared memory -- the axes differ from pair to pair, so this is a
// gather -- and serve all heads from there; a CTA takes several tokens, so that
// the three loads that follow one another before its first product (position,
// table, value) are waited for once.  With few tokens a token's rows are dealt
// over several CTAs, one row a thread.
//
// B200: 32768 tokens of 64 + 8 + 8 heads of 128, bf16, rotated and written
// into the cache in 212 us, 6.4 TB/s: the rate of a plain copy.
//
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "decode_attention_b200.h"
#include "decode_gemm_b200.h"
#include "sm100.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxThreads = 1024;        // a head of 2048 values, one by one
constexpr int kCtasPerSm = 5;            // 48 registers a thread (32768 tokens of 80 heads: 212 us; 4 CTAs 224)
constexpr int kRowsPerThread = 8;        // wanted, with tokens enough
constexpr int kMaxTokens = 64;           // of a CTA
constexpr int kMaxTrig = 4096;           // floats of cos and sin of a CTA's tokens (16 KiB)

struct E4m3 {
  uint8_t bits;
};

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ void from_float(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_float(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_float(float& d, float v) { d = v; }
// Saturating (+-448), to nearest even, NaN stays NaN.
__device__ __forceinline__ void from_float(E4m3& d, float v) {
  d.bits = static_cast<uint8_t>(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3));
}
__device__ __forceinline__ uint16_t e4m3_pair(float lo, float hi) {
  return static_cast<uint16_t>(__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3));
}

// N values as one access, 16-bit ones in pairs: the compiler keeps what is on
// its way packed (as single values, bf16 took 16 registers more).
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};
template <int N>
struct alignas(4 * N) Words {
  uint32_t w[N];
};
template <typename T, int N>
struct Packed {
  static constexpr bool kPairs = sizeof(T) == 2 && N % 2 == 0;
  typename std::conditional<kPairs, Words<(N + 1) / 2>, Vec<T, N>>::type raw;
};

__device__ __forceinline__ float2 pair_of(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 pair_of(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pair_from(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pair_from(float lo, float hi, __half) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

template <typename T, int N>
__device__ __forceinline__ Packed<T, N> load(const T* p) {
  return *reinterpret_cast<const Packed<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ void unpack(const Packed<T, N>& p, float (&x)[N]) {
  if constexpr (Packed<T, N>::kPairs) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 f = pair_of(p.raw.w[i], T{});
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float(p.raw.v[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float (&x)[N]) {
  if constexpr (Packed<T, N>::kPairs) {
    Words<(N + 1) / 2> o;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) o.w[i] = pair_from(x[2 * i], x[2 * i + 1], T{});
    *reinterpret_cast<Words<(N + 1) / 2>*>(p) = o;
  } else if constexpr (std::is_same<T, E4m3>::value && N % 2 == 0) {
    Vec<uint16_t, N / 2> o;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) o.v[i] = e4m3_pair(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<Vec<uint16_t, N / 2>*>(p) = o;
  } else {
    Vec<T, N> o;
#pragma unroll
    for (int i = 0; i < N; ++i) from_float(o.v[i], x[i]);
    *reinterpret_cast<Vec<T, N>*>(p) = o;
  }
}

// (u, w) turned.  Which product is rounded is spelled out, so that every
// variant of the kernel gives the same bits.
__device__ __forceinline__ void turn(float& x, float& y, float u, float w, float c, float s) {
  x = __fmaf_rn(-w, s, __fmul_rn(u, c));
  y = __fmaf_rn(u, s, __fmul_rn(w, c));
}

struct Geometry {
  int units;              // units a row
  int rows;               // rows a token: heads + kv_heads (k) + kv_heads (v)
  int slots;              // rows that a CTA's threads cover at once
  int tokens;             // tokens a CTA takes
  int pieces;             // CTAs that a token's rows are dealt over (tokens == 1)
  // Byte strides (token, head): a row's address is two 32 x 32 -> 64 bit
  // multiply-adds.
  int q[2], k[2], v[2], q_out[2], k_out[2];
};

template <typename P>
__device__ __forceinline__ P* at(P* base, int t, int token_stride, int row, int head_stride) {
  using Byte = typename std::conditional<std::is_const<P>::value, const char, char>::type;
  return reinterpret_cast<P*>(reinterpret_cast<Byte*>(base) + static_cast<long long>(t) * token_stride +
                              static_cast<long long>(row) * head_stride);
}

// kThreads threads, or for heads of more than 2 * kThreads values that are
// taken one by one, as many as a row has units.
template <typename T, typename C, int VE, bool HALF>
__global__ void __launch_bounds__(VE == 1 ? kMaxThreads : kThreads, VE == 1 ? 1 : kCtasPerSm)
    rotary_kernel(const __grid_constant__ dg_rotary_args a, const __grid_constant__ Geometry g) {
  constexpr bool kCached = !std::is_same<C, void>::value;
  __shared__ __align__(16) float trig[kMaxTrig];     // [token][cos of rot/2 pairs, sin of rot/2 pairs]
  __shared__ int2 place[kMaxTokens];                 // cache page and offset, page -1: none

  dg::sm100::griddep_launch_dependents();
  dg::sm100::griddep_wait();

  const int tid = static_cast<int>(threadIdx.x);
  const int slot = tid / g.units, unit = tid - slot * g.units;
  const unsigned group = blockIdx.x / static_cast<unsigned>(g.pieces);
  const int piece = static_cast<int>(blockIdx.x - group * static_cast<unsigned>(g.pieces));
  const int t0 = static_cast<int>(group) * g.tokens;
  const int tokens = min(g.tokens, a.tokens - t0);
  const int half = a.rot >> 1;
  const int q_rows = a.heads, qk_rows = a.heads + a.kv_heads;
  const bool rotates = unit < a.rot / (2 * VE);
  // A unit's two vectors in a row that turns, and in one that passes (v).
  const int first_r = rotates && HALF ? unit * VE : unit * 2 * VE;
  const int second_r = rotates && HALF ? first_r + half : first_r + VE;
  const int first_v = unit * 2 * VE, second_v = first_v + VE;

  auto fetch = [&](int tok, int row, Packed<T, VE>& lo, Packed<T, VE>& hi) {
    const bool is_q = row < q_rows, is_v = row >= qk_rows;
    const T* src = at(static_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k), t0 + tok,
                      is_q ? g.q[0] : is_v ? g.v[0] : g.k[0], row - (is_q ? 0 : is_v ? qk_rows : q_rows),
                      is_q ? g.q[1] : is_v ? g.v[1] : g.k[1]);
    const int second = is_v ? second_v : second_r;
    lo = load<T, VE>(src + (is_v ? first_v : first_r));
    if (second < a.head_dim) hi = load<T, VE>(src + second);
  };
  // (tok, row) -> this thread's next.
  const int step = g.slots * g.pieces;
  auto next = [&](int& tok, int& row) {
    row += step;
    while (row >= g.rows && tok < tokens) {
      row -= g.rows;
      ++tok;
    }
  };

  int tok = 0, row = slot + piece * g.slots - step;
  next(tok, row);
  if (g.pieces > 1 && tok > 0) tok = tokens;         // a dealt token's rows are done in one round
  const bool idle = slot >= g.slots;
  Packed<T, VE> lo{}, hi{};
  if (!idle && tok < tokens) fetch(tok, row, lo, hi);

  for (int i = tid; i < tokens * half; i += static_cast<int>(blockDim.x)) {
    const int tk = i / half, pair = i - tk * half;
    const int axis = (a.axis_of[pair >> 4] >> ((pair & 15) * 2)) & 3;
    const long long from = axis * a.position_stride + t0 + tk;
    const long long p = a.position_64 != 0 ? static_cast<const long long*>(a.positions)[from]
                                           : static_cast<const int*>(a.positions)[from];
    float c = __int_as_float(0x7fffffff), s = c;     // NaN
    if (p >= 0 && p < a.max_position) {
      c = a.cos_sin[p * a.rot + pair];
      s = a.cos_sin[p * a.rot + half + pair];
    } else if (a.status != nullptr) {
      atomicCAS(a.status, 0, DG_ERR_POSITION);
    }
    trig[tk * a.rot + pair] = c;
    trig[tk * a.rot + half + pair] = a.inverse != 0 ? -s : s;
  }
  if constexpr (kCached) {
    for (int i = tid; i < tokens; i += static_cast<int>(blockDim.x)) {
      const long long row_at = a.slots[t0 + i];
      long long page = -1, offset = 0;
      if (row_at >= static_cast<long long>(a.num_pages) * a.page_size) {
        if (a.status != nullptr) atomicCAS(a.status, 0, DG_ERR_SLOT);
      } else if (row_at >= 0) {
        page = (row_at >> 32) == 0 ? static_cast<unsigned>(row_at) / static_cast<unsigned>(a.page_size)
                                   : row_at / a.page_size;
        offset = row_at - page * a.page_size;
      }
      place[i] = make_int2(static_cast<int>(page), static_cast<int>(offset));
    }
  }
  __syncthreads();
  if (idle) return;

  while (tok < tokens) {
    const int r = row, tk = tok;
    const bool is_q = r < q_rows, is_v = r >= qk_rows;
    const int first = is_v ? first_v : first_r, second = is_v ? second_v : second_r;
    const bool both = second < a.head_dim;           // a row's last passing vector can stand alone
    float x[VE], y[VE];
    unpack<T, VE>(lo, x);
    unpack<T, VE>(hi, y);
    next(tok, row);
    if (g.pieces > 1) tok = tokens;
    if (tok < tokens) fetch(tok, row, lo, hi);

    if (rotates && !is_v) {
      float c[VE], s[VE];
      const float* cs = trig + tk * a.rot + unit * VE;
      constexpr int W = VE < 4 ? VE : 4;
#pragma unroll
      for (int j = 0; j < VE; j += W) {
        const Vec<float, W> u = *reinterpret_cast<const Vec<float, W>*>(cs + j);
        const Vec<float, W> w = *reinterpret_cast<const Vec<float, W>*>(cs + half + j);
#pragma unroll
        for (int l = 0; l < W; ++l) {
          c[j + l] = u.v[l];
          s[j + l] = w.v[l];
        }
      }
      if constexpr (HALF) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float u = x[j], w = y[j];
          turn(x[j], y[j], u, w, c[j], s[j]);
        }
      } else {
        // 2 * VE consecutive values: pair j is values 2j and 2j + 1.
        float z[2 * VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          z[j] = x[j];
          z[VE + j] = y[j];
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float u = z[2 * j], w = z[2 * j + 1];
          turn(z[2 * j], z[2 * j + 1], u, w, c[j], s[j]);
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          x[j] = z[j];
          y[j] = z[VE + j];
        }
      }
    }
    if (is_q || (!is_v && a.k_out != nullptr)) {
      T* dst = at(static_cast<T*>(is_q ? a.q_out : a.k_out), t0 + tk, is_q ? g.q_out[0] : g.k_out[0],
                  is_q ? r : r - q_rows, is_q ? g.q_out[1] : g.k_out[1]);
      store<T, VE>(dst + first, x);
      if (both) store<T, VE>(dst + second, y);
    }
    if constexpr (kCached) {
      const int2 where = place[tk];
      if (is_q || where.x < 0) continue;
      const int head = r - (is_v ? qk_rows : q_rows);
      const long long* st = is_v ? a.v_cache_stride : a.k_cache_stride;
      C* cache = static_cast<C*>(is_v ? a.v_cache : a.k_cache) + where.x * st[0] + where.y * st[1] +
                 head * st[2];
      if constexpr (std::is_same<C, E4m3>::value) {
        const float* scales = is_v ? a.v_scale : a.k_scale;
        if (scales != nullptr) {
          const float scale = scales[head];
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            x[j] = x[j] / scale;
            y[j] = y[j] / scale;
          }
        }
      }
      store<C, VE>(cache + first, x);
      if (both) store<C, VE>(cache + second, y);
    }
  }
}

bool multiple(long long stride, int n) { return stride % n == 0; }

// Byte strides of one tensor as ints; false where they do not fit.
bool bytes_of(const void* p, const long long (&stride)[2], int size, int (&out)[2]) {
  for (int i = 0; i < 2; ++i) {
    const long long b = p == nullptr ? 0 : stride[i] * size;
    if (b < 0 || b > 0x7fffffffLL) return false;
    out[i] = static_cast<int>(b);
  }
  return true;
}

// Whether every access can be `ve` values wide.
bool fits(const dg_rotary_args& a, int ve, int size, int cache_size) {
  if ((a.rot / 2) % ve != 0 || a.head_dim % ve != 0) return false;
  const void* p[5] = {a.q, a.k, a.v, a.q_out, a.k_out};
  const long long* s[5] = {a.q_stride, a.k_stride, a.v_stride, a.q_out_stride, a.k_out_stride};
  for (int i = 0; i < 5; ++i) {
    if (p[i] == nullptr) continue;
    if (reinterpret_cast<uintptr_t>(p[i]) % static_cast<uintptr_t>(ve * size) != 0) return false;
    if (!multiple(s[i][0], ve) || !multiple(s[i][1], ve)) return false;
  }
  if (a.k_cache != nullptr) {
    const void* c[2] = {a.k_cache, a.v_cache};
    const long long* cs[2] = {a.k_cache_stride, a.v_cache_stride};
    for (int i = 0; i < 2; ++i) {
      if (reinterpret_cast<uintptr_t>(c[i]) % static_cast<uintptr_t>(ve * cache_size) != 0) return false;
      for (int j = 0; j < 3; ++j)
        if (!multiple(cs[i][j], ve)) return false;
    }
  }
  return true;
}

using Kernel = void (*)(const dg_rotary_args, const Geometry);

template <typename T, int VE, bool HALF>
Kernel pick_pairing(const dg_rotary_args& a) {
  if (a.k_cache == nullptr) return rotary_kernel<T, void, VE, HALF>;
  if constexpr (!std::is_same<T, float>::value) {
    if (a.cache_type == DG_TYPE_E4M3) return rotary_kernel<T, E4m3, VE, HALF>;
    return rotary_kernel<T, T, VE, HALF>;
  } else {
    return nullptr;
  }
}

template <typename T, int VE>
Kernel pick_cache(const dg_rotary_args& a) {
  return a.pairing == DG_PAIR_HALF ? pick_pairing<T, VE, true>(a) : pick_pairing<T, VE, false>(a);
}

// 16 bytes a vector where everything is aligned for it; 8 bytes serve rotated
// widths that are a multiple of 8 only (40 of a head of 80); else one by one.
template <typename T>
Kernel pick(const dg_rotary_args& a, int cache_size, int* ve) {
  constexpr int kWide = 16 / static_cast<int>(sizeof(T));
  *ve = kWide;
  if (fits(a, kWide, sizeof(T), cache_size)) return pick_cache<T, kWide>(a);
  if constexpr (kWide == 8) {
    *ve = 4;
    if (fits(a, 4, sizeof(T), cache_size)) return pick_cache<T, 4>(a);
  }
  *ve = 1;
  return pick_cache<T, 1>(a);
}

bool refused(const dg_rotary_args& a) {
  if (a.tokens < 1 || a.heads < 0 || a.kv_heads < 0 || a.heads + a.kv_heads < 1 || a.head_dim < 2 || a.head_dim > 2 * kMaxThreads || a.rot < 2 ||
      a.rot % 2 != 0 || a.rot > a.head_dim || a.rot > DG_MAX_ROT || a.max_position < 1)
    return true;
  if (a.type != DG_TYPE_BF16 && a.type != DG_TYPE_FP16 && a.type != DG_TYPE_FP32) return true;
  if (a.pairing != DG_PAIR_HALF && a.pairing != DG_PAIR_ADJACENT) return true;
  if (a.positions == nullptr || a.cos_sin == nullptr || a.position_stride < 0) return true;
  if ((a.heads > 0) != (a.q != nullptr) || (a.q != nullptr) != (a.q_out != nullptr)) return true;
  if ((a.kv_heads > 0) != (a.k != nullptr)) return true;
  const uintptr_t value = a.type == DG_TYPE_FP32 ? 3 : 1, place = a.position_64 != 0 ? 7 : 3;
  const void* values[] = {a.q, a.k, a.v, a.q_out, a.k_out};
  for (const void* p : values)
    if ((reinterpret_cast<uintptr_t>(p) & value) != 0) return true;
  const void* words[] = {a.cos_sin, a.k_scale, a.v_scale, a.status};
  for (const void* p : words)
    if ((reinterpret_cast<uintptr_t>(p) & 3u) != 0) return true;
  if ((reinterpret_cast<uintptr_t>(a.positions) & place) != 0) return true;
  const bool cached = a.k_cache != nullptr;
  if (cached != (a.v_cache != nullptr) || cached != (a.v != nullptr)) return true;
  if (a.k != nullptr && a.k_out == nullptr && !cached) return true;
  if (a.k == nullptr && (a.k_out != nullptr || cached)) return true;
  if (cached) {
    if (a.slots == nullptr || a.page_size < 1 || a.num_pages < 1) return true;
    if (a.type == DG_TYPE_FP32 || (a.cache_type != a.type && a.cache_type != DG_TYPE_E4M3)) return true;
    if ((reinterpret_cast<uintptr_t>(a.slots) & 7u) != 0) return true;
    if (a.cache_type != DG_TYPE_E4M3 &&
        ((reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache)) & 1u) != 0)
      return true;
    if (a.cache_type != DG_TYPE_E4M3 && (a.k_scale != nullptr || a.v_scale != nullptr)) return true;
  }
  return false;
}

}  // namespace

extern "C" int dg_rotary(const dg_rotary_args* args, void* stream, int pdl_attr) {
  if (args == nullptr || refused(*args)) return cudaErrorInvalidValue;
  const dg_rotary_args& a = *args;
  int ve = 1;
  const int cache_size = a.cache_type == DG_TYPE_E4M3 ? 1 : 2;
  const Kernel fn = a.type == DG_TYPE_FP32 ? pick<float>(a, cache_size, &ve)
                    : a.type == DG_TYPE_FP16 ? pick<__half>(a, cache_size, &ve)
                                             : pick<__nv_bfloat16>(a, cache_size, &ve);
  if (fn == nullptr) return cudaErrorInvalidValue;

  Geometry g;
  const int size = a.type == DG_TYPE_FP32 ? 4 : 2;
  if (!bytes_of(a.q, a.q_stride, size, g.q) || !bytes_of(a.k, a.k_stride, size, g.k) ||
      !bytes_of(a.v, a.v_stride, size, g.v) || !bytes_of(a.q_out, a.q_out_stride, size, g.q_out) ||
      !bytes_of(a.k_out, a.k_out_stride, size, g.k_out))
    return cudaErrorInvalidValue;
  const long long rows = static_cast<long long>(a.heads) + a.kv_heads + (a.v != nullptr ? a.kv_heads : 0);
  if (rows > (1 << 24)) return cudaErrorInvalidValue;
  g.units = (a.head_dim + 2 * ve - 1) / (2 * ve);
  const int threads = g.units <= kThreads ? kThreads : (g.units + 31) / 32 * 32;
  g.rows = static_cast<int>(rows);
  g.slots = threads / g.units;
  // A decode step has fewer tokens than the GPU has SMs: one row a thread
  // then, so that its latency is one row's.  Else whole tokens, about
  // kRowsPerThread rows a thread, in whole waves of the GPU.
  const int sms = dg_num_sms() > 0 ? dg_num_sms() : 148;
  g.pieces = 1;
  g.tokens = 1;
  if (a.tokens <= 2 * sms) {
    g.pieces = (g.rows + g.slots - 1) / g.slots;
  } else {
    const long long wanted = (static_cast<long long>(g.slots) * kRowsPerThread + g.rows - 1) / g.rows;
    const long long places = static_cast<long long>(sms) * kCtasPerSm;
    long long waves = a.tokens / (places * wanted);
    if (waves < 1) waves = 1;
    const long long tokens = (a.tokens + places * waves - 1) / (places * waves);
    g.tokens = static_cast<int>(tokens < kMaxTokens ? tokens : kMaxTokens);
    if (g.tokens > kMaxTrig / a.rot) g.tokens = kMaxTrig / a.rot;
    if (g.tokens < 1) g.tokens = 1;
  }
  const long long groups = (static_cast<long long>(a.tokens) + g.tokens - 1) / g.tokens;
  const long long ctas = groups * g.pieces;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;

  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1]{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (pdl_attr) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, fn, a, g);
}
