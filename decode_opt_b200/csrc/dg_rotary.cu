// SPDX-License-Identifier: MIT
//
// dg_rotary.cu -- rotary positions with several axes (forward and inverse)
// and the write of keys and values into a paged cache
// (include/decode_attention_b200.h gives the definition).
//
// Pure traffic: every value is read once and written once, 3 multiply-adds a
// pair.  The unit of work ("task") is 2 * VE values of one row (a row = one
// head of one token's q, k or v): the two 16-byte vectors whose values pair
// up, so that a rotation never crosses threads and an output may be its
// input.  Tasks are numbered through a token's rows and a CTA takes a group
// of whole tokens (or, with few tokens, a piece of one), so that neighbouring
// lanes read neighbouring vectors whatever the head counts are.  cos and sin
// are fetched once per token and pair into shared memory -- the axes differ
// from pair to pair, so this is a gather -- and serve all heads from there.

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
constexpr int kMaxTableFloats = 8192;    // cos and sin of one CTA's tokens (32 KiB)

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

// N values as one access.
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load(const T* p) {
  return *reinterpret_cast<const Vec<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float (&x)[N]) {
  Vec<T, N> o;
#pragma unroll
  for (int i = 0; i < N; ++i) from_float(o.v[i], x[i]);
  *reinterpret_cast<Vec<T, N>*>(p) = o;
}

struct Geometry {
  int tokens_per_cta;     // whole tokens a CTA takes
  int units;              // tasks a row
  int tasks;              // tasks a token
  int pieces;             // CTAs a token is split over (tokens_per_cta == 1)
  int rows;               // rows a token: heads + kv_heads (k) + kv_heads (v)
};

template <typename T, typename C, int VE>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ dg_rotary_args a,
                                                          const Geometry g) {
  __shared__ __align__(16) float trig[kMaxTableFloats];
  dg::sm100::griddep_launch_dependents();
  dg::sm100::griddep_wait();

  const int tid = static_cast<int>(threadIdx.x);
  const int half = a.rot >> 1;
  const int group = static_cast<int>(blockIdx.x / static_cast<unsigned>(g.pieces));
  const int piece = static_cast<int>(blockIdx.x - static_cast<unsigned>(group) * static_cast<unsigned>(g.pieces));
  const int t0 = group * g.tokens_per_cta;
  const int tokens = min(g.tokens_per_cta, a.tokens - t0);

  // trig[token][0, half) = cos, [half, rot) = +-sin of that pair's axis.
  for (int i = tid; i < tokens * half; i += kThreads) {
    const int tok = i / half, pair = i - tok * half;
    const int axis = (a.axis_of[pair >> 4] >> ((pair & 15) * 2)) & 3;
    const long long at = axis * a.position_stride + t0 + tok;
    const long long p = a.position_64 != 0 ? static_cast<const long long*>(a.positions)[at]
                                           : static_cast<const int*>(a.positions)[at];
    float c = __int_as_float(0x7fffffff), s = c;     // NaN
    if (p >= 0 && p < a.max_position) {
      const float* row = a.cos_sin + p * a.rot;
      c = __ldg(row + pair);
      s = __ldg(row + half + pair);
    } else if (a.status != nullptr) {
      atomicCAS(a.status, 0, DG_ERR_POSITION);
    }
    trig[tok * a.rot + pair] = c;
    trig[tok * a.rot + half + pair] = a.inverse != 0 ? -s : s;
  }
  __syncthreads();

  const int rotated_units = a.rot / (2 * VE);
  const int all = tokens * g.tasks;
  for (int i = tid + piece * kThreads; i < all; i += kThreads * g.pieces) {
    const int tok = i / g.tasks, task = i - tok * g.tasks;
    const int row = task / g.units, unit = task - row * g.units;
    const long long t = t0 + tok;
    const bool is_q = row < a.heads;
    const bool is_v = row >= a.heads + a.kv_heads;
    const int head = is_q ? row : (is_v ? row - a.heads - a.kv_heads : row - a.heads);

    const T* src = is_q ? static_cast<const T*>(a.q) + t * a.q_stride[0] + head * a.q_stride[1]
                        : is_v ? static_cast<const T*>(a.v) + t * a.v_stride[0] + head * a.v_stride[1]
                               : static_cast<const T*>(a.k) + t * a.k_stride[0] + head * a.k_stride[1];
    // The task's two vectors.
    const bool turns = !is_v && unit < rotated_units;
    const int first = turns ? (a.pairing == DG_PAIR_HALF ? unit * VE : unit * 2 * VE) : unit * 2 * VE;
    const int second = turns && a.pairing == DG_PAIR_HALF ? first + half : first + VE;
    const bool both = second < a.head_dim;   // a row's last passing vector can stand alone
    float x[VE], y[VE];
    {
      const Vec<T, VE> lo = load<T, VE>(src + first);
#pragma unroll
      for (int j = 0; j < VE; ++j) x[j] = to_float(lo.v[j]);
      if (both) {
        const Vec<T, VE> hi = load<T, VE>(src + second);
#pragma unroll
        for (int j = 0; j < VE; ++j) y[j] = to_float(hi.v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) y[j] = 0.0f;
      }
    }
    if (turns) {
      const Vec<float, (VE < 4 ? VE : 4)>* cs;
      float c[VE], s[VE];
      const float* base = trig + tok * a.rot + unit * VE;
      constexpr int W = VE < 4 ? VE : 4;
#pragma unroll
      for (int j = 0; j < VE; j += W) {
        cs = reinterpret_cast<const Vec<float, W>*>(base + j);
#pragma unroll
        for (int l = 0; l < W; ++l) c[j + l] = cs->v[l];
        cs = reinterpret_cast<const Vec<float, W>*>(base + half + j);
#pragma unroll
        for (int l = 0; l < W; ++l) s[j + l] = cs->v[l];
      }
      if (a.pairing == DG_PAIR_HALF) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float u = x[j], w = y[j];
          x[j] = u * c[j] - w * s[j];
          y[j] = w * c[j] + u * s[j];
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
          z[2 * j] = u * c[j] - w * s[j];
          z[2 * j + 1] = w * c[j] + u * s[j];
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          x[j] = z[j];
          y[j] = z[VE + j];
        }
      }
    }
    T* dst = is_q ? (a.q_out != nullptr ? static_cast<T*>(a.q_out) + t * a.q_out_stride[0] + head * a.q_out_stride[1]
                                        : nullptr)
                  : (!is_v && a.k_out != nullptr
                         ? static_cast<T*>(a.k_out) + t * a.k_out_stride[0] + head * a.k_out_stride[1]
                         : nullptr);
    if (dst != nullptr) {
      store<T, VE>(dst + first, x);
      if (both) store<T, VE>(dst + second, y);
    }
    if constexpr (!std::is_same<C, void>::value) {
      if (is_q) continue;
      const long long slot = a.slots[t];
      if (slot < 0) continue;
      if (slot >= static_cast<long long>(a.num_pages) * a.page_size) {
        if (a.status != nullptr) atomicCAS(a.status, 0, DG_ERR_SLOT);
        continue;
      }
      const long long page = slot / a.page_size, offset = slot - page * a.page_size;
      const long long* st = is_v ? a.v_cache_stride : a.k_cache_stride;
      C* cache = static_cast<C*>(is_v ? a.v_cache : a.k_cache) + page * st[0] + offset * st[1] + head * st[2];
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

template <typename T, int VE>
Kernel pick_cache(const dg_rotary_args& a) {
  if (a.k_cache == nullptr) return rotary_kernel<T, void, VE>;
  if constexpr (!std::is_same<T, float>::value) {
    if (a.cache_type == DG_TYPE_E4M3) return rotary_kernel<T, E4m3, VE>;
    return rotary_kernel<T, T, VE>;
  } else {
    return nullptr;
  }
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
  if (a.tokens < 1 || a.heads < 0 || a.kv_heads < 0 || a.heads + a.kv_heads < 1 || a.head_dim < 2 || a.rot < 2 ||
      a.rot % 2 != 0 || a.rot > a.head_dim || a.rot > DG_MAX_ROT || a.max_position < 1)
    return true;
  if (a.type != DG_TYPE_BF16 && a.type != DG_TYPE_FP16 && a.type != DG_TYPE_FP32) return true;
  if (a.pairing != DG_PAIR_HALF && a.pairing != DG_PAIR_ADJACENT) return true;
  if (a.positions == nullptr || a.cos_sin == nullptr || a.position_stride < 0) return true;
  if ((a.heads > 0) != (a.q != nullptr) || (a.q != nullptr) != (a.q_out != nullptr)) return true;
  if ((a.kv_heads > 0) != (a.k != nullptr)) return true;
  const bool cached = a.k_cache != nullptr;
  if (cached != (a.v_cache != nullptr) || cached != (a.v != nullptr)) return true;
  if (a.k != nullptr && a.k_out == nullptr && !cached) return true;
  if (a.k == nullptr && (a.k_out != nullptr || cached)) return true;
  if (cached) {
    if (a.slots == nullptr || a.page_size < 1 || a.num_pages < 1) return true;
    if (a.type == DG_TYPE_FP32 || (a.cache_type != a.type && a.cache_type != DG_TYPE_E4M3)) return true;
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
  const long long rows = static_cast<long long>(a.heads) + a.kv_heads + (a.v != nullptr ? a.kv_heads : 0);
  g.units = (a.head_dim + 2 * ve - 1) / (2 * ve);
  const long long tasks = rows * g.units;
  if (tasks > (1 << 24)) return cudaErrorInvalidValue;
  g.rows = static_cast<int>(rows);
  g.tasks = static_cast<int>(tasks);
  // About two tasks a thread: whole tokens while there are CTAs enough, else
  // a token's tasks spread over several CTAs so that a decode step uses more
  // than `tokens` SMs.
  const int sms = dg_num_sms() > 0 ? dg_num_sms() : 148;
  g.tokens_per_cta = static_cast<int>(2 * kThreads / tasks);
  if (g.tokens_per_cta > kMaxTableFloats / a.rot) g.tokens_per_cta = kMaxTableFloats / a.rot;
  if (g.tokens_per_cta < 1 || a.tokens <= 2 * sms) g.tokens_per_cta = 1;
  g.pieces = 1;
  if (a.tokens <= 2 * sms) g.pieces = static_cast<int>((tasks + kThreads - 1) / kThreads);
  const long long groups = (static_cast<long long>(a.tokens) + g.tokens_per_cta - 1) / g.tokens_per_cta;
  const long long ctas = groups * g.pieces;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;

  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1]{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
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
