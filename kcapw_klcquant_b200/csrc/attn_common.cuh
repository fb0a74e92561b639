// Shared pieces of the attention kernels: 16-bit element types, exponentials
// in base 2, the cache layout and the argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cmath>

#include "klc_common.cuh"

namespace klc {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxBatch = 4096;  // sequences per decode call (each CTA keeps 16 bytes of plan per sequence)

// kTopLog2: the softmax numerators are made up to 2^kTopLog2, not up to 1, and the sums carry the same factor.  f16 has
// 5 exponent bits: with numerators up to 1 those below 2^-14 lose bits and those below 2^-25 vanish, though a long context
// has many of them (a score 18 below the row's largest is 2^-26), while 2^1 .. 2^15 lie unused.  bf16 has fp32's range.
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr uint32_t kMmaFormat = 1;  // tcgen05 kind::f16 operand format field
  static constexpr float kTopLog2 = 0.f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
};
template <>
struct Elem<__half> {
  static constexpr uint32_t kMmaFormat = 0;
  static constexpr float kTopLog2 = 15.f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Maxima that keep a NaN: a row with a score that is not a number must not pass for one without keys.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A row's share of the softmax over some of its keys: a reference m at or
// below the running maximum (in units of log2), the sum l of 2^(s - m) and the
// unnormalised output.
// Joining shares k: m = max m_k, l = sum l_k 2^(m_k - m), o likewise.  An
// attention sink is one more key of weight 2^sink without a value.  m = -inf
// says that the share has no key: a NaN score makes m or l a NaN, never that.
//
// 1 / denominator and the log-sum-exp (natural log) of a finished row whose
// keys gave (m, l), with the head's sink when there is one.  A row that sees
// no key has l = 0: its output is 0 and its log-sum-exp the sink's (or -inf).
__device__ __forceinline__ void finish_row(float m, float l, bool has_sink, float sink_log2, float* inv, float* lse) {
  float top = m, sum = l, to_top = 1.f;
  if (has_sink) {
    top = fmaxf(m, sink_log2);
    to_top = m == -INFINITY ? 0.f : exp2f(m - top);
    sum = l * to_top + (sink_log2 == -INFINITY ? 0.f : exp2f(sink_log2 - top));
  }
  *inv = sum > 0.f || sum != sum ? to_top / sum : 0.f;  // a NaN stays a NaN
  *lse = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

inline int check_heads(const char* who, int dtype, int heads, int kv_heads, int head_dim) {
  const std::string w(who);
  if (dtype != KLC_BF16 && dtype != KLC_F16) return fail(KLC_ERR_INVALID, w + ": dtype must be KLC_BF16 or KLC_F16");
  if (head_dim != 64 && head_dim != 128) return fail(KLC_ERR_UNSUPPORTED, w + ": head_dim must be 64 or 128");
  if (kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0)
    return fail(KLC_ERR_INVALID, w + ": heads must be a positive multiple of kv_heads");
  if (heads / kv_heads > 64) return fail(KLC_ERR_UNSUPPORTED, w + ": at most 64 query heads per key head");
  if (kv_heads > 4096) return fail(KLC_ERR_UNSUPPORTED, w + ": at most 4096 key heads");
  return KLC_OK;
}

inline int check_scale(const char* who, float scale) {
  if (!(scale > 0.f) || !std::isfinite(scale)) return fail(KLC_ERR_INVALID, std::string(who) + ": scale must be finite and > 0");
  return KLC_OK;
}

// Raises a kernel's dynamic shared memory limit, once per device (a call on each launch costs host time).
struct SmemLimit {
  std::atomic<uint64_t> done{0};  // bit d: device d
  int raise(const void* kernel, size_t bytes) {
    int dev = 0;
    KLC_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (bit != 0 && (done.load(std::memory_order_relaxed) & bit) != 0) return KLC_OK;
    KLC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
    done.fetch_or(bit, std::memory_order_relaxed);
    return KLC_OK;
  }
};

inline bool page_size_ok(int ps) { return ps == 16 || ps == 32 || ps == 64 || ps == 128; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace attn
}  // namespace klc
