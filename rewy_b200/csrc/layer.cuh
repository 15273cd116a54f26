// What the kernels around a recurrence share (conv.cu, selective_scan.cu, norms.cu, delta_step.cu): element types, groups of
// elements between memory and FP32 registers, the activations, and the host-side checks of their entry points.
#pragma once
#include <cuda_fp16.h>
#include <cstdio>
#include <type_traits>
#include "common.cuh"

namespace rewy {

using half_t = __half;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(half_t x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ half_t from_f32<half_t>(float x) { return __float2half_rn(x); }

// V consecutive elements as they lie in memory; accesses of up to 16 bytes
template <class T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ void load_pack(Pack<T, V>& d, const T* p) {
  constexpr int BYTES = sizeof(T) * V;
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; i++) reinterpret_cast<uint4*>(&d)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else if constexpr (BYTES == 8) {
    *reinterpret_cast<uint2*>(&d) = __ldg(reinterpret_cast<const uint2*>(p));
  } else if constexpr (BYTES == 4) {
    *reinterpret_cast<uint32_t*>(&d) = __ldg(reinterpret_cast<const uint32_t*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) d.v[i] = p[i];
  }
}
template <class T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& s) {
  constexpr int BYTES = sizeof(T) * V;
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; i++) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&s)[i];
  } else if constexpr (BYTES == 8) {
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(&s);
  } else if constexpr (BYTES == 4) {
    *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(&s);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) p[i] = s.v[i];
  }
}
template <class T, int V>
__device__ __forceinline__ void zero_pack(Pack<T, V>& d) {
#pragma unroll
  for (int i = 0; i < V; i++) d.v[i] = from_f32<T>(0.f);
}
// All elements of a group as FP32 and back, two 16-bit elements per instruction
template <class T, int V>
__device__ __forceinline__ void to_floats(float (&f)[V], const Pack<T, V>& p) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = to_f32(p.v[i]);
  } else {
    static_assert(V % 2 == 0, "pairs");
#pragma unroll
    for (int i = 0; i < V / 2; i++) {
      const uint32_t u = reinterpret_cast<const uint32_t*>(&p)[i];
      if constexpr (std::is_same_v<T, bf16>) {
        f[2 * i] = __uint_as_float(u << 16);
        f[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
      } else {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u));
        f[2 * i] = x.x; f[2 * i + 1] = x.y;
      }
    }
  }
}
template <class T, int V>
__device__ __forceinline__ void from_floats(Pack<T, V>& p, const float (&f)[V]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; i++) p.v[i] = from_f32<T>(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; i++) {
      uint32_t u;
      if constexpr (std::is_same_v<T, bf16>) {
        u = pack_bf16(f[2 * i], f[2 * i + 1]);
      } else {
        const __half2 x = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        u = *reinterpret_cast<const uint32_t*>(&x);
      }
      reinterpret_cast<uint32_t*>(&p)[i] = u;
    }
  }
}
// V elements of which the first `valid` exist; `wide`: the address is aligned for whole accesses
template <class T, int V>
__device__ __forceinline__ void load_some(Pack<T, V>& d, const T* p, int valid, bool wide) {
  if (wide && valid >= V) {
    load_pack<T, V>(d, p);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; i++) d.v[i] = i < valid ? p[i] : from_f32<T>(0.f);
}
template <class T, int V>
__device__ __forceinline__ void store_some(T* p, const Pack<T, V>& s, int valid, bool wide) {
  if (wide && valid >= V) {
    store_pack<T, V>(p, s);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; i++)
    if (i < valid) p[i] = s.v[i];
}

// A parameter (weights, biases, scales): its own type, read once per thread
__device__ __forceinline__ float param_at(const void* p, int dtype, long long i) {
  if (dtype == REWY_F32) return static_cast<const float*>(p)[i];
  if (dtype == REWY_BF16) return to_f32(static_cast<const bf16*>(p)[i]);
  return to_f32(static_cast<const half_t*>(p)[i]);
}
__device__ __forceinline__ void param_store(void* p, int dtype, long long i, float x) {
  if (dtype == REWY_F32) static_cast<float*>(p)[i] = x;
  else if (dtype == REWY_BF16) static_cast<bf16*>(p)[i] = from_f32<bf16>(x);
  else static_cast<half_t*>(p)[i] = from_f32<half_t>(x);
}

__device__ __forceinline__ float ex2(float x) {  // 2 ulp, results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {  // 1 ulp
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two FP32 values in a register pair: one instruction for both
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 pair(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ F2 both(float x) { return pair(x, x); }
__device__ __forceinline__ float2 halves(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 neg2(F2 a) {
  const float2 h = halves(a);
  return pair(-h.x, -h.y);
}
__device__ __forceinline__ float sum_halves(F2 a) {
  const float2 h = halves(a);
  return h.x + h.y;
}
template <class T, int V>
__device__ __forceinline__ void to_pairs(F2 (&x)[V / 2], const Pack<T, V>& p) {
  float f[V];
  to_floats(f, p);
#pragma unroll
  for (int i = 0; i < V / 2; i++) x[i] = pair(f[2 * i], f[2 * i + 1]);
}
template <class T, int V>
__device__ __forceinline__ void from_pairs(Pack<T, V>& p, const F2 (&x)[V / 2]) {
  float f[V];
#pragma unroll
  for (int i = 0; i < V / 2; i++) {
    const float2 h = halves(x[i]);
    f[2 * i] = h.x; f[2 * i + 1] = h.y;
  }
  from_floats(p, f);
}
__device__ __forceinline__ F2 ex2_2(F2 a) {
  const float2 h = halves(a);
  return pair(ex2(h.x), ex2(h.y));
}
constexpr float LOG2E = 1.4426950408889634f;
// 1 / (1 + e^-x): e^-x overflows to infinity and its reciprocal to 0 for very negative x, as the sigmoid does
__device__ __forceinline__ float sigmoid_fast(float x) { return rcp_fast(1.f + ex2(-LOG2E * x)); }
// softplus(x) = max(x, 0) + log(1 + e^-|x|), the logarithm as 2 atanh(s), s = e / (2 + e) <= 1/3 (series to s^13: 1.4e-8 of the
// value); sig: its derivative, from the same exponential
__device__ __forceinline__ float softplus_fast(float x, float& sig) {
  const float e = ex2(-LOG2E * fabsf(x)), r = rcp_fast(1.f + e);
  sig = x >= 0.f ? r : e * r;
  const float s = e * rcp_fast(2.f + e), z = s * s;
  float p = fmaf(z, 1.f / 13, 1.f / 11);
  p = fmaf(z, p, 1.f / 9);
  p = fmaf(z, p, 1.f / 7);
  p = fmaf(z, p, 1.f / 5);
  p = fmaf(z, p, 1.f / 3);
  p = fmaf(z, p, 1.f);
  return fmaxf(x, 0.f) + 2.f * s * p;
}

// Sequence of a packed batch that holds token t: the last s with cu[s] <= t
__device__ __forceinline__ int packed_sequence(const int* cu, int num_seqs, int t) {
  int lo = 0, hi = num_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// The state of a pool that row b of a batch of single tokens works on, -1 if its index lies outside the pool; and whether an earlier
// row has the same index, which is asked by all threads of a block together, after they have asked for their part of the state:
// then the row is skipped like one without a state.
__device__ __forceinline__ long long slot_at(const void* slots, int slots_are_i64, int i) {
  return slots_are_i64 ? static_cast<const long long*>(slots)[i] : (long long)static_cast<const int*>(slots)[i];
}
__device__ __forceinline__ long long pool_row(const void* slots, int slots_are_i64, int b, long long pool) {
  const long long mine = slots == nullptr ? b : slot_at(slots, slots_are_i64, b);
  return mine < 0 || mine >= pool ? -1 : mine;
}
__device__ __forceinline__ bool row_repeats(const void* slots, int slots_are_i64, int b, long long mine) {
  if (slots == nullptr || mine < 0) return false;   // the same for all threads
  bool again = false;
  for (int i = threadIdx.x; i < b; i += blockDim.x) again |= slot_at(slots, slots_are_i64, i) == mine;
  return __syncthreads_or(again);
}

inline bool unaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
inline int element_bytes(int dtype) { return dtype == REWY_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == REWY_BF16 || dtype == REWY_F16 || dtype == REWY_F32; }
inline int launched(const char* what, int n = 1) {
  count_launch(n);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return REWY_OK;
  char msg[200];
  snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
  return report_error(REWY_ERR_LAUNCH, msg);
}
// f(T()) with T the element type
template <class F>
inline void with_type(int dtype, F&& f) {
  if (dtype == REWY_BF16) f(bf16());
  else if (dtype == REWY_F16) f(half_t());
  else f(float());
}

}  // namespace rewy

#define LAYER_REQUIRE(ok, code, text) \
  do {                                \
    if (!(ok)) return report_error(code, text); \
  } while (0)
