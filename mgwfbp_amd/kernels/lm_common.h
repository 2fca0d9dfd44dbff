// Shared by the language-model kernels (embedding, token loss, gradient
// clip): 16-byte accesses at any element alignment, conversions, and the
// wave64 reductions.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <torch/extension.h>
#include <c10/hip/HIPStream.h>
#include <cstdint>

#define CHECK_HIP(x)                                                         \
  do {                                                                       \
    hipError_t err__ = (x);                                                  \
    TORCH_CHECK(err__ == hipSuccess, "HIP error: ",                          \
                hipGetErrorString(err__));                                   \
  } while (0)

namespace mgx {

// Rows of an odd width start anywhere, so no vector access here assumes
// more than the element's own alignment: gfx950 does global 16-byte
// accesses at any address, and the compiler emits one dwordx4 for these.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

__device__ __forceinline__ u32x4 load16(const void* p) {
  return *static_cast<const u32x4_any*>(p);
}
__device__ __forceinline__ void store16(void* p, u32x4 v) {
  *static_cast<u32x4_any*>(p) = v;
}

// The same past the 256 MB cache, for what is read or written once and does
// not fit there anyhow. A load that takes a line of that cache has to wait
// until what was written there before has gone to memory: streams of 256
// and 800 MB behind written ones were read at 2.9 and 4.5 TB/s, past the
// cache at 6.4 and 6.9; copies gain 7% (5.9 to 6.3 TB/s, both ways).
__device__ __forceinline__ u32x4 load16_past(const void* p) {
  return __builtin_nontemporal_load(static_cast<const u32x4_any*>(p));
}
__device__ __forceinline__ void store16_past(void* p, u32x4 v) {
  __builtin_nontemporal_store(v, static_cast<u32x4_any*>(p));
}

// One element type: how many sit in 16 bytes, and both conversions. Only
// the rounding to the 16-bit types loses anything: half a step, to even.
template <typename T> struct Elem;

template <> struct Elem<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ u32x4 minus_inf() {
    return u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
  }
  static __device__ __forceinline__ float get(u32x4 v, int i) {
    return __uint_as_float(v[i]);
  }
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]),
                 __float_as_uint(f[2]), __float_as_uint(f[3])};
  }
};

template <> struct Elem<__hip_bfloat16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ u32x4 minus_inf() {
    return u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
  }
  static __device__ __forceinline__ float get(u32x4 v, int i) {
    const uint32_t w = v[i >> 1];
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ float up(__hip_bfloat16 x) {
    return __bfloat162float(x);
  }
  static __device__ __forceinline__ __hip_bfloat16 down(float x) {
    return __float2bfloat16(x);
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(
          (f32x2{f[2 * i], f[2 * i + 1]}), bf16x2));
    return v;
  }
};

template <> struct Elem<__half> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ u32x4 minus_inf() {
    return u32x4{0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u};
  }
  static __device__ __forceinline__ float get(u32x4 v, int i) {
    const uint32_t w = v[i >> 1];
    return static_cast<float>(__builtin_bit_cast(
        _Float16, static_cast<uint16_t>((i & 1) ? (w >> 16) : w)));
  }
  static __device__ __forceinline__ float up(__half x) {
    return __half2float(x);
  }
  static __device__ __forceinline__ __half down(float x) {
    return __float2half(x);
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(
          (f32x2{f[2 * i], f[2 * i + 1]}), f16x2));
    return v;
  }
};

// Calls f with a value of the tensor's element type, for the three types
// that the kernels take.
template <typename F>
void with_elem(at::ScalarType t, const char* what, F&& f) {
  switch (t) {
    case at::kFloat: f(float{}); break;
    case at::kBFloat16: f(__hip_bfloat16{}); break;
    case at::kHalf: f(__half{}); break;
    default:
      TORCH_CHECK_TYPE(false, what, " must be float32, bfloat16 or float16, "
                       "not ", t);
  }
}

// A launch counts its threads in 32 bits.
inline dim3 grid_of(long blocks, long threads, const char* what) {
  TORCH_CHECK_VALUE(blocks * threads < (1L << 32), "too many ", what,
                    " for one call");
  return dim3((unsigned)blocks);
}

inline hipStream_t current_stream() {
  return c10::hip::getCurrentHIPStream().stream();
}

}  // namespace mgx
