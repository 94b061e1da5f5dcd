// Feature types of the row operators (experts, routing, norms, dropout): fp16,
// bf16 and fp32 in memory, fp32 in registers, in chunks of 16 bytes.
#pragma once

#include "common.hpp"

#include <type_traits>

#include "../../../include/spira_hip.h"

namespace spira_hip {

typedef float floatx4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4_t __attribute__((ext_vector_type(4)));

template <class T> constexpr int kVec = 16 / static_cast<int>(sizeof(T));  // values per chunk

template <class T> __device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }
// (to nearest, ties to even)
template <class T> __device__ __forceinline__ T from_float(float v) { return static_cast<T>(v); }

// Rows of odd widths and views start at any element: the chunk's type claims an
// element's alignment only, and the hardware takes 16 bytes at any address in
// one access.
typedef uint32_t uintx4_a2_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t uintx4_a4_t __attribute__((ext_vector_type(4), aligned(4)));
template <class T> using Unaligned = std::conditional_t<sizeof(T) == 2, uintx4_a2_t, uintx4_a4_t>;
template <class T> struct Packed {
  T v[kVec<T>];
};
template <class T> struct Chunk {
  float v[kVec<T>];
};

// n: how many of the chunk's values lie inside the row (any number; values
// past it are zero, or not written)
template <class T> __device__ __forceinline__ uintx4_t load_raw(const T *p, int64_t n) {
  uintx4_t raw = {0, 0, 0, 0};
  if (n >= kVec<T>) {
    raw = *reinterpret_cast<const Unaligned<T> *>(p);
  } else if (n > 0) {  // (few lanes; those wholly past the row skip it)
    Packed<T> r;
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) r.v[i] = i < n ? p[i] : static_cast<T>(0.f);
    raw = __builtin_bit_cast(uintx4_t, r);
  }
  return raw;
}
template <class T> __device__ __forceinline__ Chunk<T> unpack(uintx4_t raw) {
  const Packed<T> r = __builtin_bit_cast(Packed<T>, raw);
  Chunk<T> c;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) c.v[i] = to_float(r.v[i]);
  return c;
}
template <class T> __device__ __forceinline__ Chunk<T> load_chunk(const T *p, int64_t n) {
  return unpack<T>(load_raw(p, n));
}
template <class T> __device__ __forceinline__ void store_chunk(T *p, int64_t n, const Chunk<T> &c) {
  Packed<T> r;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) r.v[i] = from_float<T>(c.v[i]);
  if (n >= kVec<T>) {
    *reinterpret_cast<Unaligned<T> *>(p) = __builtin_bit_cast(uintx4_t, r);
  } else if (n > 0) {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (i < n) p[i] = r.v[i];
  }
}

// sum over groups of G consecutive lanes (a power of two up to 64), the same in
// every lane of the group
template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// y[t] = sum_j h[slots[t, j]] over the slots in [0, rows), y in `dtype` (route.hip)
int sum_slots(const float *h, int64_t rows, const int32_t *slots, int64_t tokens, int k, int c, int dtype, void *y,
              hipStream_t stream);

// A launch has fewer than 2^32 threads (in x): of more, some do not run, and no error
// says so.
inline bool launchable(int64_t blocks, int64_t threads) { return blocks * threads < (int64_t(1) << 32); }
// launch(first block, blocks) for so many blocks of 256 in all, in slices of 2^23
// (a kernel that walks its blocks instead takes 5 % longer: dropout of 200k x 96
// 20.1 us, 19.1 this way)
template <class F> int in_slices(int64_t blocks, F &&launch) {
  constexpr int64_t most = int64_t(1) << 23;
  for (int64_t first = 0; first < blocks; first += most) {
    launch(first, dim3(static_cast<uint32_t>(blocks - first < most ? blocks - first : most)));
    SPIRA_HIP_LAUNCH_CHECK();
  }
  return kOk;
}

// f(T{}) for the storage type that `dtype` names
template <class F> int with_type(int dtype, F &&f) {
  switch (dtype) {
    case SPIRA_F16: return f(static_cast<_Float16>(0));
    case SPIRA_BF16: return f(static_cast<__bf16>(0.f));
    case SPIRA_F32: return f(0.f);
    default: set_error("dtype must be fp16, bf16 or fp32"); return kInvalidArgument;
  }
}

}  // namespace spira_hip
