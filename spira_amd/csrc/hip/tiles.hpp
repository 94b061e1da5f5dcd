// What the kernels that tile rows share: groups of rows and their parts, found on
// the device, and loads that write LDS themselves.
#pragma once

#include "numeric.hpp"

namespace spira_hip {

namespace tiles {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) short4v lds_short4;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) uintx4_t lds_chunk;
typedef __attribute__((address_space(3))) uint32_t lds_word;

// ---------------------------------------------------------------------------
// groups
// ---------------------------------------------------------------------------
struct Groups {
  const int32_t *offsets;  // [count + 1]
  int count;
  int64_t rows;
};

struct Part {
  int group;  // -1: the index lies past the last part, `begin` parts after it
  int64_t begin, end;
};

__device__ __forceinline__ int64_t bound(const Groups &g, int i) {
  const int64_t v = g.offsets[i];
  return v < 0 ? 0 : v > g.rows ? g.rows : v;
}

// Part `index` of the groups cut into parts of `size` rows, in group order; the
// same on every lane of the wave.  Lanes count the parts of 64 groups at a time.
__device__ __forceinline__ Part find_part(const Groups &g, int size, int64_t index) {
  const int lane = lane_id();
  int64_t before = 0;
  for (int first = 0; first < g.count; first += 64) {
    const int e = first + lane;
    const int64_t lo = e < g.count ? bound(g, e) : 0, hi = e < g.count ? bound(g, e + 1) : 0;
    const int parts = hi > lo ? static_cast<int>((hi - lo + size - 1) / size) : 0;
    int upto = parts;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int u = __shfl_up(upto, o, 64);
      if (lane >= o) upto += u;
    }
    const uint64_t past = ballot(before + upto > index);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int64_t nth = index - before - (__shfl(upto, at, 64) - __shfl(parts, at, 64));
      const int64_t begin = __shfl(lo, at, 64) + nth * size, end = __shfl(hi, at, 64);
      return {uniform(first + at), uniform(begin), uniform(begin + size < end ? begin + size : end)};
    }
    before += __shfl(upto, 63, 64);
  }
  return {-1, uniform(index - before), 0};
}

// the first part of group `group`, and how many it has
__device__ __forceinline__ void parts_of(const Groups &g, int size, int group, int64_t &first, int64_t &count) {
  const int lane = lane_id();
  int64_t sum = 0;
  for (int e = lane; e < group; e += 64) {
    const int64_t n = bound(g, e + 1) - bound(g, e);
    sum += n > 0 ? (n + size - 1) / size : 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  const int64_t n = bound(g, group + 1) - bound(g, group);
  first = sum;
  count = n > 0 ? (n + size - 1) / size : 0;
}

// parts of all groups
__device__ __forceinline__ int64_t count_parts(const Groups &g, int size) {
  int64_t first, count;
  parts_of(g, size, g.count - 1, first, count);
  return first + count;
}

// ---------------------------------------------------------------------------
// loads
// ---------------------------------------------------------------------------
// Four 16-bit values of 16 lanes, transposed: lane i of the 16 gets value i % 4
// of lanes i / 4 + {0, 4, 8, 12}.
__device__ __forceinline__ short4v read_tr(const char *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(const_cast<char *>(p)));
}
__device__ __forceinline__ short4v read_tr(lds_char *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)p);
}

constexpr uint32_t kOutOfRange = 0x80000000u;
constexpr int64_t kBufferLimit = int64_t(1) << 31;

// A buffer descriptor: base, bytes, raw.
__device__ __forceinline__ uintx4_t buffer(const void *base, int64_t bytes) {
  const int64_t n = bytes < 0 ? 0 : bytes < kBufferLimit ? bytes : kBufferLimit - 1;
  const auto at = reinterpret_cast<uint64_t>(base);
  return {uniform(static_cast<uint32_t>(at)), uniform(static_cast<uint32_t>(at >> 32) & 0xFFFFu),
          uniform(static_cast<uint32_t>(n)), 0x00020000u};
}
// 1 KB to LDS, 16 bytes from each lane's offset.  In assembly, and waited for by
// the ring alone: the compiler's own count of such loads is not kept over the
// ring's loop, it would wait for all of them once a turn.  (No register is
// written.  What loads the compiler itself waits for, it waits longer.)
__device__ __forceinline__ void load_lds(uintx4_t from, uint32_t offset, lds_void *to) {
  const uint32_t at = uniform(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(at), "v"(offset), "s"(from) : "memory", "m0");
}
__device__ __forceinline__ void load_lds(uintx4_t from, uint32_t offset, char *to) {
  load_lds(from, offset, (lds_void *)to);
}
// 256 bytes, 4 from each lane's offset
__device__ __forceinline__ void load_lds_word(uintx4_t from, uint32_t offset, void *to) {
  const uint32_t at = uniform(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void *)to)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(at), "v"(offset), "s"(from) : "memory", "m0");
}
// Until all but the last N loads have landed and this wave's LDS reads are done,
// then the block's barrier.
template <int N> __device__ __forceinline__ void wait_loads_and_meet() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt(0)

}  // namespace tiles

}  // namespace spira_hip
