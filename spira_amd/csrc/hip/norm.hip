// The end of a residual block and the entry of the next (gfx950), one row of
// features at a time:
//
//   z = h / sqrt(mean(h^2) + eps) * w        (or z = h, without w)
//   r = x + s g z                            (g: none, [C], [N, 1] or [N, C], raw or through a sigmoid)
//   n = r / sqrt(mean(r^2) + eps) * w_next   (or none; without h, r = x: the entry norm alone)
//
// Everything in fp32 from the loads on, each output rounded once (n comes from
// the unrounded r).  A row is held in registers by G lanes, NV chunks of 16
// bytes each, so that the forward pass reads x, h and the gate once and writes
// r and n.  The backward pass reads them again with the two gradients and makes
// r anew: saving it would cost the bytes that reading x costs, and a rounding.
// Sums over the rows (the gradients of w, w_next and a gate per channel) stay in
// registers over all rows of a block, then go over the blocks in a fixed order:
// no atomics, the same result on every call.
//
// Bound by memory.
#include "numeric.hpp"

#include <algorithm>

namespace spira_hip {

namespace norm {

enum Gate { kNone = 0, kChannel = 1, kRow = 2, kFull = 3 };

struct Args {
  const void *x, *h, *w, *gate, *w_next;
  int64_t n;
  int c, gate_form, sigmoid;
  float scale, eps;
  void *r, *next;
  float *inv_h, *inv_r;  // 1 / root mean squares of the rows, kept for the gradient (or null)
  // backward
  const void *dr, *dnext;
  void *dx, *dh, *dgate;
  float *partial;  // [blocks, 3, c]: w, w_next, gate per channel
};

// sum over the G lanes of a row; with more than a wave, over the whole block
template <int G> __device__ __forceinline__ float row_sum(float v, float *shared) {
  if constexpr (G <= 64) {
    return group_sum<G>(v);
  } else {
    v = group_sum<64>(v);
    __syncthreads();  // (the sum before is read)
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0;
#pragma unroll
    for (int i = 0; i < G / 64; ++i) s += shared[i];
    return s;
  }
}

template <class T, int NV> struct Row {
  float v[NV][kVec<T>];
};
// a row as it lies in memory: half the registers, unpacked where it is used
template <int NV> struct Raw {
  uintx4_t v[NV];
};

template <class T, int G, int NV>
__device__ __forceinline__ Raw<NV> load_row(const void *base, int64_t row, int c, int lane) {
  Raw<NV> r;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (lane + i * G) * kVec<T>;
    r.v[i] = load_raw(static_cast<const T *>(base) + row * c + at, base ? c - at : 0);
  }
  return r;
}

template <class T, int NV> __device__ __forceinline__ Row<T, NV> unpack_row(const Raw<NV> &raw) {
  Row<T, NV> r;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Chunk<T> k = unpack<T>(raw.v[i]);
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) r.v[i][j] = k.v[j];
  }
  return r;
}

template <class T, int G, int NV>
__device__ __forceinline__ void store_row(void *base, int64_t row, int c, int lane, const Row<T, NV> &r) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (lane + i * G) * kVec<T>;
    Chunk<T> k;
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) k.v[j] = r.v[i][j];
    store_chunk(static_cast<T *>(base) + row * c + at, c - at, k);
  }
}

// f(i, j) over the lane's values
template <class T, int NV, class F> __device__ __forceinline__ void each(F &&f) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) f(i, j);
}

// For 16 bits the hardware's exponential and reciprocal, good to one unit each: at
// |v| up to 20 within 3e-6 of the value, a hundredth of an output's rounding (the
// library's take 17 us of a 16k x 1024 call).  For fp32 that would be tens of units:
// the library's exponential and a rounded division (16k x 1024 forward 64.5 -> 67.5 us).
template <class T> __device__ __forceinline__ float sigmoid(float v) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * v));
  else return 1.f / (1.f + expf(-v));
}

// a row's part of the gate as it lies in memory: its channels, or its one value
template <class T, int G, int NV>
__device__ __forceinline__ Raw<NV> load_gate(const Args &a, int64_t row, int lane) {
  if (a.gate_form == kFull) return load_row<T, G, NV>(a.gate, row, a.c, lane);
  Raw<NV> g{};
  if (a.gate_form == kRow) g.v[0] = load_raw(static_cast<const T *>(a.gate) + row, 1);
  return g;
}
// the gate's values, through its sigmoid if it has one; `channel`: a gate per channel
template <class T, int NV>
__device__ __forceinline__ Row<T, NV> gate_of(const Args &a, const Raw<NV> &own, const Raw<NV> &channel) {
  Row<T, NV> g;
  if (a.gate_form == kNone) {
    each<T, NV>([&](int i, int j) { g.v[i][j] = 1.f; });
    return g;
  }
  g = unpack_row<T>(a.gate_form == kChannel ? channel : own);
  if (a.gate_form == kRow) {
    const float v = g.v[0][0];
    each<T, NV>([&](int i, int j) { g.v[i][j] = v; });
  }
  if (a.sigmoid) each<T, NV>([&](int i, int j) { g.v[i][j] = sigmoid<T>(g.v[i][j]); });
  return g;
}

// Each group of lanes walks rows, with the next row's loads under way while it
// computes; weights stay in registers.  (Every group takes as many turns, so that
// a block's barriers meet.)
template <class T, int G, int NV, int NT>
__global__ __launch_bounds__(NT) void forward_kernel(const Args a) {
  __shared__ float shared[NT / 64];
  constexpr int RPB = NT / G;
  const int lane = threadIdx.x % G;
  const float inv_c = 1.f / static_cast<float>(a.c);
  const int64_t turn = gridDim.x * static_cast<int64_t>(RPB);
  const Raw<NV> w_raw = load_row<T, G, NV>(a.w, 0, a.c, lane), next_raw = load_row<T, G, NV>(a.w_next, 0, a.c, lane);
  const Raw<NV> channel = load_row<T, G, NV>(a.gate_form == kChannel ? a.gate : nullptr, 0, a.c, lane);
  int64_t first = blockIdx.x * static_cast<int64_t>(RPB);
  Raw<NV> x, h, gate;
  const auto fetch = [&](int64_t from) {
    const int64_t row = std::min<int64_t>(from + threadIdx.x / G, a.n - 1);
    x = load_row<T, G, NV>(a.x, row, a.c, lane);
    if (a.h) {
      h = load_row<T, G, NV>(a.h, row, a.c, lane);
      gate = load_gate<T, G, NV>(a, row, lane);
    }
  };
  fetch(first);
  for (; first < a.n; first += turn) {
    const int64_t row = first + threadIdx.x / G;
    const bool there = row < a.n;
    Row<T, NV> r = unpack_row<T>(x), z = unpack_row<T>(h);
    const Raw<NV> own = gate;
    if (first + turn < a.n) fetch(first + turn);
    if (a.h) {
      if (a.w) {
        float ss = 0;
        each<T, NV>([&](int i, int j) { ss += z.v[i][j] * z.v[i][j]; });
        const float inv = rsqrtf(row_sum<G>(ss, shared) * inv_c + a.eps);
        if (there && a.inv_h && lane == 0) a.inv_h[row] = inv;
        const Row<T, NV> w = unpack_row<T>(w_raw);
        each<T, NV>([&](int i, int j) { z.v[i][j] *= inv * w.v[i][j]; });
      }
      const Row<T, NV> g = gate_of<T>(a, own, channel);
      each<T, NV>([&](int i, int j) { r.v[i][j] += a.scale * g.v[i][j] * z.v[i][j]; });
      if (there) store_row<T, G, NV>(a.r, row, a.c, lane, r);
    }
    if (a.next) {
      float ss = 0;
      each<T, NV>([&](int i, int j) { ss += r.v[i][j] * r.v[i][j]; });
      // (lanes past the row hold zeros)
      const float inv = rsqrtf(row_sum<G>(ss, shared) * inv_c + a.eps);
      if (there && a.inv_r && lane == 0) a.inv_r[row] = inv;
      const Row<T, NV> w = unpack_row<T>(next_raw);
      each<T, NV>([&](int i, int j) { r.v[i][j] *= inv * w.v[i][j]; });
      if (there) store_row<T, G, NV>(a.next, row, a.c, lane, r);
    }
  }
}

// CHANNEL: a gate per channel, whose gradient is a sum over the rows
template <class T, int G, int NV, int NT, bool CHANNEL>
__global__ __launch_bounds__(NT) void backward_kernel(const Args a) {
  constexpr int RPB = NT / G, VEC = kVec<T>, NW = NT / 64;
  __shared__ float shared[NW];
  __shared__ float sums[NT > G ? NW * G * NV * VEC : 1];
  const int lane = threadIdx.x % G;
  const float inv_c = 1.f / static_cast<float>(a.c);
  const int64_t turn = gridDim.x * static_cast<int64_t>(RPB);
  const Raw<NV> w_raw = load_row<T, G, NV>(a.w, 0, a.c, lane), next_raw = load_row<T, G, NV>(a.w_next, 0, a.c, lane);
  const Raw<NV> channel = load_row<T, G, NV>(CHANNEL ? a.gate : nullptr, 0, a.c, lane);
  Row<T, NV> dw{}, dw_next{}, dg_sum{};
  int64_t first = blockIdx.x * static_cast<int64_t>(RPB);
  Raw<NV> x, h, gate, dr, dnext;
  float inv_h, inv_r;
  const auto fetch = [&](int64_t from) {
    const int64_t row = std::min<int64_t>(from + threadIdx.x / G, a.n - 1);
    x = load_row<T, G, NV>(a.x, row, a.c, lane);
    if (a.h) {
      h = load_row<T, G, NV>(a.h, row, a.c, lane);
      gate = load_gate<T, G, NV>(a, row, lane);
    }
    dr = load_row<T, G, NV>(a.dr, row, a.c, lane);
    if (a.dnext) dnext = load_row<T, G, NV>(a.dnext, row, a.c, lane);
    inv_h = a.w ? a.inv_h[row] : 1.f;
    inv_r = a.dnext ? a.inv_r[row] : 1.f;
  };
  fetch(first);
  for (; first < a.n; first += turn) {
    const int64_t row = first + threadIdx.x / G;
    const bool there = row < a.n;
    Row<T, NV> r = unpack_row<T>(x), d = unpack_row<T>(dr), hh{}, g{};
    const float ih = inv_h, ir = inv_r;
    if (a.h) {
      hh = unpack_row<T>(h);
      g = gate_of<T>(a, gate, channel);
      // (z is w hhat, or h)
      const Row<T, NV> w = unpack_row<T>(w_raw);
      each<T, NV>([&](int i, int j) {
        hh.v[i][j] *= ih;
        r.v[i][j] += a.scale * g.v[i][j] * (a.w ? hh.v[i][j] * w.v[i][j] : hh.v[i][j]);
      });
    }
    Row<T, NV> dn = unpack_row<T>(dnext);
    if (first + turn < a.n) fetch(first + turn);
    if (a.dnext) {
      const Row<T, NV> w = unpack_row<T>(next_raw);
      float s = 0;
      each<T, NV>([&](int i, int j) {
        r.v[i][j] *= ir;
        if (there) dw_next.v[i][j] += dn.v[i][j] * r.v[i][j];
        dn.v[i][j] *= w.v[i][j];
        s += dn.v[i][j] * r.v[i][j];
      });
      s = row_sum<G>(s, shared) * inv_c;
      each<T, NV>([&](int i, int j) { d.v[i][j] += ir * (dn.v[i][j] - r.v[i][j] * s); });
    }
    if (there && a.dx) store_row<T, G, NV>(a.dx, row, a.c, lane, d);
    if (!a.h) continue;
    // d becomes dz, g the gate's gradient
    float along = 0;
    {
      const Row<T, NV> w = unpack_row<T>(w_raw);
      each<T, NV>([&](int i, int j) {
        const float dz = a.scale * g.v[i][j] * d.v[i][j];
        float dg = a.scale * (a.w ? hh.v[i][j] * w.v[i][j] : hh.v[i][j]) * d.v[i][j];
        if (a.sigmoid) dg *= g.v[i][j] * (1.f - g.v[i][j]);
        g.v[i][j] = dg;
        along += dg;
        d.v[i][j] = dz;
      });
    }
    if constexpr (CHANNEL) {
      if (there) each<T, NV>([&](int i, int j) { dg_sum.v[i][j] += g.v[i][j]; });
    } else if (a.gate_form == kFull) {
      if (there && a.dgate) store_row<T, G, NV>(a.dgate, row, a.c, lane, g);
    } else if (a.gate_form == kRow) {
      along = row_sum<G>(along, shared);
      if (there && a.dgate && lane == 0) static_cast<T *>(a.dgate)[row] = from_float<T>(along);
    }
    if (a.w) {
      const Row<T, NV> w = unpack_row<T>(w_raw);
      float s = 0;
      each<T, NV>([&](int i, int j) {
        if (there) dw.v[i][j] += d.v[i][j] * hh.v[i][j];
        d.v[i][j] *= w.v[i][j];
        s += d.v[i][j] * hh.v[i][j];
      });
      s = row_sum<G>(s, shared) * inv_c;
      each<T, NV>([&](int i, int j) { d.v[i][j] = ih * (d.v[i][j] - hh.v[i][j] * s); });
    }
    if (there && a.dh) store_row<T, G, NV>(a.dh, row, a.c, lane, d);
  }
  if (!a.partial) return;
  auto out = [&](Row<T, NV> v, int which) {
    float *p = a.partial + (blockIdx.x * static_cast<int64_t>(3) + which) * a.c;
    if constexpr (NT > G) {
      // the block's groups: first those of a wave, then the waves in order
      if constexpr (G < 64)
        each<T, NV>([&](int i, int j) {
#pragma unroll
          for (int o = G; o < 64; o *= 2) v.v[i][j] += __shfl_xor(v.v[i][j], o, 64);
        });
      __syncthreads();
      if ((threadIdx.x & 63) < G)
        each<T, NV>([&](int i, int j) { sums[((threadIdx.x >> 6) * NV + i) * G * VEC + lane * VEC + j] = v.v[i][j]; });
      __syncthreads();
      for (int k = threadIdx.x; k < NV * G * VEC && k < a.c; k += NT) {
        float s = 0;
#pragma unroll
        for (int q = 0; q < NW; ++q) s += sums[q * NV * G * VEC + k];
        p[k] = s;
      }
    } else {
      each<T, NV>([&](int i, int j) {
        const int at = (lane + i * G) * VEC + j;
        if (at < a.c) p[at] = v.v[i][j];
      });
    }
  };
  if (a.w) out(dw, 0);
  if (a.dnext) out(dw_next, 1);
  if constexpr (CHANNEL) out(dg_sum, 2);
}

// columns of the blocks' sums: 16 columns a block, 64 threads to each, joined in
// a fixed tree
template <class T>
__global__ __launch_bounds__(1024) void columns_kernel(const float *partial, int blocks, int c, void *o0, void *o1,
                                                       void *o2) {
  __shared__ float s[64][17];
  void *o = blockIdx.y == 0 ? o0 : blockIdx.y == 1 ? o1 : o2;
  if (!o) return;
  const int col = blockIdx.x * 16 + threadIdx.x % 16, q = threadIdx.x / 16;
  float v = 0;
  if (col < c)
    for (int b = q; b < blocks; b += 64) v += partial[(b * static_cast<int64_t>(3) + blockIdx.y) * c + col];
  s[q][threadIdx.x % 16] = v;
  __syncthreads();
  for (int half = 32; half > 0; half /= 2) {
    if (q < half) s[q][threadIdx.x % 16] += s[q + half][threadIdx.x % 16];
    __syncthreads();
  }
  if (q == 0 && col < c) static_cast<T *>(o)[col] = from_float<T>(s[0][threadIdx.x]);
}

// f(lanes, chunks a lane, threads a block) of the smallest shape that holds c values
template <class T, class F> int with_shape(int c, F &&f) {
  using std::integral_constant;
  const int chunks = static_cast<int>(div_up(c, kVec<T>));
#define SPIRA_SHAPE(G, NV, NT) \
  if (chunks <= G * NV) return f(integral_constant<int, G>{}, integral_constant<int, NV>{}, integral_constant<int, NT>{})
  SPIRA_SHAPE(8, 1, 256);
  SPIRA_SHAPE(16, 1, 256);
  SPIRA_SHAPE(32, 1, 256);
  SPIRA_SHAPE(64, 1, 256);
  SPIRA_SHAPE(64, 2, 256);
  SPIRA_SHAPE(256, 1, 256);
  SPIRA_SHAPE(256, 2, 256);
  SPIRA_SHAPE(1024, 1, 1024);
  SPIRA_SHAPE(1024, 2, 1024);
  if constexpr (sizeof(T) == 4) SPIRA_SHAPE(1024, 4, 1024);
#undef SPIRA_SHAPE
  set_error("gated_residual_norm: rows of more than 16384 channels");
  return kInvalidArgument;
}

// Blocks: what the CUs hold at once, each walking rows.  The backward pass's write
// their partial sums of the columns.
static int64_t forward_blocks(int64_t n, int rows_per_block) {
  return std::min<int64_t>(div_up(n, rows_per_block), 2048);
}
static int64_t backward_blocks(int64_t n, int rows_per_block) {
  return std::min<int64_t>(div_up(n, rows_per_block), 512);
}

static int check(int64_t n, int c, const void *x, const void *w, const void *h, const void *gate, int gate_form) {
  SPIRA_HIP_REQUIRE(n >= 0 && n < (int64_t(1) << 31), "gated_residual_norm: bad number of rows");
  SPIRA_HIP_REQUIRE(c > 0 && c <= 16384, "gated_residual_norm: needs 1 to 16384 channels");
  SPIRA_HIP_REQUIRE(n == 0 || x, "gated_residual_norm: null features");
  SPIRA_HIP_REQUIRE(gate_form >= kNone && gate_form <= kFull && (n == 0 || (gate_form == kNone) == (gate == nullptr)),
                    "gated_residual_norm: the gate does not fit its form");
  // (tensors without rows may have no address)
  SPIRA_HIP_REQUIRE(n == 0 || h || (!w && !gate), "gated_residual_norm: a norm or gate of no update");
  return kOk;
}

}  // namespace norm

}  // namespace spira_hip

using namespace spira_hip;

extern "C" {

int spira_hip_gated_residual_norm(const void *x, const void *h, int64_t n, int c, int dtype, const void *weight,
                                  const void *gate, int gate_form, int gate_sigmoid, float scale,
                                  const void *next_weight, float eps, void *r, void *next, float *inv_h, float *inv_r,
                                  hipStream_t stream) {
  if (int rc = norm::check(n, c, x, weight, h, gate, gate_form)) return rc;
  if (n == 0) return kOk;
  SPIRA_HIP_REQUIRE((next == nullptr) == (next_weight == nullptr) && (r == nullptr) == (h == nullptr) && (r || next),
                    "gated_residual_norm: outputs and inputs do not fit");
  norm::Args a{};
  a.x = x; a.h = h; a.w = weight; a.gate = gate; a.w_next = next_weight;
  a.n = n; a.c = c; a.gate_form = gate_form; a.sigmoid = gate_sigmoid; a.scale = scale; a.eps = eps;
  a.r = r; a.next = next; a.inv_h = inv_h; a.inv_r = inv_r;
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return norm::with_shape<T>(c, [&](auto G, auto NV, auto NT) -> int {
      constexpr int g = decltype(G)::value, nt = decltype(NT)::value;
      hipLaunchKernelGGL((norm::forward_kernel<T, g, decltype(NV)::value, nt>), dim3(norm::forward_blocks(n, nt / g)), dim3(nt), 0,
                         stream, a);
      SPIRA_HIP_LAUNCH_CHECK();
      return kOk;
    });
  });
}

int spira_hip_gated_residual_norm_backward_workspace(int64_t n, int c, int dtype, size_t *bytes) {
  SPIRA_HIP_REQUIRE(n >= 0 && c > 0, "gated_residual_norm: bad sizes");
  return with_type(dtype, [&](auto t) -> int {
    return norm::with_shape<decltype(t)>(c, [&](auto G, auto, auto NT) -> int {
      constexpr int rows = decltype(NT)::value / decltype(G)::value;
      *bytes = static_cast<size_t>(norm::backward_blocks(n, rows)) * 3 * c * sizeof(float);
      return kOk;
    });
  });
}

int spira_hip_gated_residual_norm_backward(const void *x, const void *h, int64_t n, int c, int dtype,
                                           const void *weight, const void *gate, int gate_form, int gate_sigmoid,
                                           float scale, const void *next_weight, const float *inv_h,
                                           const float *inv_r, const void *dr, const void *dnext, void *dx, void *dh,
                                           void *dweight, void *dgate, void *dnext_weight, void *workspace,
                                           size_t workspace_bytes, hipStream_t stream) {
  if (int rc = norm::check(n, c, x, weight, h, gate, gate_form)) return rc;
  SPIRA_HIP_REQUIRE(n == 0 || ((!weight || inv_h) && (!dnext || (inv_r && next_weight))),
                    "gated_residual_norm_backward: needs the forward pass's root mean squares");
  norm::Args a{};
  a.x = x; a.h = h; a.w = weight; a.gate = gate; a.w_next = next_weight;
  a.n = n; a.c = c; a.gate_form = gate_form; a.sigmoid = gate_form != norm::kNone && gate_sigmoid;
  a.scale = scale;
  a.inv_h = const_cast<float *>(inv_h); a.inv_r = const_cast<float *>(inv_r);
  a.dr = dr; a.dnext = dnext; a.dx = dx; a.dh = dh; a.dgate = dgate;
  const bool channel = gate_form == norm::kChannel;
  if (!dnext && n > 0) dnext_weight = nullptr;  // (no rows: zeros)
  const bool sums = (weight && dweight) || dnext_weight || (channel && dgate);
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return norm::with_shape<T>(c, [&](auto G, auto NV, auto NT) -> int {
      constexpr int g = decltype(G)::value, nt = decltype(NT)::value;
      const int64_t blocks = norm::backward_blocks(n, nt / g);
      if (sums) {
        SPIRA_HIP_REQUIRE(workspace_bytes >= static_cast<size_t>(blocks) * 3 * c * sizeof(float) &&
                              (workspace || blocks == 0),
                          "gated_residual_norm_backward: workspace too small");
        a.partial = static_cast<float *>(workspace);
      }
      if (n > 0) {
        if (channel)
          hipLaunchKernelGGL((norm::backward_kernel<T, g, decltype(NV)::value, nt, true>), dim3(blocks), dim3(nt), 0,
                             stream, a);
        else
          hipLaunchKernelGGL((norm::backward_kernel<T, g, decltype(NV)::value, nt, false>), dim3(blocks), dim3(nt), 0,
                             stream, a);
        SPIRA_HIP_LAUNCH_CHECK();
      }
      if (sums) {
        hipLaunchKernelGGL(norm::columns_kernel<T>, dim3(div_up(c, 16), 3), dim3(1024), 0, stream, a.partial,
                           static_cast<int>(blocks), c, weight ? dweight : nullptr, dnext_weight,
                           channel ? dgate : nullptr);
        SPIRA_HIP_LAUNCH_CHECK();
      }
      return kOk;
    });
  });
}

}  // extern "C"
