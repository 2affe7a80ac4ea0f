// rows.h — what the row kernels of a training step share on gfx950: vector
// loads and stores of fp32 or bf16 rows, sums over the lanes of a head or a
// block, launch checks.
#pragma once

#include "common.h"
#include "../../include/agpt_attn.h"

#include <cstdio>

namespace agpt_rows {

using agpt::bf16_t;
using agpt::block_x;
using agpt::block_y;

__device__ __forceinline__ int thread_x() { return static_cast<int>(__builtin_amdgcn_workitem_id_x()); }

// V consecutive elements as fp32, in one load (V a power of two, 16 bytes at most, aligned to its own size).
template <int V>
__device__ __forceinline__ void load_row(const float* __restrict__ p, float (&x)[V]) {
  if constexpr (V % 4 == 0) {
    agpt::load_vec<V>(p, x);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = p[i];
  }
}
template <int V>
__device__ __forceinline__ void load_row(const bf16_t* __restrict__ p, float (&x)[V]) {
  if constexpr (V % 4 == 0) {
    agpt::load_vec<V>(p, x);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = agpt::to_f32(p[i]);
  }
}

template <int V>
__device__ __forceinline__ void store_row(float* __restrict__ p, const float (&x)[V]) {
  if constexpr (V % 4 == 0) {
    agpt::store_vec<V>(p, x);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = x[i];
  }
}
// Rounded once, to the nearest bf16 (ties to even).
template <int V>
__device__ __forceinline__ void store_row(bf16_t* __restrict__ p, const float (&x)[V]) {
  if constexpr (V == 8) {
    *reinterpret_cast<uint4*>(p) = uint4{agpt::pack2_bf16(x[0], x[1]), agpt::pack2_bf16(x[2], x[3]),
                                         agpt::pack2_bf16(x[4], x[5]), agpt::pack2_bf16(x[6], x[7])};
  } else if constexpr (V == 4) {
    *reinterpret_cast<uint2*>(p) = uint2{agpt::pack2_bf16(x[0], x[1]), agpt::pack2_bf16(x[2], x[3])};
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i].bits = static_cast<uint16_t>(agpt::pack2_bf16(x[i], 0.0f));
  }
}

// V elements as they are in memory, loaded in one piece: what a row that is still
// on its way takes in registers.
template <typename T, int V>
struct Raw {
  static constexpr int kWords = V * static_cast<int>(sizeof(T)) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* __restrict__ p) {
    if constexpr (kWords == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
      static_assert(kWords == 2, "8 or 16 bytes");
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x; w[1] = v.y;
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void get(float (&x)[V]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        x[i] = __uint_as_float(w[i / 2] << 16);
        x[i + 1] = __uint_as_float(w[i / 2] & 0xffff0000u);
      }
    }
  }
};

template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xf, 0xf, false));
}

// Sum over aligned runs of L lanes (a power of two up to 64), the same bits
// in every lane of the run: pair swap, quad reverse, half-row and row mirror,
// then exchanges across 16 and 32 lanes.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (L > 1) v += dpp<0xB1>(v);
  if constexpr (L > 2) v += dpp<0x1B>(v);
  if constexpr (L > 4) v += dpp<0x141>(v);
  if constexpr (L > 8) v += dpp<0x140>(v);
  if constexpr (L > 16) v += __shfl_xor(v, 16);
  if constexpr (L > 32) v += __shfl_xor(v, 32);
  return v;
}

inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

inline int launch_status(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return AGPT_OK;
  char msg[160];
  snprintf(msg, sizeof(msg), "%s: launch failed: %s", what, hipGetErrorString(e));
  return agpt_internal_set_error(AGPT_ERR_DEVICE, msg);
}

inline int invalid(const char* what, const char* why) {
  char msg[240];
  snprintf(msg, sizeof(msg), "%s: %s", what, why);
  return agpt_internal_set_error(AGPT_ERR_INVALID_ARG, msg);
}

// out[j] = sum over n rows of part[., j], j < cols (row stride `ld`, a
// multiple of 4, at least cols; out 16-byte aligned), in a fixed order: one workgroup per 64 columns, 16
// lanes x float4 across them and 64 row slots down the rows, slot s summing
// rows s, s + 64, ...; the slots are folded in order.
constexpr int kFoldThreads = 1024;
__device__ __forceinline__ void fold_columns(const float* __restrict__ part, int64_t ld, int n, int cols, int blk,
                                             float* __restrict__ out) {
  __shared__ float4 red[kFoldThreads / 16][16];
  const int tid = thread_x(), c4 = tid & 15, slot = tid >> 4, col = blk * 64 + c4 * 4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < cols) {
    const float* p = part + col;
#pragma unroll 8
    for (int q = slot; q < n; q += kFoldThreads / 16) {
      const float4 v = *reinterpret_cast<const float4*>(p + q * ld);
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
  }
  red[slot][c4] = a;
  __syncthreads();
  // 64 slots -> 8 -> 1, each in slot order
  if (slot < 8) {
    a = red[slot * 8][c4];
    for (int t = 1; t < 8; ++t) {
      const float4 v = red[slot * 8 + t][c4];
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
  }
  __syncthreads();
  if (slot < 8) red[slot][c4] = a;
  __syncthreads();
  if (slot == 0 && col < cols) {
    for (int t = 1; t < 8; ++t) {
      const float4 v = red[t][c4];
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
    if (col + 4 <= cols) {
      *reinterpret_cast<float4*>(out + col) = a;
    } else {
      const float v[4] = {a.x, a.y, a.z, a.w};
      for (int i = 0; col + i < cols; ++i) out[col + i] = v[i];
    }
  }
}

}  // namespace agpt_rows
