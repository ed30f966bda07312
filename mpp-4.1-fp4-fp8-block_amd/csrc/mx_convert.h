// mx_convert.h - loads and stores of f32, f16 and bf16 values (MX_DTYPE_*), as f32.
#pragma once

#include "../../include/mxfp4hip.h"
#include "mx_device.h"

namespace mx {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ float load_as_f32(const void* p, size_t i) {
  if constexpr (DT == MX_DTYPE_F32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == MX_DTYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
  else return (float)static_cast<const __bf16*>(p)[i];
}

// One rounding, to nearest even.
template <int DT>
__device__ __forceinline__ void store_from_f32(void* p, size_t i, float v) {
  if constexpr (DT == MX_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if constexpr (DT == MX_DTYPE_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
  else static_cast<__bf16*>(p)[i] = (__bf16)v;
}

// N = 8 (16-byte aligned) or 1 values
template <int DT, int N>
__device__ __forceinline__ void load_n_as_f32(const void* p, size_t i, float* v) {
  if constexpr (N == 1) {
    v[0] = load_as_f32<DT>(p, i);
  } else if constexpr (DT == MX_DTYPE_F32) {
    const v4f* q = reinterpret_cast<const v4f*>(static_cast<const float*>(p) + i);
    const v4f lo = q[0], hi = q[1];
#pragma unroll
    for (int u = 0; u < 4; u++) { v[u] = lo[u]; v[u + 4] = hi[u]; }
  } else if constexpr (DT == MX_DTYPE_F16) {
    const v8h h = *reinterpret_cast<const v8h*>(static_cast<const _Float16*>(p) + i);
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = (float)h[u];
  } else {
    const v8bf h = *reinterpret_cast<const v8bf*>(static_cast<const __bf16*>(p) + i);
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = (float)h[u];
  }
}

template <int DT, int N>
__device__ __forceinline__ void store_n_from_f32(void* p, size_t i, const float* v) {
  if constexpr (N == 1) {
    store_from_f32<DT>(p, i, v[0]);
  } else if constexpr (DT == MX_DTYPE_F32) {
    v4f* q = reinterpret_cast<v4f*>(static_cast<float*>(p) + i);
    q[0] = v4f{v[0], v[1], v[2], v[3]};
    q[1] = v4f{v[4], v[5], v[6], v[7]};
  } else if constexpr (DT == MX_DTYPE_F16) {
    v8h h;
#pragma unroll
    for (int u = 0; u < 8; u++) h[u] = (_Float16)v[u];
    *reinterpret_cast<v8h*>(static_cast<_Float16*>(p) + i) = h;
  } else {
    v8bf h;
#pragma unroll
    for (int u = 0; u < 8; u++) h[u] = (__bf16)v[u];
    *reinterpret_cast<v8bf*>(static_cast<__bf16*>(p) + i) = h;
  }
}

// Eight values at any address of their type, or the `left` that there still are (the
// others: 0, not stored).
template <int DT>
__device__ __forceinline__ void load_some_as_f32(const void* p, size_t i, int left, float* v) {
  constexpr int SIZE = DT == MX_DTYPE_F32 ? 4 : 2;
  if (left >= 8) {
    __attribute__((aligned(16))) uint8_t raw[8 * SIZE];
    __builtin_memcpy(raw, static_cast<const uint8_t*>(p) + i * SIZE, sizeof raw);
    load_n_as_f32<DT, 8>(raw, 0, v);
    return;
  }
#pragma unroll
  for (int u = 0; u < 8; u++) v[u] = u < left ? load_as_f32<DT>(p, i + u) : 0.0f;
}
template <int DT>
__device__ __forceinline__ void store_some_from_f32(void* p, size_t i, int left, const float* v) {
  constexpr int SIZE = DT == MX_DTYPE_F32 ? 4 : 2;
  if (left >= 8) {
    __attribute__((aligned(16))) uint8_t raw[8 * SIZE];
    store_n_from_f32<DT, 8>(raw, 0, v);
    __builtin_memcpy(static_cast<uint8_t*>(p) + i * SIZE, raw, sizeof raw);
    return;
  }
#pragma unroll
  for (int u = 0; u < 8; u++)
    if (u < left) store_from_f32<DT>(p, i + u, v[u]);
}

}  // namespace mx
