// pcx_project.h -- what the two halves of the boards' projection share: pcx_project.hip (the product) and
// pcx_project_grad.hip (its gradients).  The mathematics is at the top of pcx_project.hip.
#pragma once

#include "pcx_internal.h"

#include <cstring>

namespace pcx {
namespace project {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));

constexpr int QUAD = 32;   // cells a lane pair reads at a time (16 bytes a lane)
constexpr int SLOTS = 512; // workgroups of 256 threads the chip holds at two per CU

struct Shape {
  int64_t n, row_stride;
  int64_t layer_offset[PCX_POST_MAX_DEPTH];  // stacked: where a layer lies within a board, -1: nowhere (all zero)
  int32_t cells, layers, hidden;
  int32_t groups;     // groups of four along the summed axis per cell
  int32_t parts;      // of a weight: 1, or 3 for float32
  int32_t quads;      // ceil(cells / 32)
  int32_t tiles;      // ceil(hidden / 32)
  int32_t stacked, activation, dtype;
  uint8_t chars[PCX_POST_MAX_DEPTH];
};

int make_shape(const pcx_project_desc* d, Shape* s, const char* who);
uint64_t backward_bytes(const Shape& s);
inline int elem_size(int dtype) { return dtype == PCX_F32 ? 4 : 2; }
inline bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// The first cell of a 32-cell quad.  The last quad of a larger board ends with the board (it begins inside the quad before
// it, and counts only what that one does not), so that no load needs a guard.
__host__ __device__ __forceinline__ int quad_start(int quad, int cells) {
  const int last = cells > QUAD ? cells - QUAD : 0;
  return quad * QUAD < last ? quad * QUAD : last;
}

template <int DT> struct Num;
template <> struct Num<PCX_F32> {
  typedef float T;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Num<PCX_F16> {
  typedef _Float16 T;
  static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};
template <> struct Num<PCX_BF16> {
  typedef __bf16 T;
  static __device__ __forceinline__ float get(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};

// Part `p` of a number in `parts` bfloat16 numbers: the upper 16 bits of what the earlier parts left over -- cut off, not
// rounded, so that nothing overflows and three parts hold all 24 bits -- and the last of fewer parts rounded.  Infinities
// and NaN are whole in part 0.
__device__ __forceinline__ uint16_t part_of(float w, int p, int parts) {
  uint32_t u = __float_as_uint(w);
  if ((u & 0x7F800000u) == 0x7F800000u) return p ? 0 : (uint16_t)((u >> 16) | ((u & 0x7FFFFFu) ? 0x40u : 0u));
  for (int i = 0; i < p; ++i) {
    w -= __uint_as_float(u & 0xFFFF0000u);
    u = __float_as_uint(w);
  }
  if (p == parts - 1) return __builtin_bit_cast(uint16_t, (__bf16)w);
  return (uint16_t)(u >> 16);
}

// The kernel's (one) argument where the runtime put it.  Its arrays are indexed there: indexed in the argument itself, the
// compiler copies the whole structure into every lane's scratch memory.
template <typename A>
__device__ __forceinline__ const __attribute__((address_space(4))) A* argument() {
  return (const __attribute__((address_space(4))) A*)__builtin_amdgcn_kernarg_segment_ptr();
}

template <bool F16>
__device__ __forceinline__ f32x16 dense_step(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 16 bytes a lane straight from memory into LDS: lane i's land at lds + 16 i (lds: the same for the whole wave).
__device__ __forceinline__ void copy_in(const uint8_t* from, uint8_t* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
// What copy_in() fetched has arrived, for every wave of the workgroup, and nobody reads the buffer of the stage before.
// NEWER: how many requests at least were made after the copies that are waited for (requests complete in order).
template <int NEWER>
__device__ __forceinline__ void stage_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NEWER) : "memory"); }

// Bytes c .. c + 3 of a board of fewer than 32 cells; zeros past its end, which is never read (the last byte is, again: four
// loads without branches, none of which waits for another).
__device__ __forceinline__ uint32_t edge_dword(const uint8_t* row, int c, int cells) {
  uint32_t v = 0;
  for (int i = 0; i < 4; ++i)
    v |= (uint32_t)row[c + i < cells ? c + i : cells - 1] << (8 * i);
  return c + 4 <= cells ? v : c < cells ? v & ((1u << (8 * (cells - c))) - 1u) : 0u;
}

}  // namespace project
}  // namespace pcx
