// pcx_project.hip -- the first layer of a policy, read from the boards: act(features . weight^T + bias) + residual, where
// `features` is the 0/1 stack of layers that rendering.ObservationToFeatureArray would write (rendering.py:545-661), and
// the gradients of its weight and bias.  The stack is never stored: the kernels expand it from the boards' characters
// (or from stacked uint8 layers, where layers overlap) in the registers that feed the matrix units.
//
// Mathematics.  With x[b][l][c] = 1 where board b shows character l at cell c:
//   z[b][h] = sum_{l,c} x[b][l][c] w[h][l][c] + bias[h],   y = act(z) + residual,
//   dz = dy act'(z),   dw[h][l][c] = sum_b dz[b][h] x[b][l][c],   dbias[h] = sum_b dz[b][h].
// A cell shows one character, so of the four features (four layers of one cell) at most one is set: the left operand is
// 2:4 sparse along the summed axis by construction, and v_smfmac_f32_32x32x32 multiplies it at 3,750 TFLOP/s where the
// dense v_mfma_f32_32x32x16 gives 2,270 (both measured here, register operands only).  Overlapping layers use the same
// instruction with two layers to a group of four (the other two weights are zero): the dense rate, one kernel.
// A set feature is the number 2 -- the bit pattern 0x4000 in bfloat16 AND in float16 -- so that expanding a feature pair
// is one shift and one mask; the other operand is halved instead (float16, whose small numbers have no bit to spare and
// whose sums cannot leave float32's range: the sum is), which is exact down to the last subnormal bit.  float32 weights
// are split into three bfloat16 parts (8 + 8 + 8 bits: none is lost), and every product is exact, so they cost three
// passes and no accuracy.  All sums are float32.
#include "pcx_internal.h"

#include <cstring>

using pcx::set_error;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));

constexpr int STEPS = 4;         // matrix steps (32 features each) a workgroup stages at a time
constexpr int FRAG = 2048;       // bytes of one right operand: 32 features x 32 hidden units x 2
constexpr int QUAD = 32;         // cells a lane pair reads at a time (16 bytes a lane)
constexpr int BLK = 64;          // boards per stage of the weight gradient

struct Shape {
  int64_t n, row_stride;
  int64_t layer_offset[PCX_POST_MAX_DEPTH];  // stacked: where a layer lies within a board, -1: nowhere (all zero)
  int32_t cells, layers, hidden;
  int32_t groups;     // groups of four along the summed axis per cell
  int32_t parts;      // 1, or 3 for float32 weights
  int32_t quads;      // ceil(cells / 32)
  int32_t tiles;      // ceil(hidden / 32)
  int32_t stacked, activation, dtype;
  uint8_t chars[PCX_POST_MAX_DEPTH];
};

int elem_size(int dtype) { return dtype == PCX_F32 ? 4 : 2; }

int make_shape(const pcx_project_desc* d, Shape* s, const char* who) {
  if (!d) return set_error(PCX_E_INVALID, "%s: null description", who);
  if (d->dtype != PCX_F32 && d->dtype != PCX_F16 && d->dtype != PCX_BF16)
    return set_error(PCX_E_INVALID, "%s: the weights are float32, float16 or bfloat16", who);
  if (d->activation < PCX_ACT_NONE || d->activation > PCX_ACT_GELU) return set_error(PCX_E_INVALID, "%s: unknown activation", who);
  if (d->cells < 1 || d->cells > 1 << 20 || d->n_layers < 1 || d->n_layers > PCX_POST_MAX_DEPTH || d->hidden < 1 || d->hidden > 1 << 16)
    return set_error(PCX_E_INVALID, "%s: cells, layers or hidden units out of range", who);
  if (d->n < 0 || d->n > (int64_t)1 << 31) return set_error(PCX_E_INVALID, "%s: %lld boards", who, (long long)d->n);
  if (d->row_stride < 0) return set_error(PCX_E_INVALID, "%s: negative stride", who);
  if (!d->stacked)
    for (int i = 0; i < d->n_layers; ++i)
      for (int j = 0; j < i; ++j)
        if (d->chars[i] == d->chars[j]) return set_error(PCX_E_INVALID, "%s: layer '%c' twice", who, d->chars[i]);
  s->n = d->n; s->row_stride = d->row_stride;
  memcpy(s->layer_offset, d->layer_offset, sizeof s->layer_offset);
  s->cells = d->cells; s->layers = d->n_layers; s->hidden = d->hidden;
  s->groups = d->stacked ? (d->n_layers + 1) / 2 : (d->n_layers + 3) / 4;
  s->parts = d->dtype == PCX_F32 ? 3 : 1;
  s->quads = (d->cells + QUAD - 1) / QUAD;
  s->tiles = (d->hidden + 31) / 32;
  s->stacked = d->stacked != 0; s->activation = d->activation; s->dtype = d->dtype;
  memcpy(s->chars, d->chars, sizeof s->chars);
  if ((int64_t)s->quads * 4 * s->groups * s->parts * s->tiles > (int64_t)1 << 27)
    return set_error(PCX_E_INVALID, "%s: the weight is too large", who);
  return 0;
}

// ---------------------------------------------------------------- numbers

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

// Part `p` of a float32 as bfloat16 bits: the upper 16 bits of what the earlier parts left over (cut off, not rounded, so
// that nothing overflows and three parts hold all 24 bits).  Infinities and NaN are whole in part 0.
__device__ __forceinline__ uint16_t part_of(float w, int p) {
  uint32_t u = __float_as_uint(w);
  if ((u & 0x7F800000u) == 0x7F800000u) return p ? 0 : (uint16_t)((u >> 16) | ((u & 0x7FFFFFu) ? 0x40u : 0u));
  for (int i = 0; i < p; ++i) {
    w -= __uint_as_float(u & 0xFFFF0000u);
    u = __float_as_uint(w);
  }
  return (uint16_t)(u >> 16);
}

// The 16 bits of one weight or gradient as the matrix unit takes it, and what its sums are multiplied by: a feature is 2.
template <int DT> constexpr float SCALE = DT == PCX_F16 ? 0.5f : 1.0f;
template <int DT>
__device__ __forceinline__ uint16_t operand_bits(float v, int part) {
  if constexpr (DT == PCX_F32) {
    return part_of(0.5f * v, part);
  } else {
    const typename Num<DT>::T r = Num<DT>::put(DT == PCX_F16 ? v : 0.5f * v);
    return __builtin_bit_cast(uint16_t, r);
  }
}

__device__ __forceinline__ void activate(int act, float z, float* y, float* slope) {
  if (act == PCX_ACT_RELU) {
    *y = z > 0.0f ? z : (z != z ? z : 0.0f); *slope = z > 0.0f ? 1.0f : 0.0f;
  } else if (act == PCX_ACT_SILU) {
    const float s = 1.0f / (1.0f + expf(-z));
    *y = z * s; *slope = s * (1.0f + z * (1.0f - s));
  } else if (act == PCX_ACT_TANH) {
    const float t = tanhf(z);
    *y = t; *slope = 1.0f - t * t;
  } else if (act == PCX_ACT_GELU) {
    const float cdf = 0.5f * (1.0f + erff(z * 0.70710678118654752f));
    *y = z * cdf; *slope = cdf + z * expf(-0.5f * z * z) * 0.3989422804014327f;
  } else {
    *y = z; *slope = 1.0f;
  }
}

// ---------------------------------------------------------------- laying the weight out

// Step order: (quad of 32 cells, octet j, group g, part) for characters, (quad, g, j, part) for stacked layers.  Within a
// step the instruction sums 32 features; lane (column c, half hb) holds 16 of them, element e standing for cell
// 32 q + 16 (e / 8) + 4 j + 2 hb + (e % 8) / 4 and position e % 4 of group g (measured lane layout of the instruction:
// the sparse side's half A covers features 16 A .. 16 A + 15, the dense side's element e feature 16 (e / 8) + 8 hb + e % 8).
// One thread writes the 16 bytes of half a lane's elements; the two halves of a lane are 1 KB apart, so that the LDS reads
// of a wave are contiguous.
template <int DT>
__global__ __launch_bounds__(256) void pcx_project_layout(Shape s, const typename Num<DT>::T* __restrict__ w, u32x4* __restrict__ packed) {
  const int64_t total = (int64_t)s.quads * 4 * s.groups * s.parts * s.tiles * 128;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int lane = (int)(i & 63), e8 = (int)((i >> 6) & 1);
    int64_t f = i >> 7;
    const int tile = (int)(f % s.tiles); f /= s.tiles;
    const int part = (int)(f % s.parts); f /= s.parts;
    int j, g;
    if (s.stacked) { j = (int)(f & 3); f >>= 2; g = (int)(f % s.groups); f /= s.groups; }
    else { g = (int)(f % s.groups); f /= s.groups; j = (int)(f & 3); f >>= 2; }
    const int q = (int)f, h = tile * 32 + (lane & 31), hb = lane >> 5;
    uint32_t word[4] = {0, 0, 0, 0};
    if (h < s.hidden) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int cell = q * QUAD + e8 * 16 + j * 4 + hb * 2 + (e >> 2), pos = e & 3;
        const int layer = s.stacked ? (pos < 2 ? g * 2 + pos : s.layers) : g * 4 + pos;
        if (cell < s.cells && layer < s.layers) {
          const float v = Num<DT>::get(w[((int64_t)h * s.layers + layer) * s.cells + cell]);
          word[e >> 1] |= (uint32_t)operand_bits<DT>(v, part) << (16 * (e & 1));
        }
      }
    }
    u32x4 out = {word[0], word[1], word[2], word[3]};
    packed[i] = out;
  }
}

// ---------------------------------------------------------------- the product

struct ForwardArgs {
  Shape s;
  const uint8_t* boards;
  const uint8_t* packed;
  const void* bias;      // or null
  const void* residual;  // [n][hidden], or null
  void* out;             // [n][hidden]
  void* slope;           // act'(z) [n][hidden] for the backward pass, or null
  float* partial;        // [splits][n][hidden]: raw sums when the cells are divided among workgroups
  int32_t splits, mblocks, nblocks, chunk;
  int32_t wide;          // hidden is a multiple of four and every array aligned for it
};

// One 32-bit word of up to four cells; cells past the end read as the last ones do (their weights are zero) and never as
// memory that is not this board's.
__device__ __forceinline__ uint32_t edge_dword(const uint8_t* row, int c, int cells) {
  uint32_t v = 0;
  if (c + 4 <= cells) { __builtin_memcpy(&v, row + c, 4); return v; }
  for (int i = 0; i < 4; ++i)
    if (c + i < cells) v |= (uint32_t)row[c + i] << (8 * i);
  return v;
}
__device__ __forceinline__ u32x4 load_cells(const uint8_t* row, int c, int cells) {
  u32x4 v;
  if (c + 16 <= cells) { __builtin_memcpy(&v, row + c, 16); return v; }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = edge_dword(row, c + 4 * i, cells);
  return v;
}
// bit 6 of every byte that is not zero
__device__ __forceinline__ uint32_t set_bytes(uint32_t b) {
  return (((((b & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | b) >> 1) & 0x40404040u);
}

// 16 bytes a lane straight from memory into LDS: lane i's land at lds + 16 i (lds: the same for the whole wave).
__device__ __forceinline__ void copy_in(const uint8_t* from, uint8_t* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

template <bool F16>
__device__ __forceinline__ f32x16 sparse_step(u32x4 a, u32x8 b, f32x16 c, int index) {
  if constexpr (F16)
    return __builtin_amdgcn_smfmac_f32_32x32x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x16, b), c, index, 0, 0);
  else
    return __builtin_amdgcn_smfmac_f32_32x32x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x16, b), c, index, 0, 0);
}

// Bias, activation and residual on up to four neighbouring sums of one board (count < 4 at the last columns; `wide`: the
// rows keep four elements aligned).
template <int DT>
__device__ __forceinline__ void finish(const ForwardArgs& a, int64_t row, int col, const float* sum, int count, bool wide) {
  typedef typename Num<DT>::T T;
  struct __align__(4 * sizeof(T)) Four { T v[4]; };
  const int64_t at = row * a.s.hidden + col;
  Four bias = {}, res = {}, out, slope;
  const T* const pb = reinterpret_cast<const T*>(a.bias);
  const T* const pr = reinterpret_cast<const T*>(a.residual);
  T* const po = reinterpret_cast<T*>(a.out);
  T* const ps = reinterpret_cast<T*>(a.slope);
  if (pb)
    for (int i = 0; i < count; ++i) bias.v[i] = pb[col + i];
  if (pr) {
    if (wide) res = *reinterpret_cast<const Four*>(pr + at);
    else
      for (int i = 0; i < count; ++i) res.v[i] = pr[at + i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y, d;
    activate(a.s.activation, sum[i] + (pb ? Num<DT>::get(bias.v[i]) : 0.0f), &y, &d);
    if (pr) y += Num<DT>::get(res.v[i]);
    out.v[i] = Num<DT>::put(y);
    slope.v[i] = Num<DT>::put(d);
  }
  if (wide) {
    *reinterpret_cast<Four*>(po + at) = out;
    if (ps) *reinterpret_cast<Four*>(ps + at) = slope;
  } else {
    for (int i = 0; i < count; ++i) {
      po[at + i] = out.v[i];
      if (ps) ps[at + i] = slope.v[i];
    }
  }
}

// A wave holds MT x NT tiles of 32 x 32 sums; 4 / WN waves lie along the boards and WN along the hidden units.
template <int DT, bool STACKED, int MT, int NT, int WN>
__global__ __launch_bounds__(256, 2) void pcx_project_forward_kernel(ForwardArgs a) {
  constexpr int FR = NT * WN;                 // right operands per step
  constexpr int STAGE = STEPS * FR * FRAG;
  constexpr int DMA = STAGE / 4096;           // 1 KB copies per wave and stage
  constexpr int MROWS = (4 / WN) * MT * 32;
  const Shape& s = a.s;
  extern __shared__ __align__(16) uint8_t lds[];
  uint32_t* const lut = reinterpret_cast<uint32_t*>(lds + 2 * STAGE);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // consecutive tiles of a board block go to one XCD (workgroup i runs on XCD i % 8), whose L2 then serves the boards once
  const uint32_t id = (blockIdx.x & 7u) * (uint32_t)a.chunk + (blockIdx.x >> 3);
  if (id >= (uint32_t)a.mblocks * a.nblocks * a.splits) return;
  const int nb = (int)(id % (uint32_t)a.nblocks);
  const uint32_t rest = id / (uint32_t)a.nblocks;
  const int split = (int)(rest % (uint32_t)a.splits), mb = (int)(rest / (uint32_t)a.splits);
  if constexpr (!STACKED) {
    // character -> bit g (16 + g): a feature of group g in its low (high) slot; bits 8..11: the two slots' positions.
    // The two positions of a group ascend: (p, 3) with the feature in the low slot for p < 3, (0, 3) in the high one for 3.
    uint32_t v = 4u << 8;  // (0, 1)
    for (int l = 0; l < s.layers; ++l)
      if (s.chars[l] == tid) {
        const int p = l & 3, g = l >> 2;
        v = p < 3 ? (1u << g) | ((uint32_t)(p | 12) << 8) : (1u << (16 + g)) | (12u << 8);
      }
    lut[tid] = v;
  }
  const int q0 = (int)((int64_t)s.quads * split / a.splits), q1 = (int)((int64_t)s.quads * (split + 1) / a.splits);
  const int per_quad = 4 * s.groups * s.parts, stages = (q1 - q0) * per_quad / STEPS;
  const int tile0 = nb * FR, live = s.tiles - tile0 < FR ? s.tiles - tile0 : FR;
  const uint8_t* const src = a.packed + ((int64_t)q0 * per_quad * s.tiles + tile0) * FRAG;
  const int wm = wave / WN, wn = wave % WN, half = lane >> 5;
  const int64_t row0 = (int64_t)mb * MROWS + wm * MT * 32;
  const uint8_t* row[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    int64_t r = row0 + m * 32 + (lane & 31);
    row[m] = a.boards + (r < s.n ? r : s.n - 1) * s.row_stride;
  }
  auto stage_in = [&](int st) {
    uint8_t* const dst = lds + (st & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < DMA; ++i) {
      const int k = wave * DMA + i, step = k / (2 * FR), off = k % (2 * FR);  // 1 KB pieces of the stage, 2 FR of them to a step
      if (off < 2 * live)
        copy_in(src + ((int64_t)(st * STEPS + step) * s.tiles) * FRAG + off * 1024 + lane * 16, dst + k * 1024);
    }
  };
  f32x16 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[m][t][i] = 0.0f;
  constexpr int PL = STACKED ? 2 : 1;  // board words in flight: one plane of characters, or a group's two layers
  u32x4 cur[MT][PL], nxt[MT][PL];
  auto fetch = [&](int q, int g) {
    const int c = q * QUAD + half * 16;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if constexpr (STACKED) {
#pragma unroll
        for (int l = 0; l < 2; ++l) {
          nxt[m][l] = u32x4{0, 0, 0, 0};
          if (2 * g + l < s.layers && s.layer_offset[2 * g + l] >= 0) nxt[m][l] = load_cells(row[m] + s.layer_offset[2 * g + l], c, s.cells);
        }
      } else {
        nxt[m][0] = load_cells(row[m], c, s.cells);
      }
    }
  };
  uint32_t word[MT][4];  // the cells' feature bits
  int index[MT];
  u32x4 left[MT];
  int q = q0, g = 0, j = 0, part = 0;
  fetch(q0, 0);
  stage_in(0);
  for (int st = 0; st < stages; ++st) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // this stage has arrived, and nobody reads the buffer of the one before any more
    if (st + 1 < stages) stage_in(st + 1);
    const uint8_t* const base = lds + (st & 1) * STAGE + wn * NT * FRAG + lane * 16;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      if (part == 0) {
        if constexpr (STACKED) {
          if (j == 0) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int l = 0; l < 2; ++l) cur[m][l] = nxt[m][l];
            if (g + 1 < s.groups) fetch(q, g + 1);
            else if (q + 1 < q1) fetch(q + 1, 0);
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint32_t lo = set_bytes(cur[m][0][0]), hi = set_bytes(cur[m][1][0]);
            left[m][0] = __builtin_amdgcn_perm(hi, lo, 0x040C000Cu);
            left[m][1] = __builtin_amdgcn_perm(hi, lo, 0x050C010Cu);
            left[m][2] = __builtin_amdgcn_perm(hi, lo, 0x060C020Cu);
            left[m][3] = __builtin_amdgcn_perm(hi, lo, 0x070C030Cu);
            index[m] = 0x4444;
#pragma unroll
            for (int l = 0; l < 2; ++l) { cur[m][l][0] = cur[m][l][1]; cur[m][l][1] = cur[m][l][2]; cur[m][l][2] = cur[m][l][3]; }
          }
        } else {
          if (g == 0) {
            if (j == 0) {
#pragma unroll
              for (int m = 0; m < MT; ++m) cur[m][0] = nxt[m][0];
              if (q + 1 < q1) fetch(q + 1, 0);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const uint32_t d = cur[m][0][0];
              cur[m][0][0] = cur[m][0][1]; cur[m][0][1] = cur[m][0][2]; cur[m][0][2] = cur[m][0][3];
              index[m] = 0;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                word[m][c] = lut[(d >> (8 * c)) & 255u];
                index[m] |= (int)(((word[m][c] >> 8) & 15u) << (4 * c));
              }
            }
          }
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int c = 0; c < 4; ++c) left[m][c] = (word[m][c] << (14 - g)) & 0x40004000u;
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint8_t* const at = base + (k * FR + t) * FRAG;
        const u32x4 b0 = *reinterpret_cast<const u32x4*>(at), b1 = *reinterpret_cast<const u32x4*>(at + 1024);
        const u32x8 right = {b0[0], b0[1], b0[2], b0[3], b1[0], b1[1], b1[2], b1[3]};
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m][t] = sparse_step<DT == PCX_F16>(left[m], right, acc[m][t], index[m]);
      }
      if (++part == s.parts) {
        part = 0;
        if constexpr (STACKED) { if (++j == 4) { j = 0; if (++g == s.groups) { g = 0; ++q; } } }
        else { if (++g == s.groups) { g = 0; if (++j == 4) { j = 0; ++q; } } }
      }
    }
  }
  // Out through LDS, 32 boards at a time and each wave by itself: a lane then has four neighbouring hidden units of one
  // board, and a wave writes whole rows of its tile.
  constexpr int PITCH = NT * 32 + 4, LANES = NT * 8;  // lanes per row
  __syncthreads();
  float* const mine = reinterpret_cast<float*>(lds) + wave * 32 * PITCH;
  const int col0 = (tile0 + wn * NT) * 32 + (lane % LANES) * 4;
  const int count = a.s.hidden - col0 < 4 ? a.s.hidden - col0 : 4;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) mine[(8 * (i >> 2) + 4 * half + (i & 3)) * PITCH + t * 32 + (lane & 31)] = SCALE<DT> * acc[m][t][i];
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 64 / LANES) {
      const int r = r0 + lane / LANES;
      const int64_t board = row0 + m * 32 + r;
      const float4 v = *reinterpret_cast<const float4*>(mine + r * PITCH + (lane % LANES) * 4);
      const float sum[4] = {v.x, v.y, v.z, v.w};
      if (board >= s.n || count <= 0) continue;
      if (a.splits > 1) {
        float* const to = a.partial + ((int64_t)split * s.n + board) * s.hidden + col0;
        if (a.wide) *reinterpret_cast<float4*>(to) = v;
        else
          for (int i = 0; i < count; ++i) to[i] = sum[i];
      } else {
        finish<DT>(a, board, col0, sum, count, a.wide);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The cells' partial sums joined in a fixed order, and the epilogue.
template <int DT>
__global__ __launch_bounds__(256) void pcx_project_join(ForwardArgs a) {
  const int quads = (a.s.hidden + 3) / 4;
  const int64_t total = a.s.n * quads, plane = a.s.n * a.s.hidden;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / quads;
    const int col = (int)(i - row * quads) * 4, count = a.s.hidden - col < 4 ? a.s.hidden - col : 4;
    const float* from = a.partial + row * a.s.hidden + col;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < a.splits; ++k, from += plane) {
      if (a.wide) {
        const float4 v = *reinterpret_cast<const float4*>(from);
        sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
      } else {
        for (int c = 0; c < count; ++c) sum[c] += from[c];
      }
    }
    finish<DT>(a, row, col, sum, count, a.wide);
  }
}

// ---------------------------------------------------------------- the gradients

struct BackwardArgs {
  Shape s;
  const uint8_t* boards;
  const void* grad_out;  // [n][hidden]
  const void* slope;     // [n][hidden], or null: no activation
  uint8_t* frags;        // dz as left operands: [ceil(n / 64) * 4][htiles][parts][64 lanes][8]
  float* bias_part;      // [bias_blocks][hidden]
  float* partial;        // [splits][hidden][layers][cells]
  void* grad_weight;     // or null
  void* grad_bias;       // or null
  int32_t blocks;        // ceil(n / 64)
  int32_t htiles;        // tiles of 32 hidden units, a whole number of workgroup tiles
  int32_t bias_blocks, splits, cell_blocks, layer_blocks, hblocks, chunk;
};

// dz = dy act'(z), turned round into the matrix unit's left operand (32 hidden units x 16 boards), and its column sums.
// dz is rounded to the weights' type -- what a framework that stores it between two operators does -- and summed for the
// bias before that rounding; float32 keeps all its bits in three parts.
template <int DT>
__global__ __launch_bounds__(256) void pcx_project_turn(BackwardArgs a) {
  typedef typename Num<DT>::T T;
  const Shape& s = a.s;
  __shared__ float tile[BLK][65];
  const int tid = threadIdx.x, h0 = blockIdx.y * 64;
  const T* const dy = reinterpret_cast<const T*>(a.grad_out);
  const T* const sl = reinterpret_cast<const T*>(a.slope);
  float total = 0.0f;
  for (int b = blockIdx.x; b < a.blocks; b += gridDim.x) {
    for (int i = tid; i < BLK * 64; i += 256) {
      const int r = i >> 6, c = i & 63;
      const int64_t gr = (int64_t)b * BLK + r;
      float v = 0.0f;
      if (gr < s.n && h0 + c < s.hidden) {
        const int64_t at = gr * s.hidden + h0 + c;
        v = Num<DT>::get(dy[at]);
        if (sl) v *= Num<DT>::get(sl[at]);
      }
      tile[r][c] = v;
    }
    __syncthreads();
    if (tid < 64) {
      float t = 0.0f;
      for (int r = 0; r < BLK; ++r) t += tile[r][tid];
      total += t;
    }
    if (a.frags)
      for (int i = tid; i < 4 * 2 * 64; i += 256) {
        const int lane = i & 63, ht = (i >> 6) & 1, kb = i >> 7;
        const int tile_h = blockIdx.y * 2 + ht;
        if (tile_h >= a.htiles) continue;
        for (int p = 0; p < s.parts; ++p) {
          u32x4 w = {0, 0, 0, 0};
#pragma unroll
          for (int e = 0; e < 8; ++e)
            w[e >> 1] |= (uint32_t)operand_bits<DT>(tile[kb * 16 + (lane >> 5) * 8 + e][ht * 32 + (lane & 31)], p) << (16 * (e & 1));
          reinterpret_cast<u32x4*>(a.frags)[((((int64_t)b * 4 + kb) * a.htiles + tile_h) * s.parts + p) * 64 + lane] = w;
        }
      }
    __syncthreads();
  }
  if (tid < 64 && h0 + tid < s.hidden && a.grad_bias) a.bias_part[(int64_t)blockIdx.x * s.hidden + h0 + tid] = total;
}

template <bool F16>
__device__ __forceinline__ f32x16 dense_step(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// dw[h][l][c] over a run of boards: a workgroup owns NH tiles of hidden units x 32 cells x 8 layers (two layers a wave).
// The right operand is the feature bit of 8 consecutive boards at one cell: the boards are turned round once per stage
// into LDS as a word of layer bits per (cell, board), from which every layer's operand is one shift and one mask.
template <int DT, bool STACKED, int NH>
__global__ __launch_bounds__(256, 2) void pcx_project_weight_grad(BackwardArgs a) {
  constexpr int PARTS = DT == PCX_F32 ? 3 : 1;
  constexpr int STAGE = 4 * NH * PARTS * 1024;
  constexpr int PITCH = BLK + 8;                // words per cell: 16-byte reads of one wave spread over the banks
  constexpr int MASKS = 32 * PITCH * 2;
  const Shape& s = a.s;
  extern __shared__ __align__(16) uint8_t lds[];
  uint16_t* const lut = reinterpret_cast<uint16_t*>(lds + 2 * STAGE + 2 * MASKS);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const uint32_t tiles = (uint32_t)a.cell_blocks * a.layer_blocks * a.hblocks;
  // the tiles of one run of boards go to one XCD, whose L2 then serves dz and the boards once
  const uint32_t id = (blockIdx.x & 7u) * (uint32_t)a.chunk + (blockIdx.x >> 3);
  if (id >= tiles * (uint32_t)a.splits) return;
  const int split = (int)(id / tiles);
  uint32_t t = id % tiles;
  const int hb = (int)(t % (uint32_t)a.hblocks); t /= (uint32_t)a.hblocks;
  const int lb = (int)(t % (uint32_t)a.layer_blocks), cb = (int)(t / (uint32_t)a.layer_blocks);
  const int l0 = lb * 8, c0 = cb * 32;
  if constexpr (!STACKED) {
    uint32_t v = 0;
    for (int l = 0; l < 8; ++l)
      if (l0 + l < s.layers && s.chars[l0 + l] == tid) v = 128u << l;
    lut[tid] = (uint16_t)v;
  }
  const int b0 = (int)((int64_t)a.blocks * split / a.splits), b1 = (int)((int64_t)a.blocks * (split + 1) / a.splits);
  auto stage_in = [&](int b) {
    uint8_t* const dst = lds + (b & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < NH * PARTS; ++i) {
      const int k = wave * NH * PARTS + i, kb = k / (NH * PARTS), off = k % (NH * PARTS);
      copy_in(a.frags + ((((int64_t)b * 4 + kb) * a.htiles + hb * NH) * PARTS + off) * 1024 + lane * 16, dst + k * 1024);
    }
  };
  // a thread turns two boards x four cells round
  const int pair = tid >> 3, cell = (tid & 7) * 4;
  constexpr int PL = STACKED ? 8 : 1;
  uint32_t raw[2][PL];
  auto fetch = [&](int b) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t gr = (int64_t)b * BLK + pair * 2 + r;
      const uint8_t* const at = a.boards + (gr < s.n ? gr : s.n - 1) * s.row_stride;  // (boards past the end meet dz = 0)
#pragma unroll
      for (int l = 0; l < PL; ++l) {
        raw[r][l] = 0;
        if (c0 + cell >= s.cells) continue;
        if constexpr (STACKED) {
          if (l0 + l < s.layers && s.layer_offset[l0 + l] >= 0) raw[r][l] = edge_dword(at + s.layer_offset[l0 + l], c0 + cell, s.cells);
        } else {
          raw[r][l] = edge_dword(at, c0 + cell, s.cells);
        }
      }
    }
  };
  auto turn = [&](int b) {
    uint8_t* const dst = lds + 2 * STAGE + (b & 1) * MASKS;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t m[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if constexpr (STACKED) {
          m[r] = 0;
#pragma unroll
          for (int l = 0; l < 8; ++l) m[r] |= ((raw[r][l] >> (8 * c)) & 255u) ? 128u << l : 0u;
        } else {
          m[r] = lut[(raw[r][0] >> (8 * c)) & 255u];
        }
      }
      *reinterpret_cast<uint32_t*>(dst + ((cell + c) * PITCH + pair * 2) * 2) = m[0] | (m[1] << 16);
    }
  };
  f32x16 acc[2][NH];
#pragma unroll
  for (int l = 0; l < 2; ++l)
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[l][h][i] = 0.0f;
  if (b0 < b1) {
    fetch(b0);
    stage_in(b0);
  }
  __syncthreads();  // the table
  if (b0 < b1) turn(b0);
  const bool work = l0 + wave * 2 < s.layers;
  const int shift = 7 - wave * 2;
  for (int b = b0; b < b1; ++b) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (b + 1 < b1) {
      fetch(b + 1);
      stage_in(b + 1);
    }
    if (work) {
      const uint8_t* const dz = lds + (b & 1) * STAGE + lane * 16;
      const uint8_t* const masks = lds + 2 * STAGE + (b & 1) * MASKS + ((lane & 31) * PITCH + half * 8) * 2;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        const u32x4 m = *reinterpret_cast<const u32x4*>(masks + kb * 32);
        u32x4 right[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          right[0][e] = (m[e] << shift) & 0x40004000u;
          right[1][e] = (m[e] << (shift - 1)) & 0x40004000u;
        }
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int p = 0; p < PARTS; ++p) {
            const u32x4 left = *reinterpret_cast<const u32x4*>(dz + ((kb * NH + h) * PARTS + p) * 1024);
            acc[0][h] = dense_step<DT == PCX_F16>(left, right[0], acc[0][h]);
            acc[1][h] = dense_step<DT == PCX_F16>(left, right[1], acc[1][h]);
          }
      }
    }
    if (b + 1 < b1) turn(b + 1);
  }
  const int c = c0 + (lane & 31);
  if (c >= s.cells) return;
#pragma unroll
  for (int l = 0; l < 2; ++l) {
    const int layer = l0 + wave * 2 + l;
    if (layer >= s.layers) continue;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int unit = (hb * NH + h) * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
        if (unit < s.hidden) a.partial[(((int64_t)split * s.hidden + unit) * s.layers + layer) * s.cells + c] = SCALE<DT> * acc[l][h][i];
      }
  }
}

// The runs' partial sums joined in a fixed order.
template <int DT>
__global__ __launch_bounds__(256) void pcx_project_weight_join(BackwardArgs a) {
  typedef typename Num<DT>::T T;
  const int64_t total = (int64_t)a.s.hidden * a.s.layers * a.s.cells;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    float sum = 0.0f;
    for (int k = 0; k < a.splits; ++k) sum += a.partial[(int64_t)k * total + i];
    reinterpret_cast<T*>(a.grad_weight)[i] = Num<DT>::put(sum);
  }
}
template <int DT>
__global__ __launch_bounds__(256) void pcx_project_bias_join(BackwardArgs a) {
  typedef typename Num<DT>::T T;
  __shared__ float part[4][64];
  const int h = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  float sum = 0.0f;
  if (h < a.s.hidden)
    for (int k = w; k < a.bias_blocks; k += 4) sum += a.bias_part[(int64_t)k * a.s.hidden + h];
  part[w][threadIdx.x & 63] = sum;
  __syncthreads();
  if (w == 0 && h < a.s.hidden)
    reinterpret_cast<T*>(a.grad_bias)[h] = Num<DT>::put((part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]));
}

// ---------------------------------------------------------------- plans

struct ForwardPlan { int mt, nt, wn, mblocks, nblocks, splits; uint64_t bytes; };
constexpr int SLOTS = 512;  // workgroups of 256 threads the chip holds at two per CU

ForwardPlan plan_forward(const Shape& s) {
  ForwardPlan p;
  if (s.n <= 512) { p.mt = 1; p.nt = 1; p.wn = 4; }
  else if (s.tiles >= 3) { p.mt = 4; p.nt = 2; p.wn = 2; }
  else if (s.tiles == 2) { p.mt = 4; p.nt = 2; p.wn = 1; }
  else { p.mt = 4; p.nt = 1; p.wn = 1; }
  const int rows = (4 / p.wn) * p.mt * 32, cols = p.nt * p.wn;
  p.mblocks = (int)((s.n + rows - 1) / rows);
  p.nblocks = (s.tiles + cols - 1) / cols;
  const int64_t groups = (int64_t)p.mblocks * p.nblocks;
  int64_t splits = groups >= SLOTS / 2 ? 1 : SLOTS / groups;
  if (splits > s.quads) splits = s.quads;
  p.splits = (int)splits;
  p.bytes = splits > 1 ? (uint64_t)splits * s.n * s.hidden * 4 : 0;
  return p;
}

struct BackwardPlan { int nh, htiles, hblocks, cell_blocks, layer_blocks, splits, bias_blocks, blocks; uint64_t frag_bytes, bias_bytes, part_bytes; };

BackwardPlan plan_backward(const Shape& s) {
  BackwardPlan p;
  p.nh = s.tiles >= 3 ? 4 : s.tiles;
  p.hblocks = (s.tiles + p.nh - 1) / p.nh;
  p.htiles = p.hblocks * p.nh;
  p.cell_blocks = (s.cells + 31) / 32;
  p.layer_blocks = (s.layers + 7) / 8;
  p.blocks = (int)((s.n + BLK - 1) / BLK);
  const int64_t tiles = (int64_t)p.hblocks * p.cell_blocks * p.layer_blocks;
  int64_t splits = SLOTS / tiles;
  if (splits > p.blocks) splits = p.blocks;
  if (splits < 1) splits = 1;
  p.splits = (int)splits;
  p.bias_blocks = p.blocks < 256 ? p.blocks : 256;
  p.frag_bytes = (uint64_t)p.blocks * 4 * p.htiles * s.parts * 1024;
  p.bias_bytes = ((uint64_t)p.bias_blocks * s.hidden * 4 + 255) & ~255ull;
  p.part_bytes = (uint64_t)p.splits * s.hidden * s.layers * s.cells * 4;
  return p;
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

template <int DT, bool STACKED, int MT, int NT, int WN>
int forward_go(const ForwardArgs& a, unsigned grid, hipStream_t st) {
  constexpr int ROWS_OUT = 4 * 32 * (NT * 32 + 4) * 4, STAGES = 2 * STEPS * NT * WN * FRAG + 1024;
  constexpr int LDS = ROWS_OUT > STAGES ? ROWS_OUT : STAGES;
  auto* const kernel = &pcx_project_forward_kernel<DT, STACKED, MT, NT, WN>;
  if (LDS > 65536) PCX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), LDS, st, a);
  return 0;
}
template <int DT, bool STACKED>
int forward_shape(const ForwardArgs& a, const ForwardPlan& p, unsigned grid, hipStream_t st) {
  if (p.mt == 1) return forward_go<DT, STACKED, 1, 1, 4>(a, grid, st);
  if (p.wn == 2) return forward_go<DT, STACKED, 4, 2, 2>(a, grid, st);
  if (p.nt == 2) return forward_go<DT, STACKED, 4, 2, 1>(a, grid, st);
  return forward_go<DT, STACKED, 4, 1, 1>(a, grid, st);
}
template <int DT>
int forward_type(const ForwardArgs& a, const ForwardPlan& p, unsigned grid, hipStream_t st) {
  if (int rc = a.s.stacked ? forward_shape<DT, true>(a, p, grid, st) : forward_shape<DT, false>(a, p, grid, st)) return rc;
  if (p.splits > 1) {
    const int64_t wgs = (a.s.n * ((a.s.hidden + 3) / 4) + 255) / 256;
    hipLaunchKernelGGL((pcx_project_join<DT>), dim3((unsigned)(wgs < 2048 ? wgs : 2048)), dim3(256), 0, st, a);
  }
  return 0;
}

template <int DT, bool STACKED, int NH>
int grad_go(const BackwardArgs& a, unsigned grid, hipStream_t st) {
  constexpr int PARTS = DT == PCX_F32 ? 3 : 1;
  constexpr int LDS = 2 * 4 * NH * PARTS * 1024 + 2 * 32 * (BLK + 8) * 2 + 512;
  auto* const kernel = &pcx_project_weight_grad<DT, STACKED, NH>;
  if (LDS > 65536) PCX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), LDS, st, a);
  return 0;
}
template <int DT, bool STACKED>
int grad_shape(const BackwardArgs& a, const BackwardPlan& p, unsigned grid, hipStream_t st) {
  if (p.nh == 4) return grad_go<DT, STACKED, 4>(a, grid, st);
  if (p.nh == 2) return grad_go<DT, STACKED, 2>(a, grid, st);
  return grad_go<DT, STACKED, 1>(a, grid, st);
}
template <int DT>
int backward_type(BackwardArgs& a, const BackwardPlan& p, hipStream_t st) {
  const unsigned hcols = (unsigned)((p.htiles + 1) / 2);
  hipLaunchKernelGGL((pcx_project_turn<DT>), dim3((unsigned)p.bias_blocks, hcols), dim3(256), 0, st, a);
  if (a.grad_weight) {
    const int64_t groups = (int64_t)p.cell_blocks * p.layer_blocks * p.hblocks * p.splits;
    a.chunk = (int32_t)((groups + 7) / 8);
    const unsigned grid = (unsigned)a.chunk * 8u;
    if (int rc = a.s.stacked ? grad_shape<DT, true>(a, p, grid, st) : grad_shape<DT, false>(a, p, grid, st)) return rc;
    const int64_t wgs = ((int64_t)a.s.hidden * a.s.layers * a.s.cells + 255) / 256;
    hipLaunchKernelGGL((pcx_project_weight_join<DT>), dim3((unsigned)(wgs < 4096 ? wgs : 4096)), dim3(256), 0, st, a);
  }
  if (a.grad_bias) hipLaunchKernelGGL((pcx_project_bias_join<DT>), dim3((unsigned)((a.s.hidden + 63) / 64)), dim3(256), 0, st, a);
  return 0;
}

int check_boards(const Shape& s, const uint8_t* boards, const char* who) {
  if (s.n && !boards) return set_error(PCX_E_INVALID, "%s: no boards", who);
  return 0;
}

}  // namespace

extern "C" {

int pcx_project_sizes(const pcx_project_desc* d, uint64_t* packed_bytes, uint64_t* forward_bytes, uint64_t* backward_bytes) {
  Shape s;
  if (int rc = make_shape(d, &s, "pcx_project_sizes")) return rc;
  if (packed_bytes) *packed_bytes = (uint64_t)s.quads * 4 * s.groups * s.parts * s.tiles * FRAG;
  if (forward_bytes) *forward_bytes = s.n ? plan_forward(s).bytes : 0;
  if (backward_bytes) {
    *backward_bytes = 0;
    if (s.n) {
      const BackwardPlan p = plan_backward(s);
      *backward_bytes = p.frag_bytes + p.bias_bytes + p.part_bytes;
    }
  }
  return 0;
}

int pcx_project_pack(const pcx_project_desc* d, const void* weight, void* packed, void* stream) {
  Shape s;
  if (int rc = make_shape(d, &s, "pcx_project_pack")) return rc;
  if (!weight || !packed || misaligned(packed, 16) || misaligned(weight, elem_size(s.dtype)))
    return set_error(PCX_E_INVALID, "pcx_project_pack: null or misaligned pointer");
  const int64_t wgs = ((int64_t)s.quads * 4 * s.groups * s.parts * s.tiles * 128 + 255) / 256;
  const dim3 grid((unsigned)(wgs < 8192 ? wgs : 8192)), block(256);
  hipStream_t st = (hipStream_t)stream;
  u32x4* const out = reinterpret_cast<u32x4*>(packed);
  if (s.dtype == PCX_F32) hipLaunchKernelGGL((pcx_project_layout<PCX_F32>), grid, block, 0, st, s, reinterpret_cast<const float*>(weight), out);
  else if (s.dtype == PCX_F16) hipLaunchKernelGGL((pcx_project_layout<PCX_F16>), grid, block, 0, st, s, reinterpret_cast<const _Float16*>(weight), out);
  else hipLaunchKernelGGL((pcx_project_layout<PCX_BF16>), grid, block, 0, st, s, reinterpret_cast<const __bf16*>(weight), out);
  PCX_HIP(hipGetLastError());
  return 0;
}

int pcx_project_forward(const pcx_project_desc* d, const uint8_t* boards, const void* packed, const void* bias, const void* residual,
                        void* out, void* slope, void* workspace, uint64_t workspace_bytes, void* stream) {
  Shape s;
  if (int rc = make_shape(d, &s, "pcx_project_forward")) return rc;
  if (int rc = check_boards(s, boards, "pcx_project_forward")) return rc;
  if (!s.n) return 0;
  const int es = elem_size(s.dtype);
  if (!packed || !out || misaligned(packed, 16) || misaligned(out, es) || misaligned(bias, es) || misaligned(residual, es) || misaligned(slope, es))
    return set_error(PCX_E_INVALID, "pcx_project_forward: null or misaligned pointer");
  const ForwardPlan p = plan_forward(s);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes || misaligned(workspace, 16)))
    return set_error(PCX_E_INVALID, "pcx_project_forward: the workspace needs %llu bytes, 16-byte aligned", (unsigned long long)p.bytes);
  ForwardArgs a{s, boards, reinterpret_cast<const uint8_t*>(packed), bias, residual, out, slope, reinterpret_cast<float*>(workspace),
                p.splits, p.mblocks, p.nblocks, 0, 0};
  a.wide = s.hidden % 4 == 0 && !misaligned(out, 4 * es) && !misaligned(residual, 4 * es) && !misaligned(slope, 4 * es);
  const int64_t groups = (int64_t)p.mblocks * p.nblocks * p.splits;
  if (groups >= (int64_t)1 << 23) return set_error(PCX_E_INVALID, "pcx_project_forward: too many boards for one call");
  a.chunk = (int32_t)((groups + 7) / 8);
  const unsigned grid = (unsigned)a.chunk * 8u;
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (s.dtype == PCX_F32) rc = forward_type<PCX_F32>(a, p, grid, st);
  else if (s.dtype == PCX_F16) rc = forward_type<PCX_F16>(a, p, grid, st);
  else rc = forward_type<PCX_BF16>(a, p, grid, st);
  if (rc) return rc;
  PCX_HIP(hipGetLastError());
  return 0;
}

int pcx_project_backward(const pcx_project_desc* d, const uint8_t* boards, const void* grad_out, const void* slope, void* grad_weight,
                         void* grad_bias, void* workspace, uint64_t workspace_bytes, void* stream) {
  Shape s;
  if (int rc = make_shape(d, &s, "pcx_project_backward")) return rc;
  if (int rc = check_boards(s, boards, "pcx_project_backward")) return rc;
  if (!s.n) return set_error(PCX_E_INVALID, "pcx_project_backward: no boards (their gradients are zero)");
  if (!grad_weight && !grad_bias) return 0;
  const int es = elem_size(s.dtype);
  if (!grad_out || misaligned(grad_out, es) || misaligned(slope, es) || misaligned(grad_weight, es) || misaligned(grad_bias, es))
    return set_error(PCX_E_INVALID, "pcx_project_backward: null or misaligned pointer");
  if (s.activation != PCX_ACT_NONE && !slope) return set_error(PCX_E_INVALID, "pcx_project_backward: the activation's slopes are missing");
  const BackwardPlan p = plan_backward(s);
  if ((int64_t)p.hblocks * p.cell_blocks * p.layer_blocks * p.splits >= (int64_t)1 << 23) return set_error(PCX_E_INVALID, "pcx_project_backward: the weight is too large");
  if (!workspace || workspace_bytes < p.frag_bytes + p.bias_bytes + p.part_bytes || misaligned(workspace, 16))
    return set_error(PCX_E_INVALID, "pcx_project_backward: the workspace needs %llu bytes, 16-byte aligned",
                     (unsigned long long)(p.frag_bytes + p.bias_bytes + p.part_bytes));
  uint8_t* const ws = reinterpret_cast<uint8_t*>(workspace);
  BackwardArgs a{s, boards, grad_out, s.activation == PCX_ACT_NONE ? nullptr : slope, grad_weight ? ws : nullptr,
                 reinterpret_cast<float*>(ws + p.frag_bytes), reinterpret_cast<float*>(ws + p.frag_bytes + p.bias_bytes), grad_weight, grad_bias,
                 p.blocks, p.htiles, p.bias_blocks, p.splits, p.cell_blocks, p.layer_blocks, p.hblocks, 0};
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (s.dtype == PCX_F32) rc = backward_type<PCX_F32>(a, p, st);
  else if (s.dtype == PCX_F16) rc = backward_type<PCX_F16>(a, p, st);
  else rc = backward_type<PCX_BF16>(a, p, st);
  if (rc) return rc;
  PCX_HIP(hipGetLastError());
  return 0;
}

}  // extern "C"
