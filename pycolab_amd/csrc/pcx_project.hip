// pcx_project.hip -- the first layer of a policy, read from the boards: act(features . weight^T + bias) + residual, where
// `features` is the 0/1 stack of layers that rendering.ObservationToFeatureArray would write (rendering.py:545-661).  The
// stack is never stored: the kernel expands it from the boards' characters (or from stacked uint8 layers, where layers
// overlap) in the registers that feed the matrix units.  pcx_project_grad.hip has the gradients.
//
// Mathematics.  With x[b][l][c] = 1 where board b shows character l at cell c:
//   z[b][h] = sum_{l,c} x[b][l][c] w[h][l][c] + bias[h],   y = act(z) + residual,
//   dz = dy act'(z),   dw[h][l][c] = sum_b dz[b][h] x[b][l][c],   dbias[h] = sum_b dz[b][h].
// A cell shows one character, so of the four features (four layers of one cell) at most one is set: the left operand is
// 2:4 sparse along the summed axis by construction, and v_smfmac_f32_32x32x32 multiplies it at 3,750 TFLOP/s where the
// dense v_mfma_f32_32x32x16 gives 2,270 (both measured here, register operands only).  Overlapping layers take the dense one,
// 8 cells x 2 layers at a time.
// A set feature is the number 2 -- the bit pattern 0x4000 in bfloat16 AND in float16 -- so that expanding a feature pair
// is one shift and one mask; the other operand is halved instead (float16, whose small numbers have no bit to spare and
// whose sums cannot leave float32's range: the sum is), which is exact down to the last subnormal bit.  float32 weights
// are split into three bfloat16 parts (8 + 8 + 8 bits: none is lost), and every product is exact, so they cost three
// passes and no accuracy.  All sums are float32.
#include "pcx_project.h"

#include <type_traits>

namespace pcx {
namespace project {

int make_shape(const pcx_project_desc* d, Shape* s, const char* who) {
  if (!d) return set_error(PCX_E_INVALID, "%s: null description", who);
  if (d->dtype != PCX_F32 && d->dtype != PCX_F16 && d->dtype != PCX_BF16)
    return set_error(PCX_E_INVALID, "%s: the weights are float32, float16 or bfloat16", who);
  if (d->activation < PCX_ACT_NONE || d->activation > PCX_ACT_GELU) return set_error(PCX_E_INVALID, "%s: unknown activation", who);
  if (d->cells < 1 || d->cells > 1 << 20 || d->n_layers < 1 || d->n_layers > PCX_POST_MAX_DEPTH || d->hidden < 1 || d->hidden > 1 << 16)
    return set_error(PCX_E_INVALID, "%s: cells, layers or hidden units out of range", who);
  if (d->n < 0 || d->n > (int64_t)1 << 31) return set_error(PCX_E_INVALID, "%s: %lld boards", who, (long long)d->n);
  if (d->row_stride < 0) return set_error(PCX_E_INVALID, "%s: negative stride", who);
  if (d->stacked)
    for (int i = 0; i < d->n_layers; ++i)
      if (d->layer_offset[i] >= (int64_t)1 << 31) return set_error(PCX_E_INVALID, "%s: a layer 2 GB or more from its board", who);
  if (!d->stacked)
    for (int i = 0; i < d->n_layers; ++i)
      for (int j = 0; j < i; ++j)
        if (d->chars[i] == d->chars[j]) return set_error(PCX_E_INVALID, "%s: layer '%c' twice", who, d->chars[i]);
  s->n = d->n; s->row_stride = d->row_stride;
  memcpy(s->layer_offset, d->layer_offset, sizeof s->layer_offset);
  s->cells = d->cells; s->layers = d->n_layers; s->hidden = d->hidden;
  // characters: more than 16 layers are two blocks of four groups, one after the other
  s->groups = d->stacked ? (d->n_layers + 1) / 2 : d->n_layers > 16 ? 8 : (d->n_layers + 3) / 4;
  s->parts = d->dtype == PCX_F32 ? 3 : 1;
  s->quads = (d->cells + QUAD - 1) / QUAD;
  s->tiles = (d->hidden + 31) / 32;
  s->stacked = d->stacked != 0; s->activation = d->activation; s->dtype = d->dtype;
  memcpy(s->chars, d->chars, sizeof s->chars);
  if ((int64_t)s->quads * 4 * s->groups * s->parts * s->tiles > (int64_t)1 << 27)
    return set_error(PCX_E_INVALID, "%s: the weight is too large", who);
  return 0;
}

}  // namespace project
}  // namespace pcx

using namespace pcx::project;
using pcx::set_error;

namespace {

// bytes of one right operand: 32 features x 32 hidden units x 2, of stacked layers 16 x 32 x 2
__host__ __device__ constexpr int frag_bytes(bool stacked) { return stacked ? 1024 : 2048; }

// What a sum of the matrix unit is multiplied by: a feature is 2, and all weights but float16 ones are laid out halved.
template <int DT> constexpr float SCALE = DT == PCX_F16 ? 0.5f : 1.0f;

template <int ACT>
__device__ __forceinline__ void activate(float z, float* y, float* slope) {
  if constexpr (ACT == PCX_ACT_RELU) {
    *y = z < 0.0f ? 0.0f : z; *slope = z <= 0.0f ? 0.0f : 1.0f;  // (a NaN stays one)
  } else if constexpr (ACT == PCX_ACT_SILU) {
    const float s = 1.0f / (1.0f + expf(-z));
    *y = z * s; *slope = s * (1.0f + z * (1.0f - s));
  } else if constexpr (ACT == PCX_ACT_TANH) {
    const float t = tanhf(z);
    *y = t; *slope = 1.0f - t * t;
  } else if constexpr (ACT == PCX_ACT_GELU) {
    const float cdf = 0.5f * (1.0f + erff(z * 0.70710678118654752f));
    *y = z * cdf; *slope = cdf + z * expf(-0.5f * z * z) * 0.3989422804014327f;
  } else {
    *y = z; *slope = 1.0f;
  }
}

// ---------------------------------------------------------------- laying the weight out

// Step order: characters (block of four groups, quad of 32 cells, octet j, part, group g of the block), stacked layers
// (quad, group, part, octet).  Within a step the instruction sums 32 features; lane (column c, half hb) holds 16 of them,
// element e standing for cell start + 16 (e / 8) + 4 j + 2 hb + (e % 8) / 4 of the quad and position e % 4 of the group
// (the lane layout of the instruction, measured: the sparse side's half A covers features 16 A .. 16 A + 15, the dense
// side's element e feature 16 (e / 8) + 8 hb + e % 8).  The 16 bytes of elements 0..7 and of 8..15 of a lane are 1 KB apart,
// so that a wave's LDS reads are contiguous.  The dense instruction of stacked layers sums 16 features: element e of a
// lane's 8 stands for cell start + 16 hb + 4 j + e / 2 and layer e % 2 of the group.  A workgroup turns one quad of one group and tile round through LDS, so that
// the weight is read in runs of 32 cells (a direct gather took 52 us for 5.6 million float32 weights; this one 23).
template <int DT>
__global__ __launch_bounds__(256) void pcx_project_layout(Shape s, const typename Num<DT>::T* __restrict__ w, u32x4* __restrict__ packed) {
  __shared__ float in[32][4 * 33 + 1];  // (an odd pitch: 32 hidden units in 32 banks)
  const int q = blockIdx.x, g = blockIdx.y, tile = blockIdx.z;
  const int start = quad_start(q, s.cells), mine = q * QUAD - start;  // (cells before `mine` belong to the quad before)
  {  // (what does not exist is read as its neighbour and dropped: 16 loads in flight, not one after the other)
    const int c = threadIdx.x & 31, pos = (threadIdx.x >> 5) & 3, cell = start + c;
    const int layer = s.stacked ? (pos < 2 ? g * 2 + pos : s.layers) : g * 4 + pos;
    const bool real = c >= mine && cell < s.cells && layer < s.layers;
    const typename Num<DT>::T* const from = w + (layer < s.layers ? layer : 0) * (int64_t)s.cells + (cell < s.cells ? cell : 0);
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int h = tile * 32 + i * 2 + (threadIdx.x >> 7);
      v[i] = Num<DT>::get(from[(int64_t)(h < s.hidden ? h : s.hidden - 1) * s.layers * s.cells]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) in[i * 2 + (threadIdx.x >> 7)][pos * 33 + c] = real && tile * 32 + i * 2 + (int)(threadIdx.x >> 7) < s.hidden ? v[i] : 0.0f;
  }
  __syncthreads();
  const int per = s.stacked || s.groups < 4 ? s.groups : 4;  // groups per block
  const int e8s = s.stacked ? 0 : 1;  // (the runs of 8 elements a lane has: 1 << e8s)
  for (int i = threadIdx.x; i < (4 * s.parts * 64) << e8s; i += 256) {
    const int lane = i & 63, e8 = (i >> 6) & e8s, j = (i >> (6 + e8s)) & 3, part = i >> (8 + e8s), hb = lane >> 5;
    u32x4 out = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = s.stacked ? in[lane & 31][(e & 1) * 33 + hb * 16 + j * 4 + (e >> 1)] : in[lane & 31][(e & 3) * 33 + e8 * 16 + j * 4 + hb * 2 + (e >> 2)];
      uint32_t bits;
      if constexpr (DT == PCX_F16) bits = __builtin_bit_cast(uint16_t, (_Float16)v);
      else bits = part_of(0.5f * v, part, s.parts);
      out[e >> 1] |= bits << (16 * (e & 1));
    }
    int64_t step;
    if (s.stacked) step = (((int64_t)g * s.quads + q) * s.parts + part) * 4 + j;
    else step = ((((int64_t)(g / per) * s.quads + q) * 4 + j) * s.parts + part) * per + g % per;
    packed[((step * s.tiles + tile) << (6 + e8s)) + e8 * 64 + lane] = out;
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

// How many octets of a quad a stage holds: as many as leave two workgroups of four waves a CU, or one of eight.
constexpr int octets_per_stage(int parts, int groups, int waves) {
  return parts > 1 ? 1 : groups == 1 ? 4 : groups == 2 ? (waves == 8 ? 4 : 2) : groups == 4 && waves == 8 ? 2 : 1;
}
constexpr int steps_per_stage(int parts, int groups, int waves) {
  return groups == 0 ? (parts > 1 ? 4 : 8) : octets_per_stage(parts, groups, waves) * (parts == 3 && groups == 1 ? 3 : 1) * groups;
}
// bit 6 of every byte that is not zero
__device__ __forceinline__ uint32_t set_bytes(uint32_t b) {
  return (((((b & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | b) >> 1) & 0x40404040u);
}

template <bool F16>
__device__ __forceinline__ f32x16 sparse_step(u32x4 a, u32x8 b, f32x16 c, int index) {
  if constexpr (F16)
    return __builtin_amdgcn_smfmac_f32_32x32x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x16, b), c, index, 0, 0);
  else
    return __builtin_amdgcn_smfmac_f32_32x32x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x16, b), c, index, 0, 0);
}

// Four neighbouring elements of a row.
template <typename T> struct __align__(4 * sizeof(T)) Four { T v[4]; };
template <typename T>
__device__ __forceinline__ Four<T> load_four(const T* from, int count, bool wide) {
  Four<T> f = {};
  if (wide) return *reinterpret_cast<const Four<T>*>(from);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) f.v[i] = from[i];
  return f;
}
template <typename T>
__device__ __forceinline__ void store_four(T* to, Four<T> f, int count, bool wide) {
  if (wide) { *reinterpret_cast<Four<T>*>(to) = f; return; }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) to[i] = f.v[i];
}
// Bias, activation and residual on up to four neighbouring sums of one board, `at` elements into out (count < 4 at the last
// columns; a.wide: the rows keep four elements aligned).
template <int DT, int ACT>
__device__ __forceinline__ void finish(const ForwardArgs& a, int64_t at, const float* sum, Four<typename Num<DT>::T> bias,
                                       Four<typename Num<DT>::T> res, int count) {
  typedef typename Num<DT>::T T;
  Four<T> out;
  float slope[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y;
    activate<ACT>(sum[i] + Num<DT>::get(bias.v[i]), &y, &slope[i]);
    out.v[i] = Num<DT>::put(a.residual ? y + Num<DT>::get(res.v[i]) : y);
  }
  store_four(reinterpret_cast<T*>(a.out) + at, out, count, a.wide);
  if (!a.slope) return;
  // relu's slopes are 0 and 1 in any type; the others keep float32, so that the gradients lose nothing but their own rounding
  if constexpr (ACT == PCX_ACT_RELU) {
    Four<T> k;
#pragma unroll
    for (int i = 0; i < 4; ++i) k.v[i] = Num<DT>::put(slope[i]);
    store_four(reinterpret_cast<T*>(a.slope) + at, k, count, a.wide);
  } else {
    store_four(reinterpret_cast<float*>(a.slope) + at, Four<float>{{slope[0], slope[1], slope[2], slope[3]}}, count, a.wide);
  }
}
// f with the activation as a constant
template <typename F>
__device__ __forceinline__ void by_activation(int act, F f) {
  switch (act) {
    case PCX_ACT_RELU: f(std::integral_constant<int, PCX_ACT_RELU>()); break;
    case PCX_ACT_SILU: f(std::integral_constant<int, PCX_ACT_SILU>()); break;
    case PCX_ACT_TANH: f(std::integral_constant<int, PCX_ACT_TANH>()); break;
    case PCX_ACT_GELU: f(std::integral_constant<int, PCX_ACT_GELU>()); break;
    default: f(std::integral_constant<int, PCX_ACT_NONE>()); break;
  }
}

// A wave holds MT x NT tiles of 32 x 32 sums; WM waves lie along the boards and WN along the hidden units.  G: groups of
// a block of characters (1..4), 0: stacked layers.  The weights of a stage are copied into LDS one stage ahead, the boards'
// bytes into registers one quad ahead; a workgroup's waves share the weights, each wave expands its own boards.
template <int DT, int G, int MT, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void pcx_project_forward_kernel(ForwardArgs a) {
  constexpr bool STACKED = G == 0;
  constexpr int PARTS = DT == PCX_F32 ? 3 : 1;
  constexpr int FR = NT * WN;                                                              // right operands per step
  constexpr int WAVES = WM * WN;
  constexpr int OCT = STACKED ? 4 : octets_per_stage(PARTS, G, WAVES);                     // octets per stage
  constexpr int PS = !STACKED && PARTS == 3 && G == 1 ? 3 : 1;                             // parts per stage
  constexpr int STEPS = steps_per_stage(PARTS, G, WAVES);                                  // matrix steps per stage
  constexpr int FRAG = frag_bytes(STACKED), PF = FRAG / 1024;
  constexpr int STAGE = STEPS * FR * FRAG;
  constexpr int PIECES = STAGE / 1024;        // 1 KB copies per stage
  constexpr int MROWS = WM * MT * 32;
  const Shape& s = a.s;
  __shared__ uint32_t lut[STACKED ? 1 : 256];
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // consecutive tiles of a board block go to one XCD (workgroup i runs on XCD i % 8), whose L2 then serves the boards once
  const uint32_t id = (blockIdx.x & 7u) * (uint32_t)a.chunk + (blockIdx.x >> 3);
  if (id >= (uint32_t)a.mblocks * a.nblocks * a.splits) return;
  const int nb = (int)(id % (uint32_t)a.nblocks);
  const uint32_t rest = id / (uint32_t)a.nblocks;
  const int split = (int)(rest % (uint32_t)a.splits), mb = (int)(rest / (uint32_t)a.splits);
  const int blocks = STACKED ? s.groups : (s.groups + 3) / 4;
  // A block's table by character: bits 0..3 and again 4..7 the positions of the two slots of a group -- they ascend: (p, 3)
  // with the feature in the low slot for p < 3, (0, 3) with it in the high one for 3 -- and bit 14 - g (30 - g) a feature of
  // group g in its low (high) slot.  (Two words a character save 6 of 21 instructions a cell quad and lose 6 % to the
  // wider LDS reads.)
  auto write_table = [&](int b) {  // (the caller has the workgroup's barriers around it)
    if (tid < 256) lut[tid] = 0x44u;  // (0, 1), none
    __syncthreads();
    const int l = b * 16 + tid, p = l & 3, g = (l >> 2) & 3;
    if (tid < 16 && l < s.layers) lut[argument<ForwardArgs>()->s.chars[l]] = p < 3 ? (0x4000u >> g) | (uint32_t)((p | 12) * 0x11) : (0x40000000u >> g) | 0xCCu;
  };
  // the run of (block, quad) units of this split (STACKED: a block is a group)
  const int units = blocks * s.quads;
  const int u0 = (int)((int64_t)units * split / a.splits), u1 = (int)((int64_t)units * (split + 1) / a.splits);
  const int per_unit = 4 * PARTS * (STACKED ? 1 : G), stages = ((u1 - u0) * per_unit + STEPS - 1) / STEPS;
  const int tile0 = nb * FR, live = s.tiles - tile0 < FR ? s.tiles - tile0 : FR;
  const uint8_t* const src = a.packed + ((int64_t)u0 * per_unit * s.tiles + tile0) * FRAG + lane * 16;
  const int wm = wave / WN, wn = wave % WN, half = lane >> 5;
  const int64_t row0 = (int64_t)mb * MROWS + wm * MT * 32;
  const uint8_t* row[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t r = row0 + m * 32 + (lane & 31);
    row[m] = a.boards + (r < s.n ? r : s.n - 1) * s.row_stride;
  }
  auto stage_in = [&](int st) {
    uint8_t* const dst = lds + (st & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < (PIECES + WAVES - 1) / WAVES; ++i) {
      const int k = wave + WAVES * i, step = k / (PF * FR), off = k % (PF * FR);  // PF FR pieces of 1 KB to a step
      if (k < PIECES && off < PF * live) copy_in(src + ((int64_t)(st * STEPS + step) * s.tiles) * FRAG + off * 1024, dst + k * 1024);
    }
  };
  f32x16 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[m][t][i] = 0.0f;
  u32x4 left[MT];
  int index[MT];
  // One matrix step: step k of the stage at `base`.  The right operands are read one ahead, the first of a stage in
  // front of it.
  typename std::conditional<STACKED, u32x4, u32x8>::type ahead;
  auto read_right = [&](const uint8_t* base, int i) {
    const uint8_t* const at = base + ((i / NT) * FR + i % NT) * FRAG;
    const u32x4 b0 = *reinterpret_cast<const u32x4*>(at);
    if constexpr (STACKED) {
      ahead = b0;
    } else {
      const u32x4 b1 = *reinterpret_cast<const u32x4*>(at + 1024);
      ahead = u32x8{b0[0], b0[1], b0[2], b0[3], b1[0], b1[1], b1[2], b1[3]};
    }
  };
  auto multiply = [&](const uint8_t* base, int k) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const auto right = ahead;
      if (k * NT + t + 1 < STEPS * NT) read_right(base, k * NT + t + 1);
#pragma unroll
      for (int m = 0; m < MT; ++m)
        if constexpr (STACKED) acc[m][t] = dense_step<DT == PCX_F16>(left[m], right, acc[m][t]);
        else acc[m][t] = sparse_step<DT == PCX_F16>(left[m], right, acc[m][t], index[m]);
    }
  };
  auto stage_base = [&](int st) { return lds + (st & 1) * STAGE + wn * NT * FRAG + lane * 16; };
  const bool small = s.cells < QUAD;
  auto load16 = [&](const uint8_t* at, int c) {
    u32x4 v;
    if (small) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = edge_dword(at, c + 4 * i, s.cells);
    } else {
      __builtin_memcpy(&v, at + c, 16);
    }
    return v;
  };
  // A stage's weights must have arrived, the boards' bytes requested after them need not: `loose` says that they were.
  constexpr int LOADS = STACKED ? 4 * MT : MT;
  bool loose = false;
  auto arrive = [&]() {
    if (loose) stage_barrier<LOADS>();
    else stage_barrier<0>();
    loose = false;
  };
  int st = 0;
  if constexpr (STACKED) {
    // The two layers of a (group, quad) unit, DEPTH - 1 units ahead: a unit is only 4 matrix steps, a trip to memory many.
    // All quads of two layers follow each other, so that a board's bytes are read in the order in which they lie.
    constexpr int DEPTH = 4;
    // Layers lie at any byte: a lane reads the five aligned words around its 16 bytes (an aligned word never leaves the page
    // of the byte that is wanted) and shifts them when they are used; loads at odd bytes took 42 us where these take 38.
    struct Bytes { u32x4 v; uint32_t more, by; };
    auto load_bytes = [&](const uint8_t* at, int c) {
      Bytes x;
      if (small) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[i] = edge_dword(at, c + 4 * i, s.cells);
        x.more = x.by = 0;
      } else {
        at += c;
        x.by = (uint32_t)reinterpret_cast<uintptr_t>(at) & 3u;
        const uint32_t* const words = reinterpret_cast<const uint32_t*>(at - x.by);
        __builtin_memcpy(&x.v, words, 16);
        x.more = words[x.by ? 4 : 3];
      }
      return x;
    };
    Bytes ring[DEPTH][MT][2];
    uint32_t on[DEPTH][2];  // 0 where the layer does not exist: its bytes are then the board's first
    int fq = u0 % s.quads, fg = u0 / s.quads, fetched = u0;
    auto fetch = [&](Bytes (&to)[MT][2], uint32_t (&keep)[2]) {
      const bool last = ++fetched >= u1;  // (then the last unit again: the same number of requests for every one)
      const int c = quad_start(fq, s.cells) + half * 16;
#pragma unroll
      for (int l = 0; l < 2; ++l) {
        const int layer = 2 * fg + l;
        const int64_t off = layer < s.layers ? argument<ForwardArgs>()->s.layer_offset[layer] : -1;
        keep[l] = off >= 0 ? 0xFFFFFFFFu : 0u;
#pragma unroll
        for (int m = 0; m < MT; ++m) to[m][l] = load_bytes(row[m] + (off >= 0 ? off : 0), c);
      }
      if (!last && ++fq == s.quads) { fq = 0; ++fg; }
    };
#pragma unroll
    for (int k = 0; k < DEPTH - 1; ++k) fetch(ring[k], on[k]);
    stage_in(0);
    stage_barrier<0>();
    const uint8_t* base = nullptr;
    const int total = u1 - u0;
#pragma unroll 1
    for (int i = 0; i < total; i += DEPTH)
#pragma unroll
      for (int k = 0; k < DEPTH; ++k) {
        if (i + k >= total) break;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          constexpr int PER = STEPS / 4;  // (PARTS = 1: units per stage)
          if (PARTS > 1 || k % PER == 0) {
            // a stage's weights must be here, the boards' bytes asked for behind it may be on their way
            if (small || (PARTS > 1 && part != 1)) stage_barrier<0>();
            else stage_barrier<PER * LOADS>();
            if (st + 1 < stages) stage_in(st + 1);
            asm volatile("" ::: "memory");
            base = stage_base(st);
            ++st;
          }
          if (part == 0) fetch(ring[(k + DEPTH - 1) % DEPTH], on[(k + DEPTH - 1) % DEPTH]);
          if (PARTS > 1 || k % PER == 0) read_right(base, 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              uint32_t b[2];
#pragma unroll
              for (int l = 0; l < 2; ++l) {
                const Bytes& x = ring[k][m][l];
                b[l] = set_bytes(__builtin_amdgcn_alignbyte(j < 3 ? x.v[j < 3 ? j + 1 : 3] : x.more, x.v[j], x.by)) & on[k][l];
              }
              const uint32_t lo = b[0], hi = b[1];
              left[m][0] = __builtin_amdgcn_perm(hi, lo, 0x040C000Cu);
              left[m][1] = __builtin_amdgcn_perm(hi, lo, 0x050C010Cu);
              left[m][2] = __builtin_amdgcn_perm(hi, lo, 0x060C020Cu);
              left[m][3] = __builtin_amdgcn_perm(hi, lo, 0x070C030Cu);
            }
            multiply(base, PARTS > 1 ? j : k % (STEPS / 4) * 4 + j);
          }
        }
      }
  } else {
    u32x4 cur[MT], nxt[MT];
    auto fetch = [&](int u) {
      const int q = u < s.quads ? u : u - s.quads, c = quad_start(q, s.cells) + half * 16;
#pragma unroll
      for (int m = 0; m < MT; ++m) nxt[m] = load16(row[m], c);
      loose = !small;
    };
    fetch(u0);
    stage_in(0);
    loose = false;
    write_table(u0 < s.quads ? 0 : 1);
    __syncthreads();
#pragma unroll 1
    for (int u = u0; u < u1; ++u) {
      if (u == s.quads && u > u0) {  // (the second block of a stack of more than 16 layers)
        __syncthreads();
        write_table(1);
        __syncthreads();
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) cur[m] = nxt[m];
      uint32_t word[MT][4];  // the cells' feature bits
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j % OCT == 0) {
          arrive();
          if (st + 1 < stages) stage_in(st + 1);
          asm volatile("" ::: "memory");
          if (j == 0 && u + 1 < u1) fetch(u + 1);
          read_right(stage_base(st), 0);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int c = 0; c < 4; ++c) word[m][c] = lut[(cur[m][j] >> (8 * c)) & 255u];
          const uint32_t lo = (word[m][0] & 0x0Fu) | (word[m][1] & 0xF0u), hi = (word[m][2] & 0x0Fu) | (word[m][3] & 0xF0u);
          index[m] = (int)(lo | hi << 8);
        }
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          if (part && part % PS == 0) {
            arrive();
            if (st + 1 < stages) stage_in(st + 1);
            read_right(stage_base(st), 0);
          }
          const uint8_t* const base = stage_base(st);
#pragma unroll
          for (int g = 0; g < G; ++g) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int c = 0; c < 4; ++c) left[m][c] = (word[m][c] << g) & 0x40004000u;
            multiply(base, ((j % OCT) * PS + part % PS) * G + g);
          }
          if ((part + 1) % PS == 0 && (PARTS > 1 || (j + 1) % OCT == 0)) ++st;
        }
      }
    }
  }
  // Out through LDS, 32 boards at a time and each wave by itself: a lane then has four neighbouring hidden units of one
  // board, and a wave writes whole rows of its tile.  The residual's rows are on their way one tile ahead and wait in LDS
  // too (loaded where they are used, every row cost its own trip to memory: 583 us against 315 for 262,144 boards of 300 cells x 8 layers).
  typedef typename Num<DT>::T T;
  constexpr int PITCH = NT * 32 + 4, LANES = NT * 8, ROUNDS = 32 * LANES / 64;  // lanes per row, rows per lane
  __syncthreads();
  float* const mine = reinterpret_cast<float*>(lds) + wave * 32 * PITCH;
  Four<T>* const kept = reinterpret_cast<Four<T>*>(lds + WAVES * 32 * PITCH * 4) + wave * ROUNDS * 64 + lane;
  const int col0 = (tile0 + wn * NT) * 32 + (lane % LANES) * 4;
  const int count = s.hidden - col0 < 4 ? s.hidden - col0 : 4;
  const bool whole = a.splits == 1;
  const T* const residual = whole ? reinterpret_cast<const T*>(a.residual) : nullptr;
  Four<T> bias = {}, res[ROUNDS] = {};
  if (whole && a.bias && count > 0) bias = load_four(reinterpret_cast<const T*>(a.bias) + col0, count, false);
  const T* from = residual + (row0 + lane / LANES) * s.hidden + col0;
  auto fetch_residual = [&](int m) {
    if (!residual || count <= 0) return;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const int64_t board = row0 + m * 32 + i * (64 / LANES) + lane / LANES;
      if (board < s.n) res[i] = load_four(from, count, a.wide);
      from += (64 / LANES) * s.hidden;
    }
  };
  fetch_residual(0);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) mine[(8 * (i >> 2) + 4 * half + (i & 3)) * PITCH + t * 32 + (lane & 31)] = SCALE<DT> * acc[m][t][i];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) kept[i * 64] = res[i];
    if (m + 1 < MT) fetch_residual(m + 1);
    __builtin_amdgcn_wave_barrier();
    const int64_t first = row0 + m * 32 + lane / LANES;
    const int rows = count <= 0 ? 0 : s.n - first < 32 ? (int)(s.n - first) : 32;  // (from this lane's first row on)
    if (whole) {
      by_activation(s.activation, [&](auto act) {
        int64_t at = first * s.hidden + col0;
#pragma unroll 1
        for (int i = 0; i < ROUNDS; ++i, at += (64 / LANES) * s.hidden) {
          const float4 v = *reinterpret_cast<const float4*>(mine + (i * (64 / LANES) + lane / LANES) * PITCH + (lane % LANES) * 4);
          const float sum[4] = {v.x, v.y, v.z, v.w};
          if (i * (64 / LANES) < rows) finish<DT, decltype(act)::value>(a, at, sum, bias, kept[i * 64], count);
        }
      });
    } else {
      float* to = a.partial + ((int64_t)split * s.n + first) * s.hidden + col0;
#pragma unroll 1
      for (int i = 0; i < ROUNDS; ++i, to += (64 / LANES) * s.hidden) {
        const float4 v = *reinterpret_cast<const float4*>(mine + (i * (64 / LANES) + lane / LANES) * PITCH + (lane % LANES) * 4);
        if (i * (64 / LANES) < rows) store_four(to, Four<float>{{v.x, v.y, v.z, v.w}}, count, a.wide);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The cells' partial sums joined in a fixed order, and the epilogue.
template <int DT>
__global__ __launch_bounds__(256) void pcx_project_join(ForwardArgs a) {
  typedef typename Num<DT>::T T;
  const int64_t plane = a.s.n * a.s.hidden;
  if (!a.wide) {  // rows that do not keep four sums aligned: one a lane (four guarded ones: 31 us for 101 boards x
                  // 19 units, this way 4)
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < plane; i += (int64_t)gridDim.x * 256) {
      Four<T> bias = {}, res = {};
      if (a.bias) bias.v[0] = reinterpret_cast<const T*>(a.bias)[i % a.s.hidden];
      if (a.residual) res.v[0] = reinterpret_cast<const T*>(a.residual)[i];
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const float* from = a.partial + i;
#pragma unroll 8
      for (int k = 0; k < a.splits; ++k, from += plane) sum[0] += *from;
      by_activation(a.s.activation, [&](auto act) { finish<DT, decltype(act)::value>(a, i, sum, bias, res, 1); });
    }
    return;
  }
  const int quads = a.s.hidden / 4;
  const int64_t total = a.s.n * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / quads;
    const int col = (int)(i - row * quads) * 4;
    const float* from = a.partial + row * a.s.hidden + col;
    Four<T> bias = {}, res = {};
    if (a.bias) bias = load_four(reinterpret_cast<const T*>(a.bias) + col, 4, false);
    if (a.residual) res = load_four(reinterpret_cast<const T*>(a.residual) + row * a.s.hidden + col, 4, true);
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int k = 0; k < a.splits; ++k, from += plane) {
      const Four<float> v = load_four(from, 4, true);
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[c] += v.v[c];
    }
    by_activation(a.s.activation, [&](auto act) { finish<DT, decltype(act)::value>(a, row * a.s.hidden + col, sum, bias, res, 4); });
  }
}

// ---------------------------------------------------------------- plan

struct ForwardPlan { int mt, nt, wm, wn, mblocks, nblocks, splits; uint64_t bytes; };

ForwardPlan plan_forward(const Shape& s) {
  ForwardPlan p;
  // 4 x 2 tiles a wave make the most of a weight in LDS and of an expanded board.  Eight waves share a weight where the
  // boards fill the chip with them (the weight then leaves L2 half as often); where they do not fill it with four, a wave
  // takes 2 x 2 tiles, and only then are the cells divided: joining costs 8 bytes a sum and part.
  // But every 128 boards fetch the weight anew, from beyond an XCD's 4 MB of L2 if it is large: from some 400 MB of that on
  // (boards times the weight's bytes) eight waves of 512 boards stay, with the cells divided more often.  Float32 weights of
  // 4,005 cells, 7 layers and 200 units: 2,048 boards 80 -> 69 us, 16,384 boards 749 -> 334; bfloat16 ones of 480 cells, 14
  // layers and 512 units: 8,192 boards 70 -> 63, 4,096 boards 40 where eight waves take 51.
  const int64_t packed = (int64_t)s.quads * 4 * s.groups * s.parts * s.tiles * frag_bytes(s.stacked);
  p.mt = 4;
  p.nt = 2;
  p.wn = s.tiles >= 3 ? 2 : 1;
  p.wm = 4 / p.wn;
  const int64_t nblocks = (s.tiles + 2 * p.wn - 1) / (2 * p.wn);
  // Stacked layers wait for the boards' bytes more than for the matrix units: small tiles of sums leave room for twice the
  // waves (32,768 boards, 11 layers of 110 cells, 128 units: 2 x 2 tiles and four waves 47 us, 1 x 2 45, with eight 42).
  if (s.stacked) { p.mt = 1; p.wm = 4; }
  else if (s.n <= 512) { p.mt = p.nt = p.wm = 1; p.wn = 4; }
  else if (p.wn == 2 && (s.n * nblocks >= 512 * 192 || s.n * packed >= (int64_t)50 << 30)) p.wm = 4;
  else if ((s.n + 128 * p.wm - 1) / (128 * p.wm) * nblocks < SLOTS / 2) p.mt = 2;
  const int rows = p.wm * p.mt * 32, cols = p.nt * p.wn;
  p.mblocks = (int)((s.n + rows - 1) / rows);
  p.nblocks = (s.tiles + cols - 1) / cols;
  const int64_t groups = (int64_t)p.mblocks * p.nblocks;
  const int64_t slots = p.wm * p.wn == 8 ? SLOTS / 2 : SLOTS;
  int64_t splits = groups > slots / 2 ? 1 : slots / groups;
  const int64_t units = (int64_t)s.quads * (s.stacked ? s.groups : 1);
  if (splits > units) splits = units;
  p.splits = (int)splits;
  p.bytes = splits > 1 ? (uint64_t)splits * s.n * s.hidden * 4 : 0;
  return p;
}

template <int DT, int G, int MT, int NT, int WM, int WN>
int forward_go(const ForwardArgs& a, unsigned grid, hipStream_t st) {
  constexpr int PARTS = DT == PCX_F32 ? 3 : 1, WAVES = WM * WN;
  constexpr int STEPS = steps_per_stage(PARTS, G, WAVES);
  constexpr int ROWS_OUT = WAVES * 32 * (NT * 32 + 4) * 4 + WAVES * 32 * NT * 32 * (DT == PCX_F32 ? 4 : 2), STAGES = 2 * STEPS * NT * WN * frag_bytes(G == 0);
  constexpr int LDS = ROWS_OUT > STAGES ? ROWS_OUT : STAGES;
  auto* const kernel = &pcx_project_forward_kernel<DT, G, MT, NT, WM, WN>;
  if (LDS + 1024 > 65536) PCX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * WAVES), LDS, st, a);
  return 0;
}
template <int DT, int G>
int forward_shape(const ForwardArgs& a, const ForwardPlan& p, unsigned grid, hipStream_t st) {
  if (p.mt == 1) return forward_go<DT, G, 1, 1, 1, 4>(a, grid, st);
  if (p.wm * p.wn == 8) return forward_go<DT, G, 4, 2, 4, 2>(a, grid, st);
  if (p.wn == 2) return p.mt == 4 ? forward_go<DT, G, 4, 2, 2, 2>(a, grid, st) : forward_go<DT, G, 2, 2, 2, 2>(a, grid, st);
  return p.mt == 4 ? forward_go<DT, G, 4, 2, 4, 1>(a, grid, st) : forward_go<DT, G, 2, 2, 4, 1>(a, grid, st);
}
template <int DT>
int forward_type(const ForwardArgs& a, const ForwardPlan& p, unsigned grid, hipStream_t st) {
  int rc;
  if (a.s.stacked) rc = p.wn == 2 ? forward_go<DT, 0, 1, 2, 4, 2>(a, grid, st) : forward_go<DT, 0, 1, 2, 4, 1>(a, grid, st);
  else if (a.s.groups == 1) rc = forward_shape<DT, 1>(a, p, grid, st);
  else if (a.s.groups == 2) rc = forward_shape<DT, 2>(a, p, grid, st);
  else if (a.s.groups == 3) rc = forward_shape<DT, 3>(a, p, grid, st);
  else rc = forward_shape<DT, 4>(a, p, grid, st);
  if (rc) return rc;
  if (p.splits > 1) {
    const int64_t wgs = (a.s.n * (a.wide ? a.s.hidden / 4 : a.s.hidden) + 255) / 256;
    hipLaunchKernelGGL((pcx_project_join<DT>), dim3((unsigned)(wgs < 2048 ? wgs : 2048)), dim3(256), 0, st, a);
  }
  return 0;
}

}  // namespace

extern "C" {

int pcx_project_sizes(const pcx_project_desc* d, uint64_t* packed_bytes, uint64_t* forward_bytes, uint64_t* backward_bytes) {
  Shape s;
  if (int rc = make_shape(d, &s, "pcx_project_sizes")) return rc;
  if (packed_bytes) *packed_bytes = ((uint64_t)s.quads * s.groups + s.stacked) * 4 * s.parts * s.tiles * frag_bytes(s.stacked);
  if (forward_bytes) *forward_bytes = s.n ? plan_forward(s).bytes : 0;
  if (backward_bytes) *backward_bytes = s.n ? pcx::project::backward_bytes(s) : 0;
  return 0;
}

int pcx_project_pack(const pcx_project_desc* d, const void* weight, void* packed, void* stream) {
  Shape s;
  if (int rc = make_shape(d, &s, "pcx_project_pack")) return rc;
  if (!weight || !packed || misaligned(packed, 16) || misaligned(weight, elem_size(s.dtype)))
    return set_error(PCX_E_INVALID, "pcx_project_pack: null or misaligned pointer");
  const dim3 grid((unsigned)s.quads, (unsigned)s.groups, (unsigned)s.tiles), block(256);
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
  if (!s.n) return 0;
  if (!boards) return set_error(PCX_E_INVALID, "pcx_project_forward: no boards");
  const int es = elem_size(s.dtype), ss = s.activation == PCX_ACT_RELU ? es : 4;
  if (!packed || !out || misaligned(packed, 16) || misaligned(out, es) || misaligned(bias, es) || misaligned(residual, es) || misaligned(slope, ss))
    return set_error(PCX_E_INVALID, "pcx_project_forward: null or misaligned pointer");
  const ForwardPlan p = plan_forward(s);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes || misaligned(workspace, 16)))
    return set_error(PCX_E_INVALID, "pcx_project_forward: the workspace needs %llu bytes, 16-byte aligned", (unsigned long long)p.bytes);
  ForwardArgs a{s, boards, reinterpret_cast<const uint8_t*>(packed), bias, residual, out, slope, reinterpret_cast<float*>(workspace),
                p.splits, p.mblocks, p.nblocks, 0, 0};
  a.wide = s.hidden % 4 == 0 && !misaligned(out, 4 * es) && !misaligned(residual, 4 * es) && !misaligned(slope, 4 * ss);
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

}  // extern "C"
