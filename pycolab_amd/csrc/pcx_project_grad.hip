// pcx_project_grad.hip -- the gradients of pcx_project.hip's weight and bias: dz = dy act'(z), dw[h][l][c] = sum over the
// boards that show character l at cell c of dz[.][h], dbias = sum of dz.  Three launches: dz turned round into matrix
// operands (with the bias' sums on the way), the product over runs of boards, and the joining of the runs in a fixed order.
//
// What dz keeps: without an activation, and after a relu, it is dy or 0 and needs no rounding.  After the others it is a
// product that a framework storing it between two operators would round to the weights' type; here it is carried in two
// bfloat16 parts (17 bits), so that a gradient over few boards is as good as its own rounding.  float32: three parts, all bits.
#include "pcx_project.h"

using namespace pcx::project;
using pcx::set_error;

namespace {

constexpr int BLK = 64;          // boards per stage

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
  int32_t wide;          // rows of grad_out and slope keep 16 elements aligned
};

// What dz's parts are made of: 1: the weights' own 16-bit type, 2 or 3: bfloat16.
int dz_parts(const Shape& s) { return s.dtype == PCX_F32 ? 3 : s.activation == PCX_ACT_NONE || s.activation == PCX_ACT_RELU ? 1 : 2; }
// A feature is 2, so dz is halved; float16 operands are not, their sums are.
template <bool F16> constexpr float SCALE = F16 ? 0.5f : 1.0f;

template <int DT, int PARTS>
__global__ __launch_bounds__(256) void pcx_project_turn(BackwardArgs a) {
  typedef typename Num<DT>::T T;
  const Shape& s = a.s;
  __shared__ float tile[BLK][65];
  __shared__ float sums[4][64];
  const int tid = threadIdx.x, h0 = blockIdx.y * 64;
  const T* const dy = reinterpret_cast<const T*>(a.grad_out);
  const T* const sl = reinterpret_cast<const T*>(a.slope);
  const float* const sl32 = reinterpret_cast<const float*>(a.slope);
  const bool relu = s.activation == PCX_ACT_RELU;
  // (relu lets a gradient through or not: an infinite one that it stops is no NaN.  Its slopes are 0 and 1; any others, of a
  // caller who does not say which activation it was, multiply.)
  auto passes = [](T g, T k) { return Num<DT>::get(k) != 0.0f ? Num<DT>::get(g) * Num<DT>::get(k) : 0.0f; };
  const int r = tid >> 2, c0 = (tid & 3) * 16;  // a thread reads 16 neighbouring hidden units of one board
  float total = 0.0f;
  for (int b = blockIdx.x; b < a.blocks; b += gridDim.x) {
    const int64_t gr = (int64_t)b * BLK + r, at = gr * s.hidden + h0 + c0;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.0f;
    if (gr < s.n) {
      if (a.wide && h0 + c0 + 16 <= s.hidden) {
        struct __align__(16) Sixteen { T v[16]; } q;
        q = *reinterpret_cast<const Sixteen*>(dy + at);
        if (!sl) {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = Num<DT>::get(q.v[i]);
        } else if (relu) {
          const Sixteen k = *reinterpret_cast<const Sixteen*>(sl + at);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = passes(q.v[i], k.v[i]);
        } else {
          struct __align__(16) Floats { float v[16]; } k = *reinterpret_cast<const Floats*>(sl32 + at);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = Num<DT>::get(q.v[i]) * k.v[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (h0 + c0 + i < s.hidden) {
            v[i] = Num<DT>::get(dy[at + i]);
            if (sl && relu) v[i] = passes(dy[at + i], sl[at + i]);
            else if (sl) v[i] *= sl32[at + i];
          }
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) tile[r][c0 + i] = v[i];
    __syncthreads();
    if (a.grad_bias) {
#pragma unroll
      for (int i = 0; i < 16; ++i) total += tile[(tid >> 6) * 16 + i][tid & 63];
    }
    if (a.frags) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = tid + k * 256, lane = i & 63, ht = (i >> 6) & 1, kb = i >> 7;
        const int tile_h = blockIdx.y * 2 + ht;
        if (tile_h >= a.htiles) continue;
        float d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = tile[kb * 16 + (lane >> 5) * 8 + e][ht * 32 + (lane & 31)];
        u32x4* const to = reinterpret_cast<u32x4*>(a.frags) + ((((int64_t)b * 4 + kb) * a.htiles + tile_h) * PARTS) * 64 + lane;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          u32x4 w = {0, 0, 0, 0};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            uint32_t bits;
            if constexpr (DT == PCX_F16 && PARTS == 1) bits = __builtin_bit_cast(uint16_t, (_Float16)d[e]);
            else bits = part_of(0.5f * d[e], p, PARTS);
            w[e >> 1] |= bits << (16 * (e & 1));
          }
          to[p * 64] = w;
        }
      }
    }
    __syncthreads();
  }
  if (!a.grad_bias) return;
  sums[tid >> 6][tid & 63] = total;
  __syncthreads();
  if (tid >= 64 || h0 + tid >= s.hidden) return;
  const float sum = (sums[0][tid] + sums[1][tid]) + (sums[2][tid] + sums[3][tid]);
  if (a.bias_blocks > 1) a.bias_part[(int64_t)blockIdx.x * s.hidden + h0 + tid] = sum;
  else reinterpret_cast<T*>(a.grad_bias)[h0 + tid] = Num<DT>::put(sum);  // (whole: nothing to join)
}

// dw[h][l][c] over a run of boards: a workgroup owns NH tiles of hidden units x 32 cells x up to 2 LW layers (NH = 1: 4 LW).
// The sum runs over boards, along which the features are not sparse: the dense instruction.  Its right operand is the
// feature bit of 8 consecutive boards at one cell: the boards are turned round once per stage into LDS as a word of layer
// bits per (cell, board), from which every layer's operand is one shift and one mask.  A wave takes LW layers x half the
// hidden units (2 layers x all units: float32 gradients of 2,048 boards of 4,005 cells 10 us slower).  65,536 boards of 300 cells x 8
// layers x 256 units take 77 us, and 89 for some 20 ms after the GPU was idle, until its clocks have settled.  Of those 89 the
// instructions alone take 47 (1.8 PFLOP/s): the masks' way through the LDS after each barrier adds 11, dz's copies and the
// boards' turning, which the other workgroup's products hide in part, 26, and the partial sums, as many as all registers of
// the card hold, 8.
// Blocks of dz in LDS, one in use: three where that leaves room for two workgroups a CU, else two (dz in two or three parts;
// one workgroup with three instead: 2,048 boards of 4,005 cells, float32 gradients 130 us against 105, 65,536 of 300 with
// gelu and bfloat16 ones 216 against 166, the turning and joining included).
template <int PARTS, int NH>
struct Stage {
  static constexpr int BYTES = 4 * NH * PARTS * 1024, MASKS = 32 * (BLK + 8) * 2, RING = 3 * BYTES + 2 * MASKS + 512 <= 80 * 1024 ? 3 : 2;
  static constexpr int LDS = RING * BYTES + 2 * MASKS + 512;
};
template <bool F16, int PARTS, bool STACKED, int NH, int LW>
__global__ __launch_bounds__(256, 2) void pcx_project_weight_grad(BackwardArgs a) {
  constexpr int STAGE = Stage<PARTS, NH>::BYTES, RING = Stage<PARTS, NH>::RING;
  constexpr int PITCH = BLK + 8;                // words per cell: 16-byte reads of one wave spread over the banks
  constexpr int MASKS = Stage<PARTS, NH>::MASKS;
  constexpr int WH = NH == 1 ? 1 : 2, HW = NH / WH, WL = 4 / WH, LAYERS = WL * LW;  // waves along hidden units and layers
  const Shape& s = a.s;
  extern __shared__ __align__(16) uint8_t lds[];
  uint16_t* const lut = reinterpret_cast<uint16_t*>(lds + RING * STAGE + 2 * MASKS);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const uint32_t tiles = (uint32_t)a.cell_blocks * a.layer_blocks * a.hblocks;
  // the tiles of one run of boards go to one XCD, whose L2 then serves dz and the boards once
  const uint32_t id = (blockIdx.x & 7u) * (uint32_t)a.chunk + (blockIdx.x >> 3);
  if (id >= tiles * (uint32_t)a.splits) return;
  const int split = (int)(id / tiles);
  uint32_t t = id % tiles;
  const int hb = (int)(t % (uint32_t)a.hblocks); t /= (uint32_t)a.hblocks;
  const int lb = (int)(t % (uint32_t)a.layer_blocks), cb = (int)(t / (uint32_t)a.layer_blocks);
  const int l0 = lb * LAYERS, c0 = quad_start(cb, s.cells);
  if constexpr (!STACKED) {
    lut[tid] = 0;
    __syncthreads();
    if (tid < LAYERS && l0 + tid < s.layers) lut[argument<BackwardArgs>()->s.chars[l0 + tid]] = (uint16_t)(1u << (14 - tid));
  }
  const int b0 = (int)((int64_t)a.blocks * split / a.splits), b1 = (int)((int64_t)a.blocks * (split + 1) / a.splits);
  const uint8_t* const src = a.frags + (int64_t)hb * NH * PARTS * 1024 + lane * 16;
  auto stage_in = [&](int b) {
    uint8_t* const dst = lds + (b - b0) % RING * STAGE;
#pragma unroll
    for (int i = 0; i < NH * PARTS; ++i) {
      const int k = wave * NH * PARTS + i;  // (piece i of board step `wave`)
      copy_in(src + ((((int64_t)(b < b1 ? b : b1 - 1) * 4 + wave) * a.htiles) * PARTS + i) * 1024, dst + k * 1024);
    }
  };
  // a thread turns two boards x four cells round
  const int pair = tid >> 3, cell = (tid & 7) * 4;
  const bool small = s.cells < QUAD;
  constexpr int PL = STACKED ? LAYERS : 1;
  int32_t offset[PL];  // STACKED: of this block's layers within a board, -1: nowhere (a board is less than 2 GB)
#pragma unroll
  for (int l = 0; l < PL; ++l) offset[l] = !STACKED ? 0 : l0 + l < s.layers ? (int32_t)argument<BackwardArgs>()->s.layer_offset[l0 + l] : -1;
  auto fetch = [&](int b, uint32_t* raw) {  // [board of the pair][layer]
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t gr = (int64_t)b * BLK + pair * 2 + r;
      const uint8_t* const at = a.boards + (gr < s.n ? gr : s.n - 1) * s.row_stride;  // (boards past the end meet dz = 0)
#pragma unroll
      for (int l = 0; l < PL; ++l) {
        uint32_t v = 0;
        if (small) {
          if (offset[l] >= 0) v = edge_dword(at + offset[l], cell, s.cells);
        } else {
          __builtin_memcpy(&v, at + (offset[l] >= 0 ? offset[l] : 0) + c0 + cell, 4);
        }
        raw[r * PL + l] = v;
      }
    }
  };
  auto turn = [&](int b, const uint32_t* raw, int c) {  // (of the thread's four cells the one numbered c)
    uint8_t* const dst = lds + RING * STAGE + (b & 1) * MASKS;
    uint32_t m[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (STACKED) {
        m[r] = 0;
#pragma unroll
        for (int l = 0; l < PL; ++l) m[r] |= offset[l] >= 0 && ((raw[r * PL + l] >> (8 * c)) & 255u) ? 1u << (14 - l) : 0u;
      } else {
        m[r] = lut[(raw[r] >> (8 * c)) & 255u];
      }
    }
    *reinterpret_cast<uint32_t*>(dst + ((cell + c) * PITCH + pair * 2) * 2) = m[0] | (m[1] << 16);
  };
  f32x16 acc[LW][HW];
#pragma unroll
  for (int l = 0; l < LW; ++l)
#pragma unroll
    for (int h = 0; h < HW; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[l][h][i] = 0.0f;
  const int wl = wave % WL, wh = wave / WL;
  // One block of boards: the block after the next is asked for, the next one's boards are turned round, this one's products
  // are formed.  Blocks past the run's end are its last block again: they land in stages that nobody reads.
  auto step = [&](int b, const uint32_t* next, uint32_t* later) {
    // block b's dz and block b + 1's boards must be here; what was asked for since then may be on its way
    if constexpr (RING == 3) {
      stage_barrier<NH * PARTS>();
      fetch(b + 2, later);
      stage_in(b + 2);
    } else {
      if (small) stage_barrier<0>();
      else stage_barrier<2 * PL>();
      stage_in(b + 1);
      asm volatile("" ::: "memory");
      fetch(b + 2, later);
    }
    const uint8_t* const dz = lds + (b - b0) % RING * STAGE + lane * 16;
    const uint8_t* const masks = lds + RING * STAGE + (b & 1) * MASKS + ((lane & 31) * PITCH + half * 8) * 2;
#pragma unroll
    for (int c = 0; c < 4; ++c) turn(b + 1, next, c);
    __builtin_amdgcn_s_setprio(1);  // (a wave that multiplies goes before the other workgroup's that turn: 94 -> 89 us)
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const u32x4 m = *reinterpret_cast<const u32x4*>(masks + kb * 32);
      u32x4 right[LW];
#pragma unroll
      for (int l = 0; l < LW; ++l)
#pragma unroll
        for (int e = 0; e < 4; ++e) right[l][e] = (m[e] << (wl * LW + l)) & 0x40004000u;
#pragma unroll
      for (int h = 0; h < HW; ++h)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          const u32x4 left = *reinterpret_cast<const u32x4*>(dz + ((kb * NH + wh * HW + h) * PARTS + p) * 1024);
#pragma unroll
          for (int l = 0; l < LW; ++l) acc[l][h] = dense_step<F16>(left, right[l], acc[l][h]);
        }
    }
    __builtin_amdgcn_s_setprio(0);
  };
  uint32_t even[2 * PL], odd[2 * PL];
  if (b0 < b1) {
    fetch(b0, even);
    stage_in(b0);
    if constexpr (RING == 3) fetch(b0 + 1, odd), stage_in(b0 + 1);
    else fetch(b0 + 1, odd);
    __syncthreads();  // the table
#pragma unroll
    for (int c = 0; c < 4; ++c) turn(b0, even, c);
#pragma unroll 1
    for (int b = b0; b < b1; b += 2) {
      step(b, odd, even);
      if (b + 1 >= b1) break;
      step(b + 1, even, odd);
    }
    stage_barrier<0>();  // (no copy may land after the workgroup's end)
  }
  const int c = c0 + (lane & 31);
  if (c < cb * QUAD || c >= s.cells) return;  // (the block before owns the cells this one shares with it)
#pragma unroll
  for (int l = 0; l < LW; ++l) {
    const int layer = l0 + wl * LW + l;
    if (layer >= s.layers) continue;
#pragma unroll
    for (int h = 0; h < HW; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int unit = (hb * NH + wh * HW + h) * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
        if (unit >= s.hidden) continue;
        const int64_t at = ((int64_t)unit * s.layers + layer) * s.cells + c;
        const float v = SCALE<F16> * acc[l][h][i];
        if (a.splits > 1) a.partial[(int64_t)split * s.hidden * s.layers * s.cells + at] = v;
        else if (PARTS == 3) reinterpret_cast<float*>(a.grad_weight)[at] = v;  // (whole: nothing to join)
        else if (F16 || (PARTS == 2 && s.dtype == PCX_F16)) reinterpret_cast<_Float16*>(a.grad_weight)[at] = Num<PCX_F16>::put(v);
        else reinterpret_cast<__bf16*>(a.grad_weight)[at] = Num<PCX_BF16>::put(v);
      }
  }
}

// The runs' partial sums joined in a fixed order; the last workgroups join the bias' sums.
template <int DT>
__global__ __launch_bounds__(256) void pcx_project_grad_join(BackwardArgs a, int weight_blocks) {
  typedef typename Num<DT>::T T;
  if ((int)blockIdx.x < weight_blocks) {
    const int64_t total = (int64_t)a.s.hidden * a.s.layers * a.s.cells;
    T* const out = reinterpret_cast<T*>(a.grad_weight);
    if ((total & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0) {
      struct __align__(4 * sizeof(T)) Four { T v[4]; };
      for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < total; i += (int64_t)weight_blocks * 1024) {
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < a.splits; ++k) {
          const float4 v = *reinterpret_cast<const float4*>(a.partial + (int64_t)k * total + i);
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        *reinterpret_cast<Four*>(out + i) = Four{{Num<DT>::put(sum.x), Num<DT>::put(sum.y), Num<DT>::put(sum.z), Num<DT>::put(sum.w)}};
      }
    } else {
      for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)weight_blocks * 256) {
        float sum = 0.0f;
        for (int k = 0; k < a.splits; ++k) sum += a.partial[(int64_t)k * total + i];
        out[i] = Num<DT>::put(sum);
      }
    }
    return;
  }
  __shared__ float part[16][16];
  const int h = ((int)blockIdx.x - weight_blocks) * 16 + (threadIdx.x & 15), w = threadIdx.x >> 4;
  float sum = 0.0f;
  if (h < a.s.hidden)
    for (int k = w; k < a.bias_blocks; k += 16) sum += a.bias_part[(int64_t)k * a.s.hidden + h];
  part[w][threadIdx.x & 15] = sum;
  __syncthreads();
  if (w || h >= a.s.hidden) return;
  for (int k = 1; k < 16; ++k) sum += part[k][threadIdx.x];
  reinterpret_cast<T*>(a.grad_bias)[h] = Num<DT>::put(sum);
}

// ---------------------------------------------------------------- plan

struct BackwardPlan { int nh, lw, htiles, hblocks, cell_blocks, layer_blocks, splits, bias_blocks, blocks, parts; uint64_t frag_bytes, bias_bytes, part_bytes; };

BackwardPlan plan_backward(const Shape& s) {
  BackwardPlan p;
  p.parts = dz_parts(s);
  p.nh = p.parts == 3 ? (s.tiles >= 2 ? 2 : 1) : s.tiles >= 3 ? 4 : s.tiles;  // (dz in three parts: two workgroups' LDS)
  p.hblocks = (s.tiles + p.nh - 1) / p.nh;
  p.htiles = p.hblocks * p.nh;
  p.cell_blocks = s.quads;
  // Eight layers a workgroup, or four where that pads fewer (one tile of hidden units: always eight).
  const int pad8 = (s.layers + 7) / 8 * 8, pad4 = (s.layers + 3) / 4 * 4;
  p.lw = pad4 < pad8 || p.nh == 1 ? 2 : 4;
  const int per = (p.nh == 1 ? 4 : 2) * p.lw;
  p.layer_blocks = (s.layers + per - 1) / per;
  p.blocks = (int)((s.n + BLK - 1) / BLK);
  const int64_t tiles = (int64_t)p.hblocks * p.cell_blocks * p.layer_blocks;
  int64_t splits = SLOTS / tiles;
  if (splits > p.blocks) splits = p.blocks;
  if (splits < 1) splits = 1;
  p.splits = (int)splits;
  p.bias_blocks = p.blocks < 512 ? p.blocks : 512;
  p.frag_bytes = (uint64_t)p.blocks * 4 * p.htiles * p.parts * 1024;
  p.bias_bytes = ((uint64_t)p.bias_blocks * s.hidden * 4 + 255) & ~255ull;
  p.part_bytes = p.splits > 1 ? (uint64_t)p.splits * s.hidden * s.layers * s.cells * 4 : 0;
  return p;
}

template <bool F16, int PARTS, bool STACKED, int NH, int LW>
int grad_go(const BackwardArgs& a, unsigned grid, hipStream_t st) {
  constexpr int LDS = Stage<PARTS, NH>::LDS;
  auto* const kernel = &pcx_project_weight_grad<F16, PARTS, STACKED, NH, LW>;
  if (LDS > 65536) PCX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), LDS, st, a);
  return 0;
}
template <bool F16, int PARTS, bool STACKED>
int grad_shape(const BackwardArgs& a, const BackwardPlan& p, unsigned grid, hipStream_t st) {
  if (p.nh == 1) return grad_go<F16, PARTS, STACKED, 1, 2>(a, grid, st);
  if (p.nh == 2) return p.lw == 4 ? grad_go<F16, PARTS, STACKED, 2, 4>(a, grid, st) : grad_go<F16, PARTS, STACKED, 2, 2>(a, grid, st);
  if constexpr (PARTS == 3) return set_error(PCX_E_INVALID, "pcx_project_backward: no such tile");
  else return p.lw == 4 ? grad_go<F16, PARTS, STACKED, 4, 4>(a, grid, st) : grad_go<F16, PARTS, STACKED, 4, 2>(a, grid, st);
}
template <int DT, int PARTS>
int backward_parts(BackwardArgs& a, const BackwardPlan& p, hipStream_t st) {
  constexpr bool F16 = DT == PCX_F16 && PARTS == 1;
  hipLaunchKernelGGL((pcx_project_turn<DT, PARTS>), dim3((unsigned)p.bias_blocks, (unsigned)((p.htiles + 1) / 2)), dim3(256), 0, st, a);
  int weight_blocks = 0;
  if (a.grad_weight) {
    const int64_t groups = (int64_t)p.cell_blocks * p.layer_blocks * p.hblocks * p.splits;
    a.chunk = (int32_t)((groups + 7) / 8);
    const unsigned grid = (unsigned)a.chunk * 8u;
    if (int rc = a.s.stacked ? grad_shape<F16, PARTS, true>(a, p, grid, st) : grad_shape<F16, PARTS, false>(a, p, grid, st)) return rc;
    const int64_t wgs = ((int64_t)a.s.hidden * a.s.layers * a.s.cells + 1023) / 1024;
    if (a.splits > 1) weight_blocks = (int)(wgs < 4096 ? wgs : 4096);
  }
  const int bias_blocks = a.grad_bias && a.bias_blocks > 1 ? (a.s.hidden + 15) / 16 : 0;
  if (weight_blocks + bias_blocks)
    hipLaunchKernelGGL((pcx_project_grad_join<DT>), dim3((unsigned)(weight_blocks + bias_blocks)), dim3(256), 0, st, a, weight_blocks);
  return 0;
}
template <int DT>
int backward_type(BackwardArgs& a, const BackwardPlan& p, hipStream_t st) {
  if constexpr (DT == PCX_F32) return backward_parts<DT, 3>(a, p, st);
  else return p.parts == 1 ? backward_parts<DT, 1>(a, p, st) : backward_parts<DT, 2>(a, p, st);
}

}  // namespace

uint64_t pcx::project::backward_bytes(const Shape& s) {
  const BackwardPlan p = plan_backward(s);
  return p.frag_bytes + p.bias_bytes + p.part_bytes;
}

extern "C" int pcx_project_backward(const pcx_project_desc* d, const uint8_t* boards, const void* grad_out, const void* slope, void* grad_weight,
                                    void* grad_bias, void* workspace, uint64_t workspace_bytes, void* stream) {
  Shape s;
  if (int rc = make_shape(d, &s, "pcx_project_backward")) return rc;
  if (!s.n) return set_error(PCX_E_INVALID, "pcx_project_backward: no boards (their gradients are zero)");
  if (!boards) return set_error(PCX_E_INVALID, "pcx_project_backward: no boards");
  if (!grad_weight && !grad_bias) return 0;
  const int es = elem_size(s.dtype), ss = s.activation == PCX_ACT_RELU ? es : 4;
  if (!grad_out || misaligned(grad_out, es) || misaligned(slope, ss) || misaligned(grad_weight, es) || misaligned(grad_bias, es))
    return set_error(PCX_E_INVALID, "pcx_project_backward: null or misaligned pointer");
  if (s.activation != PCX_ACT_NONE && !slope) return set_error(PCX_E_INVALID, "pcx_project_backward: the activation's slopes are missing");
  const BackwardPlan p = plan_backward(s);
  if ((int64_t)p.hblocks * p.cell_blocks * p.layer_blocks * p.splits >= (int64_t)1 << 23)
    return set_error(PCX_E_INVALID, "pcx_project_backward: the weight is too large");
  if (!workspace || workspace_bytes < p.frag_bytes + p.bias_bytes + p.part_bytes || misaligned(workspace, 16))
    return set_error(PCX_E_INVALID, "pcx_project_backward: the workspace needs %llu bytes, 16-byte aligned",
                     (unsigned long long)(p.frag_bytes + p.bias_bytes + p.part_bytes));
  uint8_t* const ws = reinterpret_cast<uint8_t*>(workspace);
  BackwardArgs a{s, boards, grad_out, s.activation == PCX_ACT_NONE ? nullptr : slope, grad_weight ? ws : nullptr,
                 reinterpret_cast<float*>(ws + p.frag_bytes), reinterpret_cast<float*>(ws + p.frag_bytes + p.bias_bytes), grad_weight, grad_bias,
                 p.blocks, p.htiles, p.bias_blocks, p.splits, p.cell_blocks, p.layer_blocks, p.hblocks, 0, 0};
  a.wide = s.hidden % 16 == 0 && !misaligned(grad_out, 16) && !misaligned(a.slope, 16);
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (s.dtype == PCX_F32) rc = backward_type<PCX_F32>(a, p, st);
  else if (s.dtype == PCX_F16) rc = backward_type<PCX_F16>(a, p, st);
  else rc = backward_type<PCX_BF16>(a, p, st);
  if (rc) return rc;
  PCX_HIP(hipGetLastError());
  return 0;
}
