// Expert products with weights of 4 bits and a scale (and zero point) per group of 32, 64 or 128: no counterpart in the reference.
//
//   out[r, n] = act( sum_G s[e, n, G] * ( sum over k of G of q[e, n, k] * x[r, k]  -  z[e, n, G] * sum over k of G of x[r, k] ) + bias[e, n] )
//
// for the rows r of expert e (rows are packed by expert, their counts read from the device; or named by row entries, and read from
// the cells).  q is 0 .. 15, z a whole number, 8 where there is none.
//
// Weights are laid out once as the matrix instruction reads them (include/brt_hip.h has the bytes): a wavefront's load of 16 bytes a
// lane is 1 KB in one piece, 16 rows of 128 columns, and word j of a lane its fragment of the j-th v_mfma_f32_16x16x32.  The four bits of a
// weight as a byte are an e4m3 number, q * 2^-9, all sixteen of them (below 8 they are subnormal, from 8 on normal of the same
// spacing), so that a word becomes a fragment of bf16 or fp16 in one shift, two masks and four conversions, exactly.  The rows stay in their
// type; fp32 rows are split into three bf16 parts (8 bits each: all of them, down to 2^-133) and take three instructions.  A group's products are summed
// by the matrix unit on top of -z times its sum of x, which one more instruction with a constant fragment leaves in the
// result's layout, and the group's sum is scaled in fp32 by one multiply-add.  So nothing but the result is rounded below fp32.
//   Elements of the range of fp32 are multiplied by q * 2^-15: before the scale a group may add up to 128 * 255 times as much as its
// largest element, which is then still within the range, and so are the sums of scaled groups whose results are.  The results are multiplied
// by 2^15 where the bias is added; the matrix unit keeps subnormal numbers, and those products are whole multiples of 2^-148.
//   The weight fragment is the first operand: a lane holds results of one row and four neighbouring columns.
#include <algorithm>
#include <type_traits>

#include "packed_rows.hpp"

namespace brt {
namespace {

constexpr int kB = 128;              // columns of a block of the weights' layout
constexpr int kMostRows = 1 << 24;   // 65 times as many are added up in 32 bits
constexpr long kMostThreads = 1l << 32;  // of a launch
constexpr int kMostColumns = 1 << 28;  // and experts and elements of a row: rounded up to tiles they are counted in 32 bits

struct Int4Args {
  const void* x;         // [P, K], or with entries [T, K]
  const int* entries;    // [P] 1-based entries t * per_cell + j + 1 of the rows, or null
  const uint8_t* w;      // [E, tiles, KB, 1024]
  const void* scales;    // [E, tiles, G, 16] of s_dtype
  const uint8_t* zeros;  // [E, tiles, G, 16] or null
  const int* loads;      // [E]
  const void* bias;      // [E, N] of bias_dtype or null
  void* out;             // [P, N] of out_dtype
  int s_dtype, bias_dtype, out_dtype, act;
  int E, P, N, K, KB, G, T, per_cell, tiles, tiles_n, blocks;
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// What weights are multiplied by, and the results of their products with rows of that type divided by.
template <int XDT>
constexpr float kWeightUnit = XDT == BRT_F16 ? 1.0f : 0x1p-15f;

// Eight weights of a word, as the numbers 0 .. 15 in such units: the low halves of its bytes are elements 0 .. 3, the high ones 4 .. 7.
template <int XDT>
__device__ __forceinline__ auto weights_of(uint32_t word) {
  constexpr float kUnit = 512.0f * kWeightUnit<XDT>;
  const int lo = static_cast<int>(word & 0x0f0f0f0fu), hi = static_cast<int>((word >> 4) & 0x0f0f0f0fu);
  if constexpr (XDT == BRT_F16) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, kUnit, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, kUnit, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, kUnit, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, kUnit, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  } else {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, kUnit, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, kUnit, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, kUnit, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, kUnit, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
}

// Eight elements of a row as the second operand; fp32 as the sum of three bf16 parts.
template <int XDT>
struct RowPart {
  static constexpr int kUnits = XDT == BRT_F32 ? 2 : 1, kParts = XDT == BRT_F32 ? 3 : 1;
  using Type = std::conditional_t<XDT == BRT_F16, f16x8, bf16x8>;
  Type part[kParts];
  __device__ __forceinline__ explicit RowPart(const u32x4* raw) {
    if constexpr (XDT == BRT_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = __uint_as_float(raw[i / 4][i % 4]);
        part[0][i] = static_cast<__bf16>(v);
        const float rest = v - static_cast<float>(part[0][i]);
        part[1][i] = static_cast<__bf16>(rest);
        part[2][i] = static_cast<__bf16>(rest - static_cast<float>(part[1][i]));
      }
    } else {
      part[0] = __builtin_bit_cast(Type, raw[0]);
    }
  }
};

__device__ __forceinline__ f32x4 multiply(const bf16x8& w, const bf16x8& x, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply(const f16x8& w, const f16x8& x, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(w, x, c, 0, 0, 0);
}
template <int XDT, typename W>
__device__ __forceinline__ f32x4 multiply(const W& w, const RowPart<XDT>& x, f32x4 c) {
#pragma unroll
  for (int p = RowPart<XDT>::kParts - 1; p >= 0; --p) c = multiply(w, x.part[p], c);  // (the small parts first)
  return c;
}
template <int XDT, typename W>
__device__ __forceinline__ f32x4 multiply(const RowPart<XDT>& x, const W& w, f32x4 c) {
#pragma unroll
  for (int p = RowPart<XDT>::kParts - 1; p >= 0; --p) c = multiply(x.part[p], w, c);
  return c;
}

// The scale that was loaded as `bits`.
__device__ __forceinline__ float scale_of(uint32_t bits, int dtype) {
  return dtype == BRT_F32 ? __uint_as_float(bits) : dtype == BRT_F16 ? f16_to_float(bits) : bf16_to_float(bits);
}

template <int COUNT>
__device__ __forceinline__ void scales_of(const uint32_t (&bits)[COUNT], int dtype, float (&s)[COUNT]) {
  if (dtype == BRT_F32) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) s[i] = __uint_as_float(bits[i]);
  } else if (dtype == BRT_F16) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) s[i] = f16_to_float(bits[i]);
  } else {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) s[i] = bf16_to_float(bits[i]);
  }
}

// GELU of an fp32 result: the fit that the other products share is off by up to 4.3e-6, which 16 bits hide and fp32 shows.
__device__ __forceinline__ float gelu_f32(float v) {
  const float b = __builtin_elementwise_maximum(v, -1e30f);  // (0 * inf; NaN stays)
  return 0.5f * b * (1.0f + erff(b * 0.70710678118654752f));
}
template <int ACT, int OUT>
__device__ __forceinline__ float activated_for(float v) {
  if constexpr (ACT == BRT_ACT_GELU && OUT == BRT_F32) return gelu_f32(v);
  else return activated<ACT>(v);
}
__device__ __forceinline__ float activated_for(float v, int act, int out_dtype) {
  return act == BRT_ACT_GELU && out_dtype == BRT_F32 ? gelu_f32(v) : activated(v, act);
}

// Four results of a row, columns n .. n + 3 (n < N), rounded and stored.  Rows of any N begin at any element: the four leave in one store
// all the same, which need not be aligned to more than an element.
typedef u32x4 u32x4_at_4 __attribute__((aligned(4)));
typedef u32x2 u32x2_at_2 __attribute__((aligned(2)));
template <int OUT>
__device__ __forceinline__ void store_four(const Int4Args& a, size_t row, int n, const float (&v)[4]) {
  char* const to = static_cast<char*>(a.out) + (row * a.N + n) * elem_bytes(OUT);
  if (n + 4 <= a.N) {
    if constexpr (OUT == BRT_F32) {
      *reinterpret_cast<u32x4_at_4*>(to) = u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    } else {
      *reinterpret_cast<u32x2_at_2*>(to) = u32x2{float_to_half_bits<OUT>(v[0]) | float_to_half_bits<OUT>(v[1]) << 16,
                                                 float_to_half_bits<OUT>(v[2]) | float_to_half_bits<OUT>(v[3]) << 16};
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    const float one[1] = {v[q]};
    if (n + q < a.N) pack_store<OUT, 1>(to + q * elem_bytes(OUT), one);
  }
}

// Row `row` of the packed layout: its elements, or null where it stands for none (padding of a path: a row of zeros).
template <int XDT>
__device__ __forceinline__ const char* row_of(const Int4Args& a, int row) {
  long at = row;
  if (a.entries != nullptr) {
    const int word = a.entries[row], cell = a.per_cell > 1 ? (word - 1) / a.per_cell : word - 1;
    if (word < 1 || cell >= a.T) return nullptr;
    at = cell;
  }
  return static_cast<const char*>(a.x) + at * a.K * elem_bytes(XDT);
}

// Few rows per expert: the weights are streamed once and set the time.  A workgroup takes 16 NT columns and 16 rows; its W
// wavefronts take blocks of 128 columns in turn, weights and rows straight into the fragments' registers, and add up their sums through
// LDS.  The rows are the first operand here: a lane holds results of one column, whose scale and zero point are one register each.
//   (Back to back.)  256 rows of 64 experts 4096 -> 1024 30 us, 139 MB at 4.6 TB/s (a large copy's rate is 5.2): memory.  1 row 2048 -> 8192
// 5.0 us and 48 rows of 8 experts 1024 -> 4096 7.4 us, of which the bytes take 1.7 and 3.6: a launch, the loads and two dependent rounds of requests.
// Two blocks of a wavefront in flight instead of one, or two and four row blocks a workgroup, which share the weights, gained nothing.
//   fp32 rows: 333 rows of 12 experts 776 -> 1001, groups of 32, 12.5 us: two rounds of requests as well, the rows' splitting
// (over again for every 16 NT columns) and three products in place of one between them; vector units 0.22 of the time, matrix units 0.06.
template <int XDT, int GJ, int NT, int W>
__global__ __launch_bounds__(W * 64) void int4_few_rows_kernel(Int4Args a) {
  using Part = RowPart<XDT>;
  using Weights = decltype(weights_of<XDT>(0));
  constexpr int kGroups = 4 / GJ;  // of a block; GJ fragments share a group
  __shared__ float s_part[W][NT][16][17];  // [row][column], a column of padding
  const int lane = lane_id(), g = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int block = blockIdx.x / a.tiles_n, tile0 = (blockIdx.x - block * a.tiles_n) * NT, n0 = tile0 * 16;
  const Block at = find_block(a, block, 4);
  if (at.rows == 0) return;
  const char* const row = row_of<XDT>(a, at.row0 + min(c16, at.rows - 1));
  const bool whole_rows = __ballot(row == nullptr) == 0;
  // the biases of the tiles that this wavefront finishes, four lanes a row of a tile and four columns each: fetched ahead of the weights,
  // not behind the last barrier
  constexpr int kFinished = (NT + W - 1) / W;
  const int r = lane >> 2, c4 = (lane & 3) * 4;
  float bias[kFinished][4];
#pragma unroll
  for (int f = 0; f < kFinished; ++f) biases<4>(a, at.e, n0 + (wave + f * W) % NT * 16 + c4, bias[f]);

  f32x4 acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  Weights minus_one;
#pragma unroll
  for (int i = 0; i < 8; ++i) minus_one[i] = -kWeightUnit<XDT>;
  for (int kb = wave; kb < a.KB; kb += W) {
    u32x4 raw_w[NT], raw_x[4 * Part::kUnits];
    uint32_t raw_s[NT][kGroups], raw_z[NT][kGroups];
    size_t one[NT][kGroups];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const size_t tile = static_cast<size_t>(at.e) * a.tiles + min(tile0 + j, a.tiles - 1);
      raw_w[j] = *reinterpret_cast<const u32x4*>(a.w + (tile * a.KB + kb) * 1024 + lane * 16);
#pragma unroll
      for (int h = 0; h < kGroups; ++h) one[j][h] = (tile * a.G + min(kb * kGroups + h, a.G - 1)) * 16 + c16, raw_z[j][h] = 8;
    }
#pragma unroll
    for (int l = 0; l < 4 * Part::kUnits; ++l) {
      const int k = kb * kB + l / Part::kUnits * 32 + g * 8;
      const char* const from = row + static_cast<size_t>(k) * elem_bytes(XDT) + l % Part::kUnits * 16;
      if (whole_rows && kb * kB + kB <= a.K) {
        raw_x[l] = *reinterpret_cast<const u32x4*>(from);
      } else {
        raw_x[l] = zero_unit<16>();
        if (k < a.K && row != nullptr) raw_x[l] = *reinterpret_cast<const u32x4*>(from);  // (K is a multiple of 8)
      }
    }
    if (a.s_dtype == BRT_F32) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < kGroups; ++h) raw_s[j][h] = static_cast<const uint32_t*>(a.scales)[one[j][h]];
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < kGroups; ++h) raw_s[j][h] = static_cast<const uint16_t*>(a.scales)[one[j][h]];
    }
    if (a.zeros != nullptr) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < kGroups; ++h) raw_z[j][h] = a.zeros[one[j][h]];
    }
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f}, part[NT];  // sum: minus the rows' sums over the group, in every column
#pragma unroll
      for (int p = 0; p < GJ; ++p) sum = multiply(Part(&raw_x[(h * GJ + p) * Part::kUnits]), minus_one, sum);
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) part[j][q] = static_cast<float>(raw_z[j][h]) * sum[q];
#pragma unroll
      for (int p = 0; p < GJ; ++p) {
        const Part x(&raw_x[(h * GJ + p) * Part::kUnits]);
#pragma unroll
        for (int j = 0; j < NT; ++j) part[j] = multiply(x, weights_of<XDT>(raw_w[j][h * GJ + p]), part[j]);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float s = scale_of(raw_s[j][h], a.s_dtype);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[j][q] = __builtin_fmaf(part[j][q], s, acc[j][q]);
      }
    }
  }

#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) s_part[wave][j][g * 4 + q][c16] = acc[j][q];
  __syncthreads();
#pragma unroll
  for (int f = 0; f < kFinished; ++f) {
    const int j = wave + f * W, n = n0 + j * 16 + c4;
    if (j >= NT || r >= at.rows || n >= a.N) continue;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += s_part[w][j][r][c4 + q];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = activated_for(__builtin_fmaf(v[q], 1.0f / kWeightUnit<XDT>, bias[f][q]), a.act, a.out_dtype);
    const size_t to = static_cast<size_t>(at.row0) + r;
    if (a.out_dtype == BRT_F32) store_four<BRT_F32>(a, to, n, v);
    else if (a.out_dtype == BRT_F16) store_four<BRT_F16>(a, to, n, v);
    else store_four<BRT_BF16>(a, to, n, v);
  }
}

template <int XDT, int GJ, int NT, int W>
int launch_few_rows(Int4Args& a, hipStream_t st) {
  const long blocks = static_cast<long>(a.P) / 16 + std::min(a.E, a.P);
  a.tiles_n = (a.tiles + NT - 1) / NT;
  if (blocks * a.tiles_n * (W * 64) >= kMostThreads) return fail(BRT_E_UNSUPPORTED, "too many tiles");
  hipLaunchKernelGGL((int4_few_rows_kernel<XDT, GJ, NT, W>), dim3(static_cast<unsigned>(blocks * a.tiles_n)), dim3(W * 64), 0, st, a);
  return check_launch("int4_few_rows_kernel");
}
// Tiles of 16 x 16 results: experts' last row blocks are taken as half full, and every expert to have rows where there are as many rows.
long small_tiles(const Int4Args& a) {
  const long used = std::min(a.E, a.P);
  return (a.P > 8l * a.E ? std::max(used, (a.P + 15l) / 16 + (a.E > 1 ? used / 2 : 0)) : used) * a.tiles;
}
// Columns of a workgroup (16 NT) and wavefronts that share its K (W), by the tiles that there are to deal out and the blocks of K.  Few
// tiles: as many wavefronts as possible on each; many: more columns to a wavefront, which fetches the rows once for all of them.  (us, bf16
// rows; NT, W) 1 row 2048 -> 8192: 2, 8 5.0, 1, 16 6.6, 4, 4 8.1; 1 row 8192 -> 1024: 1, 16 6.4, 2, 8 8.9; 64 rows 4096 -> 4096: 4, 8 10.2, 2, 8
// 13.1; 4 rows of 4 experts 4096 -> 4096: 2, 8 8.9, 4, 8 9.7; 48 rows of 8 1024 -> 4096: 2, 4 7.4, 4, 8 7.8, 2, 8 8.3; 128 rows of 32
// 1024 -> 4096: 4, 2 16.0, 2, 4 18.7, 4, 8 19.9, 1, 8 27; 128 of 32 4096 -> 1024: 4, 8 16.5, 4, 4 18.2, 4, 2 25.
struct FewRows {
  int tiles, waves;  // NT, W
};
FewRows few_rows_of(const Int4Args& a, int x_dtype) {
  const long tiles = small_tiles(a);
  if (tiles < 384) return {1, a.KB >= 32 && tiles <= 256 ? 16 : 8};
  // About one row block to an expert: no other workgroup reads its weights, and 32 columns a workgroup deal them out more evenly than 64 (111
  // of 408 drawn shapes: 0.93 of the time in the mean, 0.77 to 1.12).  The borders matter little: from 2048 to 4096 tiles and 16 to 48 blocks of
  // K the mean of 958 shapes moves by 0.3 %.  Not for fp32 rows, which every workgroup splits anew (24 shapes: 0.94 of the time with 64 columns).
  const bool alone = x_dtype != BRT_F32 && a.P <= 8l * a.E && (tiles <= 1024 || (tiles <= 4096 && a.KB < 24));
  if (tiles < 640 || a.KB < 4 || alone) return {2, a.KB >= 8 && tiles <= 1024 ? 8 : a.KB >= 4 ? 4 : 2};
  if (a.KB >= 8 && tiles <= 2048) return {4, 8};
  return {4, a.KB >= 16 || a.KB <= 4 || tiles <= 4096 ? 4 : 2};
}
template <int XDT, int GJ>
int launch_few_rows(Int4Args& a, hipStream_t st) {
  const FewRows by = few_rows_of(a, XDT);
  switch (by.tiles * 100 + by.waves) {
    case 116: return launch_few_rows<XDT, GJ, 1, 16>(a, st);
    case 108: return launch_few_rows<XDT, GJ, 1, 8>(a, st);
    case 208: return launch_few_rows<XDT, GJ, 2, 8>(a, st);
    case 204: return launch_few_rows<XDT, GJ, 2, 4>(a, st);
    case 202: return launch_few_rows<XDT, GJ, 2, 2>(a, st);
    case 408: return launch_few_rows<XDT, GJ, 4, 8>(a, st);
    case 404: return launch_few_rows<XDT, GJ, 4, 4>(a, st);
    default: return launch_few_rows<XDT, GJ, 4, 2>(a, st);
  }
}

// Row blocks of all experts (blocks of 1 << bits rows; at most `most`, which the host has made the grid for).
__device__ __forceinline__ int count_blocks(const Int4Args& a, int bits, int most) {
  const int lane = lane_id();
  int blocks = 0;
  for (int base = 0; base < a.E; base += kWave) {
    const int given = a.loads[min(base + lane, a.E - 1)];
    const int m = base + lane < a.E ? min(max(given, 0), a.P) : 0;
    blocks = min(blocks + read_lane(wave_inclusive_scan((m + (1 << bits) - 1) >> bits), kWave - 1), most);
  }
  return blocks;
}

// Many rows per expert: tiles of 64 rows and 128 NT columns, eight wavefronts, 16 NT columns and all rows each: a weight is unpacked once a
// workgroup, and not held in LDS.  Rows go straight into LDS, two blocks of 128 columns ahead, weights and scales into registers one block
// ahead.  The groups' sums of x are made for the block ahead by half of the wavefronts, 16 rows each, and pass through LDS;
// -scale * zero times them, for four groups at a time, is a product of its own in fp32 (v_mfma_f32_16x16x4_f32): the vector units, which
// unpack and scale beside the matrix units, have no part in it.
//   Two workgroups of 8 wavefronts fit a CU (125 registers, 66 KB), which hides the loads and the barrier: 64 x 256 tiles took four
// wavefronts of twice the columns 76 us where these take 65 (4096 rows of 32 experts 1024 -> 4096), and as long as them where the matrix
// units' power sets the time (16384 rows of 8 experts 4096 -> 4096, groups of 128: 575 us, 956 TFLOP/s; 612 on another card).  There the products alone take
// 357 us; without the unpacking and scaling the kernel takes as long as with them, without the loads 140 us less, without the sums and
// their product 46 less (groups of 64, of which there are twice as many: 667 us in all).
constexpr int kTileWaves = 8;
template <int XDT, int GJ, int NT>
__global__ __launch_bounds__(kTileWaves * 64, 2) void int4_tiles_kernel(Int4Args a) {
  using Part = RowPart<XDT>;
  using W = decltype(weights_of<XDT>(0));
  static_assert(elem_bytes(XDT) == 2, "a chunk of 16 bytes is a lane's part of a fragment");
  constexpr int MT = 4, BM = 16 * MT, kGroups = 4 / GJ, kStages = 3;
  constexpr int kBits = 6;  // log2 of BM
  constexpr int kRow = kB * elem_bytes(XDT), kChunks = kRow / 16, kRowsOfLoad = 64 / kChunks;  // of a row in LDS; rows of a load
  constexpr int XL = BM / kRowsOfLoad / kTileWaves;  // loads of a wavefront and block
  constexpr int kStage = BM * kRow;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // of the last eight groups: the rows' sums, and a wavefront's scales and their products with the zero points
  float* const s_sums = reinterpret_cast<float*>(smem + kStages * kStage);  // [8][BM]
  float* const s_scales = s_sums + 8 * BM + (threadIdx.x >> 6) * (2 * 8 * 16 * NT);  // [8][16 NT]
  float* const s_zeros = s_scales + 8 * 16 * NT;                                      // [8][16 NT]
  const int lane = lane_id(), g = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Tiles are dealt out in runs, one per XCD: neighbours in the list, four row blocks wide, share rows and weights in its L2.
  const int blocks = count_blocks(a, kBits, a.blocks);
  const int tiles = blocks * a.tiles_n, run = (tiles + kXcds - 1) / kXcds;
  const int turn = blockIdx.x / kXcds, t = blockIdx.x % kXcds * run + turn;
  if (turn >= run || t >= tiles) return;
  constexpr int kPatch = 4;
  const int patch = t / (kPatch * a.tiles_n), in = t - patch * kPatch * a.tiles_n, wide = min(kPatch, blocks - patch * kPatch);
  const Block found = find_block(a, patch * kPatch + in % wide, kBits);
  if (found.rows == 0) return;
  const int e = __builtin_amdgcn_readfirstlane(found.e), row0 = __builtin_amdgcn_readfirstlane(found.row0), rows = __builtin_amdgcn_readfirstlane(found.rows);
  const int tile0 = in / wide * (kTileWaves * NT) + wave * NT;

  // Slot s of LDS row r holds chunk s ^ (r & 15) of that row: the 16 rows that are read together at one chunk cover all banks.
  const uint32_t row_bytes = static_cast<uint32_t>(a.K) * elem_bytes(XDT);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem)));
  i32x4 rx;
  if (a.entries != nullptr) rx = make_rsrc(a.x, static_cast<size_t>(a.T) * row_bytes);
  else rx = make_rsrc(static_cast<const char*>(a.x) + static_cast<size_t>(row0) * row_bytes, static_cast<size_t>(rows) * row_bytes);
  uint32_t from[XL], chunk_at[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int r = (wave * XL + i) * kRowsOfLoad + lane / kChunks;
    chunk_at[i] = ((lane % kChunks) ^ (r & 15)) * 16;
    from[i] = kNowhere;
    if (r < rows) {
      if (a.entries == nullptr) {
        from[i] = r * row_bytes + chunk_at[i];
      } else {
        const int word = a.entries[row0 + r], cell = a.per_cell > 1 ? (word - 1) / a.per_cell : word - 1;
        if (word >= 1 && cell < a.T) from[i] = cell * row_bytes + chunk_at[i];
      }
    }
  }
  auto request = [&](int kb, int stage) {
    const uint32_t to = lds0 + stage, start = kb * kRow;
    if (start + kRow <= row_bytes) {
#pragma unroll
      for (int i = 0; i < XL; ++i) load_to_lds(rx, from[i], start, to + (wave * XL + i) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < XL; ++i) load_to_lds(rx, start + chunk_at[i] >= row_bytes ? kNowhere : from[i], start, to + (wave * XL + i) * 1024);
    }
  };
  struct Loaded {
    u32x4 w[NT];
    uint32_t s[kGroups];  // of the wavefront's column `lane`
    uint8_t z[kGroups];
  };
  // (tiles behind the last hold what that one does; groups behind the last, whose rows are zeros, a scale of zero)
  const size_t first = static_cast<size_t>(e) * a.tiles + min(tile0, a.tiles - 1);
  const int left = a.tiles - 1 - min(tile0, a.tiles - 1);
  const uint8_t* const w0 = a.w + first * a.KB * 1024;
  const int s_bytes = a.s_dtype == BRT_F32 ? 4 : 2;
  const uint32_t s_place = min(g % NT, left) * a.G * 16 + c16;  // (lane l has column l % (16 NT))
  const int s_extent = (min(NT - 1, left) + 1) * a.G * 16;
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(a.scales)) + first * a.G * 16 * s_bytes, 0, s_extent * s_bytes, 0x00020000);
  // (without zero points: nothing is in reach, which reads as zeros)
  const __amdgpu_buffer_rsrc_t rz = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.zeros) + first * a.G * 16, 0, a.zeros != nullptr ? s_extent : 0, 0x00020000);
  const float z_least = a.zeros != nullptr ? 0.0f : 8.0f;
  auto load = [&](int kb, Loaded& to) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
      to.w[j] = *reinterpret_cast<const u32x4*>(w0 + (static_cast<size_t>(min(j, left)) * a.KB + kb) * 1024 + static_cast<uint32_t>(lane * 16));
    uint32_t place[kGroups];
#pragma unroll
    for (int h = 0; h < kGroups; ++h) place[h] = kb * kGroups + h < a.G ? s_place : kNowhere / 4;
    if (a.s_dtype == BRT_F32) {
#pragma unroll
      for (int h = 0; h < kGroups; ++h) to.s[h] = __builtin_amdgcn_raw_buffer_load_b32(rs, place[h] * 4, (kb * kGroups + h) * 64, 0);
    } else {
#pragma unroll
      for (int h = 0; h < kGroups; ++h) to.s[h] = __builtin_amdgcn_raw_buffer_load_b16(rs, place[h] * 2, (kb * kGroups + h) * 32, 0);
    }
#pragma unroll
    for (int h = 0; h < kGroups; ++h) to.z[h] = __builtin_amdgcn_raw_buffer_load_b8(rz, a.zeros != nullptr ? place[h] : kNowhere, (kb * kGroups + h) * 16, 0);
  };
  auto keep_scales = [&](int kb, const Loaded& of) {
    float s[kGroups];
    scales_of(of.s, a.s_dtype, s);
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      const int at = ((kb * kGroups + h) & 7) * 16 * NT + lane % (16 * NT);
      s_scales[at] = s[h], s_zeros[at] = -(static_cast<float>(of.z[h]) + z_least) * s[h];
    }
  };
  // fragment p of 16 rows from row r0 of a stage
  uint32_t part_at[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) part_at[p] = c16 * kRow + ((p * 4 + g) ^ c16) * 16;
  auto part_of = [&](int stage, int r0, int p) { return Part(reinterpret_cast<const u32x4*>(smem + (part_at[p] + stage) + r0 * kRow)); };
  W one;
#pragma unroll
  for (int i = 0; i < 8; ++i) one[i] = kWeightUnit<XDT>;
  auto sum_up = [&](int kb, int stage) {
    if (wave >= MT) return;
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int p = 0; p < GJ; ++p) sum = multiply(one, part_of(stage, wave * 16, h * GJ + p), sum);
      s_sums[((kb * kGroups + h) & 7) * BM + wave * 16 + c16] = sum[0];  // (four lanes hold and write the same)
    }
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  Loaded now;
  request(0, 0);
  if (a.KB > 1) request(1, kStage);
  load(0, now);
  keep_scales(0, now);
  wait_loads_but<0>();
  __syncthreads();
  sum_up(0, 0);
  int stage = 0, stage1 = kStage, stage2 = 2 * kStage;  // of this block and the two after it
#pragma unroll 1
  for (int kb = 0; kb < a.KB; ++kb) {
    wait_loads_but<0>();
    __syncthreads();  // the block after this one has landed, its sums' place and the stage of the one before are free
    // groups four by four: their zero points come off when the last of them is at hand
    const int group = ((kb * kGroups) & ~3) + g;
    const bool correct = ((kb + 1) * kGroups & 3) == 0 || kb + 1 == a.KB;
    if (kb + 2 < a.KB) request(kb + 2, stage2);
    Loaded next;
    load(min(kb + 1, a.KB - 1), next);
    sum_up(kb + 1, stage1);  // (behind the last block: of what the stage holds, for a place that is not read)
    // fragment by fragment: the next one's weights are unpacked and its rows fetched beside this one's products
    W w[2][NT];
    Part x[2][MT] = {{part_of(stage, 0, 0), part_of(stage, 16, 0), part_of(stage, 32, 0), part_of(stage, 48, 0)}, {part_of(stage, 0, 1), part_of(stage, 16, 1), part_of(stage, 32, 1), part_of(stage, 48, 1)}};
    f32x4 part[MT][NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) w[0][j] = weights_of<XDT>(now.w[j][0]);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      if (p > 0 && p < 3) {
#pragma unroll
        for (int i = 0; i < MT; ++i) x[(p + 1) & 1][i] = part_of(stage, i * 16, p + 1);
      }
      if (p < 3) {
#pragma unroll
        for (int j = 0; j < NT; ++j) w[(p + 1) & 1][j] = weights_of<XDT>(now.w[j][p + 1]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[i][j] = multiply(w[p & 1][j], x[p & 1][i], p % GJ == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : part[i][j]);
      if (p % GJ == GJ - 1) {
        f32x4 s[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) s[j] = *reinterpret_cast<const f32x4*>(s_scales + ((kb * kGroups + p / GJ) & 7) * 16 * NT + j * 16 + g * 4);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][j][q] = __builtin_fmaf(part[i][j][q], s[j][q], acc[i][j][q]);
            asm volatile("" : "+v"(acc[i][j]));  // (left alone, the compiler puts the additions off, and the parts do not fit)
          }
      }
    }
    if (correct) {
      float off[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) off[j] = group < a.G ? s_zeros[(group & 7) * 16 * NT + j * 16 + c16] : 0.0f;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float sum = group < (kb + 1) * kGroups ? s_sums[(group & 7) * BM + i * 16 + c16] : 0.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(off[j], sum, acc[i][j], 0, 0, 0);
      }
    }
    now = next;
    keep_scales(kb + 1, now);
    const int free = stage;
    stage = stage1, stage1 = stage2, stage2 = free;
  }

  auto store = [&](auto act, auto out) {
    constexpr int ACT = decltype(act)::value, OUT = decltype(out)::value;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = (tile0 + j) * 16 + g * 4;
      float bias[4];
      biases<4>(a, e, min(n, a.N - 1), bias);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = activated_for<ACT, OUT>(__builtin_fmaf(acc[i][j][q], 1.0f / kWeightUnit<XDT>, bias[q]));
        if (i * 16 + c16 < rows && n < a.N) store_four<OUT>(a, static_cast<size_t>(row0) + i * 16 + c16, n, v);
      }
    }
  };
  auto with_act = [&](auto out) {
    if (a.act == BRT_ACT_GELU) store(std::integral_constant<int, BRT_ACT_GELU>{}, out);
    else if (a.act == BRT_ACT_RELU) store(std::integral_constant<int, BRT_ACT_RELU>{}, out);
    else store(std::integral_constant<int, BRT_ACT_NONE>{}, out);
  };
  if (a.out_dtype == BRT_F32) with_act(std::integral_constant<int, BRT_F32>{});
  else if (a.out_dtype == BRT_F16) with_act(std::integral_constant<int, BRT_F16>{});
  else with_act(std::integral_constant<int, BRT_BF16>{});
}

template <int XDT, int GJ, int NT>
int launch_tiles(Int4Args& a, hipStream_t st) {
  constexpr int BM = 64, kBytes = 3 * BM * kB * elem_bytes(XDT) + 8 * BM * 4 + kTileWaves * 2 * 8 * 16 * NT * 4;
  const auto fn = int4_tiles_kernel<XDT, GJ, NT>;
  a.tiles_n = (a.tiles + kTileWaves * NT - 1) / (kTileWaves * NT);
  // an expert adds at most one row block that it does not fill
  const long blocks = static_cast<long>(a.P) / BM + std::min(a.E, a.P), grid = (blocks * a.tiles_n + kXcds - 1) / kXcds * kXcds;
  if (grid * (kTileWaves * 64) >= kMostThreads) return fail(BRT_E_UNSUPPORTED, "too many tiles");
  a.blocks = static_cast<int>(blocks);
  if (const int rc = allow_dynamic_lds(reinterpret_cast<const void*>(fn), kBytes); rc != BRT_OK) return rc;
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(grid)), dim3(kTileWaves * 64), kBytes, st, a);
  return check_launch("int4_tiles_kernel");
}

// Which kernel takes 16-bit rows, by what each is estimated to take (us): few rows, or 64 x 128 and 64 x 256 tiles.  The first fetches the
// weights again for every 16 rows, 5300 tiles of 16 x 16 x 128 a microsecond with the chip full; the others take a time per block of 128
// columns, waiting for loads while there is a workgroup to a CU at most, multiplying beyond (us, groups of 128): 64 rows 4096 -> 4096
// 10 and 31 / 43; 600 rows of 2 experts 4096 -> 4096 56 and 45 / 45; 1024 rows of 16 1024 -> 4096 33 and 25 / 24; 8192 of 64 2048 -> 2048 211
// and 127 / 102.  (Over 400 shapes, 32 to 20000 rows of 1 to 64 experts, 512 to 8192 -> 256 to 8192, the choice takes 0.4 % longer in the mean than the
// best of the three, 1.29 times at worst: 281 rows of 16 1024 -> 5120.)
enum RowsKind { kFewRows = 16, kTiles128 = 128, kTiles256 = 256 };
RowsKind rows_kind(const Int4Args& a, int group, int x_dtype) {
  if (x_dtype == BRT_F32) return kFewRows;  // (the tiles would split them again in every wavefront: 4096 rows of 64 experts 2048 -> 2048 197 us, 283)
  // (the tiles address 64 rows, or all cells, in 31 bits)
  const long row = static_cast<long>(a.K) * elem_bytes(x_dtype), reach = std::max(64l, a.entries != nullptr ? a.T : 0l) * row;
  if (reach >= (1l << 31) - (1 << 16) || (a.entries != nullptr && a.T == 0)) return kFewRows;
  const double used = std::min(a.E, a.P), blocks = std::max(used, a.P / 64.0 + used / 2);
  const double by_group = group == 32 ? 1.25 : group == 64 ? 1.1 : 1.0;
  double least = 2.5 + static_cast<double>(small_tiles(a)) * a.KB / 5300;
  RowsKind kind = kFewRows;
  auto consider = [&](RowsKind of, int columns, double alone, double full) {
    const double rounds = blocks * ((a.N + columns - 1) / columns) / (kXcds * kCusPerXcd);
    const double time = 2.0 + a.KB * by_group * std::max(alone, full * rounds);
    if (time < least) least = time, kind = of;
  };
  consider(kTiles128, 128, 0.87, 0.69);
  consider(kTiles256, 256, 1.36, 1.15);
  return kind;
}

template <int XDT, int GJ>
int launch(Int4Args& a, hipStream_t st) {
  if constexpr (XDT != BRT_F32) {
    switch (rows_kind(a, 32 * GJ, XDT)) {
      case kTiles128: return launch_tiles<XDT, GJ, 1>(a, st);
      case kTiles256: return launch_tiles<XDT, GJ, 2>(a, st);
      default: break;
    }
  }
  return launch_few_rows<XDT, GJ>(a, st);
}
template <int XDT>
int launch(Int4Args& a, int group, hipStream_t st) {
  if (group == 32) return launch<XDT, 1>(a, st);
  if (group == 64) return launch<XDT, 2>(a, st);
  return launch<XDT, 4>(a, st);
}

bool is_type(int dtype) { return dtype == BRT_F32 || dtype == BRT_F16 || dtype == BRT_BF16; }

}  // namespace
}  // namespace brt

using namespace brt;

extern "C" int brt_hip_grouped_gemm_int4_kernel(int x_dtype, int T, int group, int E, int P, int N, int K) {
  if (!is_type(x_dtype) || (group != 32 && group != 64 && group != 128) || E <= 0 || P <= 0 || N <= 0 || K <= 0) return BRT_E_INVALID;
  Int4Args a{};
  static const int kRoutes = 0;
  a.entries = T >= 0 ? &kRoutes : nullptr;  // (whether there are any is all that is asked)
  a.T = T; a.E = E; a.P = P; a.N = N; a.K = K; a.KB = (K + kB - 1) / kB; a.tiles = (N + 15) / 16;
  return rows_kind(a, group, x_dtype);
}

extern "C" int brt_hip_grouped_gemm_int4_few_rows(int x_dtype, int E, int P, int N, int K) {
  if (!is_type(x_dtype) || E <= 0 || P <= 0 || N <= 0 || K <= 0) return BRT_E_INVALID;
  Int4Args a{};
  a.E = E; a.P = P; a.N = N; a.K = K; a.KB = (K + kB - 1) / kB; a.tiles = (N + 15) / 16;
  const FewRows by = few_rows_of(a, x_dtype);
  return by.tiles * 100 + by.waves;
}

extern "C" int brt_hip_grouped_gemm_int4(const void* x, int x_dtype, const int32_t* row_entries, int entries_per_cell, int T,
                                         const void* w, const void* scales, int scale_dtype, const uint8_t* zeros, int group,
                                         const int32_t* loads, const void* bias, int bias_dtype, void* out, int out_dtype, int E, int P,
                                         int N, int K, int activation, void* stream) {
  if (E <= 0 || P < 0 || N < 0 || K < 0) return fail(BRT_E_INVALID, "bad shape E=%d P=%d N=%d K=%d", E, P, N, K);
  if (group != 32 && group != 64 && group != 128) return fail(BRT_E_UNSUPPORTED, "groups of %d elements", group);
  if (!is_type(x_dtype) || !is_type(out_dtype) || !is_type(scale_dtype) || (bias && !is_type(bias_dtype)))
    return fail(BRT_E_UNSUPPORTED, "dtypes %d, %d, %d, %d are not supported", x_dtype, out_dtype, scale_dtype, bias_dtype);
  if (activation != BRT_ACT_NONE && activation != BRT_ACT_GELU && activation != BRT_ACT_RELU)
    return fail(BRT_E_UNSUPPORTED, "activation %d is not supported", activation);
  if (row_entries && (entries_per_cell < 1 || T < 0)) return fail(BRT_E_INVALID, "bad shape k=%d T=%d", entries_per_cell, T);
  if (P == 0 || N == 0) return BRT_OK;
  if (K == 0) return fail(BRT_E_UNSUPPORTED, "rows of no elements");
  if ((!x && !(row_entries && T == 0)) || !w || !scales || !loads || !out) return fail(BRT_E_INVALID, "null argument");
  if (K % 8 != 0 || !aligned(x, 16) || (static_cast<long>(K) * elem_bytes(x_dtype)) % 16 != 0)
    return fail(BRT_E_UNSUPPORTED, "rows must be whole, aligned units of 8 elements (K=%d)", K);
  if (!aligned(w, 16) || !aligned(scales, 16) || !aligned(zeros, 4)) return fail(BRT_E_UNSUPPORTED, "weights and scales must be aligned to 16 bytes");
  if (P >= kMostRows) return fail(BRT_E_UNSUPPORTED, "more than %d rows", kMostRows - 1);
  if (E > kMostColumns || N > kMostColumns || K > kMostColumns) return fail(BRT_E_UNSUPPORTED, "more than %d columns, elements or experts", kMostColumns);
  Int4Args a{};
  a.x = x; a.entries = row_entries; a.per_cell = entries_per_cell; a.T = T; a.w = static_cast<const uint8_t*>(w);
  a.scales = scales; a.s_dtype = scale_dtype; a.zeros = zeros; a.loads = loads; a.bias = bias; a.bias_dtype = bias_dtype;
  a.out = out; a.out_dtype = out_dtype; a.act = activation;
  a.E = E; a.P = P; a.N = N; a.K = K; a.KB = (K + kB - 1) / kB; a.G = (K + group - 1) / group; a.tiles = (N + 15) / 16;
  hipStream_t st = as_stream(stream);
  if (x_dtype == BRT_F32) return launch<BRT_F32>(a, group, st);
  if (x_dtype == BRT_F16) return launch<BRT_F16>(a, group, st);
  return launch<BRT_BF16>(a, group, st);
}
