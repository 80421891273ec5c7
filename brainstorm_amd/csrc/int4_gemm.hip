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
// type; fp32 rows are split into three bf16 parts (8 bits each: all of them) and take three instructions.  A group's products are summed
// by the matrix unit on top of -z times its sum of x, which one more instruction with a constant fragment leaves in the
// result's layout, and the group's sum is scaled in fp32 by one multiply-add.  So nothing but the result is rounded below fp32.
//   The weight fragment is the first operand: a lane holds results of one row and four neighbouring columns.
#include <algorithm>
#include <type_traits>

#include "packed_rows.hpp"

namespace brt {
namespace {

constexpr int kB = 128;              // columns of a block of the weights' layout
constexpr int kMostRows = 1 << 24;   // 65 times as many are added up in 32 bits
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

// Eight weights of a word, as the numbers 0 .. 15: the low halves of its bytes are elements 0 .. 3, the high ones 4 .. 7.
template <int XDT>
__device__ __forceinline__ auto weights_of(uint32_t word) {
  const int lo = static_cast<int>(word & 0x0f0f0f0fu), hi = static_cast<int>((word >> 4) & 0x0f0f0f0fu);
  if constexpr (XDT == BRT_F16) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  } else {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true);
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

// Four values of the layout's 16 columns of a group.
struct Four {
  u32x4 raw;
};
__device__ __forceinline__ Four load_four(const void* base, int dtype, size_t at) {
  Four f{};
  if (dtype == BRT_F32) {
    f.raw = *reinterpret_cast<const u32x4*>(static_cast<const float*>(base) + at);
  } else {
    const u32x2 half = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(base) + at);
    f.raw[0] = half[0], f.raw[1] = half[1];
  }
  return f;
}
__device__ __forceinline__ f32x4 values_of(const Four& f, int dtype) {
  f32x4 v;
  if (dtype == BRT_F32) {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = __uint_as_float(f.raw[q]);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t h = q % 2 ? f.raw[q / 2] >> 16 : f.raw[q / 2] & 0xffffu;
      v[q] = dtype == BRT_F16 ? f16_to_float(h) : bf16_to_float(h);
    }
  }
  return v;
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

// Few rows per expert: the weights are streamed once and set the time.  A workgroup takes 16 NT columns and 16 MT rows; its W
// wavefronts take blocks of 128 columns in turn, weights and rows straight into the fragments' registers, the next block's requested
// while this one is multiplied, and add up their sums through LDS.
template <int XDT, int GJ, int MT, int NT, int W>
__global__ __launch_bounds__(W * 64) void int4_few_rows_kernel(Int4Args a) {
  using Part = RowPart<XDT>;
  constexpr int kGroups = 4 / GJ;  // of a block; GJ fragments share a group
  constexpr int kBits = MT == 1 ? 4 : MT == 2 ? 5 : 6;
  __shared__ f32x4 s_part[W][NT * MT][64];
  const int lane = lane_id(), g = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int block = blockIdx.x / a.tiles_n, tile0 = (blockIdx.x - block * a.tiles_n) * NT, n0 = tile0 * 16;
  const Block at = find_block(a, block, kBits);
  if (at.rows == 0) return;
  const char* row[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) row[i] = row_of<XDT>(a, at.row0 + min(i * 16 + c16, at.rows - 1));
  // the biases of the tiles that this wavefront finishes: fetched ahead of the weights, not behind the last barrier
  constexpr int kFinished = (MT * NT + W - 1) / W;
  float bias[kFinished][4];
#pragma unroll
  for (int f = 0; f < kFinished; ++f) biases<4>(a, at.e, n0 + (wave + f * W) % NT * 16 + g * 4, bias[f]);

  struct Loaded {
    u32x4 w[NT], x[MT][4 * Part::kUnits];
    Four s[NT][kGroups];
    uint32_t z[NT][kGroups];
  };
  auto load = [&](int kb, Loaded& to) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const size_t tile = static_cast<size_t>(at.e) * a.tiles + min(tile0 + j, a.tiles - 1);
      to.w[j] = *reinterpret_cast<const u32x4*>(a.w + (tile * a.KB + kb) * 1024 + lane * 16);
#pragma unroll
      for (int h = 0; h < kGroups; ++h) {
        const size_t four = (tile * a.G + min(kb * kGroups + h, a.G - 1)) * 16 + g * 4;
        to.s[j][h] = load_four(a.scales, a.s_dtype, four);
        to.z[j][h] = a.zeros != nullptr ? *reinterpret_cast<const uint32_t*>(a.zeros + four) : 0x08080808u;
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int l = 0; l < 4 * Part::kUnits; ++l) {
        const int k = kb * kB + l / Part::kUnits * 32 + g * 8;
        const bool there = k < a.K && row[i] != nullptr;  // (K is a multiple of 8)
        to.x[i][l] = zero_unit<16>();
        if (there) to.x[i][l] = *reinterpret_cast<const u32x4*>(row[i] + static_cast<size_t>(k) * elem_bytes(XDT) + l % Part::kUnits * 16);
      }
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  decltype(weights_of<XDT>(0)) minus_one;
#pragma unroll
  for (int i = 0; i < 8; ++i) minus_one[i] = -1.0f;

  Loaded now;
  if (wave < a.KB) load(wave, now);
  for (int kb = wave; kb < a.KB; kb += W) {
    Loaded next;
    if (kb + W < a.KB) load(kb + W, next);
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      decltype(weights_of<XDT>(0)) w[NT][GJ];
      f32x4 s[NT];
      float z[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        s[j] = values_of(now.s[j][h], a.s_dtype);
#pragma unroll
        for (int q = 0; q < 4; ++q) z[j][q] = static_cast<float>((now.z[j][h] >> (8 * q)) & 0xffu);
#pragma unroll
        for (int p = 0; p < GJ; ++p) w[j][p] = weights_of<XDT>(now.w[j][h * GJ + p]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f}, part[NT];  // sum: minus the row's sum over the group, in all four
#pragma unroll
        for (int p = 0; p < GJ; ++p) sum = multiply(minus_one, Part(&now.x[i][(h * GJ + p) * Part::kUnits]), sum);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) part[j][q] = z[j][q] * sum[q];
#pragma unroll
        for (int p = 0; p < GJ; ++p) {
          const Part x(&now.x[i][(h * GJ + p) * Part::kUnits]);
#pragma unroll
          for (int j = 0; j < NT; ++j) part[j] = multiply(w[j][p], x, part[j]);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][j][q] = __builtin_fmaf(part[j][q], s[j][q], acc[i][j][q]);
      }
    }
    now = next;
  }

#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) s_part[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  const bool whole = a.N % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
#pragma unroll
  for (int f = 0; f < kFinished; ++f) {
    const int p = wave + f * W;
    if (p >= MT * NT) break;
    f32x4 sum = s_part[0][p][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) sum += s_part[w][p][lane];
    const int r = p / NT * 16 + c16, n = n0 + p % NT * 16 + g * 4;
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = activated_for(sum[q] + bias[f][q], a.act, a.out_dtype);
    if (r < at.rows && n < a.N) store_part<4>(a, static_cast<size_t>(at.row0) + r, n, whole, v);
  }
}

template <int XDT, int GJ, int MT, int NT, int W>
int launch_few_rows(Int4Args& a, hipStream_t st) {
  constexpr int kRows = 16 * MT;
  const long blocks = static_cast<long>(a.P) / kRows + std::min(a.E, a.P);
  a.tiles_n = (a.tiles + NT - 1) / NT;
  if (blocks * a.tiles_n >= (1l << 31)) return fail(BRT_E_UNSUPPORTED, "too many tiles");
  hipLaunchKernelGGL((int4_few_rows_kernel<XDT, GJ, MT, NT, W>), dim3(static_cast<unsigned>(blocks * a.tiles_n)), dim3(W * 64), 0, st, a);
  return check_launch("int4_few_rows_kernel");
}
template <int XDT, int GJ>
int launch_few_rows(Int4Args& a, hipStream_t st) {
  const long tiles = static_cast<long>(std::min(a.E, a.P)) * a.tiles;
  if constexpr (XDT != BRT_F32)
    if (a.P > 16 && a.P > 10l * a.E) return launch_few_rows<XDT, GJ, 2, 2, 8>(a, st);
  if (tiles < 512) return launch_few_rows<XDT, GJ, 1, 1, 8>(a, st);
  return launch_few_rows<XDT, GJ, 1, 2, 8>(a, st);
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

// Many rows per expert: 64 x 256 tiles, four wavefronts, 64 columns and all rows each: a weight is unpacked once a workgroup, and not held in
// LDS.  Rows go straight into LDS, two blocks of 128 columns ahead, weights and scales into registers one block ahead.  The groups'
// sums of x are made for the block ahead by a quarter of its rows a wavefront, and pass through LDS; -scale * zero times them, for four
// groups at a time, is a product of its own in fp32 (v_mfma_f32_16x16x4_f32): the vector units, which unpack and scale beside the matrix
// units, have no part in it.
template <int XDT, int GJ>
__global__ __launch_bounds__(256, XDT == BRT_F32 ? 1 : 2) void int4_tiles_kernel(Int4Args a) {
  using Part = RowPart<XDT>;
  using W = decltype(weights_of<XDT>(0));
  constexpr int MT = 4, BM = 16 * MT, NT = 4, kGroups = 4 / GJ, kStages = 3;
  constexpr int kBits = 6;
  constexpr int kRow = kB * elem_bytes(XDT), kChunks = kRow / 16, kRowsOfLoad = 64 / kChunks;  // of a row in LDS; rows of a load
  constexpr int XL = BM / kRowsOfLoad / 4;  // loads of a wavefront and block
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
  const int tile0 = in / wide * 16 + wave * NT;

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
  auto request = [&](int kb) {
    const uint32_t to = lds0 + kb % kStages * kStage, start = kb * kRow;
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
    uint32_t s[kGroups], z[kGroups];  // of the wavefront's column `lane`
  };
  auto load = [&](int kb, Loaded& to) {
    const size_t first = static_cast<size_t>(e) * a.tiles;
#pragma unroll
    for (int j = 0; j < NT; ++j)
      to.w[j] = *reinterpret_cast<const u32x4*>(a.w + ((first + min(tile0 + j, a.tiles - 1)) * a.KB + kb) * 1024 + lane * 16);
    size_t one[kGroups];
#pragma unroll
    for (int h = 0; h < kGroups; ++h)
      one[h] = ((first + min(tile0 + g, a.tiles - 1)) * a.G + min(kb * kGroups + h, a.G - 1)) * 16 + c16;
    if (a.s_dtype == BRT_F32) {
#pragma unroll
      for (int h = 0; h < kGroups; ++h) to.s[h] = static_cast<const uint32_t*>(a.scales)[one[h]];
    } else {
#pragma unroll
      for (int h = 0; h < kGroups; ++h) to.s[h] = static_cast<const uint16_t*>(a.scales)[one[h]];
    }
#pragma unroll
    for (int h = 0; h < kGroups; ++h) to.z[h] = 8;
    if (a.zeros != nullptr) {
#pragma unroll
      for (int h = 0; h < kGroups; ++h) to.z[h] = a.zeros[one[h]];
    }
  };
  auto keep_scales = [&](int kb, const Loaded& of) {
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      const int at = (kb * kGroups + h & 7) * 16 * NT + lane;
      const float s = a.s_dtype == BRT_F32 ? __uint_as_float(of.s[h]) : a.s_dtype == BRT_F16 ? f16_to_float(of.s[h]) : bf16_to_float(of.s[h]);
      s_scales[at] = s, s_zeros[at] = -static_cast<float>(of.z[h]) * s;
    }
  };
  // fragment p of a block, of 16 rows from row r0
  auto part_of = [&](int kb, int r0, int p) {
    const char* const row = smem + kb % kStages * kStage + (r0 + c16) * kRow;
    u32x4 raw[Part::kUnits];
#pragma unroll
    for (int u = 0; u < Part::kUnits; ++u) raw[u] = *reinterpret_cast<const u32x4*>(row + ((((p * 4 + g) * Part::kUnits + u) ^ c16) * 16));
    return Part(raw);
  };
  W one;
#pragma unroll
  for (int i = 0; i < 8; ++i) one[i] = 1.0f;
  auto sum_up = [&](int kb) {
    const int r0 = wave * (BM / 4);
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int p = 0; p < GJ; ++p) sum = multiply(one, part_of(kb, r0, h * GJ + p), sum);
      if (g == 0) s_sums[((kb * kGroups + h) & 7) * BM + r0 + c16] = sum[0];
    }
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  Loaded now;
  request(0);
  if (a.KB > 1) request(1);
  load(0, now);
  keep_scales(0, now);
  wait_loads_but<0>();
  __syncthreads();
  sum_up(0);
#pragma unroll 1
  for (int kb = 0; kb < a.KB; ++kb) {
    wait_loads_but<0>();
    __syncthreads();  // the block after this one has landed, its sums' place and the stage of the one before are free
    // groups four by four: their zero points come off when the last of them is at hand
    const int group = (kb * kGroups & ~3) + g;
    const bool correct = ((kb + 1) * kGroups & 3) == 0 || kb + 1 == a.KB;
    if (kb + 2 < a.KB) request(kb + 2);
    Loaded next;
    if (kb + 1 < a.KB) {
      load(kb + 1, next);
      sum_up(kb + 1);
    }
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      W w[NT][GJ];
      f32x4 s[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        s[j] = *reinterpret_cast<const f32x4*>(s_scales + (kb * kGroups + h & 7) * 16 * NT + j * 16 + g * 4);
#pragma unroll
        for (int p = 0; p < GJ; ++p) w[j][p] = weights_of<XDT>(now.w[j][h * GJ + p]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        f32x4 part[NT];
#pragma unroll
        for (int p = 0; p < GJ; ++p) {
          const Part x = part_of(kb, i * 16, h * GJ + p);
#pragma unroll
          for (int j = 0; j < NT; ++j) part[j] = multiply(w[j][p], x, p == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : part[j]);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][j][q] = __builtin_fmaf(part[j][q], s[j][q], acc[i][j][q]);
      }
      // (the sums are complete here: left alone, the compiler puts off the additions of all groups, whose parts do not fit)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) asm volatile("" : "+v"(acc[i][j]));
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
    if (kb + 1 < a.KB) keep_scales(kb + 1, now);
  }

  const bool whole = a.N % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
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
        for (int q = 0; q < 4; ++q) v[q] = activated_for<ACT, OUT>(acc[i][j][q] + bias[q]);
        char* const to = static_cast<char*>(a.out) + ((static_cast<size_t>(row0) + i * 16 + c16) * a.N + n) * elem_bytes(OUT);
        if (i * 16 + c16 >= rows || n >= a.N) continue;
        if (whole) {
          pack_store<OUT, 4>(to, v);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float one[1] = {v[q]};
            if (n + q < a.N) pack_store<OUT, 1>(to + q * elem_bytes(OUT), one);
          }
        }
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

template <int XDT, int GJ>
int launch_tiles(Int4Args& a, hipStream_t st) {
  constexpr int BM = 64, kBytes = 3 * BM * kB * elem_bytes(XDT) + 8 * BM * 4 + 4 * 2 * 8 * 64 * 4;
  const auto fn = int4_tiles_kernel<XDT, GJ>;
  if (const int rc = allow_dynamic_lds(reinterpret_cast<const void*>(fn), kBytes); rc != BRT_OK) return rc;
  a.tiles_n = (a.tiles + 15) / 16;
  // an expert adds at most one row block that it does not fill
  const long blocks = static_cast<long>(a.P) / BM + std::min(a.E, a.P);
  if (blocks * a.tiles_n >= (1l << 31) - kXcds) return fail(BRT_E_UNSUPPORTED, "too many tiles");
  a.blocks = static_cast<int>(blocks);
  const long grid = (blocks * a.tiles_n + kXcds - 1) / kXcds * kXcds;
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(grid)), dim3(256), kBytes, st, a);
  return check_launch("int4_tiles_kernel");
}

bool few_rows(const Int4Args& a, int x_dtype) {
  // (the tiles address 64 rows, or all cells, in 31 bits)
  const long row = static_cast<long>(a.K) * elem_bytes(x_dtype), reach = a.entries != nullptr ? a.T * row : 64 * row;
  if (reach >= (1l << 31) - (1 << 16) || (a.entries != nullptr && a.T == 0)) return true;
  return a.P <= 16 || a.P <= 16l * a.E;
}
template <int XDT, int GJ>
int launch(Int4Args& a, hipStream_t st) {
  if (few_rows(a, XDT)) return launch_few_rows<XDT, GJ>(a, st);
  return launch_tiles<XDT, GJ>(a, st);
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
