// Expert products in 8-bit floating point (OCP e4m3) with one fp32 scale per block of 128: no counterpart in the reference.
//
//   out[r, n] = act( sum_kb sx[r, kb] * sw[e, n / 128, kb] * (sum over the 128 k of block kb of xq[r, k] * wq[e, n, k]) + bias[e, n] )
//
// for the rows r of expert e (rows are packed by expert, their counts read from the device).  Rows are scaled per 1 x 128,
// weights per 128 x 128.  One v_mfma_f32_16x16x128_f8f6f4 sums exactly one block of K: it is issued with a zero addend, and
// its 4 results per lane are scaled into the fp32 accumulator by one multiply-add each.  The weight fragment is the first
// operand, so that a lane holds results of ONE row: the scale of a row tile is one register, sx * sw.
//
// The 8-bit matrix instructions align the products that they add at once (at most 16) to the largest and drop what lies more than
// 13 bits below it; between such groups they add in fp32.  On normal data a block's sum is off by 1.3e-5 of the result's norm: a
// hundredth of a bf16 rounding, a sixteenth of an fp16 one (behind a second quantization and product, whose rows it turns at borders of
// e4m3, 1.66e-3 of a bf16 result's norm become 1.96e-3).  An fp32 result would show it, so there, unless asked otherwise,
// the operands are widened to bf16 in registers (exactly) and multiplied by v_mfma_f32_16x16x32_bf16, off by 1.2e-8 (of fp32 rows,
// with their quantization: 48 of 8 experts 1024 -> 4096 10.2 us, 8-bit instruction 9.9; 8192 of 64 1024 -> 4096 130 and 101; 16384 of
// 8 4096 -> 4096 606 and 371).
#include <algorithm>
#include <type_traits>

#include "packed_rows.hpp"

namespace brt {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kB = 128;            // elements of a scale block, bytes of a K-step
constexpr float kMax = 448.0f;     // the largest e4m3 value
constexpr float kLeast = 0x1p-100f;  // blocks whose largest value is below this are scaled as if it were this
constexpr int kPatchRows = 4;
constexpr int kMostRows = 1 << 24;   // 65 times as many are added up in 32 bits
constexpr int kMostColumns = 1 << 30;  // and experts: rounded up to tiles they are counted in 32 bits
constexpr int kMostExperts = 512;  // whose row blocks a workgroup keeps in LDS

// ------------------------------------------------------------------------------------- quantization
// A block's largest magnitude as the bits of its magnitude (integers order them, NaN on top) -> its scale and the inverse.
__device__ __forceinline__ void scale_of(uint32_t top_bits, float* scale, float* inverse) {
  float top = __uint_as_float(top_bits);
  top = top_bits < __float_as_uint(kLeast) ? kLeast : top;  // (not fmaxf: NaN stays)
  *scale = top / kMax;
  *inverse = 1.0f / top * kMax;
}
__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }
// four values as e4m3, round to nearest even
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// rows [P, K] -> q [P, pitch] (zeros behind K) and scales [KB][P].  Eight lanes a block, 16 elements a lane, so a wavefront
// reads 8 rows of one block: 256-byte pieces of 16-bit rows, and writes 8 scales that lie side by side.  Bound by memory: 16384 x 4096
// bf16 33 us (203 MB, 6.2 TB/s), 8192 x 1024 6.9.
template <int DT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const void* __restrict__ x, uint8_t* __restrict__ q,
                                                            float* __restrict__ scales, int P, int K, int pitch, int KB) {
  constexpr int NE = 16 / elem_bytes(DT), NU = 16 / NE;
  const int lane = lane_id();
  const long wave = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int kb = static_cast<int>(wave % KB);
  const long row = wave / KB * 8 + (lane >> 3);
  if (row >= P) return;
  const int k = kb * kB + (lane & 7) * 16;
  float v[16];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    float part[NE];
    u32x4 w = zero_unit<16>();
    if (k < K) w = *(reinterpret_cast<const u32x4*>(static_cast<const char*>(x) + (row * K + k) * elem_bytes(DT)) + u);
    unpack<DT, 16>(w, part);
#pragma unroll
    for (int i = 0; i < NE; ++i) v[u * NE + i] = part[i];
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, magnitude(v[i]));
  top = static_cast<uint32_t>(segment_all_reduce(static_cast<int>(top), 8, [](int a, int b) { return max(a, b); }));
  float scale, inverse;
  scale_of(top, &scale, &inverse);
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pack4(v[4 * i] * inverse, v[4 * i + 1] * inverse, v[4 * i + 2] * inverse, v[4 * i + 3] * inverse);
  *reinterpret_cast<u32x4*>(q + row * pitch + k) = o;
  if ((lane & 7) == 0) scales[static_cast<size_t>(kb) * P + row] = scale;
}

// ------------------------------------------------------------------------------------------ products
struct Fp8Args {
  const void* x;       // e4m3 rows of `pitch` bytes (few-rows kernel: also rows of x_dtype that it quantizes itself)
  const float* sx;     // [KB][P]
  const uint8_t* w;    // [E, N, K]
  const float* sw;     // [E, NB, KB]
  const int* loads;    // [E]
  const void* bias;    // [E, N] of bias_dtype or null
  void* out;           // [P, N] of out_dtype, or with out_scales e4m3 [P, NB * 128]
  float* out_scales;   // [NB][P] or null
  int pitch, bias_dtype, out_dtype, act, exact;
  int E, P, N, K, KB, NB, tiles_n;
};

__device__ __forceinline__ f32x4 multiply(const i32x8& w, const i32x8& x) {
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, zero, 0, 0, 0, 0, 0, 0);
}

// The same from bf16 instructions: 8 bytes of both fragments at a time, widened exactly.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ bf16x8 widened(int lo, int hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
struct Wide {
  bf16x8 part[4];
};
__device__ __forceinline__ Wide widened(const i32x8& v) {
  return {widened(v[0], v[1]), widened(v[2], v[3]), widened(v[4], v[5]), widened(v[6], v[7])};
}
__device__ __forceinline__ f32x4 multiply(const Wide& w, const Wide& x) {
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int p = 0; p < 4; ++p) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.part[p], x.part[p], sum, 0, 0, 0);
  return sum;
}
template <bool EXACT>
__device__ __forceinline__ auto operand(const i32x8& v) {
  if constexpr (EXACT) return widened(v);
  else return v;
}

// The products of a K-step on their way into the accumulators: while one is on the matrix pipe, the one three before it is scaled
// and added (two before it: 16384 rows of 8 experts 4096 -> 4096 276 us, three 265, four to six the same).  What is left of a K-step
// is added while the next one's fragments come, with its scales still.  (sched_barrier keeps the order: left alone the compiler puts
// each addition behind its product and waits for it.)
template <int MT, int NT>
struct Pipe {
  static constexpr int kBehind = 3;
  f32x4 held[kBehind + 1];
  __device__ __forceinline__ Pipe() { clear(); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int p = 0; p <= kBehind; ++p) held[p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  __device__ __forceinline__ void add(int p, f32x4 (&acc)[MT][NT], const float (&s)[MT]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[p % MT][p / MT][q] = __builtin_fmaf(held[p % (kBehind + 1)][q], s[p % MT], acc[p % MT][p / MT][q]);
  }
  __device__ __forceinline__ void put(int p, const f32x4& product, f32x4 (&acc)[MT][NT], const float (&s)[MT]) {
    held[p % (kBehind + 1)] = product;
    if (p >= kBehind) add(p - kBehind, acc, s);
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ void drain(f32x4 (&acc)[MT][NT], const float (&s)[MT]) {
#pragma unroll
    for (int p = MT * NT - kBehind; p < MT * NT; ++p) add(p, acc, s);
  }
};

// Results of one row as they are stored: biased, activated, rounded.
template <int ACT, int OUT>
__device__ __forceinline__ void finish8(const Fp8Args& a, size_t row, int n, bool whole, const float (&bias)[8], float (&v)[8]) {
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = activated<ACT>(v[q] + bias[q]);
  const size_t at = row * a.N + n;
  char* const to = static_cast<char*>(a.out) + at * elem_bytes(OUT);
  if (whole) {
    // (streaming stores: 16384 rows of 8 experts 4096 -> 4096 bf16 292 -> 274 us; fp32 results of 16384 rows 1024 -> 2048 69 -> 75)
    pack_store<OUT, 8, OUT != BRT_F32>(to, v);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (n + q < a.N) {
        const float one[1] = {v[q]};
        pack_store<OUT, 1>(to + q * elem_bytes(OUT), one);
      }
  }
}

// The results of a wavefront: MT x NT tiles from row r0 of the block and column n0, tile columns as the kernels below deal them.
template <int MT, int NT, bool EXACT>
__device__ __forceinline__ void store_tile(const Fp8Args& a, const Block& at, int r0, int n0, f32x4 (&acc)[MT][NT]) {
  const int lane = lane_id(), g = lane >> 4, c16 = lane & 15;
  const bool whole = a.N % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  auto store = [&](auto act, auto out) {
#pragma unroll
    for (int j = 0; j < NT; j += 2) {
      const int n = n0 + (j >> 2) * 64 + ((j >> 1) & 1) * 32 + g * 8;
      float bias[8];
      biases<8>(a, at.e, n, bias);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int r = r0 + i * 16 + c16;
        float v[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = acc[i][j][q], v[4 + q] = acc[i][j + 1][q];
        if (r < at.rows && n < a.N)
          finish8<decltype(act)::value, decltype(out)::value>(a, static_cast<size_t>(at.row0) + r, n, whole, bias, v);
      }
    }
  };
  auto with_act = [&](auto out) {
    if (a.act == BRT_ACT_GELU) store(std::integral_constant<int, BRT_ACT_GELU>{}, out);
    else if (a.act == BRT_ACT_RELU) store(std::integral_constant<int, BRT_ACT_RELU>{}, out);
    else store(std::integral_constant<int, BRT_ACT_NONE>{}, out);
  };
  if (EXACT || a.out_dtype == BRT_F32) with_act(std::integral_constant<int, BRT_F32>{});
  else if (a.out_dtype == BRT_F16) with_act(std::integral_constant<int, BRT_F16>{});
  else with_act(std::integral_constant<int, BRT_BF16>{});
}

// The same results rounded to bf16 and quantized: what quantize_rows makes of them, without their way through memory.  A scale
// block is the columns of one wavefront (NT = 8) or of two neighbours (NT = 4), which exchange their largest values through
// `exchange` ([WN][BM] words); every wavefront of the workgroup calls it.
template <int ACT, int MT, int NT, int BM, int WN>
__device__ __forceinline__ void store_blocks(const Fp8Args& a, const Block& at, int r0, int n0, int wn, uint32_t* exchange, f32x4 (&acc)[MT][NT]) {
  static_assert(NT == 8 || (NT == 4 && WN % 2 == 0), "a block of 128 columns belongs to one wavefront or two");
  const int lane = lane_id(), g = lane >> 4, c16 = lane & 15;
  uint32_t top[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) top[i] = 0;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = n0 + (j >> 2) * 64 + ((j >> 1) & 1) * 32 + g * 8 + (j & 1) * 4;
    float bias[4];
    biases<4>(a, at.e, min(n, a.N - 1), bias);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        // (columns behind the last are zero; the value is held as the bf16 it was rounded to)
        const float v = n + q < a.N ? bf16_to_float(float_to_bf16(activated<ACT>(acc[i][j][q] + bias[q]))) : 0.0f;
        acc[i][j][q] = v;
        top[i] = max(top[i], magnitude(v));
      }
    __builtin_amdgcn_sched_barrier(0);  // (the biases of all columns at once do not fit beside the accumulators)
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    top[i] = max(top[i], static_cast<uint32_t>(__shfl_xor(static_cast<int>(top[i]), 16, kWave)));
    top[i] = max(top[i], static_cast<uint32_t>(__shfl_xor(static_cast<int>(top[i]), 32, kWave)));
  }
  if constexpr (NT == 4) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
      if (g == 0) exchange[wn * BM + r0 + i * 16 + c16] = top[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i) top[i] = max(top[i], exchange[(wn ^ 1) * BM + r0 + i * 16 + c16]);
  }
  const int nb = n0 / kB;
  uint8_t* const out = static_cast<uint8_t*>(a.out);
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = r0 + i * 16 + c16;
    if (r >= at.rows || nb >= a.NB) continue;
    const size_t row = static_cast<size_t>(at.row0) + r;
    float scale, inverse;
    scale_of(top[i], &scale, &inverse);
    if (g == 0 && n0 % kB == 0) a.out_scales[static_cast<size_t>(nb) * a.P + row] = scale;
#pragma unroll
    for (int j = 0; j < NT; j += 2) {
      u32x2 o;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        o[h] = pack4(acc[i][j + h][0] * inverse, acc[i][j + h][1] * inverse, acc[i][j + h][2] * inverse, acc[i][j + h][3] * inverse);
      *reinterpret_cast<u32x2*>(out + row * (static_cast<size_t>(a.NB) * kB) + n0 + (j >> 2) * 64 + ((j >> 1) & 1) * 32 + g * 8) = o;
    }
  }
}

// BM x BN tiles, WM x WN wavefronts, STAGES K-steps of 128 bytes in LDS.  Operands and scales go straight into LDS; a K-step is
// requested STAGES - 1 steps before it is multiplied, into the stage that was read last.  A workgroup stays for several tiles, and
// its requests run on through their boundaries: a tile of 1024 elements has eight K-steps, and starting anew (which expert, the
// first K-step) took as long as half of them.  The list of row blocks is kept in LDS for that.
//
// Bound by the matrix pipe beside the additions and the requests: 16384 rows of 8 experts 4096 -> 4096 265 us by itself (2.07 PFLOP/s; the
// same instructions from registers alone 3.6, the requests cost 40 to 60 us of it), 276 behind the quantization, 309 into an fp32 result; by
// the weights' way from memory with fewer rows: 8192 of 64 experts 1024 -> 4096 with GELU 81 us, of which the weights' 268 MB are 52.
template <int BM_BITS, int BN, int WM, int WN, int STAGES, bool GO_ROUND, bool EXACT, bool BLOCKS>
__global__ __launch_bounds__(WM* WN * 64, 2) void fp8_tiles_kernel(Fp8Args a) {
  constexpr int BM = 1 << BM_BITS, WAVES = WM * WN;
  constexpr int MT = BM / WM / 16, NT = BN / WN / 16;  // 16 x 16 tiles of a wavefront
  constexpr int XL = BM / 8 / WAVES, WL = BN / 8 / WAVES;  // loads of a wavefront and K-step, 8 rows each
  constexpr int kLoads = XL + WL + 1;                      // ... and one of scales: of 64 rows, or of a wavefront's columns
  constexpr int kRowScales = (BM + BN) * kB, kColumnScales = kRowScales + BM * 4;
  constexpr int kStage = kColumnScales + WN * 256;
  static_assert(NT % 4 == 0 && XL >= 1 && WL >= 1 && kB % (BN / WN) == 0, "a wavefront's columns share a scale block");
  static_assert(BM >= 64 && WAVES >= BM / 64 + WN, "a wavefront fetches the scales of 64 rows or of its columns");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int* const s_blocks = reinterpret_cast<int*>(smem + STAGES * kStage);  // [E] row blocks up to an expert and its own
  int* const s_rows = s_blocks + a.E;                                    // [E] rows likewise
  uint32_t* const s_tops = reinterpret_cast<uint32_t*>(s_rows + a.E);    // [WN][BM], where results are quantized
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  if (wave == 0) {
    int carry_b = 0, carry_m = 0;
    for (int base = 0; base < a.E; base += kWave) {
      const int given = a.loads[min(base + lane, a.E - 1)];
      const int m = base + lane < a.E ? min(max(given, 0), a.P) : 0;  // (loads as in find_block; here no block is without rows)
      const int sum_m = carry_m + wave_inclusive_scan(m), incl_m = min(sum_m, a.P);
      const int incl_b = carry_b + wave_inclusive_scan((incl_m - min(sum_m - m, a.P) + BM - 1) >> BM_BITS);
      if (base + lane < a.E) s_blocks[base + lane] = incl_b, s_rows[base + lane] = incl_m;
      carry_b = read_lane(incl_b, kWave - 1);
      carry_m = read_lane(incl_m, kWave - 1);
    }
  }
  __syncthreads();
  const int blocks = __builtin_amdgcn_readfirstlane(s_blocks[a.E - 1]);
  // Tiles are dealt out in runs, one per XCD and round; four row blocks wide, so that a run shares both operands in its L2.
  const int run = gridDim.x / kXcds, per = kPatchRows * a.tiles_n;
  // Where a last round has work for half of the workgroups at most, its tiles are dealt out by the halves of their rows: those have
  // one wavefront of each SIMD at work (the second halves of tiles that have none are left out; nothing follows them).
  constexpr bool kHalves = WAVES == 8;
  const long real = static_cast<long>(blocks) * a.tiles_n, whole = kHalves && real % gridDim.x * 2 <= gridDim.x ? real / gridDim.x * gridDim.x : real;
  const long tiles = whole + 2 * (real - whole);
  long t = static_cast<long>(blockIdx.x % kXcds) * run + blockIdx.x / kXcds;
  struct Tile {
    int e, row0, rows, n0;
  };
  auto tile_at = [&](long at_walk) {
    const int over = static_cast<int>(at_walk - whole);
    const int t = static_cast<int>(over < 0 ? at_walk : whole + (over >> 1)), half = over < 0 ? 0 : BM / 2;
    const int group = t / per, in = t - group * per, wide = min(kPatchRows, blocks - group * kPatchRows);
    const int block = __builtin_amdgcn_readfirstlane(group * kPatchRows + in % wide);
    int e = 0;
    for (int base = 0; base < a.E; base += kWave) {
      const unsigned long long hit = __ballot(base + lane < a.E && block < s_blocks[min(base + lane, a.E - 1)]);
      if (hit != 0) {
        e = base + __builtin_ctzll(hit);
        break;
      }
    }
    const int before = e > 0 ? s_blocks[e - 1] : 0, first = e > 0 ? s_rows[e - 1] : 0;
    const int seat0 = ((block - before) << BM_BITS) + (over & 1 ? half : 0), row0 = first + seat0;
    Tile at;
    at.e = __builtin_amdgcn_readfirstlane(e);
    at.row0 = __builtin_amdgcn_readfirstlane(row0);
    at.rows = __builtin_amdgcn_readfirstlane(min(BM - half, s_rows[e] - row0));
    at.n0 = __builtin_amdgcn_readfirstlane(in / wide * BN);
    return at;
  };
  if (t >= tiles) return;

  // Slot s of LDS row r holds chunk s ^ key(r) of that row.  The keys make any 16 rows that are read together at one chunk cover
  // all banks: 16 neighbours of x; of w the rows 8 g + r + constant, g and r in 0..3 (see the columns below).
  uint32_t ox[XL], ow[WL];
  auto x_chunk = [&](int l, int i) { return (l & 7) ^ ((((wave * XL + i) * 8 + (l >> 3)) >> 1) & 7); };
  auto w_chunk = [&](int l, int i) {
    const int r = (wave * WL + i) * 8 + (l >> 3);
    return (l & 7) ^ (((r >> 1) & 1) | ((r >> 3) & 3) << 1);
  };
#pragma unroll
  for (int i = 0; i < XL; ++i) ox[i] = ((wave * XL + i) * 8 + (lane >> 3)) * a.pitch + x_chunk(lane, i) * 16;
#pragma unroll
  for (int i = 0; i < WL; ++i) ow[i] = ((wave * WL + i) * 8 + (lane >> 3)) * a.K + w_chunk(lane, i) * 16;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem)));
  // a last K-step that K does not fill (-1: there is none): its chunks behind K are turned to nowhere
  const int part = __builtin_amdgcn_readfirstlane(a.K % kB != 0 ? a.KB - 1 : -1);
  // What is requested next: K-step ahead_kt of a tile.  Rows and columns that do not exist are past the buffers' extents: they
  // read as zeros and cost no request.  The first wavefronts bring the scales of 64 rows each, the next ones those of WN's columns.
  // With GO_ROUND a tile begins with the K-step of its number in the row of tiles: with all of them at one place of K, weight rows
  // that are a power of two apart come from the same few memory channels (300 rows of 32 experts 4096 -> 4096 149 -> 103 us, 4224 ->
  // 4096 100 either way).  Where weights are read from the L2 several times it costs 4 % and gains nothing.
  int ahead_kt = 0, ahead_left = 0;
  uint32_t into = 0;  // the stage that the request fills
  i32x4 rx, rw;
  uint64_t scales_at;
  int scales_bytes;
  constexpr int kRowWaves = BM / 64;
  const int scales_of = wave < kRowWaves + WN ? wave : 0;
  const bool column_scales = scales_of >= kRowWaves;
  const uint32_t scales_to = column_scales ? kColumnScales + (scales_of - kRowWaves) * 256 : kRowScales + scales_of * 256;
  const uint64_t scales_step = column_scales ? 4 : static_cast<uint64_t>(a.P) * 4;
  auto aim = [&](const Tile& at) {
    ahead_kt = GO_ROUND ? at.n0 / BN % a.KB : 0;
    ahead_left = a.KB;
    rx = make_rsrc(static_cast<const uint8_t*>(a.x) + static_cast<size_t>(at.row0) * a.pitch, static_cast<size_t>(at.rows) * a.pitch);
    rw = make_rsrc(a.w + (static_cast<size_t>(at.e) * a.N + at.n0) * a.K, static_cast<size_t>(min(BN, a.N - at.n0)) * a.K);
    const int column = min((at.n0 + (scales_of - kRowWaves) * (BN / WN)) / kB, a.NB - 1);
    scales_at = column_scales ? reinterpret_cast<uint64_t>(a.sw + (static_cast<size_t>(at.e) * a.NB + column) * a.KB)
                              : reinterpret_cast<uint64_t>(a.sx + at.row0 + scales_of * 64);
    if constexpr (GO_ROUND) scales_at += ahead_kt * scales_step;
    scales_bytes = column_scales ? 4 : max(0, min(64, at.rows - scales_of * 64)) * 4;
  };
  Tile at = tile_at(t);
  if (at.rows <= 0) return;
  aim(at);
  auto request = [&] {
    const uint32_t from = ahead_kt * kB, to = lds0 + into;
    into = into == (STAGES - 1) * kStage ? 0 : into + kStage;
    load_word_to_lds(make_rsrc(reinterpret_cast<const void*>(scales_at), scales_bytes), lane * 4, to + scales_to);
    scales_at += scales_step;
    if (ahead_kt != part) {
#pragma unroll
      for (int i = 0; i < XL; ++i) load_to_lds(rx, ox[i], from, to + (wave * XL + i) * 1024);
#pragma unroll
      for (int i = 0; i < WL; ++i) load_to_lds(rw, ow[i], from, to + BM * kB + (wave * WL + i) * 1024);
    } else {
      int l = lane;
      asm volatile("" : "+v"(l));  // (else what follows from it is kept in registers all through the K loop)
#pragma unroll
      for (int i = 0; i < XL; ++i)
        load_to_lds(rx, from + x_chunk(l, i) * 16 >= static_cast<uint32_t>(a.K) ? kNowhere : ox[i], from, to + (wave * XL + i) * 1024);
#pragma unroll
      for (int i = 0; i < WL; ++i)
        load_to_lds(rw, from + w_chunk(l, i) * 16 >= static_cast<uint32_t>(a.K) ? kNowhere : ow[i], from, to + BM * kB + (wave * WL + i) * 1024);
    }
  };
  // one K-step on, into the next tile of this workgroup at the end of one; false behind the last
  auto step_ahead = [&] {
    if (GO_ROUND ? --ahead_left > 0 : ahead_kt + 1 < a.KB) {
      if (++ahead_kt == a.KB && GO_ROUND) {
        ahead_kt = 0;
        scales_at -= a.KB * scales_step;
      }
      return true;
    }
    t += gridDim.x;
    if (t >= tiles) return false;
    const Tile next = tile_at(t);
    if (next.rows <= 0) return false;
    aim(next);
    return true;
  };

  const int g = lane >> 4, c16 = lane & 15;
  // Row i of tile j's weight fragment is column (j / 4) 64 + (j / 2 % 2) 32 + (i / 4) 8 + (j % 2) 4 + i % 4: the results of
  // two tiles are then 8 neighbouring columns of a lane's row, and the four lanes of a row store 64 bytes side by side.
  const int wr = wn * (BN / WN) + (c16 >> 2) * 8 + (c16 & 3), wkey = ((wr >> 1) & 1) | ((wr >> 3) & 3) << 1;
  const int wlo = BM * kB + wr * kB + ((g ^ wkey) << 4), whi = BM * kB + wr * kB + (((g + 4) ^ wkey) << 4);  // chunks g and g + 4
  const int xr = wm * (BM / WM) + c16, xkey = (c16 >> 1) & 7;
  const int xlo = xr * kB + ((g ^ xkey) << 4), xhi = xr * kB + (((g + 4) ^ xkey) << 4);
  auto column_of = [](int j) { return (j >> 2) * 64 + ((j >> 1) & 1) * 32 + (j & 1) * 4; };

  long done = t;  // (the same walk, for the tile that is multiplied)
  bool more = true;  // there is a K-step that has not been requested
  auto request_ahead = [&] {
    if (more) {
      request();
      more = step_ahead();
    }
  };
  // A K-step begins with its requests, but with 256 rows with the fragments' reads, which the requests' arrivals would hold up
  // (16384 rows of 8 experts 4096 -> 4096 385 us the other way round, 327 so; 64 x 64 tiles 15 % the other way).  A wavefront without
  // rows only fetches (8192 rows of 64 experts 1024 -> 4096 86.6 -> 84.6 us, 400 of 8 15.5 -> 14.8, in 256-row tiles 20.2 -> 16.8).
  constexpr bool kRequestsFirst = BM <= 128;
#pragma unroll
  for (int q = 0; q < STAGES - 1; ++q) request_ahead();
  using Operand = decltype(operand<EXACT>(i32x8{}));
  uint32_t stage_at = 0;
  f32x4 acc[MT][NT];
  float s[MT];
  Pipe<MT, NT> pipe;
  for (;;) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      s[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const bool live = at.rows > wm * (BM / WM);
#pragma unroll 1
    for (int kt = 0; kt < a.KB; ++kt) {
      // (of the loads behind this K-step's all but STAGES - 2 steps' have been requested; behind the last request the count is less)
      if (STAGES == 2 || !more) wait_loads_but<0>();
      else wait_loads_but<(STAGES - 2) * kLoads>();
      block_barrier();
      const char* const stage = smem + stage_at;
      stage_at = stage_at == (STAGES - 1) * kStage ? 0 : stage_at + kStage;
      auto fragment = [&](int lo_at, int hi_at) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(stage + lo_at), hi = *reinterpret_cast<const i32x4*>(stage + hi_at);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      };
      if (kRequestsFirst || !live) request_ahead();
      if (!live) continue;
      i32x8 w = fragment(wlo, whi), x_read[MT];
      float s_read[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) x_read[i] = fragment(xlo + i * 16 * kB, xhi + i * 16 * kB);
#pragma unroll
      for (int i = 0; i < MT; ++i) s_read[i] = *reinterpret_cast<const float*>(stage + kRowScales + (xr + i * 16) * 4);
      const float scale = *reinterpret_cast<const float*>(stage + kColumnScales + wn * 256);
      if constexpr (!kRequestsFirst) request_ahead();
      __builtin_amdgcn_sched_barrier(0);
      pipe.drain(acc, s);
      Operand x[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) x[i] = operand<EXACT>(x_read[i]);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const Operand at_hand = operand<EXACT>(w);
        if (j + 1 < NT) w = fragment(wlo + column_of(j + 1) * kB, whi + column_of(j + 1) * kB);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int p = j * MT + i;
          if (p == pipe.kBehind) {  // (not earlier: the first products wait for their own fragments only)
#pragma unroll
            for (int r = 0; r < MT; ++r) s[r] = s_read[r] * scale;
          }
          pipe.put(p, multiply(at_hand, x[i]), acc, s);
        }
      }
    }
    pipe.drain(acc, s);
    pipe.clear();
    const Block rows_at{at.e, at.row0, at.rows};
    if constexpr (BLOCKS) {
      auto blocks = [&](auto act) {
        store_blocks<decltype(act)::value, MT, NT, BM, WN>(a, rows_at, wm * (BM / WM), at.n0 + wn * (BN / WN), wn, s_tops, acc);
      };
      if (a.act == BRT_ACT_GELU) blocks(std::integral_constant<int, BRT_ACT_GELU>{});
      else if (a.act == BRT_ACT_RELU) blocks(std::integral_constant<int, BRT_ACT_RELU>{});
      else blocks(std::integral_constant<int, BRT_ACT_NONE>{});
    } else {
      store_tile<MT, NT, EXACT>(a, rows_at, wm * (BM / WM), at.n0 + wn * (BN / WN), acc);
    }
    done += gridDim.x;
    if (done >= tiles) return;
    at = tile_at(done);
    if (at.rows <= 0) return;
  }
}

// Few rows per expert: the weights are streamed once and set the time.  A workgroup takes 16 NT columns and 16 MT rows; its
// W wavefronts take K-steps in turn (weights straight into the fragments' registers) and add up their sums through LDS.  Rows that are
// not 8-bit yet are quantized on the way in: the 32 elements that a lane holds of its row's block are exactly its fragment, so that costs
// two exchanges among the row's four lanes and no launch of its own.  One row of 2048 -> 8192: 6.6 us (16.8 MB, 2.5 TB/s: a launch,
// the loads, and two rounds of requests, one behind the other: 16 K-steps on eight wavefronts); 48 rows of 8 experts 1024 -> 4096 with
// bias and GELU 9.9 (33.9 MB, 3.4 TB/s: one round, as many K-steps as wavefronts).
template <int XDT, int MT, int NT, int W, bool EXACT>
__global__ __launch_bounds__(W * 64) void fp8_few_rows_kernel(Fp8Args a) {
  constexpr bool kQuantized = XDT < 0;
  constexpr int kBytes = kQuantized ? 1 : elem_bytes(XDT == BRT_F32 ? BRT_F32 : BRT_F16);
  constexpr int kLoads = 2 * kBytes;  // 16-byte loads for a lane's 32 elements
  constexpr int kBits = MT == 1 ? 4 : MT == 2 ? 5 : 6;
  __shared__ f32x4 s_part[W > 1 ? W : 1][NT * MT][64];
  const int lane = lane_id(), g = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int block = blockIdx.x / a.tiles_n, n0 = (blockIdx.x - block * a.tiles_n) * 16 * NT;
  const Block at = find_block(a, block, kBits);
  if (at.rows == 0) return;
  const int pitch = a.pitch * kBytes;
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(a.x)) + static_cast<size_t>(at.row0) * pitch, 0, at.rows * pitch, 0x00020000);
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.w) + (static_cast<size_t>(at.e) * a.N + n0) * a.K, 0, min(16 * NT, a.N - n0) * a.K, 0x00020000);
  const float* sw = a.sw + (static_cast<size_t>(at.e) * a.NB + n0 / kB) * a.KB;

  // the biases of the tiles that this wavefront finishes: fetched ahead of the weights, not behind the last barrier
  constexpr int kFinished = (MT * NT + W - 1) / W;
  float bias[kFinished][4];
#pragma unroll
  for (int f = 0; f < kFinished; ++f) biases<4>(a, at.e, n0 + (wave + f * W) % NT * 16 + g * 4, bias[f]);

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  for (int kb = wave; kb < a.KB; kb += W) {
    u32x4 wv[NT][2], xv[MT][kLoads];
    float given[MT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // the lane's chunks of 16: g and g + 4
      const bool there = kb * kB + h * 64 + g * 16 < a.K;
#pragma unroll
      for (int j = 0; j < NT; ++j)
        wv[j][h] = __builtin_amdgcn_raw_buffer_load_b128(rw, there ? (j * 16 + c16) * a.K + h * 64 + g * 16 : kNowhere, kb * kB, 0);
    }
    const float scale = sw[kb];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const int h = l / kBytes;
        const bool there = kb * kB + h * 64 + g * 16 < a.K;
        xv[i][l] = __builtin_amdgcn_raw_buffer_load_b128(
            rx, there ? (i * 16 + c16) * pitch + (h * 64 + g * 16) * kBytes + (l % kBytes) * 16 : kNowhere, kb * kB * kBytes, 0);
      }
      if constexpr (kQuantized) given[i] = a.sx[static_cast<size_t>(kb) * a.P + at.row0 + min(i * 16 + c16, at.rows - 1)];
    }
    decltype(operand<EXACT>(i32x8{})) x[MT];
    float s[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      i32x8 q;
      if constexpr (kQuantized) {
#pragma unroll
        for (int l = 0; l < 2; ++l)
#pragma unroll
          for (int c = 0; c < 4; ++c) q[4 * l + c] = static_cast<int>(xv[i][l][c]);
        s[i] = given[i] * scale;
      } else {
        constexpr int NE = 16 / kBytes;
        float v[32];
        uint32_t top = 0;
#pragma unroll
        for (int l = 0; l < kLoads; ++l) {
          float part[NE];
          unpack<XDT, 16>(xv[i][l], part);
#pragma unroll
          for (int c = 0; c < NE; ++c) {
            v[l * NE + c] = part[c];
            top = max(top, magnitude(part[c]));
          }
        }
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, kWave)));
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, kWave)));
        float own, inverse;
        scale_of(top, &own, &inverse);
#pragma unroll
        for (int c = 0; c < 8; ++c)
          q[c] = static_cast<int>(pack4(v[4 * c] * inverse, v[4 * c + 1] * inverse, v[4 * c + 2] * inverse, v[4 * c + 3] * inverse));
        s[i] = own * scale;
      }
      x[i] = operand<EXACT>(q);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      i32x8 v;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) v[4 * h + c] = static_cast<int>(wv[j][h][c]);
      const auto w = operand<EXACT>(v);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const f32x4 part = multiply(w, x[i]);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][j][q] = __builtin_fmaf(part[q], s[i], acc[i][j][q]);
      }
    }
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
    const int r = p / NT * 16 + c16;
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = sum[q];
    if (r < at.rows) finish<4>(a, static_cast<size_t>(at.row0) + r, n0 + p % NT * 16 + g * 4, whole, bias[f], v);
  }
}

template <int XDT, int MT, int NT, int W, bool EXACT>
int launch_few_rows(Fp8Args& a, hipStream_t st) {
  constexpr int kRows = 16 * MT;
  const long blocks = static_cast<long>(a.P) / kRows + std::min(a.E, a.P);
  a.tiles_n = (a.N + 16 * NT - 1) / (16 * NT);
  if (blocks * a.tiles_n >= (1l << 31)) return fail(BRT_E_UNSUPPORTED, "too many tiles");
  hipLaunchKernelGGL((fp8_few_rows_kernel<XDT, MT, NT, W, EXACT>), dim3(static_cast<unsigned>(blocks * a.tiles_n)), dim3(W * 64), 0, st, a);
  return check_launch("fp8_few_rows_kernel");
}
// Rows and columns of a workgroup, wavefronts that share K.  `tiles` of 16 columns is what there is to deal
// out (the loads are on the device: every expert is taken to have rows where there are as many rows).  Few of them: as many
// wavefronts as possible on each; many: more columns to a wavefront, which quantizes the rows once for all of them.
template <int XDT, bool EXACT>
int launch_few_rows(Fp8Args& a, hipStream_t st) {
  const long tiles = static_cast<long>(std::min(a.E, a.P)) * ((a.N + 15) / 16);
  if (a.P > 16 && a.P > 10l * a.E) {
    if (tiles < 1024) return launch_few_rows<XDT, 2, 2, 8, EXACT>(a, st);
    return launch_few_rows<XDT, 2, 4, 4, EXACT>(a, st);
  }
  if (tiles < 512) return launch_few_rows<XDT, 1, 1, 16, EXACT>(a, st);
  if (tiles < 1536) return launch_few_rows<XDT, 1, 2, 8, EXACT>(a, st);
  if (tiles < 4096) return launch_few_rows<XDT, 1, 4, 8, EXACT>(a, st);
  return launch_few_rows<XDT, 1, 4, 4, EXACT>(a, st);
}
template <int XDT>
int launch_few_rows(Fp8Args& a, hipStream_t st) {
  return a.exact ? launch_few_rows<XDT, true>(a, st) : launch_few_rows<XDT, false>(a, st);
}
// Which shapes the kernel for few rows takes: those of few tiles, whose time is a launch and the chain of loads behind it.  It needs
// no launch to quantize the rows, but quantizes them again for every 16 to 64 columns (with the launch counted, us here / 64 x 128
// or 64 x 64 tiles): 1 row 1024 -> 1024 4.0 / 8; 48 rows of 8 experts 1024 -> 4096 10.0 / 11.2; 64 rows 4096 -> 4096 15.3 / 18.8; 100
// rows of 4 experts 8192 -> 1024 24.8 / 32.2; but 128 rows of 32 experts 1024 -> 4096 31.4 / 30.4, 200 of 64 768 -> 2048 23.9 / 22.3,
// 190 of 8 1024 -> 4096 15.2 / 12.4.  Beyond kMostExperts it takes everything, and reads the weights again for every 32 rows of an
// expert (512 experts on the tiles / 513 here, 1024 -> 1024: 4000 rows 114 / 128, 40000 rows 163 / 407).
bool few_rows(int P, int E, int N) {
  if (E > kMostExperts || P <= 16) return true;
  const long used = std::min(E, P);
  if (P <= 10l * E) return used * ((N + 15) / 16) <= 4096;
  return P <= 128 && ((P + 31) / 32 + used - 1) * ((N + 31) / 32) <= 320;
}

template <int BM_BITS, int BN, int WM, int WN, int STAGES, bool GO_ROUND, bool EXACT, bool BLOCKS>
int launch_tiles(Fp8Args& a, hipStream_t st) {
  constexpr int kStage = ((1 << BM_BITS) + BN) * kB + (1 << BM_BITS) * 4 + WN * 256;
  constexpr int kTops = BLOCKS && BN / WN < kB ? WN * (1 << BM_BITS) * 4 : 0;  // (a block's largest values pass between wavefronts)
  constexpr int kMost = STAGES * kStage + kMostExperts * 8 + kTops;
  constexpr int kResident = kMost <= 80 * 1024 ? 2 : 1;  // workgroups of a CU
  const auto fn = fp8_tiles_kernel<BM_BITS, BN, WM, WN, STAGES, GO_ROUND, EXACT, BLOCKS>;
  if (const int rc = allow_dynamic_lds(reinterpret_cast<const void*>(fn), kMost); rc != BRT_OK) return rc;
  a.tiles_n = (a.N + BN - 1) / BN;
  // an expert adds at most one row block that it does not fill
  const long tiles = ((static_cast<long>(a.P) >> BM_BITS) + std::min(a.E, a.P)) * a.tiles_n;
  if (tiles >= (1l << 31)) return fail(BRT_E_UNSUPPORTED, "too many tiles");
  const long grid = std::min<long>((tiles + kXcds - 1) / kXcds * kXcds, kResident * kXcds * kCusPerXcd);
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(grid)), dim3(WM * WN * 64), STAGES * kStage + a.E * 8 + kTops, st, a);
  return check_launch("fp8_tiles_kernel");
}
template <int BM_BITS, int BN, int WM, int WN, int STAGES, bool GO_ROUND = false>
int launch_tiles(Fp8Args& a, hipStream_t st) {
  if (a.out_scales != nullptr) return launch_tiles<BM_BITS, BN, WM, WN, STAGES, GO_ROUND, false, true>(a, st);
  return launch_tiles<BM_BITS, BN, WM, WN, STAGES, GO_ROUND, false, false>(a, st);
}

// Tiles by what there is to deal out, the experts' last row blocks taken as half full, and a mean load of less than 0.8 of a block as one
// block (us; without the launch that quantizes):
//   64 x 64, four stages, while they go once round the chip, two workgroups on a CU: 400 rows of 8 experts 1024 -> 4096 8.9, 64 x 128
//   12.7, but 1000 of 8 512 -> 2048 10.9 and 7.6;
//   64 x 128, three stages, likewise, and for less than 64 rows an expert: 1500 rows of 4 experts 768 -> 2048
//   9, 64 x 64 13, 128 x 256 11, 2500 of 16 4096 -> 1024 25, 128 x 256 34, but 4096 of 8 4096 -> 1024 47 and 36, 6000 of 16 1024 ->
//   1024 18 and 13; 2048 rows of 128 experts 1024 -> 2048 56, 128 x 256 58;
//   128 x 256 and 256 x 256 by the rounds over the CUs that they take (one, or the share of one and half of one), at 1.05 and 1.6 us a
//   K-step and 4 and 7.5 a tile, 6.5 and 13.5 with fp32 results: 16384 rows of 64 experts 1024 -> 4096 118 and 126, 8192 of 32 1024
//   -> 4096 61 and 63, 8192 of 32 4096 -> 1024 59 and 53, 16384 of 8 4096 -> 4096 303 and 267, 16384 of 16 1024 -> 2048 fp32 69 and 81.
enum TileKind { k64x64, k64x128, k128x128, k128x256, k256x256 };
TileKind tile_kind(int E, int P, int N, int K, int out_dtype, bool exact) {
  const long used = std::min(E, P);
  auto tiles = [&](int rows, int columns) {
    const long blocks = used == 1 ? (P + rows - 1) / rows : 5l * P <= 4l * rows * used ? used : (2l * P / rows + used + 1) / 2;
    return blocks * ((N + columns - 1) / columns);
  };
  if (tiles(64, 64) <= 512) return k64x64;
  if (exact) return k128x128;
  if (tiles(64, 128) <= 512 || P < 64l * E) return k64x128;
  const long cus = kXcds * kCusPerXcd, steps = (K + kB - 1) / kB;
  const bool f32 = out_dtype == BRT_F32;
  auto rounds = [&](long n) { return n <= cus ? cus : n + cus / 2; };  // (in CUs; a tile's time in twentieths of a microsecond)
  const long wide = rounds(tiles(256, 256)) * (32 * steps + (f32 ? 270 : 150)), half = rounds(tiles(128, 256)) * (21 * steps + (f32 ? 130 : 80));
  return wide < half ? k256x256 : k128x256;
}
bool quantizes_result(int E, int P, int N, int K, int out_dtype) {
  return !few_rows(P, E, N) && out_dtype == BRT_BF16 && tile_kind(E, P, N, K, out_dtype, false) != k64x64;
}
int launch_any_tiles(Fp8Args& a, hipStream_t st) {
  TileKind kind = tile_kind(a.E, a.P, a.N, a.K, a.out_dtype, a.exact != 0);
  // (quantizing 256 x 256 results needs more registers than there are: 8192 rows of 32 experts 1024 -> 4096 + GELU 101 us, 128 x 256 88)
  if (kind == k256x256 && a.out_scales != nullptr) kind = k128x256;
  switch (kind) {
    case k64x64: return a.exact ? launch_tiles<6, 64, 2, 1, 4, false, true, false>(a, st) : launch_tiles<6, 64, 2, 1, 4, false, false, false>(a, st);
    case k64x128: return launch_tiles<6, 128, 2, 2, 3, true>(a, st);
    case k128x128: return launch_tiles<7, 128, 2, 2, 2, false, true, false>(a, st);
    case k128x256: return launch_tiles<7, 256, 2, 4, 3>(a, st);
    default: return launch_tiles<8, 256, 4, 2, 2, false, false, false>(a, st);
  }
}

}  // namespace
}  // namespace brt

using namespace brt;

extern "C" int brt_hip_quantize_rows(const void* x, int P, int K, int dtype, void* q, int pitch, float* scales, void* stream) {
  if (P < 0 || K < 0 || pitch < (K + kB - 1l) / kB * kB) return fail(BRT_E_INVALID, "bad shape P=%d K=%d pitch=%d", P, K, pitch);
  if (dtype != BRT_F32 && dtype != BRT_F16 && dtype != BRT_BF16) return fail(BRT_E_UNSUPPORTED, "dtype %d is not supported", dtype);
  if (P == 0 || K == 0) return BRT_OK;
  if (!x || !q || !scales) return fail(BRT_E_INVALID, "null argument");
  if (K % 16 != 0 || pitch % 16 != 0 || !aligned(x, 16) || !aligned(q, 16))
    return fail(BRT_E_UNSUPPORTED, "rows must be whole, aligned units of 16 elements (K=%d)", K);
  const int KB = static_cast<int>((K + kB - 1l) / kB);
  const long waves = (static_cast<long>(P) + 7) / 8 * KB;
  if (waves >= (1l << 31)) return fail(BRT_E_UNSUPPORTED, "too many blocks");
  const dim3 grid(static_cast<unsigned>((waves + 3) / 4)), block(256);
  hipStream_t st = as_stream(stream);
  uint8_t* to = static_cast<uint8_t*>(q);
  if (dtype == BRT_F32) hipLaunchKernelGGL((quantize_rows_kernel<BRT_F32>), grid, block, 0, st, x, to, scales, P, K, pitch, KB);
  else if (dtype == BRT_F16) hipLaunchKernelGGL((quantize_rows_kernel<BRT_F16>), grid, block, 0, st, x, to, scales, P, K, pitch, KB);
  else hipLaunchKernelGGL((quantize_rows_kernel<BRT_BF16>), grid, block, 0, st, x, to, scales, P, K, pitch, KB);
  return check_launch("quantize_rows_kernel");
}

extern "C" int brt_hip_grouped_gemm_fp8_quantizes(int E, int P, int N) { return few_rows(P, E, N) ? 1 : 0; }

extern "C" int brt_hip_grouped_gemm_fp8_blocks(int E, int P, int N, int K, int out_dtype) {
  return quantizes_result(E, P, N, K, out_dtype) ? 1 : 0;
}

extern "C" int brt_hip_grouped_gemm_fp8(const void* x, int x_dtype, int pitch, const float* x_scales, const void* w,
                                        const float* w_scales, const int32_t* loads, const void* bias, int bias_dtype, void* out,
                                        int out_dtype, float* out_scales, int E, int P, int N, int K, int activation, int exact,
                                        void* stream) {
  if (E <= 0 || P < 0 || N < 0 || K < 0 || pitch < K) return fail(BRT_E_INVALID, "bad shape E=%d P=%d N=%d K=%d pitch=%d", E, P, N, K, pitch);
  const bool quantized = x_scales != nullptr;
  if (!quantized && x_dtype != BRT_F32 && x_dtype != BRT_F16 && x_dtype != BRT_BF16)
    return fail(BRT_E_UNSUPPORTED, "dtype %d is not supported", x_dtype);
  if (out_dtype != BRT_F32 && out_dtype != BRT_F16 && out_dtype != BRT_BF16) return fail(BRT_E_UNSUPPORTED, "dtype %d is not supported", out_dtype);
  if (bias && bias_dtype != BRT_F32 && bias_dtype != BRT_F16 && bias_dtype != BRT_BF16)
    return fail(BRT_E_UNSUPPORTED, "bias dtype %d is not supported", bias_dtype);
  if (activation != BRT_ACT_NONE && activation != BRT_ACT_GELU && activation != BRT_ACT_RELU)
    return fail(BRT_E_UNSUPPORTED, "activation %d is not supported", activation);
  if (exact && out_dtype != BRT_F32) return fail(BRT_E_UNSUPPORTED, "a sum of exact products goes to an fp32 result");
  if (P == 0 || N == 0) return BRT_OK;
  if (K == 0) return fail(BRT_E_UNSUPPORTED, "rows of no elements");
  if (!x || !w || !w_scales || !loads || !out) return fail(BRT_E_INVALID, "null argument");
  if (K % 16 != 0 || pitch % 16 != 0 || !aligned(x, 16) || !aligned(w, 16))
    return fail(BRT_E_UNSUPPORTED, "rows must be whole, aligned units of 16 elements (K=%d)", K);
  if (P >= kMostRows) return fail(BRT_E_UNSUPPORTED, "more than %d rows", kMostRows - 1);
  if (E > kMostColumns || N > kMostColumns) return fail(BRT_E_UNSUPPORTED, "more than %d columns or experts", kMostColumns);
  if (pitch > (1 << 20)) return fail(BRT_E_UNSUPPORTED, "rows of more than 1 Mi elements");  // (256 of them are addressed by 31 bits)
  if (out_scales && (!quantizes_result(E, P, N, K, out_dtype) || !aligned(out, 16)))
    return fail(BRT_E_UNSUPPORTED, "results of this shape are not quantized by the product's kernel");
  if (!quantized && !few_rows(P, E, N)) return fail(BRT_E_UNSUPPORTED, "rows for the wide tiles are quantized beforehand");
  Fp8Args a{};
  a.x = x; a.sx = x_scales; a.w = static_cast<const uint8_t*>(w); a.sw = w_scales; a.loads = loads;
  a.bias = bias; a.bias_dtype = bias_dtype; a.out = out; a.out_dtype = out_dtype; a.out_scales = out_scales; a.act = activation; a.exact = exact;
  a.pitch = pitch; a.E = E; a.P = P; a.N = N; a.K = K;
  a.KB = (K + kB - 1) / kB; a.NB = (N + kB - 1) / kB;
  hipStream_t st = as_stream(stream);
  if (few_rows(P, E, N)) {
    if (quantized) return launch_few_rows<-1>(a, st);
    if (x_dtype == BRT_F32) return launch_few_rows<BRT_F32>(a, st);
    if (x_dtype == BRT_F16) return launch_few_rows<BRT_F16>(a, st);
    return launch_few_rows<BRT_BF16>(a, st);
  }
  return launch_any_tiles(a, st);
}
