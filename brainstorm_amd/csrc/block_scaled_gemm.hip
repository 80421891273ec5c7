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
// three-hundredth of a bf16 rounding, a twentieth of an fp16 one.  An fp32 result would show it, so there the operands are
// widened to bf16 in registers (exactly) and multiplied by v_mfma_f32_16x16x32_bf16, whose sums are off by 1.2e-8.
#include <algorithm>

#include "grouped_gemm.hpp"
#include "rows.hpp"

namespace brt {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kB = 128;            // elements of a scale block, bytes of a K-step
constexpr float kMax = 448.0f;     // the largest e4m3 value
constexpr float kLeast = 0x1p-100f;  // blocks whose largest value is below this are scaled as if it were this
constexpr int kXcds = 8, kCusPerXcd = 32;
constexpr int kPatchRows = 4;
constexpr uint32_t kNowhere = 0x7ffffff0u;  // an offset past every extent: reads as zero, costs no request

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
// reads 8 rows of one block: 256-byte pieces of 16-bit rows, and writes 8 scales that lie side by side.
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
  void* out;           // [P, N] of out_dtype
  int pitch, bias_dtype, out_dtype, act;
  int E, P, N, K, KB, NB, tiles_n;
};

__device__ __forceinline__ i32x4 make_rsrc(const void* p, size_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(a));
  r[1] = __builtin_amdgcn_readfirstlane(static_cast<int>((a >> 32) & 0xffff));
  r[2] = __builtin_amdgcn_readfirstlane(static_cast<int>(bytes));
  r[3] = 0x00020000;
  return r;
}
// 16 bytes per lane from the buffer into LDS at lds_base + 16 * lane (M0; one wait state between its write and the load).  The
// compiler does not know that it touches LDS, nor counts it: every wait for such a load is written out.
__device__ __forceinline__ void load_to_lds(const i32x4& rsrc, uint32_t voffset, uint32_t soffset, uint32_t lds_base) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "{m0}"(lds_base), "v"(voffset), "s"(rsrc), "s"(soffset)
               : "memory");
}
__device__ __forceinline__ void wait_loads_all() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }
__device__ __forceinline__ void block_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
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

struct Block {
  int e, row0, rows;
};
// The expert and the rows of row block `block` of the list (blocks of `1 << bits` rows); rows 0: there is no such block.
__device__ __forceinline__ Block find_block(const Fp8Args& a, int block, int bits) {
  const int lane = lane_id();
  int carry_b = 0, carry_m = 0;
  for (int base = 0; base < a.E; base += kWave) {
    const int given = a.loads[min(base + lane, a.E - 1)];
    const int m = base + lane < a.E ? max(given, 0) : 0;
    const int b = (m + (1 << bits) - 1) >> bits;
    const int incl_b = carry_b + wave_inclusive_scan(b), incl_m = carry_m + wave_inclusive_scan(m);
    const unsigned long long hit = __ballot(block < incl_b);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      const int seat0 = (block - (read_lane(incl_b, src) - read_lane(b, src))) << bits;
      const int load = read_lane(m, src);
      const int row0 = read_lane(incl_m, src) - load + seat0;
      return {base + src, row0, max(0, min(min(1 << bits, load - seat0), a.P - row0))};
    }
    carry_b = read_lane(incl_b, kWave - 1);
    carry_m = read_lane(incl_m, kWave - 1);
  }
  return {0, 0, 0};
}

__device__ __forceinline__ float activated(float v, int act) {
  if (act == BRT_ACT_GELU) return gelu_erf(v);
  if (act == BRT_ACT_RELU) return fmaxf(v, 0.0f);
  return v;
}

// COUNT results of one row, columns n .. n + COUNT - 1, biased, activated, rounded and stored; `whole`: the row's pieces are
// aligned and N is a multiple of COUNT.
template <int COUNT>
__device__ __forceinline__ void finish(const Fp8Args& a, int e, size_t row, int n, bool whole, float (&v)[COUNT]) {
  if (n >= a.N) return;
  if (a.bias != nullptr) {
#pragma unroll
    for (int q = 0; q < COUNT; ++q)
      v[q] += load_gate(a.bias, a.bias_dtype, static_cast<size_t>(e) * a.N + min(n + q, a.N - 1));
  }
#pragma unroll
  for (int q = 0; q < COUNT; ++q) v[q] = activated(v[q], a.act);
  const size_t at = row * a.N + n;
  if (whole) {
    if (a.out_dtype == BRT_F32) pack_store<BRT_F32, COUNT>(static_cast<float*>(a.out) + at, v);
    else if (a.out_dtype == BRT_F16) pack_store<BRT_F16, COUNT>(static_cast<uint16_t*>(a.out) + at, v);
    else pack_store<BRT_BF16, COUNT>(static_cast<uint16_t*>(a.out) + at, v);
    return;
  }
#pragma unroll
  for (int q = 0; q < COUNT; ++q) {
    if (n + q >= a.N) break;
    if (a.out_dtype == BRT_F32) static_cast<float*>(a.out)[at + q] = v[q];
    else static_cast<uint16_t*>(a.out)[at + q] = static_cast<uint16_t>(a.out_dtype == BRT_F16 ? float_to_f16(v[q]) : float_to_bf16(v[q]));
  }
}

// BM x BN tiles, WM x WN wavefronts.  Both operands go straight into LDS, K-steps of 128 bytes in two stages: the next one is
// requested when this one has landed and is read.
template <int BM_BITS, int BN, int WM, int WN, bool EXACT>
__global__ __launch_bounds__(WM* WN * 64, 2) void fp8_tiles_kernel(Fp8Args a) {
  constexpr int BM = 1 << BM_BITS, WAVES = WM * WN;
  constexpr int MT = BM / WM / 16, NT = BN / WN / 16;  // 16 x 16 tiles of a wavefront
  constexpr int XL = BM / 8 / WAVES, WL = BN / 8 / WAVES;  // loads of a wavefront and K-step, 8 rows each
  constexpr int kStage = (BM + BN) * kB;
  static_assert(NT % 4 == 0 && XL >= 1 && WL >= 1 && kB % (BN / WN) == 0, "a wavefront's columns share a scale block");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // 32 tiles at a time per XCD, four row blocks wide, so that they share both operands in its L2
  const int xcd = blockIdx.x % kXcds, idx = blockIdx.x / kXcds;
  const int t = ((idx / kCusPerXcd) * kXcds + xcd) * kCusPerXcd + idx % kCusPerXcd;
  const int per = kPatchRows * a.tiles_n;
  const int block = __builtin_amdgcn_readfirstlane(t / per * kPatchRows + t % kPatchRows);
  const int n0 = __builtin_amdgcn_readfirstlane(t % per / kPatchRows * BN);
  const Block at = find_block(a, block, BM_BITS);
  if (at.rows == 0) return;

  const i32x4 rx = make_rsrc(static_cast<const uint8_t*>(a.x) + static_cast<size_t>(at.row0) * a.pitch, static_cast<size_t>(at.rows) * a.pitch);
  const i32x4 rw = make_rsrc(a.w + (static_cast<size_t>(at.e) * a.N + n0) * a.K, static_cast<size_t>(min(BN, a.N - n0)) * a.K);
  // Slot s of LDS row r holds chunk s ^ key(r) of that row.  The keys make any 16 rows that are read together at one chunk cover
  // all banks: 16 neighbours of x; of w the rows 8 g + r + constant, g and r in 0..3 (see the columns below).
  uint32_t ox[XL], ow[WL];
  const int sub = lane >> 3, slot = lane & 7;
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int r = (wave * XL + i) * 8 + sub;
    ox[i] = r < at.rows ? r * a.pitch + (slot ^ ((r >> 1) & 7)) * 16 : kNowhere;
  }
#pragma unroll
  for (int i = 0; i < WL; ++i) {
    const int r = (wave * WL + i) * 8 + sub;
    ow[i] = r < a.N - n0 ? r * a.K + (slot ^ (((r >> 1) & 1) | ((r >> 3) & 3) << 1)) * 16 : kNowhere;
  }
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem)));
  auto request = [&](int kt) {
    const uint32_t from = kt * kB, to = lds0 + (kt & 1) * kStage;
    if (kt == a.KB - 1 && a.K % kB != 0) {  // a last K-step that K does not fill: chunks behind K read as zeros
#pragma unroll
      for (int i = 0; i < XL; ++i) {
        const int r = (wave * XL + i) * 8 + sub;
        if (kt * kB + (slot ^ ((r >> 1) & 7)) * 16 >= a.K) ox[i] = kNowhere;
      }
#pragma unroll
      for (int i = 0; i < WL; ++i) {
        const int r = (wave * WL + i) * 8 + sub;
        if (kt * kB + (slot ^ (((r >> 1) & 1) | ((r >> 3) & 3) << 1)) * 16 >= a.K) ow[i] = kNowhere;
      }
    }
#pragma unroll
    for (int i = 0; i < XL; ++i) load_to_lds(rx, ox[i], from, to + (wave * XL + i) * 1024);
#pragma unroll
    for (int i = 0; i < WL; ++i) load_to_lds(rw, ow[i], from, to + BM * kB + (wave * WL + i) * 1024);
  };

  const int g = lane >> 4, c16 = lane & 15;
  // Row i of tile j's weight fragment is column (j / 4) 64 + (j / 2 % 2) 32 + (i / 4) 8 + (j % 2) 4 + i % 4: the results of
  // two tiles are then 8 neighbouring columns of a lane's row, and the four lanes of a row store 64 bytes side by side.
  int wrow[4], xrow[MT];  // LDS offsets
  uint32_t wkey[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = wn * (BN / WN) + (j >> 1) * 32 + (c16 >> 2) * 8 + (j & 1) * 4 + (c16 & 3);
    wrow[j] = BM * kB + r * kB;
    wkey[j] = ((r >> 1) & 1) | ((r >> 3) & 3) << 1;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) xrow[i] = (wm * (BM / WM) + i * 16 + c16) * kB;
  const uint32_t xkey = (c16 >> 1) & 7;

  const float* sx = a.sx + at.row0 + wm * (BM / WM) + c16;
  const int last_row = a.P - 1 - (at.row0 + wm * (BM / WM) + c16);
  const float* sw = a.sw + (static_cast<size_t>(at.e) * a.NB + min((n0 + wn * (BN / WN)) / kB, a.NB - 1)) * a.KB;
  float sxv[MT], swv;
  auto request_scales = [&](int kt) {
#pragma unroll
    for (int i = 0; i < MT; ++i) sxv[i] = sx[static_cast<size_t>(kt) * a.P + min(i * 16, last_row)];
    swv = sw[kt];
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  request_scales(0);
  request(0);
  for (int kt = 0; kt < a.KB; ++kt) {
    wait_loads_all();
    block_barrier();
    float s[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) s[i] = sxv[i] * swv;
    if (kt + 1 < a.KB) {
      request_scales(kt + 1);
      request(kt + 1);
    }
    const char* const stage = smem + (kt & 1) * kStage;
    decltype(operand<EXACT>(i32x8{})) x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const i32x4 lo = *reinterpret_cast<const i32x4*>(stage + xrow[i] + ((g ^ xkey) << 4));
      const i32x4 hi = *reinterpret_cast<const i32x4*>(stage + xrow[i] + (((g + 4) ^ xkey) << 4));
      x[i] = operand<EXACT>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const char* const from = stage + wrow[j & 3] + (j >> 2) * 64 * kB;
      const i32x4 lo = *reinterpret_cast<const i32x4*>(from + ((g ^ wkey[j & 3]) << 4));
      const i32x4 hi = *reinterpret_cast<const i32x4*>(from + (((g + 4) ^ wkey[j & 3]) << 4));
      const auto w = operand<EXACT>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const f32x4 part = multiply(w, x[i]);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][j][q] = __builtin_fmaf(part[q], s[i], acc[i][j][q]);
      }
    }
  }

  const bool whole = a.N % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = wm * (BM / WM) + i * 16 + c16;
    if (r >= at.rows) continue;
#pragma unroll
    for (int j = 0; j < NT; j += 2) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = acc[i][j][q], v[4 + q] = acc[i][j + 1][q];
      finish<8>(a, at.e, static_cast<size_t>(at.row0) + r, n0 + wn * (BN / WN) + (j >> 2) * 64 + ((j >> 1) & 1) * 32 + g * 8, whole, v);
    }
  }
}

template <int BM_BITS, int BN, int WM, int WN, bool EXACT = false>
int launch_tiles(Fp8Args& a, hipStream_t st) {
  constexpr int kLds = 2 * ((1 << BM_BITS) + BN) * kB;
  const auto fn = fp8_tiles_kernel<BM_BITS, BN, WM, WN, EXACT>;
  if (const int rc = allow_dynamic_lds(reinterpret_cast<const void*>(fn), kLds); rc != BRT_OK) return rc;
  a.tiles_n = (a.N + BN - 1) / BN;
  // an expert adds at most one row block that it does not fill
  const long blocks = (static_cast<long>(a.P) >> BM_BITS) + std::min(a.E, a.P);
  const long tiles = (blocks + kPatchRows - 1) / kPatchRows * kPatchRows * a.tiles_n;
  const long round = kXcds * kCusPerXcd;
  const long grid = (tiles + round - 1) / round * round;
  if (grid >= (1l << 31)) return fail(BRT_E_UNSUPPORTED, "too many tiles");
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(grid)), dim3(WM * WN * 64), kLds, st, a);
  return check_launch("fp8_tiles_kernel");
}

}  // namespace
}  // namespace brt

using namespace brt;

extern "C" int brt_hip_quantize_rows(const void* x, int P, int K, int dtype, void* q, int pitch, float* scales, void* stream) {
  if (P < 0 || K < 0 || pitch < (K + kB - 1) / kB * kB) return fail(BRT_E_INVALID, "bad shape P=%d K=%d pitch=%d", P, K, pitch);
  if (dtype != BRT_F32 && dtype != BRT_F16 && dtype != BRT_BF16) return fail(BRT_E_UNSUPPORTED, "dtype %d is not supported", dtype);
  if (P == 0 || K == 0) return BRT_OK;
  if (!x || !q || !scales) return fail(BRT_E_INVALID, "null argument");
  if (K % 16 != 0 || pitch % 16 != 0 || !aligned(x, 16) || !aligned(q, 16))
    return fail(BRT_E_UNSUPPORTED, "rows must be whole, aligned units of 16 elements (K=%d)", K);
  const int KB = (K + kB - 1) / kB;
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

extern "C" int brt_hip_grouped_gemm_fp8(const void* x, int pitch, const float* x_scales, const void* w, const float* w_scales,
                                        const int32_t* loads, const void* bias, int bias_dtype, void* out, int out_dtype, int E,
                                        int P, int N, int K, int activation, void* stream) {
  if (E <= 0 || P < 0 || N < 0 || K < 0 || pitch < K) return fail(BRT_E_INVALID, "bad shape E=%d P=%d N=%d K=%d pitch=%d", E, P, N, K, pitch);
  if (out_dtype != BRT_F32 && out_dtype != BRT_F16 && out_dtype != BRT_BF16) return fail(BRT_E_UNSUPPORTED, "dtype %d is not supported", out_dtype);
  if (bias && bias_dtype != BRT_F32 && bias_dtype != BRT_F16 && bias_dtype != BRT_BF16)
    return fail(BRT_E_UNSUPPORTED, "bias dtype %d is not supported", bias_dtype);
  if (activation != BRT_ACT_NONE && activation != BRT_ACT_GELU && activation != BRT_ACT_RELU)
    return fail(BRT_E_UNSUPPORTED, "activation %d is not supported", activation);
  if (P == 0 || N == 0) return BRT_OK;
  if (K == 0) return fail(BRT_E_UNSUPPORTED, "rows of no elements");
  if (!x || !x_scales || !w || !w_scales || !loads || !out) return fail(BRT_E_INVALID, "null argument");
  if (K % 16 != 0 || pitch % 16 != 0 || !aligned(x, 16) || !aligned(w, 16))
    return fail(BRT_E_UNSUPPORTED, "rows must be whole, aligned units of 16 elements (K=%d)", K);
  if (pitch > (1 << 22)) return fail(BRT_E_UNSUPPORTED, "rows of more than 4 Mi elements");  // (256 of them are addressed by 31 bits)
  Fp8Args a{};
  a.x = x; a.sx = x_scales; a.w = static_cast<const uint8_t*>(w); a.sw = w_scales; a.loads = loads;
  a.bias = bias; a.bias_dtype = bias_dtype; a.out = out; a.out_dtype = out_dtype; a.act = activation;
  a.pitch = pitch; a.E = E; a.P = P; a.N = N; a.K = K;
  a.KB = (K + kB - 1) / kB; a.NB = (N + kB - 1) / kB;
  if (out_dtype == BRT_F32) return launch_tiles<7, 128, 2, 2, true>(a, as_stream(stream));
  if (P > 160 * static_cast<long>(E) && N > 128) return launch_tiles<8, 256, 4, 2>(a, as_stream(stream));
  return launch_tiles<7, 128, 2, 2>(a, as_stream(stream));
}
