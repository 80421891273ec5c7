// Shared by the products of rows that are packed by expert with weights of few bits: loads straight into LDS, where an expert's
// rows are, and the epilogue.  `A` is a kernel's argument block: loads [E], P rows, N columns; bias [E, N] of bias_dtype or null; out [P, N] of
// out_dtype; act.
#pragma once

#include "grouped_gemm.hpp"
#include "rows.hpp"

namespace brt {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kXcds = 8, kCusPerXcd = 32;
constexpr uint32_t kNowhere = 0x7ffffff0u;  // an offset past every extent: reads as zero, costs no request

// The descriptor of a buffer for the loads below.  A scalar that a vector unit wrote, as these are where the compiler cannot tell that
// they are the same in all lanes, may be read by a load five wait states later, which no one counts for inline assembly: they pass here.
__device__ __forceinline__ i32x4 make_rsrc(const void* p, size_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(a));
  r[1] = __builtin_amdgcn_readfirstlane(static_cast<int>((a >> 32) & 0xffff));
  r[2] = __builtin_amdgcn_readfirstlane(static_cast<int>(bytes));
  r[3] = 0x00020000;
  asm volatile("s_nop 4" : "+s"(r));
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
// ... 4 bytes per lane, at lds_base + 4 * lane
__device__ __forceinline__ void load_word_to_lds(const i32x4& rsrc, uint32_t voffset, uint32_t lds_base) {
  asm volatile("s_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "{m0}"(lds_base), "v"(voffset), "s"(rsrc)
               : "memory");
}
// all but the last N loads of this wavefront have landed
template <int N>
__device__ __forceinline__ void wait_loads_but() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory"); }
__device__ __forceinline__ void block_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

struct Block {
  int e, row0, rows;
};
// The expert and the rows of row block `block` of the list (blocks of `1 << bits` rows); rows 0: there is no such block.  Loads are
// taken as what they can be: none below zero, no rows behind the P that there are (which are few enough for 32-bit sums).
template <typename A>
__device__ __forceinline__ Block find_block(const A& a, int block, int bits) {
  const int lane = lane_id();
  int carry_b = 0, carry_m = 0;
  for (int base = 0; base < a.E; base += kWave) {
    const int given = a.loads[min(base + lane, a.E - 1)];
    const int m = base + lane < a.E ? min(max(given, 0), a.P) : 0;
    const int b = (m + (1 << bits) - 1) >> bits;
    const int incl_b = carry_b + wave_inclusive_scan(b), incl_m = min(carry_m + wave_inclusive_scan(m), a.P);
    const unsigned long long hit = __ballot(block < incl_b);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      const int seat0 = (block - (read_lane(incl_b, src) - read_lane(b, src))) << bits;
      const int before = src > 0 ? read_lane(incl_m, src - 1) : carry_m, row0 = before + seat0;
      return {base + src, row0, max(0, min(1 << bits, read_lane(incl_m, src) - row0))};
    }
    carry_b = read_lane(incl_b, kWave - 1);
    carry_m = read_lane(incl_m, kWave - 1);
  }
  return {0, 0, 0};
}

// Activations hand NaN on: a row that holds NaN or an infinity has results of NaN, not zeros that look sound, in blocks too.
template <int ACT>
__device__ __forceinline__ float activated(float v) { return apply_act<ACT, true>(v); }
__device__ __forceinline__ float activated(float v, int act) {
  if (act == BRT_ACT_GELU) return activated<BRT_ACT_GELU>(v);
  if (act == BRT_ACT_RELU) return activated<BRT_ACT_RELU>(v);
  return v;
}

// The biases of columns n .. n + COUNT - 1 (zeros without any).
template <int COUNT, typename A>
__device__ __forceinline__ void biases(const A& a, int e, int n, float (&b)[COUNT]) {
#pragma unroll
  for (int q = 0; q < COUNT; ++q)
    b[q] = a.bias != nullptr ? load_gate(a.bias, a.bias_dtype, static_cast<size_t>(e) * a.N + min(n + q, a.N - 1)) : 0.0f;
}

// COUNT results of one row, columns n .. n + COUNT - 1, biased, activated, rounded and stored; `whole`: the row's pieces are
// aligned and N is a multiple of COUNT.
template <int COUNT, typename A>
__device__ __forceinline__ void finish(const A& a, size_t row, int n, bool whole, const float (&bias)[COUNT], float (&v)[COUNT]) {
  if (n >= a.N) return;
#pragma unroll
  for (int q = 0; q < COUNT; ++q) v[q] = activated(v[q] + bias[q], a.act);
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
}  // namespace brt
