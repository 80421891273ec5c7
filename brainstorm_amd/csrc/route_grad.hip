// Gradients of the compact route: of the gate's weights, of the rows copied to their paths, and of the rows added up to
// their cells (no counterpart in the reference, whose ops are not differentiable).
//
//   gate      w[t,j] = softmax(s[t])[id(t,j)]        ds[t,e] = p[t,e] * (G[t,e] - sum_j g[t,j] w[t,j])
//                                                     (G: g[t,j] at the chosen columns, zero elsewhere)
//   dispatch  row[r] = w[e] * x[cell(e)]              dx[t] = sum_j w[t,j] * g[row(t,j)],  dw[t,j] = <x[t], g[row(t,j)]>
//   combine   out[t] = sum_j w[t,j] * y[row(t,j)]     dy[r] = w[e] * g[cell(e)],           dw[t,j] = <y[row(t,j)], g[t]>
//
// All three are bound by memory: each operand is read once and each result written once, in one launch.  The two row
// kernels are driven by cells, not by rows: what belongs to the cell (x or dx, the gradient of the result) passes once,
// where a walk over the rows would fetch it once per path, and the sums over j and over a row's elements stay in
// registers -- no atomics, the order of every sum is fixed.  Products and sums are fp32, results are rounded once.
// Measured: dispatch 16384 cells x 1024 bf16, two rows each 21.7 us (100 MB, 4.6 TB/s), combine 32768 x 1024 bf16, two rows each,
// both gradients 50.5 us (332 MB, 6.6 TB/s); a copy of 1 GiB moves 5.1 TB/s.
#include <algorithm>

#include "gate.hpp"
#include "rows.hpp"

namespace brt {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxK = 8;  // entries per cell of the row kernels, as in combine_by_rows

// ---------------------------------------------------------------------------------------------- gate
struct GateGradArgs {
  const void* scores;
  const int* ids;
  const float* weights;
  const float* grad;
  void* out;
  int T, E, k, softmax;
  int ls;  // log2 of the lanes that share a row
};

// A row is held by 1 << ls lanes, STEPS units of V columns each (one 16-byte unit where the rows are whole units, one column
// otherwise): 16-bit scores of 128 paths take 16 lanes, so that a wavefront has four rows in flight and its reductions stay
// on the DPP network.  Bound by the issue of the exponentials and the masks: 65536 x 128 bf16 11.6 us (33.6 MB, 2.9 TB/s), of which its 5.67 M
// vector instructions at four clocks on 1024 SIMDs of 2.4 GHz are 9.2.
template <int DT, int V, int STEPS>
__global__ __launch_bounds__(kBlock) void gate_grad_kernel(GateGradArgs a) {
  using namespace std;
  const int lane = lane_id(), ls = a.ls, lpr = 1 << ls;
  const int glane = lane & (lpr - 1);
  const long wave = static_cast<long>(blockIdx.x) * (kBlock / kWave) + (threadIdx.x >> 6);
  const long row = (wave << (6 - ls)) + (lane >> ls);
  const bool live = row < a.T;
  const size_t t = live ? row : a.T - 1;
  constexpr int kBytes = V * elem_bytes(DT);
  using U = typename Unit<kBytes>::type;
  const U* __restrict__ from = static_cast<const U*>(a.scores) + t * (a.E / V);
  const int units = a.E / V;
  float p[STEPS][V], g[STEPS][V];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int u = s * lpr + glane;
    if (a.softmax) unpack<DT, kBytes>(from[min(u, units - 1)], p[s]);
#pragma unroll
    for (int v = 0; v < V; ++v) g[s][v] = 0.0f;
  }
  float dot = 0.0f;
  for (int j0 = 0; j0 < a.k; j0 += 2) {  // (two at a time: their words are fetched together)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const size_t slot = t * a.k + min(j0 + q, a.k - 1);
      const int id = j0 + q < a.k ? a.ids[slot] : -1;
      const float d = a.grad[slot], w = a.softmax ? a.weights[slot] : 0.0f;
      if (j0 + q < a.k) dot += d * w;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int c = (s * lpr + glane) * V;
#pragma unroll
        for (int v = 0; v < V; ++v) g[s][v] = c + v == id ? d : g[s][v];  // (a row's ids differ)
      }
    }
  }
  if (a.softmax) {
    float top = -INFINITY;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (s * lpr + glane < units) top = fmaxf(top, p[s][v]);
    top = segment_max(top, lpr);
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        p[s][v] = expf(p[s][v] - top);
        if (s * lpr + glane < units) sum += p[s][v];
      }
    const float inverse = 1.0f / segment_sum(sum, lpr);  // (one division a row: 65536 x 128 bf16 13.2 -> 11.6 us)
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) g[s][v] = p[s][v] * inverse * (g[s][v] - dot);
  }
  char* const to = static_cast<char*>(a.out) + t * a.E * elem_bytes(DT);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int u = s * lpr + glane;
    if (live && u < units) pack_store<DT, V>(to + static_cast<size_t>(u) * kBytes, g[s]);
  }
}

// ---------------------------------------------------------------------------------------------- rows
struct RowsGradArgs {
  const void* grad;       // dispatch: [P, cell] of the rows; combine: [T, cell] of the result
  const void* operand;    // dispatch: the cells [T, cell]; combine: the rows [P, cell] (read for grad_weights only)
  const float* weights;   // [T, k] or null
  const int* ids;         // combine: [T, k]
  const int* seat_rows;   // [T, k]
  const int* row_entries; // combine: [P]
  void* out;              // dispatch: [T, cell]; combine: [P, cell]; or null
  float* grad_weights;    // [T, k] or null
  int T, P, k, cpr;
  int cell_blocks;        // combine: workgroups that take cells, the others clear rows without an entry
};

// Units of a row into registers as fp32: 16-byte units of 16-bit elements, from a row of DT or (G32) of fp32 elements.
template <int DT, bool G32, int NE>
__device__ __forceinline__ void load_unit(const void* base, size_t unit, float (&x)[NE]) {
  if constexpr (!G32 || DT == BRT_F32) {
    unpack<DT, 16>(static_cast<const u32x4*>(base)[unit], x);
  } else {
    const f32x4* p = static_cast<const f32x4*>(base) + 2 * unit;
    const f32x4 lo = p[0], hi = p[1];
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = lo[q], x[4 + q] = hi[q];
  }
}

// The entries of a cell: row[j] (0-based) and whether the entry has one; loads are unconditional (clamped into the table).
template <int KMAX>
__device__ __forceinline__ void entries_of(const RowsGradArgs& a, size_t slot0, bool live, int (&row)[KMAX], float (&w)[KMAX],
                                           bool (&has)[KMAX]) {
#pragma unroll
  for (int j = 0; j < KMAX; ++j) row[j] = a.seat_rows[slot0 + min(j, a.k - 1)];
  if (a.weights != nullptr) {
#pragma unroll
    for (int j = 0; j < KMAX; ++j) w[j] = a.weights[slot0 + min(j, a.k - 1)];
  } else {
#pragma unroll
    for (int j = 0; j < KMAX; ++j) w[j] = 1.0f;
  }
#pragma unroll
  for (int j = 0; j < KMAX; ++j) {
    has[j] = live && j < a.k && row[j] >= 1 && row[j] <= a.P;
    row[j] = has[j] ? row[j] - 1 : 0;
    w[j] = has[j] ? w[j] : 0.0f;  // (the weight of an entry without a row may be anything)
  }
}

// dots of a cell, summed over the lanes of its group; lane j writes the j-th
template <int KMAX>
__device__ __forceinline__ void store_dots(const RowsGradArgs& a, size_t slot0, bool live, int lpr, int glane, float (&dot)[KMAX]) {
  float mine = 0.0f;
#pragma unroll
  for (int j = 0; j < KMAX; ++j) {
    const float sum = segment_sum(dot[j], lpr);
    if (glane == j) mine = sum;
    if (lpr <= j && j < a.k && live && glane == 0) a.grad_weights[slot0 + j] = sum;  // (groups of fewer lanes than entries)
  }
  if (live && glane < min(a.k, KMAX)) a.grad_weights[slot0 + glane] = mine;
}

template <int DT, int LS, int UPR, int KMAX>
__global__ __launch_bounds__(kBlock) void dispatch_grad_kernel(RowsGradArgs a) {
  constexpr int NE = 16 / elem_bytes(DT);
  constexpr int LPR = 1 << LS;
  constexpr bool kStream = LS >= 4;  // rows of more than 128 bytes are not read again here
  const int lane = lane_id(), glane = lane & (LPR - 1);
  const long wave = static_cast<long>(blockIdx.x) * (kBlock / kWave) + (threadIdx.x >> 6);
  const long t = (wave << (6 - LS)) + (lane >> LS);
  const bool live = t < a.T;
  const size_t cell = live ? t : a.T - 1, slot0 = cell * a.k;
  int row[KMAX];
  float w[KMAX], dot[KMAX];
  bool has[KMAX];
  entries_of<KMAX>(a, slot0, live, row, w, has);
#pragma unroll
  for (int j = 0; j < KMAX; ++j) dot[j] = 0.0f;
  const bool dots = a.grad_weights != nullptr;
  for (int off0 = 0; off0 < a.cpr; off0 += LPR * UPR) {
    // every load is unconditional (clamped into its array, what does not belong to the sum cleared afterwards): loads
    // under conditions of their own wait for each other
    u32x4 val[KMAX][UPR], mine[UPR];
#pragma unroll
    for (int u = 0; u < UPR; ++u) {
      const int off = min(off0 + u * LPR + glane, a.cpr - 1);
#pragma unroll
      for (int j = 0; j < KMAX; ++j) val[j][u] = static_cast<const u32x4*>(a.grad)[static_cast<size_t>(row[j]) * a.cpr + off];
    }
    if (dots) {
#pragma unroll
      for (int u = 0; u < UPR; ++u)
        mine[u] = static_cast<const u32x4*>(a.operand)[cell * a.cpr + min(off0 + u * LPR + glane, a.cpr - 1)];
    }
#pragma unroll
    for (int u = 0; u < UPR; ++u) {
      const int off = off0 + u * LPR + glane;
      float acc[NE], x[NE];
      unpack<DT, 16>(dots && off < a.cpr ? mine[u] : zero_unit<16>(), x);
#pragma unroll
      for (int q = 0; q < NE; ++q) acc[q] = 0.0f;
#pragma unroll
      for (int j = 0; j < KMAX; ++j) {
        float g[NE];
        unpack<DT, 16>(has[j] && off < a.cpr ? val[j][u] : zero_unit<16>(), g);
#pragma unroll
        for (int q = 0; q < NE; ++q) {
          acc[q] += w[j] * g[q];
          dot[j] = __builtin_fmaf(x[q], g[q], dot[j]);
        }
      }
      if (a.out != nullptr && live && off < a.cpr)
        pack_store<DT, NE, kStream>(static_cast<u32x4*>(a.out) + cell * a.cpr + off, acc);
    }
  }
  if (dots) {
    // an entry without a row was summed as 0 * x, which an x that is not finite makes NaN: its gradient is zero
#pragma unroll
    for (int j = 0; j < KMAX; ++j) dot[j] = has[j] ? dot[j] : 0.0f;
    store_dots<KMAX>(a, slot0, live, LPR, glane, dot);
  }
}

template <int DT, bool G32, int LS, int UPR, int KMAX>
__global__ __launch_bounds__(kBlock) void combine_grad_kernel(RowsGradArgs a) {
  constexpr int NE = 16 / elem_bytes(DT);
  constexpr int LPR = 1 << LS;
  constexpr bool kStream = LS >= 4;
  const int lane = lane_id(), glane = lane & (LPR - 1);
  if (static_cast<int>(blockIdx.x) >= a.cell_blocks) {
    // rows that no entry owns: zeros.  A wavefront looks at 64 of them.
    const long wave = (static_cast<long>(blockIdx.x) - a.cell_blocks) * (kBlock / kWave) + (threadIdx.x >> 6);
    const long r0 = wave * kWave, n = static_cast<long>(a.T) * a.k;
    const int entry = r0 + lane < a.P ? a.row_entries[r0 + lane] : 0;
    unsigned long long bare = __ballot(r0 + lane < a.P && (entry < 1 || entry > n));
    u32x4* const out = static_cast<u32x4*>(a.out);
    while (bare != 0) {
      const long r = r0 + __builtin_ctzll(bare);
      bare &= bare - 1;
      for (int off = lane; off < a.cpr; off += kWave) out[r * a.cpr + off] = zero_unit<16>();
    }
    return;
  }
  const long wave = static_cast<long>(blockIdx.x) * (kBlock / kWave) + (threadIdx.x >> 6);
  const long t = (wave << (6 - LS)) + (lane >> LS);
  const bool live = t < a.T;
  const size_t cell = live ? t : a.T - 1, slot0 = cell * a.k;
  int row[KMAX], id[KMAX];
  float w[KMAX], dot[KMAX];
  bool has[KMAX], use[KMAX];
#pragma unroll
  for (int j = 0; j < KMAX; ++j) id[j] = a.ids[slot0 + min(j, a.k - 1)];
  entries_of<KMAX>(a, slot0, live, row, w, has);
  // of the entries of a cell that name one path the combine adds the first one that owns a row
#pragma unroll
  for (int j = 0; j < KMAX; ++j) {
    use[j] = has[j] && id[j] != 0x7fffffff;
#pragma unroll
    for (int i = 0; i < j; ++i) use[j] = use[j] && !(has[i] && id[i] == id[j]);
    dot[j] = 0.0f;
  }
  const bool dots = a.grad_weights != nullptr;
  for (int off0 = 0; off0 < a.cpr; off0 += LPR * UPR) {
    u32x4 val[KMAX][UPR];
    float g[UPR][NE];
#pragma unroll
    for (int u = 0; u < UPR; ++u)
      load_unit<DT, G32, NE>(a.grad, cell * a.cpr + min(off0 + u * LPR + glane, a.cpr - 1), g[u]);
    if (dots) {
#pragma unroll
      for (int u = 0; u < UPR; ++u) {
        const int off = min(off0 + u * LPR + glane, a.cpr - 1);
#pragma unroll
        for (int j = 0; j < KMAX; ++j) val[j][u] = static_cast<const u32x4*>(a.operand)[static_cast<size_t>(row[j]) * a.cpr + off];
      }
    }
#pragma unroll
    for (int u = 0; u < UPR; ++u) {
      const int off = off0 + u * LPR + glane;
#pragma unroll
      for (int j = 0; j < KMAX; ++j) {
        float o[NE];
        if (dots) {
          float y[NE];
          const bool counts = use[j] && off < a.cpr;
          unpack<DT, 16>(counts ? val[j][u] : zero_unit<16>(), y);
#pragma unroll
          for (int q = 0; q < NE; ++q) dot[j] = __builtin_fmaf(y[q], counts ? g[u][q] : 0.0f, dot[j]);
        }
#pragma unroll
        for (int q = 0; q < NE; ++q) o[q] = use[j] ? w[j] * g[u][q] : 0.0f;
        if (a.out != nullptr && has[j] && off < a.cpr)
          pack_store<DT, NE, kStream>(static_cast<u32x4*>(a.out) + static_cast<size_t>(row[j]) * a.cpr + off, o);
      }
    }
  }
  if (dots) store_dots<KMAX>(a, slot0, live, LPR, glane, dot);
}

// Lanes per row by its length (16-byte units), units a lane has in flight by the entries of a cell.
template <typename F>
void with_row_shape(int cpr, int k, F&& launch) {
  using std::integral_constant;
  auto with_k = [&](auto ls, auto upr1, auto upr2) {
    if (k == 1) launch(ls, upr1, integral_constant<int, 1>{});
    else if (k == 2) launch(ls, upr2, integral_constant<int, 2>{});
    else if (k <= 4) launch(ls, integral_constant<int, 1>{}, integral_constant<int, 4>{});
    else launch(ls, integral_constant<int, 1>{}, integral_constant<int, 8>{});
  };
  constexpr integral_constant<int, 1> one;
  constexpr integral_constant<int, 2> two;
  if (cpr > kWave) with_k(integral_constant<int, 6>{}, two, two);
  else if (cpr > 32) with_k(integral_constant<int, 6>{}, one, one);
  else if (cpr > 16) with_k(integral_constant<int, 5>{}, one, one);
  else if (cpr > 8) with_k(integral_constant<int, 4>{}, one, one);
  else if (cpr > 4) with_k(integral_constant<int, 3>{}, one, one);
  else with_k(integral_constant<int, 2>{}, one, one);
}

int check_rows(RowsGradArgs& a, int T, int k, int cell, int P, int dtype, const void* const* units, int n_units) {
  if (T < 0 || k <= 0 || cell < 0 || P < 0) return fail(BRT_E_INVALID, "bad shape T=%d k=%d cell=%d P=%d", T, k, cell, P);
  if (k > kMaxK) return fail(BRT_E_UNSUPPORTED, "more than %d paths per cell", kMaxK);
  if (dtype != BRT_F32 && dtype != BRT_F16 && dtype != BRT_BF16) return fail(BRT_E_UNSUPPORTED, "dtype %d is not supported", dtype);
  if (static_cast<long>(T) * k >= (1l << 31)) return fail(BRT_E_UNSUPPORTED, "T*k >= 2^31");
  const size_t row_bytes = static_cast<size_t>(cell) * elem_bytes(dtype);
  bool whole = row_bytes % 16 == 0;
  for (int i = 0; i < n_units; ++i) whole = whole && (units[i] == nullptr || aligned(units[i], 16));
  if (!whole) return fail(BRT_E_UNSUPPORTED, "rows must be whole 16-byte units (row is %zu bytes)", row_bytes);
  a.T = T; a.P = P; a.k = k;
  a.cpr = static_cast<int>(row_bytes / 16);
  return BRT_OK;
}

// Workgroups for the cells: 64 >> ls cells a wavefront.
unsigned blocks_of_cells(int T, int ls) {
  const long cells_pb = static_cast<long>(kBlock / kWave) << (6 - ls);
  return static_cast<unsigned>((T + cells_pb - 1) / cells_pb);
}

}  // namespace
}  // namespace brt

using namespace brt;

extern "C" int brt_hip_gate_topk_grad(const void* scores, const int32_t* path_ids, const float* weights, const float* grad,
                                      void* grad_scores, int T, int E, int k, int dtype, int softmax, void* stream) {
  if (T < 0 || E <= 0 || k < 0 || k > E) return fail(BRT_E_INVALID, "bad shape T=%d E=%d k=%d", T, E, k);
  if (dtype != BRT_F32 && dtype != BRT_F16 && dtype != BRT_BF16) return fail(BRT_E_UNSUPPORTED, "dtype %d is not supported", dtype);
  if (E > 1024) return fail(BRT_E_UNSUPPORTED, "more than 1024 paths");
  if (static_cast<long>(T) * E >= (1l << 31)) return fail(BRT_E_UNSUPPORTED, "T*E >= 2^31");
  if (T == 0) return BRT_OK;
  if ((softmax && !scores) || !grad_scores || (k > 0 && (!path_ids || !grad || (softmax && !weights)))) return fail(BRT_E_INVALID, "null argument");
  GateGradArgs a{scores, path_ids, weights, grad, grad_scores, T, E, k, softmax, 0};
  const int per = 16 / elem_bytes(dtype);
  const bool units = E % per == 0 && aligned(scores, 16) && aligned(grad_scores, 16);
  const int n = units ? E / per : E;
  while ((1 << a.ls) < std::min(n, kWave)) ++a.ls;
  const long rows_pb = static_cast<long>(kBlock / kWave) << (6 - a.ls);
  const dim3 grid(static_cast<unsigned>((T + rows_pb - 1) / rows_pb)), block(kBlock);
  hipStream_t st = as_stream(stream);
#define BRT_GRAD(DT, V, STEPS) hipLaunchKernelGGL((gate_grad_kernel<DT, V, STEPS>), grid, block, 0, st, a)
#define BRT_GRAD_DT(DT, V)                                                            \
  if (units) {                                                                        \
    if (n <= kWave) BRT_GRAD(DT, V, 1); else BRT_GRAD(DT, V, 16 / V);                 \
  } else if (n <= kWave) BRT_GRAD(DT, 1, 1);                                          \
  else if (n <= 4 * kWave) BRT_GRAD(DT, 1, 4);                                        \
  else BRT_GRAD(DT, 1, 16);
  if (dtype == BRT_F32) { BRT_GRAD_DT(BRT_F32, 4) }
  else if (dtype == BRT_F16) { BRT_GRAD_DT(BRT_F16, 8) }
  else { BRT_GRAD_DT(BRT_BF16, 8) }
#undef BRT_GRAD_DT
#undef BRT_GRAD
  return check_launch("gate_grad_kernel");
}

extern "C" int brt_hip_dispatch_by_rows_grad(const void* grad_rows, const void* cells, const float* weights,
                                             const int32_t* seat_rows, void* grad_cells, float* grad_weights, int T, int k,
                                             int cell, int P, int dtype, void* stream) {
  RowsGradArgs a{};
  const void* const units[] = {grad_rows, cells, grad_cells};
  const int rc = check_rows(a, T, k, cell, P, dtype, units, 3);
  if (rc != BRT_OK) return rc;
  if (T == 0 || (!grad_cells && !grad_weights)) return BRT_OK;
  if (!seat_rows || (P > 0 && cell > 0 && !grad_rows) || (grad_weights && cell > 0 && !cells)) return fail(BRT_E_INVALID, "null argument");
  if (cell == 0) a.P = 0;
  a.grad = grad_rows; a.operand = cells; a.weights = weights; a.seat_rows = seat_rows; a.out = grad_cells; a.grad_weights = grad_weights;
  if (P == 0) a.grad = grad_cells ? grad_cells : cells;  // (entries without a row fetch the first one, and drop it)
  hipStream_t st = as_stream(stream);
#define BRT_LAUNCH(DT)                                                                                             \
  with_row_shape(a.cpr, k, [&](auto ls, auto upr, auto km) {                                                       \
    constexpr int LS = decltype(ls)::value, UPR = decltype(upr)::value, KM = decltype(km)::value;                  \
    hipLaunchKernelGGL((dispatch_grad_kernel<DT, LS, UPR, KM>), dim3(blocks_of_cells(T, LS)), dim3(kBlock), 0, st, a); \
  });
  if (dtype == BRT_F32) BRT_LAUNCH(BRT_F32)
  else if (dtype == BRT_F16) BRT_LAUNCH(BRT_F16)
  else BRT_LAUNCH(BRT_BF16)
#undef BRT_LAUNCH
  return check_launch("dispatch_grad_kernel");
}

extern "C" int brt_hip_combine_by_rows_grad(const void* grad, const void* rows, const float* weights, const int32_t* path_ids,
                                            const int32_t* seat_rows, const int32_t* row_entries, void* grad_rows,
                                            float* grad_weights, int T, int k, int cell, int P, int dtype, int grad_dtype,
                                            void* stream) {
  RowsGradArgs a{};
  const void* const units[] = {grad, rows, grad_rows};
  const int rc = check_rows(a, T, k, cell, P, dtype, units, 3);
  if (rc != BRT_OK) return rc;
  if (grad_dtype != dtype && grad_dtype != BRT_F32) return fail(BRT_E_UNSUPPORTED, "dtype pair %d -> %d is not supported", dtype, grad_dtype);
  if (!grad_rows && !grad_weights) return BRT_OK;
  if ((T > 0 && (!seat_rows || !path_ids || (cell > 0 && !grad))) || (grad_rows && P > 0 && cell > 0 && !row_entries) ||
      (grad_weights && P > 0 && cell > 0 && !rows))
    return fail(BRT_E_INVALID, "null argument");
  if (cell == 0) a.P = 0;
  a.grad = grad; a.operand = rows; a.weights = weights; a.ids = path_ids; a.seat_rows = seat_rows; a.row_entries = row_entries;
  a.out = a.P > 0 ? grad_rows : nullptr; a.grad_weights = grad_weights;
  if (P == 0) a.operand = grad;  // (entries without a row fetch the first one, and drop it)
  const unsigned clearing = a.out != nullptr ? static_cast<unsigned>((static_cast<long>(P) + kBlock - 1) / kBlock) : 0;
  hipStream_t st = as_stream(stream);
#define BRT_LAUNCH(DT, G32)                                                                                       \
  with_row_shape(a.cpr, k, [&](auto ls, auto upr, auto km) {                                                      \
    constexpr int LS = decltype(ls)::value, UPR = decltype(upr)::value, KM = decltype(km)::value;                 \
    a.cell_blocks = static_cast<int>(blocks_of_cells(T, LS));                                                     \
    if (a.cell_blocks + clearing > 0)                                                                             \
      hipLaunchKernelGGL((combine_grad_kernel<DT, G32, LS, UPR, KM>), dim3(a.cell_blocks + clearing), dim3(kBlock), 0, st, a); \
  });
  if (dtype == BRT_F32) BRT_LAUNCH(BRT_F32, false)
  else if (dtype == BRT_F16 && grad_dtype == BRT_F16) BRT_LAUNCH(BRT_F16, false)
  else if (dtype == BRT_F16) BRT_LAUNCH(BRT_F16, true)
  else if (grad_dtype == BRT_BF16) BRT_LAUNCH(BRT_BF16, false)
  else BRT_LAUNCH(BRT_BF16, true)
#undef BRT_LAUNCH
  return check_launch("combine_grad_kernel");
}
