// The losses that keep a router balanced, and their gradient (no counterpart in the reference, whose ops are not
// differentiable).  Of scores s [T,E] and the paths chosen from them, over the n cells that count:
//
//   p = softmax(s[t])      lse = log(sum exp s[t])      counts[e] = entries that name path e
//   balance = E / (n n k) * sum_e counts[e] * sum_t p[t,e]           z = 1/n * sum_t lse[t]^2
//   ds[t,e] = p[t,e] * (c[e] - sum_i c[i] p[t,i] + q lse[t])         c = g_balance E / (n n k) counts,  q = g_z 2 / n
//
// A row is held by 1 << ls lanes, STEPS units of V columns each (the longest unit of up to 16 bytes that rows are whole numbers
// of), so every lane keeps its columns for all rows of its wavefront: the column sums stay in registers, go through LDS
// once per workgroup and to memory as one vector of E per workgroup, which a second launch adds up (one launch, one workgroup, for
// small batches).  No floating-point atomics: the order of every sum follows from the sizes.  Exponents are taken of s - max, so rows of the
// type's lowest value have a softmax; a cell that does not count is read as zeros, whatever it holds.
//   What bounds it (MI355X, the least of 40 launches; their mean is up to 0.6 us more): 65536 x 128 bf16 10.4-10.8 us forward (16.8 MB, 1.6
// TB/s), 6.0-6.2 to join 256 workgroups' sums and 13.0-13.4 backward (33.6 MB, 2.5 TB/s), where the bytes alone take 3.3 and 6.5: a launch, a
// round of loads and the exchanges along a row that follow one another (four rows at a time hide part of them: the gradient takes 20.9 with one), vector instructions 0.32 and 0.23 of the time.  1024 x 16 fp32
// 7.1 + 3.4, 4099 x 60 fp16 6.4 + 5.2 + 3.6 us: launches and dependent loads, and behind them a reduction whose end one thread adds up.
#include <algorithm>

#include "gate.hpp"
#include "rows.hpp"

namespace brt {
namespace {

constexpr int kMostWaves = 16;    // of a workgroup of the losses; 8 above 512 paths, so that its column sums fit LDS
constexpr int kMostBlocks = 256;  // one per CU: the second launch reads 8 bytes per column of each
constexpr int kMostPaths = 1024;
constexpr float kLog2E = 1.44269504088896341f;

struct BalanceArgs {
  const void* scores;
  const int* ids;
  const uint8_t* counted;  // [T] or null
  float* balance;
  float* z;
  int* counts;         // [E]
  float* row_stats;    // [T, 2] max and sum of the exponentials, or null
  float* coefficients; // [E + 1] c and q of unit gradients, or null
  float* part_p;       // [blocks][columns]
  int* part_counts;    // [blocks][columns]
  float* part_z;       // [blocks]
  int* part_n;         // [blocks]
  int T, E, k, blocks;
  int columns;  // E rounded up to a multiple of 4
  int ls;  // log2 of the lanes that share a row
};

// exp(x) for x <= 0, within 2 + 1.23 |x| steps of 2^-24 (the product's rounding is up to |x| of them, the constant's 0.22 |x|): small
// exponents are exact to the last bits, where the large probabilities are
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2E); }

// Column sums and what belongs to the batch -> the losses, the counts and the gradient's coefficients; by the whole workgroup.
// column(e, &p, &count) gives the sums of a column.
template <typename F>
__device__ __forceinline__ void finish(const BalanceArgs& a, double z, long n, double* s_dot, F&& column) {
  const double entries = static_cast<double>(n) * a.k;
  const double scale = n > 0 && a.k > 0 ? a.E / (entries * n) : 0.0;
  double dot = 0.0;
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    double p;
    int count;
    column(e, &p, &count);
    dot += p * count;
    a.counts[e] = count;
    if (a.coefficients != nullptr) a.coefficients[e] = static_cast<float>(scale * count);
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) dot += __shfl_xor(dot, d, kWave);
  if (lane_id() == 0) s_dot[threadIdx.x >> 6] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int w = 0; w < static_cast<int>(blockDim.x) / kWave; ++w) sum += s_dot[w];
    *a.balance = static_cast<float>(scale * sum);
    *a.z = n > 0 ? static_cast<float>(z / n) : 0.0f;
    if (a.coefficients != nullptr) a.coefficients[a.E] = n > 0 ? static_cast<float>(2.0 / n) : 0.0f;
  }
}

template <int DT, int V, int STEPS, int ROWS>
__global__ __launch_bounds__(kMostWaves * kWave) void balance_kernel(BalanceArgs a) {
  extern __shared__ float s_p[];  // [waves][E], and the counts [E]
  const int waves = blockDim.x / kWave;
  int* const s_counts = reinterpret_cast<int*>(s_p + waves * a.E);
  __shared__ float s_z[kMostWaves];
  __shared__ int s_n[kMostWaves];
  __shared__ double s_dot[kMostWaves];
  constexpr int kBytes = V * elem_bytes(DT);
  using U = typename Unit<kBytes>::type;
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const int ls = a.ls, lpr = 1 << ls, glane = lane & (lpr - 1), per = kWave >> ls;  // rows of a wavefront side by side
  const int units = a.E / V;
  // the rows of a workgroup lie side by side; its wavefronts take them in turn, ROWS loads at a time
  const long share = (static_cast<long>(a.T) + a.blocks - 1) / a.blocks;
  const long first = min(share * blockIdx.x, static_cast<long>(a.T)), last = min(first + share, static_cast<long>(a.T));
  // entries of those rows, by path (whole numbers: their order does not matter); a thread's first one is fetched ahead of the scores
  const long entry0 = first * a.k + threadIdx.x, entries = last * a.k;
  auto path_of = [&](long i) {
    const bool there = i < entries && (a.counted == nullptr || a.counted[static_cast<uint32_t>(i) / a.k] != 0);
    const int id = there ? a.ids[i] : -1;
    return id < a.E ? id : -1;
  };
  const int path0 = path_of(entry0);
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) s_counts[e] = 0;
  __syncthreads();
  float acc[STEPS][V];
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int v = 0; v < V; ++v) acc[s][v] = 0.0f;
  float z = 0.0f;
  int n = 0;
  for (long r0 = first + wave * (per * ROWS); r0 < last; r0 += waves * per * ROWS) {
    U raw[ROWS][STEPS];
    bool use[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const long row = r0 + i * per + (lane >> ls), at = min(row, last - 1);
      use[i] = row < last && (a.counted == nullptr || a.counted[at] != 0);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) raw[i][s] = static_cast<const U*>(a.scores)[at * units + min(s * lpr + glane, units - 1)];
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const long row = r0 + i * per + (lane >> ls);
      float x[STEPS][V], top = -INFINITY;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        unpack<DT, kBytes>(use[i] ? raw[i][s] : zero_unit<kBytes>(), x[s]);
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (s * lpr + glane < units) top = fmaxf(top, x[s][v]);
      }
      top = segment_max(top, lpr);
      float sum = 0.0f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          x[s][v] = exp_of(x[s][v] - top);
          if (s * lpr + glane < units) sum += x[s][v];
        }
      sum = segment_sum(sum, lpr);
      const float inverse = use[i] ? 1.0f / sum : 0.0f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[s][v] = __builtin_fmaf(x[s][v], inverse, acc[s][v]);
      if (glane == 0 && row < last) {
        if (use[i]) {
          const float lse = top + logf(sum);
          z += lse * lse;
          ++n;
        }
        if (a.row_stats != nullptr) *reinterpret_cast<f32x2*>(a.row_stats + 2 * row) = f32x2{top, sum};
      }
    }
  }
  if (path0 >= 0) atomicAdd(&s_counts[path0], 1);
  for (long i = entry0 + blockDim.x; i < entries; i += blockDim.x) {
    const int path = path_of(i);
    if (path >= 0) atomicAdd(&s_counts[path], 1);
  }
  for (int d = lpr; d < kWave; d <<= 1) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[s][v] += __shfl_xor(acc[s][v], d, kWave);
  }
  if (lane < lpr) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (s * lpr + lane < units) s_p[wave * a.E + (s * lpr + lane) * V + v] = acc[s][v];
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) z += __shfl_xor(z, d, kWave), n += __shfl_xor(n, d, kWave);
  if (lane == 0) s_z[wave] = z, s_n[wave] = n;
  __syncthreads();
  float block_z = 0.0f;
  int block_n = 0;
  for (int w = 0; w < waves; ++w) block_z += s_z[w], block_n += s_n[w];
  auto column = [&](int e, auto* p, int* count) {
    float sum = 0.0f;
#pragma unroll 4
    for (int w = 0; w < waves; ++w) sum += s_p[w * a.E + e];
    *p = sum, *count = s_counts[e];
  };
  if (a.blocks == 1) return finish(a, block_z, block_n, s_dot, column);
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    const size_t at = static_cast<size_t>(blockIdx.x) * a.columns + e;
    column(e, &a.part_p[at], &a.part_counts[at]);
  }
  if (threadIdx.x == 0) a.part_z[blockIdx.x] = block_z, a.part_n[blockIdx.x] = block_n;
}

// The workgroups' sums added up: a thread takes four columns of every `slices`-th of them, up to eight requests of 16 bytes at once
// (256 workgroups of 128 columns 6.0 us; one column a thread 6.5).
constexpr int kJoin = 1024;
__global__ __launch_bounds__(kJoin) void balance_join_kernel(BalanceArgs a, int slices) {
  __shared__ double s_p[kJoin * 4];
  __shared__ int s_counts[kJoin * 4];
  __shared__ double s_dot[kJoin / kWave], s_z[kJoin / kWave];
  __shared__ int s_n[kJoin / kWave];
  const int width = kJoin / slices, slice = threadIdx.x / width, unit = threadIdx.x % width, units = a.columns / 4;
  double p[4] = {0.0, 0.0, 0.0, 0.0};
  int count[4] = {0, 0, 0, 0};
  if (unit < units) {
#pragma unroll 4
    for (int b = slice; b < a.blocks; b += slices) {
      const size_t at = static_cast<size_t>(b) * units + unit;
      const f32x4 more = reinterpret_cast<const f32x4*>(a.part_p)[at];
      const u32x4 counted = reinterpret_cast<const u32x4*>(a.part_counts)[at];
#pragma unroll
      for (int q = 0; q < 4; ++q) p[q] += more[q], count[q] += static_cast<int>(counted[q]);
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) s_p[threadIdx.x * 4 + q] = p[q], s_counts[threadIdx.x * 4 + q] = count[q];
  double z = 0.0;
  int n = 0;
  for (int b = threadIdx.x; b < a.blocks; b += kJoin) z += a.part_z[b], n += a.part_n[b];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) z += __shfl_xor(z, d, kWave), n += __shfl_xor(n, d, kWave);
  if (lane_id() == 0) s_z[threadIdx.x >> 6] = z, s_n[threadIdx.x >> 6] = n;
  for (int half = slices / 2; half > 0; half /= 2) {
    __syncthreads();
    if (slice < half) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        s_p[threadIdx.x * 4 + q] += s_p[(threadIdx.x + half * width) * 4 + q];
        s_counts[threadIdx.x * 4 + q] += s_counts[(threadIdx.x + half * width) * 4 + q];
      }
    }
  }
  __syncthreads();
  z = 0.0, n = 0;
  for (int w = 0; w < kJoin / kWave; ++w) z += s_z[w], n += s_n[w];
  finish(a, z, n, s_dot, [&](int column, double* sum, int* total) { *sum = s_p[column], *total = s_counts[column]; });
}

struct BalanceGradArgs {
  const void* scores;
  const uint8_t* counted;
  const float* row_stats;
  const float* coefficients;
  const float* grad_balance;  // one value each, or null
  const float* grad_z;
  void* out;
  int T, E, ls;
};

template <int DT, int V, int STEPS, int ROWS>
__global__ __launch_bounds__(256) void balance_grad_kernel(BalanceGradArgs a) {
  constexpr int kBytes = V * elem_bytes(DT);
  using U = typename Unit<kBytes>::type;
  const int lane = lane_id(), ls = a.ls, lpr = 1 << ls, glane = lane & (lpr - 1), per = kWave >> ls, units = a.E / V;
  const float by = a.grad_balance != nullptr ? *a.grad_balance : 0.0f;
  const float q = a.grad_z != nullptr ? *a.grad_z * a.coefficients[a.E] : 0.0f;
  float c[STEPS][V];
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = (s * lpr + glane) * V + v;
      c[s][v] = a.grad_balance != nullptr && e < a.E ? by * a.coefficients[e] : 0.0f;
    }
  const long wave = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const long r0 = wave * ROWS * per + (lane >> ls);
  U raw[ROWS][STEPS];
  f32x2 stats[ROWS];
  bool use[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const long at = min(r0 + i * per, static_cast<long>(a.T) - 1);
    use[i] = a.counted == nullptr || a.counted[at] != 0;
    stats[i] = reinterpret_cast<const f32x2*>(a.row_stats)[at];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) raw[i][s] = static_cast<const U*>(a.scores)[at * units + min(s * lpr + glane, units - 1)];
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const long row = r0 + i * per;
    const float top = stats[i][0], inverse = 1.0f / stats[i][1];
    float p[STEPS][V], dot = 0.0f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      unpack<DT, kBytes>(raw[i][s], p[s]);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        p[s][v] = exp_of(p[s][v] - top) * inverse;
        if (s * lpr + glane < units) dot = __builtin_fmaf(c[s][v], p[s][v], dot);
      }
    }
    dot = segment_sum(dot, lpr);
    if (a.grad_z != nullptr) dot -= q * (top + logf(stats[i][1]));
    if (row >= a.T) continue;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      float o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = use[i] ? p[s][v] * (c[s][v] - dot) : 0.0f;
      const int u = s * lpr + glane;
      if (u < units) pack_store<DT, V>(static_cast<char*>(a.out) + (static_cast<size_t>(row) * units + u) * kBytes, o);
    }
  }
}

int check_scores(int T, int E, int dtype) {
  if (T < 0 || E <= 0) return fail(BRT_E_INVALID, "bad shape T=%d E=%d", T, E);
  if (dtype != BRT_F32 && dtype != BRT_F16 && dtype != BRT_BF16) return fail(BRT_E_UNSUPPORTED, "dtype %d is not supported", dtype);
  if (E > kMostPaths) return fail(BRT_E_UNSUPPORTED, "more than %d paths", kMostPaths);
  if (static_cast<long>(T) * E >= (1l << 31)) return fail(BRT_E_UNSUPPORTED, "T*E >= 2^31");
  return BRT_OK;
}

// Lanes that share a row of n units.
int lanes_of(int n) {
  int ls = 0;
  while ((1 << ls) < std::min(n, kWave)) ++ls;
  return ls;
}

int columns_of(int E) { return (E + 3) & ~3; }

// Workgroups of the losses: one, and one launch, while that takes no longer than two (2048 x 16 fp32 10.5 us, 10.1 with two; 4096 x 16
// 16.7 and 10.3), 2048 scores each and more beyond.
int blocks_of(int T, int E) {
  const long scores = static_cast<long>(T) * E;
  if (scores <= (1 << 15)) return 1;
  return static_cast<int>(std::min<long>(kMostBlocks, (scores + (1 << 11) - 1) >> 11));
}

// The kernel of a row shape: launch(type, V, STEPS, ROWS), `lanes` the log2 of the lanes that share a row.  ROWS loads of a wavefront at a time.
template <int ROWS, typename F>
void with_scores(int dtype, int E, const void* const* rows, int n_rows, int* lanes, F&& launch) {
  using std::integral_constant;
  auto fits = [&](int V) {
    bool ok = E % V == 0;
    for (int i = 0; i < n_rows; ++i) ok = ok && aligned(rows[i], V * elem_bytes(dtype));
    return ok;
  };
  auto shape = [&](auto dt, auto v) {
    constexpr int V = decltype(v)::value;
    const int n = E / V;
    *lanes = lanes_of(n);
    if (n <= kWave) launch(dt, v, integral_constant<int, 1>{}, integral_constant<int, ROWS>{});
    else if (n <= 4 * kWave) launch(dt, v, integral_constant<int, V == 8 ? 2 : 4>{}, integral_constant<int, 1>{});
    else if constexpr (V <= 2) launch(dt, v, integral_constant<int, V == 2 ? 8 : 16>{}, integral_constant<int, 1>{});
  };
  auto type = [&](auto dt) {
    if constexpr (decltype(dt)::value != BRT_F32)
      if (fits(8)) return shape(dt, integral_constant<int, 8>{});
    if (fits(4)) return shape(dt, integral_constant<int, 4>{});
    if (fits(2)) return shape(dt, integral_constant<int, 2>{});
    return shape(dt, integral_constant<int, 1>{});
  };
  if (dtype == BRT_F32) type(integral_constant<int, BRT_F32>{});
  else if (dtype == BRT_F16) type(integral_constant<int, BRT_F16>{});
  else type(integral_constant<int, BRT_BF16>{});
}

}  // namespace
}  // namespace brt

using namespace brt;

extern "C" size_t brt_hip_balance_loss_workspace_bytes(int T, int E) {
  if (T < 0 || E <= 0 || E > kMostPaths || static_cast<long>(T) * E >= (1l << 31)) return 0;
  const int blocks = blocks_of(T, E);
  return blocks == 1 ? 0 : static_cast<size_t>(blocks) * (columns_of(E) + 1) * 8;
}

extern "C" int brt_hip_balance_loss(const void* scores, const int32_t* path_ids, const uint8_t* counted, float* balance, float* z,
                                    int32_t* counts, float* row_stats, float* coefficients, int T, int E, int k, int dtype,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check_scores(T, E, dtype); rc != BRT_OK) return rc;
  if (k < 0) return fail(BRT_E_INVALID, "bad shape k=%d", k);
  if (static_cast<long>(T) * k >= (1l << 31)) return fail(BRT_E_UNSUPPORTED, "T*k >= 2^31");
  if ((T > 0 && (!scores || (k > 0 && !path_ids))) || !balance || !z || !counts) return fail(BRT_E_INVALID, "null argument");
  if (row_stats && !aligned(row_stats, 8)) return fail(BRT_E_UNSUPPORTED, "row_stats is not aligned to 8 bytes");
  BalanceArgs a{scores, path_ids, counted, balance, z, counts, row_stats, coefficients, nullptr, nullptr, nullptr, nullptr, T, E, k, blocks_of(T, E), columns_of(E), 0};
  if (a.blocks > 1) {
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < brt_hip_balance_loss_workspace_bytes(T, E))
      return fail(BRT_E_WORKSPACE, "workspace of %zu bytes needed, got %zu", brt_hip_balance_loss_workspace_bytes(T, E), workspace_bytes);
    a.part_p = static_cast<float*>(workspace);
    a.part_counts = static_cast<int*>(workspace) + static_cast<size_t>(a.blocks) * a.columns;
    a.part_z = a.part_p + static_cast<size_t>(a.blocks) * a.columns * 2;
    a.part_n = static_cast<int*>(workspace) + static_cast<size_t>(a.blocks) * (2 * a.columns + 1);
  }
  hipStream_t st = as_stream(stream);
  const int waves = E > 512 ? kMostWaves / 2 : kMostWaves;
  with_scores<4>(dtype, E, &scores, 1, &a.ls, [&](auto dt, auto v, auto steps, auto rows) {
    hipLaunchKernelGGL((balance_kernel<decltype(dt)::value, decltype(v)::value, decltype(steps)::value, decltype(rows)::value>),
                       dim3(a.blocks), dim3(waves * kWave), (waves + 1) * E * 4, st, a);
  });
  if (const int rc = check_launch("balance_kernel"); rc != BRT_OK || a.blocks == 1) return rc;
  int slices = 1;
  while (slices < 64 && kJoin / (2 * slices) >= a.columns / 4) slices *= 2;
  hipLaunchKernelGGL(balance_join_kernel, dim3(1), dim3(kJoin), 0, st, a, slices);
  return check_launch("balance_join_kernel");
}

extern "C" int brt_hip_balance_loss_grad(const void* scores, const uint8_t* counted, const float* row_stats, const float* coefficients,
                                         const float* grad_balance, const float* grad_z, void* grad_scores, int T, int E, int dtype,
                                         void* stream) {
  if (const int rc = check_scores(T, E, dtype); rc != BRT_OK) return rc;
  if (T == 0) return BRT_OK;
  if (!scores || !row_stats || !coefficients || !grad_scores) return fail(BRT_E_INVALID, "null argument");
  if (!aligned(row_stats, 8)) return fail(BRT_E_UNSUPPORTED, "row_stats is not aligned to 8 bytes");
  BalanceGradArgs a{scores, counted, row_stats, coefficients, grad_balance, grad_z, grad_scores, T, E, 0};
  hipStream_t st = as_stream(stream);
  const void* const both[] = {scores, grad_scores};
  auto launch = [&](auto dt, auto v, auto steps, auto rows) {
    constexpr int R = decltype(rows)::value;
    const long rows_pb = static_cast<long>(4 * R) << (6 - a.ls);
    hipLaunchKernelGGL((balance_grad_kernel<decltype(dt)::value, decltype(v)::value, decltype(steps)::value, R>),
                       dim3(static_cast<unsigned>((T + rows_pb - 1) / rows_pb)), dim3(256), 0, st, a);
  };
  // (65536 x 128 bf16 12.8 us with four rows at a time, 20.9 with one; 8192 x 64 fp32 3.8 and 3.4, 4099 x 60 fp16 3.6 and 2.7)
  if (static_cast<long>(T) * E >= 1 << 20) with_scores<4>(dtype, E, both, 2, &a.ls, launch);
  else with_scores<1>(dtype, E, both, 2, &a.ls, launch);
  return check_launch("balance_grad_kernel");
}
