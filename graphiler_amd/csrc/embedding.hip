// Embedding rows and their table's gradient:
//
//   y_i = scale table[id_i],      grad_table[v] = scale sum over i with id_i = v of gy_i
//
// Both move rows, 16 bytes a lane (32 of fp32), LANES lanes a row, and are bound by that.  For the gradient the places i are
// first brought into the order of their ids (the stable counting sort of graph_prep.hip), so that every row of the table is
// the sum of rows that are named side by side: no atomics, one order, each row written once.  A row that more than kRun
// places name is cut into the runs of kRun places that the whole list is cut into; such a run holds the end of one long
// row at most and the beginning of another, whose sums a last launch adds up.
//
// 262,144 rows of 512 bf16 of a table of 32,000: 63 us, 4.8 TB/s.  Gradient of 65,536 rows of 1024, ids of a power law: 61 us for the rows,
// 15 + 6 for the long ones, 42 for the sort (eight short launches); cut at 128 places instead of 64 the longest rows held the
// launch, 74.
#include "vec8.h"

namespace ga {
namespace {

constexpr int kRun = 64;

// The id of place i, or -1 where it names no row.
__device__ __forceinline__ int64_t id_at(const void *ids, int bits, int64_t i, int64_t n_table) {
  const int64_t v = bits == 64 ? ((const int64_t *)ids)[i] : (int64_t)((const int32_t *)ids)[i];
  return v >= 0 && v < n_table ? v : -1;
}

// n values of a row that is not read again here: kept out of the caches, which hold the table.  262,144 rows of 512 bf16 of a
// table of 32,000: 78 -> 63 us.
template <typename T>
__device__ __forceinline__ void store_once(T *p, int n, const float (&f)[kVec]) {
  typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
  if (n < kVec) {
    store_group(p, n, f);
  } else if constexpr (sizeof(T) == 2) {
    any4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack_bf16(f[2 * j], f[2 * j + 1]);
    __builtin_nontemporal_store(w, reinterpret_cast<any4 *>(p));
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      any4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(f[4 * k + j]);
      __builtin_nontemporal_store(w, reinterpret_cast<any4 *>(p + 4 * k));
    }
  }
}

template <typename T, int LANES>
__global__ __launch_bounds__(kBlock) void embedding_kernel(const T *__restrict__ table, const void *__restrict__ ids, int bits,
                                                           T *__restrict__ y, int64_t n_ids, int64_t n_table, int64_t cols,
                                                           float scale) {
  constexpr int kRows = kBlock / LANES, kDeep = 4;           // rows a workgroup has at a time, a lane's rows on their way
  const int64_t col = ((int64_t)blockIdx.y * LANES + threadIdx.x % LANES) * kVec;
  const int64_t first = (int64_t)blockIdx.x * (kRows * kDeep) + threadIdx.x / LANES;
  if (col >= cols) return;
  const int n = (int)min((int64_t)kVec, cols - col);
  int64_t v[kDeep];
#pragma unroll
  for (int d = 0; d < kDeep; ++d) {
    const int64_t i = first + d * kRows;
    v[d] = i < n_ids ? id_at(ids, bits, i, n_table) : -1;
  }
  float f[kDeep][kVec];
#pragma unroll
  for (int d = 0; d < kDeep; ++d) load_group(table + max(v[d], (int64_t)0) * cols + col, v[d] < 0 ? 0 : n, f[d]);
#pragma unroll
  for (int d = 0; d < kDeep; ++d) {
    const int64_t i = first + d * kRows;
    if (i >= n_ids) break;
#pragma unroll
    for (int j = 0; j < kVec; ++j) f[d][j] *= scale;
    store_once(y + i * cols + col, n, f[d]);
  }
}

// Keys of the sort: the ids, n_table for those that name no row.
__global__ __launch_bounds__(kBlock) void embedding_keys_kernel(const void *__restrict__ ids, int bits, int64_t n_ids,
                                                                int64_t n_table, int64_t *__restrict__ keys) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n_ids; i += (int64_t)gridDim.x * kBlock) {
    const int64_t v = id_at(ids, bits, i, n_table);
    keys[i] = v < 0 ? n_table : v;
  }
}

// f += the rows of gy that places[from] ... places[to - 1] name
template <typename T>
__device__ __forceinline__ void add_rows(const T *__restrict__ gy, const int32_t *__restrict__ places, int32_t from, int32_t to,
                                         int64_t cols, int64_t col, int n, float (&f)[kVec]) {
  constexpr int kDeep = 8;
  for (int32_t s = from; s < to; s += kDeep) {
    float g[kDeep][kVec];
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
      load_group(gy + (int64_t)places[min(s + d, to - 1)] * cols + col, s + d < to ? n : 0, g[d]);
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
#pragma unroll
      for (int j = 0; j < kVec; ++j) f[j] += g[d][j];
  }
}

// Rows of the table that at most kRun places name, none included.
template <typename T, int LANES>
__global__ __launch_bounds__(kBlock) void embedding_rows_kernel(const T *__restrict__ gy, const int32_t *__restrict__ pointer,
                                                                const int32_t *__restrict__ places, T *__restrict__ grad,
                                                                int64_t n_table, int64_t cols, float scale) {
  const int64_t col = ((int64_t)blockIdx.y * LANES + threadIdx.x % LANES) * kVec;
  const int64_t row = (int64_t)blockIdx.x * (kBlock / LANES) + threadIdx.x / LANES;
  if (col >= cols || row >= n_table) return;
  const int n = (int)min((int64_t)kVec, cols - col);
  const int32_t from = pointer[row], to = pointer[row + 1];
  if (to - from > kRun) return;
  float f[kVec] = {};
  add_rows(gy, places, from, to, cols, col, n, f);
#pragma unroll
  for (int j = 0; j < kVec; ++j) f[j] *= scale;
  store_group(grad + row * cols + col, n, f);
}

// Sums of run blockIdx.x: of the long row that its first place names, and of the one that its last place names if that is
// another.
template <typename T, int LANES>
__global__ __launch_bounds__(kBlock) void embedding_runs_kernel(const T *__restrict__ gy, const int64_t *__restrict__ keys,
                                                                const int32_t *__restrict__ pointer,
                                                                const int32_t *__restrict__ places, float *__restrict__ parts,
                                                                int64_t n_ids, int64_t n_table, int64_t cols) {
  constexpr int kGroups = kBlock / LANES;
  __shared__ float sums[kGroups][LANES * kVec];
  const int64_t run0 = (int64_t)blockIdx.x * kRun;
  const int32_t begin = (int32_t)run0, end = (int32_t)min(n_ids, run0 + kRun);
  const int64_t lane_col = threadIdx.x % LANES * kVec, col = (int64_t)blockIdx.y * LANES * kVec + lane_col;
  const int n = (int)max((int64_t)0, min((int64_t)kVec, cols - col)), group = threadIdx.x / LANES;
  const int64_t row[2] = {keys[places[begin]], keys[places[end - 1]]};
  for (int k = 0; k < 2; ++k) {
    if (row[k] >= n_table || (k == 1 && row[1] == row[0])) continue;
    const int32_t from = pointer[row[k]], to = pointer[row[k] + 1];
    if (to - from <= kRun) continue;
    // the workgroup's groups of lanes take equal shares of the places, one after the other
    const int32_t a = max(from, begin), b = min(to, end), share = (b - a + kGroups - 1) / kGroups;
    float f[kVec] = {};
    add_rows(gy, places, min(b, a + group * share), min(b, a + (group + 1) * share), cols, col, n, f);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kVec; ++j) sums[group][lane_col + j] = f[j];
    __syncthreads();
    for (int c = threadIdx.x; c < LANES * kVec; c += kBlock) {
      float t = 0.0f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) t += sums[g][c];
      const int64_t at = (int64_t)blockIdx.y * LANES * kVec + c;
      if (at < cols) parts[((int64_t)blockIdx.x * 2 + k) * cols + at] = t;
    }
  }
}

// The runs of long rows added up: up to 512 rows of the table a workgroup, gridDim.x apart (ids named often tend to lie side by side),
// 64 columns blockIdx.y; eight wavefronts take equal shares of a row's runs.
template <typename T>
__global__ __launch_bounds__(8 * kWave) void embedding_join_kernel(const float *__restrict__ parts,
                                                                   const int32_t *__restrict__ pointer, T *__restrict__ grad,
                                                                   int64_t n_table, int64_t cols, float scale) {
  __shared__ float sums[8][kWave];
  __shared__ uint64_t long_rows[8];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int64_t mine = blockIdx.x + (int64_t)threadIdx.x * gridDim.x;
  const int32_t len = mine < n_table ? pointer[mine + 1] - pointer[mine] : 0;
  const uint64_t found = __ballot(len > kRun);
  if (lane == 0) long_rows[wave] = found;
  __syncthreads();
  const int64_t col = (int64_t)blockIdx.y * kWave + lane;
  uint64_t rows = long_rows[0];
  for (int part = 0;;) {
    if (!rows) {
      if (++part == 8) break;
      rows = long_rows[part];
      continue;
    }
    const int64_t row = blockIdx.x + (int64_t)(part * kWave + __ffsll((unsigned long long)rows) - 1) * gridDim.x;
    rows &= rows - 1;
    const int32_t from = pointer[row], to = pointer[row + 1];
    const int32_t first = from / kRun, last = (to - 1) / kRun, share = (last - first + 8) / 8;
    float f = 0.0f;
    if (col < cols) {
      const int32_t a = min(last + 1, first + wave * share), b = min(last + 1, first + (wave + 1) * share);
#pragma unroll 8
      for (int32_t r = a; r < b; ++r)                        // second of its first run, unless it begins with that
        f += parts[((int64_t)r * 2 + (r == first && from % kRun ? 1 : 0)) * cols + col];
    }
    sums[wave][lane] = f;
    __syncthreads();
    if (wave == 0 && col < cols) {
      float t = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) t += sums[k][lane];
      f32_to_elem(t * scale, grad[row * cols + col]);
    }
    __syncthreads();
  }
}

// Few places: a workgroup for each row of the table looks through all of them, a quarter by each wavefront in its turn, 512
// columns blockIdx.y.  One launch in the place of the sort's and the sums' eleven (us, 512 places of 64 columns, 300 rows 47 -> 9;
// 88 of 417, 26,498 rows 41 -> 14; 1024 of 512, 16,000 39 -> 16, 60,000 50 -> 49).
constexpr int64_t kFewPlaces = 1024, kFewTable = 65536;
template <typename T>
__global__ __launch_bounds__(kBlock) void embedding_few_kernel(const T *__restrict__ gy, const void *__restrict__ ids, int bits,
                                                               T *__restrict__ grad, int n_ids, int64_t cols, float scale) {
  constexpr int kWaves = kBlock / kWave, kDeep = 4;
  __shared__ float sums[kWaves][kWave * kVec];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int64_t row = blockIdx.x, col = ((int64_t)blockIdx.y * kWave + lane) * kVec;
  const int n = (int)max((int64_t)0, min((int64_t)kVec, cols - col));
  const int share = (n_ids + kWaves * kWave - 1) / (kWaves * kWave) * kWave, end = min(n_ids, (wave + 1) * share);
  float f[kVec] = {};
  for (int i0 = wave * share; i0 < end; i0 += kWave) {
    const int i = i0 + lane;
    const bool named = i < end && (bits == 64 ? ((const int64_t *)ids)[i] : (int64_t)((const int32_t *)ids)[i]) == row;
    uint64_t found = __ballot(named);
    while (found) {
      int place[kDeep];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        place[d] = found ? i0 + __ffsll((unsigned long long)found) - 1 : -1;
        found &= found - 1;
      }
      float g[kDeep][kVec];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) load_group(gy + (int64_t)max(place[d], 0) * cols + col, place[d] < 0 ? 0 : n, g[d]);
#pragma unroll
      for (int d = 0; d < kDeep; ++d)
#pragma unroll
        for (int j = 0; j < kVec; ++j) f[j] += g[d][j];
    }
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) sums[wave][j * kWave + lane] = f[j];
  __syncthreads();
  if (wave != 0 || n == 0) return;
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    f[j] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) f[j] += sums[w][j * kWave + lane];
    f[j] *= scale;
  }
  store_group(grad + row * cols + col, n, f);
}

template <typename W>
__global__ __launch_bounds__(kBlock) void embedding_zero_kernel(W *__restrict__ out, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) out[i] = 0;
}

inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

struct Plan {
  int64_t keys, pointer, places, status, parts, group;       // bytes from the workspace's start
  size_t group_bytes, bytes;
};
bool few(int64_t n_ids, int64_t n_table) { return n_ids <= kFewPlaces && n_table <= kFewTable; }
Plan plan_of(int64_t n_ids, int64_t n_table, int64_t cols) {
  Plan p;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up256(bytes);
    return here;
  };
  p.keys = take(8 * n_ids);
  p.pointer = take(4 * (n_table + 2));
  p.places = take(4 * n_ids);
  p.status = take(4);
  p.parts = take(((n_ids + kRun - 1) / kRun) * 2 * cols * 4);
  p.group_bytes = ga_group_edges_workspace_bytes(n_table + 1, n_ids);
  p.group = take((int64_t)p.group_bytes);
  p.bytes = (size_t)at;
  return p;
}

template <typename T, int LANES>
int lookup(const void *table, const void *ids, int bits, void *y, int64_t n_ids, int64_t n_table, int64_t cols, float scale,
           hipStream_t s) {
  const int64_t blocks = (n_ids + kBlock / LANES * 4 - 1) / (kBlock / LANES * 4), wide = (cols + LANES * kVec - 1) / (LANES * kVec);
  if (blocks > kMostLanes / kBlock || wide > 65535) return GA_EUNSUPPORTED;
  hipLaunchKernelGGL((embedding_kernel<T, LANES>), dim3((unsigned)blocks, (unsigned)wide), dim3(kBlock), 0, s, (const T *)table,
                     ids, bits, (T *)y, n_ids, n_table, cols, scale);
  return launch_status();
}

template <typename T, int LANES>
int sum_rows(const void *gy, const Plan &p, char *ws, void *grad, int64_t n_ids, int64_t n_table, int64_t cols, float scale,
             hipStream_t s) {
  const int64_t wide = (cols + LANES * kVec - 1) / (LANES * kVec), blocks = (n_table + kBlock / LANES - 1) / (kBlock / LANES);
  const int64_t runs = (n_ids + kRun - 1) / kRun;
  const int32_t *pointer = (const int32_t *)(ws + p.pointer), *places = (const int32_t *)(ws + p.places);
  float *parts = (float *)(ws + p.parts);
  hipLaunchKernelGGL((embedding_rows_kernel<T, LANES>), dim3((unsigned)blocks, (unsigned)wide), dim3(kBlock), 0, s,
                     (const T *)gy, pointer, places, (T *)grad, n_table, cols, scale);
  if (int rc = launch_status()) return rc;
  if (n_ids <= kRun) return GA_OK;                           // no row is long
  hipLaunchKernelGGL((embedding_runs_kernel<T, LANES>), dim3((unsigned)runs, (unsigned)wide), dim3(kBlock), 0, s, (const T *)gy,
                     (const int64_t *)(ws + p.keys), pointer, places, parts, n_ids, n_table, cols);
  if (int rc = launch_status()) return rc;
  // a small table's long rows in as many workgroups as there are (435 rows, nearly all long, 311 -> 8 us)
  const int64_t across = (cols + kWave - 1) / kWave, some = n_table < 2048 / across ? n_table : 2048 / across;
  const int64_t least = (n_table + 8 * kWave - 1) / (8 * kWave);
  hipLaunchKernelGGL((embedding_join_kernel<T>), dim3((unsigned)(some > least ? some : least), (unsigned)across), dim3(8 * kWave), 0, s,
                     parts, pointer, (T *)grad, n_table, cols, scale);
  return launch_status();
}

int check_embedding(const void *a, const void *ids, int idx_bits, const void *out, int64_t n_ids, int64_t n_table, int64_t cols,
                    float scale, int dtype, bool any_out) {
  if (n_ids < 0 || n_table < 0 || cols <= 0 || (idx_bits != 32 && idx_bits != 64)) return GA_EINVAL;
  if (!(scale - scale == 0.0f)) return GA_EINVAL;            // times the zeros of ids outside it would be NaN
  if (dtype != GA_F32 && dtype != GA_BF16) return GA_EUNSUPPORTED;
  if (cols > (1 << 20)) return GA_EUNSUPPORTED;
  if (n_ids > 0 && !ids) return GA_EINVAL;
  if (any_out && !out) return GA_EINVAL;
  const size_t e = dtype == GA_F32 ? 4 : 2;
  if (!aligned(a, e) || !aligned(out, e) || !aligned(ids, idx_bits / 8)) return GA_EALIGN;
  return GA_OK;
}

// Lanes a row: as many as its columns need, a wavefront's at most.
int lanes_of(int64_t cols) { return cols <= 8 * kVec ? 8 : cols <= 16 * kVec ? 16 : cols <= 32 * kVec ? 32 : 64; }
#define GA_BY_COLS(call, T, ...)                          \
  (lanes_of(cols) == 8    ? call<T, 8>(__VA_ARGS__)       \
   : lanes_of(cols) == 16 ? call<T, 16>(__VA_ARGS__)      \
   : lanes_of(cols) == 32 ? call<T, 32>(__VA_ARGS__)      \
                          : call<T, 64>(__VA_ARGS__))

// What the launches of a gradient hold: a workgroup for every run of the ids, and for as many rows of the table as it has groups of lanes.
bool holds(int64_t n_ids, int64_t n_table, int64_t cols) {
  constexpr int64_t blocks = kMostLanes / kBlock;
  return n_ids <= blocks * kRun && n_table <= blocks * (kBlock / lanes_of(cols));
}

}  // namespace
}  // namespace ga

extern "C" {

int ga_embedding(const void *table, const void *ids, int idx_bits, void *y, int64_t n_ids, int64_t n_table, int64_t cols,
                 float scale, int dtype, ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_embedding(table, ids, idx_bits, y, n_ids, n_table, cols, scale, dtype, n_ids > 0)) return rc;
  if (n_ids == 0) return GA_OK;
  if (n_table > 0 && !table) return GA_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  return dtype == GA_F32 ? GA_BY_COLS(lookup, float, table, ids, idx_bits, y, n_ids, n_table, cols, scale, s)
                         : GA_BY_COLS(lookup, bf16_t, table, ids, idx_bits, y, n_ids, n_table, cols, scale, s);
}

size_t ga_embedding_backward_workspace_bytes(int64_t n_ids, int64_t n_table, int64_t cols) {
  if (n_ids <= 0 || n_table <= 0 || cols <= 0 || !ga::holds(n_ids, n_table, cols)) return 0;
  return ga::few(n_ids, n_table) ? 0 : ga::plan_of(n_ids, n_table, cols).bytes;
}

int ga_embedding_backward(const void *grad_y, const void *ids, int idx_bits, void *grad_table, int64_t n_ids, int64_t n_table,
                          int64_t cols, float scale, int dtype, void *workspace, size_t workspace_bytes, ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_embedding(grad_y, ids, idx_bits, grad_table, n_ids, n_table, cols, scale, dtype, n_table > 0)) return rc;
  if (!holds(n_ids, n_table, cols)) return GA_EUNSUPPORTED;
  if (n_table == 0) return GA_OK;
  if (n_ids > 0 && !grad_y) return GA_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  if (n_ids == 0) {
    const int64_t n = n_table * cols * (dtype == GA_F32 ? 4 : 2);
    if (aligned(grad_table, 4) && n % 4 == 0) {              // whole words; else value by value
      hipLaunchKernelGGL(embedding_zero_kernel<uint32_t>, dim3(4096), dim3(kBlock), 0, s, (uint32_t *)grad_table, n / 4);
    } else {
      hipLaunchKernelGGL(embedding_zero_kernel<uint16_t>, dim3(4096), dim3(kBlock), 0, s, (uint16_t *)grad_table, n / 2);
    }
    return launch_status();
  }
  if (few(n_ids, n_table)) {
    const dim3 grid((unsigned)n_table, (unsigned)((cols + kWave * kVec - 1) / (kWave * kVec)));
    if (dtype == GA_F32)
      hipLaunchKernelGGL((embedding_few_kernel<float>), grid, dim3(kBlock), 0, s, (const float *)grad_y, ids, idx_bits,
                         (float *)grad_table, (int)n_ids, cols, scale);
    else
      hipLaunchKernelGGL((embedding_few_kernel<bf16_t>), grid, dim3(kBlock), 0, s, (const bf16_t *)grad_y, ids, idx_bits,
                         (bf16_t *)grad_table, (int)n_ids, cols, scale);
    return launch_status();
  }
  const Plan p = plan_of(n_ids, n_table, cols);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < p.bytes) return GA_EWORKSPACE;
  char *ws = (char *)workspace;
  int64_t *keys = (int64_t *)(ws + p.keys);
  const int64_t blocks = (n_ids + kBlock - 1) / kBlock;
  hipLaunchKernelGGL(embedding_keys_kernel, dim3((unsigned)(blocks > 8192 ? 8192 : blocks)), dim3(kBlock), 0, s, ids, idx_bits,
                     n_ids, n_table, keys);
  if (int rc = launch_status()) return rc;
  if (int rc = ga_group_edges(keys, nullptr, n_table + 1, n_ids, (int32_t *)(ws + p.pointer), nullptr, (int32_t *)(ws + p.places),
                              (int32_t *)(ws + p.status), ws + p.group, p.group_bytes, stream))
    return rc;
  return dtype == GA_F32 ? GA_BY_COLS(sum_rows, float, grad_y, p, ws, grad_table, n_ids, n_table, cols, scale, s)
                         : GA_BY_COLS(sum_rows, bf16_t, grad_y, p, ws, grad_table, n_ids, n_table, cols, scale, s);
}

}  // extern "C"
