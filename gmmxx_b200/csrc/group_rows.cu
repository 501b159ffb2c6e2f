// group_rows.cu -- routing: slots sorted by the component they are assigned to
// (gmmxx_group_rows), and the table of row tiles that the grouped products walk.
//
// A stable counting sort.  The slots are cut into one contiguous chunk per
// warp; every warp counts its chunk's labels into its own row of a
// [warps][K + 1] table (column K: unassigned slots), the columns are scanned
// over the warps and the totals over the components, and every warp walks its
// chunk again and places each slot at (group start) + (earlier warps' slots of
// that label) + (rank inside the warp).  Equal labels keep their slot order and
// nothing depends on the order in which warps run, so the result is the same
// in every run.
//
// Small problems (kSmallSlots slots and a [35][K + 1] table in shared memory)
// run in a single block and launch; larger ones in four launches.
#include "experts_api.cuh"

#include <algorithm>

namespace gmmxx {
namespace experts {
namespace {

constexpr int kWarps = 32;                       // warps of the one-block kernel
constexpr int64_t kSmallSlots = 32768;           // above, four launches over the whole GPU are faster
constexpr int kSmallSmem = 200 * 1024;
constexpr int64_t kChunk = 1024;                 // slots per warp of the large path, at least
constexpr int64_t kMaxWarps = 148 * 32;
constexpr int kTableSmem = 200 * 1024;       // counters of one block's warps

__device__ __forceinline__ int load_label(const void* labels, int wide, int64_t i, int K) {
  // clamped before the narrowing: a 64-bit label beyond 32 bits is unassigned too
  if (wide) {
    const long long v = static_cast<const long long*>(labels)[i];
    return (v < 0 || v >= K) ? K : (int)v;
  }
  const int v = static_cast<const int*>(labels)[i];
  return (v < 0 || v >= K) ? K : v;
}

// Slots [begin, end) of one warp, four groups of 32 in flight.  COUNT: adds
// each label to cnt.  Otherwise cnt holds the next free position per label and
// the slots are placed.
template <bool COUNT>
__device__ __forceinline__ void walk(const void* labels, int wide, int64_t begin, int64_t end, int K, int* cnt,
                                     int32_t* order) {
  const int lane = threadIdx.x & 31;
  for (int64_t i0 = begin; i0 < end; i0 += 128) {
    int lab[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = i0 + u * 32 + lane;
      lab[u] = i < end ? load_label(labels, wide, i, K) : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (COUNT) {
        if (lab[u] >= 0) atomicAdd(&cnt[lab[u]], 1);
      } else {
        const unsigned same = __match_any_sync(0xffffffffu, lab[u]);
        const int rank = __popc(same & ((1u << lane) - 1u));
        int base = 0;
        if (lab[u] >= 0) base = cnt[lab[u]];
        __syncwarp();
        if (lab[u] >= 0) {
          order[base + rank] = (int32_t)(i0 + u * 32 + lane);
          if (rank == 0) cnt[lab[u]] = base + __popc(same);
        }
        __syncwarp();
      }
    }
  }
}

// exclusive scan over the block of one value per thread (1024 threads); *total gets the sum
__device__ __forceinline__ int block_exclusive(int v, int* red, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  __syncthreads();
  if (lane == 31) red[w] = s;
  __syncthreads();
  if (w == 0) {
    int t = red[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    red[lane] = t;
  }
  __syncthreads();
  *total = red[31];
  return s - v + (w ? red[w - 1] : 0);
}

// Group starts and tile starts from the group sizes.  size(k): slots of group
// k, k == K the unassigned.  One block of 1024 threads; start[k] (may be the
// caller's shared memory) and first[k] receive K + 1 values each.
template <typename Size>
__device__ __forceinline__ void scan_groups(int K, Size size, int* start, int* first, int* first2, int32_t* offsets,
                                            int32_t* tiles, int* red) {
  int row0 = 0, tile0 = 0, pair0 = 0;
  for (int k0 = 0; k0 <= K; k0 += 1024) {
    const int k = k0 + threadIdx.x;
    const int c = k <= K ? size(k) : 0;
    const int nt = (c + kTileRows - 1) / kTileRows;
    int rows, ntiles, npairs;
    const int r = row0 + block_exclusive(c, red, &rows);
    const int t = tile0 + block_exclusive(nt, red, &ntiles);
    const int p = pair0 + block_exclusive((c + kPairRows - 1) / kPairRows, red, &npairs);
    if (k <= K) {
      start[k] = r;
      first[k] = t;
      first2[k] = p;
      offsets[k] = r;  // offsets[K]: end of the last group, start of the unassigned slots
    }
    row0 += rows;
    tile0 += ntiles;
    pair0 += npairs;
  }
  if (threadIdx.x == 0) {
    tiles[0] = tile0;
    tiles[1] = pair0;
  }
}

// Tile table: per tile of `per` rows {group, first position, rows}; the
// unassigned slots' tiles have group K and come last.  Entry t of `table`:
__device__ __forceinline__ void fill_tile(int K, const int* first, const int* start, int slots, int per, int32_t* table,
                                          int64_t t) {
  int lo = 0, hi = K;  // last k with first[k] <= t: the one whose tiles t falls in
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= t) lo = mid; else hi = mid - 1;
  }
  const int pos = start[lo] + (int)(t - first[lo]) * per;
  const int end = lo < K ? start[lo + 1] : slots;
  int32_t* e = table + t * kTileInts;
  e[0] = lo;
  e[1] = pos;
  e[2] = min(per, end - pos);
}

// both tables, the tiles [begin, ...) in steps of `step`; pairs: offset of the second
__device__ __forceinline__ void fill_tables(int K, const int* first, const int* first2, const int* start, int slots,
                                            int32_t* tiles, int64_t pairs, int64_t begin, int64_t step) {
  const int n1 = tiles[0], n2 = tiles[1];
  for (int64_t t = begin; t < n1; t += step) fill_tile(K, first, start, slots, kTileRows, tiles + kTileHeader, t);
  for (int64_t t = begin; t < n2; t += step) fill_tile(K, first2, start, slots, kPairRows, tiles + kTileHeader + pairs, t);
}

__global__ void __launch_bounds__(1024) group_rows_small_kernel(const void* labels, int wide, int slots, int K,
                                                                int32_t* order, int32_t* offsets, int32_t* tiles,
                                                                int64_t pairs) {
  extern __shared__ int sm[];
  __shared__ int red[32];
  const int K1 = K + 1, warp = threadIdx.x >> 5;
  int* table = sm;                // [kWarps][K1]
  int* start = sm + kWarps * K1;  // [K1]
  int* first = start + K1;        // [K1]
  int* first2 = first + K1;       // [K1]
  for (int i = threadIdx.x; i < kWarps * K1; i += 1024) table[i] = 0;
  __syncthreads();
  // whole 128-slot steps per warp
  const int chunk = ((slots + kWarps - 1) / kWarps + 127) / 128 * 128;
  const int begin = min(slots, warp * chunk), end = min(slots, begin + chunk);
  walk<true>(labels, wide, begin, end, K, table + warp * K1, nullptr);
  __syncthreads();
  for (int k = threadIdx.x; k < K1; k += 1024) {
    int run = 0;
    for (int w = 0; w < kWarps; ++w) {
      const int c = table[w * K1 + k];
      table[w * K1 + k] = run;
      run += c;
    }
    first[k] = run;
  }
  __syncthreads();
  scan_groups(K, [&](int k) { return first[k]; }, start, first, first2, offsets, tiles, red);
  __syncthreads();
  for (int i = threadIdx.x; i < kWarps * K1; i += 1024) table[i] += start[i % K1];
  __syncthreads();
  walk<false>(labels, wide, begin, end, K, table + warp * K1, order);
  fill_tables(K, first, first2, start, slots, tiles, pairs, threadIdx.x, 1024);
}

// rows of the table: warp w of the grid counts slots [w * chunk, (w + 1) * chunk)
__global__ void count_kernel(const void* labels, int wide, int64_t slots, int K, int64_t chunk, int nwarps,
                             int* table) {
  extern __shared__ int sm[];
  const int K1 = K + 1, warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < warps * K1; i += blockDim.x) sm[i] = 0;
  __syncthreads();
  const int64_t w = (int64_t)blockIdx.x * warps + warp;
  const int64_t begin = min(slots, w * chunk), end = min(slots, begin + chunk);
  walk<true>(labels, wide, begin, end, K, sm + warp * K1, nullptr);
  __syncthreads();
  const int rows = min(warps, nwarps - (int)blockIdx.x * warps);
  int* out = table + (int64_t)blockIdx.x * warps * K1;
  for (int i = threadIdx.x; i < rows * K1; i += blockDim.x) out[i] = sm[i];
}

// Columns of the table scanned over the warps: 32 columns per block, 32
// segments of warps; total[k] gets the column sums.
__global__ void __launch_bounds__(1024) columns_kernel(int* table, int nwarps, int K1, int* total) {
  __shared__ int part[32][33];
  const int lane = threadIdx.x & 31, seg = threadIdx.x >> 5;
  const int k = blockIdx.x * 32 + lane;
  const int per = (nwarps + 31) / 32, w0 = min(nwarps, seg * per), w1 = min(nwarps, w0 + per);
  int sum = 0;
  if (k < K1)
    for (int w = w0; w < w1; ++w) sum += table[(int64_t)w * K1 + k];
  part[seg][lane] = sum;
  __syncthreads();
  int run = 0;
  for (int s = 0; s < seg; ++s) run += part[s][lane];
  if (k < K1) {
    if (seg == 31) total[k] = run + sum;
    for (int w = w0; w < w1; ++w) {
      const int c = table[(int64_t)w * K1 + k];
      table[(int64_t)w * K1 + k] = run;
      run += c;
    }
  }
}

__global__ void __launch_bounds__(1024) totals_kernel(const int* total, int K, int* start, int* first,
                                                      int* first2, int32_t* offsets, int32_t* tiles) {
  __shared__ int red[32];
  scan_groups(K, [&](int k) { return total[k]; }, start, first, first2, offsets, tiles, red);
}

__global__ void place_kernel(const void* labels, int wide, int64_t slots, int K, int64_t chunk, int nwarps,
                             const int* table, const int* start, const int* first, const int* first2, int32_t* order,
                             int32_t* tiles, int64_t pairs) {
  extern __shared__ int sm[];
  const int K1 = K + 1, warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
  const int rows = min(warps, nwarps - (int)blockIdx.x * warps);
  const int* in = table + (int64_t)blockIdx.x * warps * K1;
  for (int i = threadIdx.x; i < rows * K1; i += blockDim.x) sm[i] = in[i] + start[i % K1];
  __syncthreads();
  const int64_t w = (int64_t)blockIdx.x * warps + warp;
  const int64_t begin = min(slots, w * chunk), end = min(slots, begin + chunk);
  walk<false>(labels, wide, begin, end, K, sm + warp * K1, order);
  fill_tables(K, first, first2, start, (int)slots, tiles, pairs, (int64_t)blockIdx.x * blockDim.x + threadIdx.x,
              (int64_t)gridDim.x * blockDim.x);
}

struct Plan {
  bool small;
  int smem;             // dynamic shared memory of the walking kernels
  int warps, blocks;    // per block, grid
  int nwarps;           // rows of the table
  int64_t chunk;
  int64_t table, total, start, first, first2, bytes;  // workspace offsets (large path)
};

Plan make_plan(int64_t slots, int64_t K) {
  Plan p{};
  const int64_t K1 = K + 1;
  const int64_t small = (kWarps + 3) * K1 * 4;
  p.small = slots <= kSmallSlots && small <= kSmallSmem;
  if (p.small) {
    p.smem = (int)small;
    p.bytes = 256;
    return p;
  }
  p.warps = (int)std::min<int64_t>(kWarps, std::max<int64_t>(1, kTableSmem / (K1 * 4)));
  const int64_t most = std::min<int64_t>(kMaxWarps, (int64_t)148 * p.warps);
  p.chunk = round_up(std::max<int64_t>(kChunk, ceil_div(slots, most)), 128);
  p.nwarps = (int)std::max<int64_t>(1, ceil_div(slots, p.chunk));
  p.blocks = (int)ceil_div(p.nwarps, p.warps);
  p.smem = (int)(p.warps * K1 * 4);
  int64_t off = 0;
  p.table = off; off += round_up((int64_t)p.nwarps * K1 * 4, 256);
  p.total = off; off += round_up(K1 * 4, 256);
  p.start = off; off += round_up(K1 * 4, 256);
  p.first = off; off += round_up(K1 * 4, 256);
  p.first2 = off; off += round_up(K1 * 4, 256);
  p.bytes = off;
  return p;
}

}  // namespace

int64_t tiles_len(int64_t slots, int64_t K) {
  return kTileHeader + kTileInts * (most_tiles(slots, K, kTileRows) + most_tiles(slots, K, kPairRows));
}

size_t group_rows_ws(int64_t slots, int64_t K) { return (size_t)make_plan(slots, K).bytes; }

int launch_group_rows(const void* labels, int wide, int64_t slots, int64_t K, int32_t* order, int32_t* offsets,
                      int32_t* tiles, char* ws, cudaStream_t st) {
  const Plan p = make_plan(slots, K);
  const int64_t pairs = kTileInts * most_tiles(slots, K, kTileRows);
  if (p.small) {
    static SmemGrants grants;
    if (int rc = allow_smem((const void*)group_rows_small_kernel, kSmallSmem, grants)) return rc;
    group_rows_small_kernel<<<1, 1024, p.smem, st>>>(labels, wide, (int)slots, (int)K, order, offsets, tiles, pairs);
    return check_launch("group_rows_small_kernel");
  }
  int* table = reinterpret_cast<int*>(ws + p.table);
  int* total = reinterpret_cast<int*>(ws + p.total);
  int* start = reinterpret_cast<int*>(ws + p.start);
  int* first = reinterpret_cast<int*>(ws + p.first);
  int* first2 = reinterpret_cast<int*>(ws + p.first2);
  static SmemGrants count_grants, place_grants;
  if (int rc = allow_smem((const void*)count_kernel, kTableSmem, count_grants)) return rc;
  if (int rc = allow_smem((const void*)place_kernel, kTableSmem, place_grants)) return rc;
  count_kernel<<<p.blocks, p.warps * 32, p.smem, st>>>(labels, wide, slots, (int)K, p.chunk, p.nwarps, table);
  if (int rc = check_launch("count_kernel")) return rc;
  columns_kernel<<<(unsigned)ceil_div(K + 1, 32), 1024, 0, st>>>(table, p.nwarps, (int)K + 1, total);
  if (int rc = check_launch("columns_kernel")) return rc;
  totals_kernel<<<1, 1024, 0, st>>>(total, (int)K, start, first, first2, offsets, tiles);
  if (int rc = check_launch("totals_kernel")) return rc;
  place_kernel<<<p.blocks, p.warps * 32, p.smem, st>>>(labels, wide, slots, (int)K, p.chunk, p.nwarps, table, start,
                                                       first, first2, order, tiles, pairs);
  return check_launch("place_kernel");
}

}  // namespace experts
}  // namespace gmmxx
