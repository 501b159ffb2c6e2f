// experts.cu -- products of rows with their component's matrix, their
// gradients, and the Newton-Schulz iteration, on the CUDA cores: 64 x 64 tiles,
// fp32 sums, one row tile per block, every type and size.
#include "experts_api.cuh"

namespace gmmxx {
namespace experts {
namespace {

constexpr int kT = 64, kKc = 16;

struct Tile {
  float a[kKc][kT + 4];
  float b[kKc][kT + 4];
};

__device__ __forceinline__ void tile_fma(const Tile& t, float acc[4][4]) {
  const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15;
#pragma unroll
  for (int kk = 0; kk < kKc; ++kk)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(t.a[kk][tr * 4 + i], t.b[kk][tc * 4 + j], acc[i][j]);
}

// out[slot] = x[slot / div] . W[k] (+ bias[k]); w_in / w_out: element strides
__global__ void __launch_bounds__(256) rows_kernel(int dt, const void* x, int div, Groups g, int n_in, int n_out,
                                                   const void* w, int64_t w_in, int64_t w_out, const void* bias,
                                                   void* out, int out_dt) {
  __shared__ Tile t;
  const int tile = blockIdx.x >> 1;
  if (tile >= g.tiles[0]) return;
  const int32_t* e = g.tiles + kTileHeader + (int64_t)tile * kTileInts;
  const int k = e[0], pos = e[1] + (blockIdx.x & 1) * kT, n = e[2] - (blockIdx.x & 1) * kT;
  if (n <= 0) return;
  const int c0 = blockIdx.y * kT;
  const int64_t wk = (int64_t)k * n_in * n_out;
  float acc[4][4] = {};
  if (k < g.K)
    for (int i0 = 0; i0 < n_in; i0 += kKc) {
      for (int i = threadIdx.x; i < kT * kKc; i += 256) {
        const int r = i / kKc, kk = i % kKc;
        t.a[kk][r] = r < n && i0 + kk < n_in ? load_x(x, (int64_t)(g.order[pos + r] / div) * n_in + i0 + kk, dt) : 0.f;
        const int c = i % kT, kb = i / kT;
        t.b[kb][c] = c0 + c < n_out && i0 + kb < n_in ? load_x(w, wk + (i0 + kb) * w_in + (c0 + c) * w_out, dt) : 0.f;
      }
      __syncthreads();
      tile_fma(t, acc);
      __syncthreads();
    }
  const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15;
  for (int i = 0; i < 4; ++i) {
    if (tr * 4 + i >= n) continue;
    const int64_t slot = g.order[pos + tr * 4 + i];
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + tc * 4 + j;
      if (c >= n_out) continue;
      float v = acc[i][j];
      if (bias != nullptr && k < g.K) v += load_x(bias, (int64_t)k * n_out + c, dt);
      store_y(out, slot * n_out + c, out_dt, v);
    }
  }
}

// gw[k] = sum over the group's slots of x^T gy
__global__ void __launch_bounds__(256) weight_kernel(int dt, const void* x, const void* gy, Groups g, int n_in,
                                                     int n_out, void* gw, int64_t w_in, int64_t w_out) {
  __shared__ Tile t;
  const int k = blockIdx.z, r0 = blockIdx.x * kT, c0 = blockIdx.y * kT;
  const int p0 = g.offsets[k], p1 = g.offsets[k + 1];
  float acc[4][4] = {};
  for (int p = p0; p < p1; p += kKc) {
    for (int i = threadIdx.x; i < kT * kKc; i += 256) {
      const int c = i % kT, kk = i / kT;
      const bool in = p + kk < p1;
      const int64_t slot = in ? g.order[p + kk] : 0;
      t.a[kk][c] = in && r0 + c < n_in ? load_x(x, slot / g.top * n_in + r0 + c, dt) : 0.f;
      t.b[kk][c] = in && c0 + c < n_out ? load_x(gy, slot * n_out + c0 + c, dt) : 0.f;
    }
    __syncthreads();
    tile_fma(t, acc);
    __syncthreads();
  }
  const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + tr * 4 + i, c = c0 + tc * 4 + j;
      if (r < n_in && c < n_out) store_y(gw, (int64_t)k * n_in * n_out + r * w_in + c * w_out, dt, acc[i][j]);
    }
}

__global__ void bias_kernel(int dt, const void* gy, Groups g, int n_out, void* gb) {
  const int k = blockIdx.y, c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= n_out) return;
  float s = 0.f;
  for (int p = g.offsets[k]; p < g.offsets[k + 1]; ++p) s += load_x(gy, (int64_t)g.order[p] * n_out + c, dt);
  store_y(gb, (int64_t)k * n_out + c, dt, s);
}

// gx[row] = sum over the row's slots, rounded once
__global__ void sum_slots_kernel(const float* part, int64_t rows, int top, int n, void* out, int dt) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= rows * n) return;
  const int64_t row = i / n, c = i % n;
  float s = 0.f;
  for (int t = 0; t < top; ++t) s += part[(row * top + t) * n + c];
  store_y(out, i, dt, s);
}

// d = alpha * (A or A^T) . (B or B^T) + beta * c for a batch; m x n x k, row-major fp32
__global__ void __launch_bounds__(256) batch_kernel(const float* a, int at, const float* b, int bt, const float* c,
                                                    float* d, int m, int n, int k, float alpha, float beta) {
  __shared__ Tile t;
  const int64_t z = blockIdx.z;
  a += z * m * k;
  b += z * n * k;
  const int r0 = blockIdx.x * kT, c0 = blockIdx.y * kT;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < k; k0 += kKc) {
    for (int i = threadIdx.x; i < kT * kKc; i += 256) {
      const int r = i % kT, kk = i / kT;
      const bool in = k0 + kk < k;
      t.a[kk][r] = in && r0 + r < m ? a[at ? (int64_t)(k0 + kk) * m + r0 + r : (int64_t)(r0 + r) * k + k0 + kk] : 0.f;
      t.b[kk][r] = in && c0 + r < n ? b[bt ? (int64_t)(c0 + r) * k + k0 + kk : (int64_t)(k0 + kk) * n + c0 + r] : 0.f;
    }
    __syncthreads();
    tile_fma(t, acc);
    __syncthreads();
  }
  const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + tr * 4 + i, cc = c0 + tc * 4 + j;
      if (r >= m || cc >= n) continue;
      const int64_t o = z * m * n + (int64_t)r * n + cc;
      d[o] = alpha * acc[i][j] + (c != nullptr ? beta * c[o] : 0.f);
    }
}

__global__ void __launch_bounds__(1024) normalise_kernel(int dt, const void* g, int64_t n, float eps, float* x) {
  __shared__ double red[32];
  const int64_t base = (int64_t)blockIdx.x * n;
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    const double v = load_x(g, base + i, dt);
    s += v * v;
  }
  s = block_sum(s, red);
  const double inv = 1.0 / (sqrt(s) + (double)eps);
  for (int64_t i = threadIdx.x; i < n; i += 1024) x[base + i] = (float)(load_x(g, base + i, dt) * inv);
}

__global__ void round_kernel(const float* x, int64_t n, void* q, int dt) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
    store_y(q, i, dt, x[i]);
}

int launch_rows(int dt, const void* x, int div, const Groups& g, int64_t n_in, int64_t n_out, const void* w,
                int64_t w_in, int64_t w_out, const void* bias, void* out, int out_dt, cudaStream_t st) {
  dim3 grid((unsigned)(2 * g.max_tiles()), (unsigned)ceil_div(n_out, kT));
  rows_kernel<<<grid, 256, 0, st>>>(dt, x, div, g, (int)n_in, (int)n_out, w, w_in, w_out, bias, out, out_dt);
  return check_launch("rows_kernel");
}

}  // namespace

size_t grouped_matmul_ws(int, const Groups&, int64_t, int64_t) { return 256; }

int launch_grouped_matmul(int dt, const void* x, const Groups& g, int64_t n_in, int64_t n_out, const void* w, int wt,
                          const void* bias, void* out, char*, cudaStream_t st) {
  return launch_rows(dt, x, g.top, g, n_in, n_out, w, wt ? 1 : n_out, wt ? n_in : 1, bias, out, dt, st);
}

size_t grouped_backward_ws(int, const Groups& g, int64_t n_in, int64_t) {
  return 256 + (g.top > 1 ? (size_t)(g.slots() * n_in * 4) : 0);
}

int launch_grouped_backward(int dt, const void* gy, const void* x, const Groups& g, int64_t n_in, int64_t n_out,
                            const void* w, int wt, void* gx, void* gw, void* gb, char* ws, cudaStream_t st) {
  if (gx != nullptr && g.rows > 0) {
    float* part = reinterpret_cast<float*>(ws);
    const bool sum = g.top > 1;
    if (int rc = launch_rows(dt, gy, 1, g, n_out, n_in, w, wt ? n_in : 1, wt ? 1 : n_out, nullptr,
                             sum ? static_cast<void*>(part) : gx, sum ? GMMXX_FLOAT32 : dt, st))
      return rc;
    if (sum) {
      sum_slots_kernel<<<(unsigned)ceil_div(g.rows * n_in, 256), 256, 0, st>>>(part, g.rows, g.top, (int)n_in, gx, dt);
      if (int rc = check_launch("sum_slots_kernel")) return rc;
    }
  }
  if (gw != nullptr) {
    dim3 grid((unsigned)ceil_div(n_in, kT), (unsigned)ceil_div(n_out, kT), (unsigned)g.K);
    weight_kernel<<<grid, 256, 0, st>>>(dt, x, gy, g, (int)n_in, (int)n_out, gw, wt ? 1 : n_out, wt ? n_in : 1);
    if (int rc = check_launch("weight_kernel")) return rc;
  }
  if (gb != nullptr) {
    bias_kernel<<<dim3((unsigned)ceil_div(n_out, 256), (unsigned)g.K), 256, 0, st>>>(dt, gy, g, (int)n_out, gb);
    if (int rc = check_launch("bias_kernel")) return rc;
  }
  return GMMXX_OK;
}

size_t orthogonalize_ws(int, int64_t batch, int64_t m, int64_t n) {
  const int64_t lo = m < n ? m : n;
  return (size_t)(4 * batch * (2 * m * n + 2 * lo * lo) + 256);
}

int launch_orthogonalize(int dt, const void* g, int64_t batch, int64_t m, int64_t n, int steps, float a, float b,
                         float c, float eps, void* q, char* ws, cudaStream_t st) {
  const int64_t lo = m < n ? m : n, hi = m < n ? n : m;
  float* x = reinterpret_cast<float*>(ws);
  float* y = x + batch * m * n;
  float* p = y + batch * m * n;
  float* r = p + batch * lo * lo;
  normalise_kernel<<<(unsigned)batch, 1024, 0, st>>>(dt, g, m * n, eps, x);
  if (int rc = check_launch("normalise_kernel")) return rc;
  for (int64_t z0 = 0; z0 < batch; z0 += 65535) {  // grid z
    const unsigned nz = (unsigned)(batch - z0 < 65535 ? batch - z0 : 65535);
    const unsigned tl = (unsigned)ceil_div(lo, kT);
    float *xs = x + z0 * m * n, *ys = y + z0 * m * n, *ps = p + z0 * lo * lo, *rs = r + z0 * lo * lo;
    for (int s = 0; s < steps; ++s) {
      const bool wide = m <= n;
      batch_kernel<<<dim3(tl, tl, nz), 256, 0, st>>>(xs, wide ? 0 : 1, xs, wide ? 1 : 0, nullptr, ps, (int)lo, (int)lo,
                                                     (int)hi, 1.f, 0.f);
      batch_kernel<<<dim3(tl, tl, nz), 256, 0, st>>>(ps, 0, ps, 0, ps, rs, (int)lo, (int)lo, (int)lo, c, b);
      dim3 grid((unsigned)ceil_div(m, kT), (unsigned)ceil_div(n, kT), nz);
      if (wide) batch_kernel<<<grid, 256, 0, st>>>(rs, 0, xs, 0, xs, ys, (int)m, (int)n, (int)lo, 1.f, a);
      else batch_kernel<<<grid, 256, 0, st>>>(xs, 0, rs, 0, xs, ys, (int)m, (int)n, (int)lo, 1.f, a);
      float* t = xs;
      xs = ys;
      ys = t;
    }
    if (int rc = check_launch("batch_kernel")) return rc;
  }
  round_kernel<<<148 * 4, 256, 0, st>>>((steps & 1) ? y : x, batch * m * n, q, dt);
  return check_launch("round_kernel");
}

}  // namespace experts
}  // namespace gmmxx
