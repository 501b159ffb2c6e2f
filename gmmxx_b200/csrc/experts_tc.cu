// experts_tc.cu -- the product kernel of the routed products and of the
// Newton-Schulz iteration, on the 5th-generation tensor cores.
//
//   D[128 x bn] = sum over k of A[128 x k] B[k x bn]      (fp32 in tensor memory)
//
// One persistent CTA per SM walks output tiles.  A TMA warp fills a ring of
// stages (64 contraction elements of A and B each, 128-byte swizzle), one
// thread issues tcgen05.mma, and eight epilogue warps drain one accumulator
// from tensor memory while the next tile's products go to the other.
//
// Routed rows of 16-bit types are never copied: four warps fetch each row where
// it lies with 16-byte cp.async into the swizzled stage, for kRows as the
// K-major A operand, for kWeights -- where the rows are the contraction -- as
// MN-major A and B operands.  (TMA's gather of four rows per instruction took
// about 80 cycles an instruction, 6 B per cycle and SM, and held the tensor pipe
// at 18 % and 7 %.)  The copies complete on the stage's mbarrier; a warp of its own
// waits for it, fences the proxies and passes the stage on (the fence costs the
// thread that issues the products 5 % of its time).  Rows behind a
// segment's last are filled with zeros; kRows fetches copies of the tile's first
// row there and does not store them.  Planes of fp32 rows are laid out sorted
// before the launch and loaded as TMA tiles; there the last stage of a kWeights
// segment also holds the next group's rows, which are zeroed in both operands
// before the products (zeroing one would leave NaN * 0).
//
// Sums.  The tensor core adds to an accumulator by cutting, not rounding: an
// addition costs about 3.4e-8 of the sum, always towards zero (measured: 8e-7
// after 24 additions of 16 products).  That is nothing beside the rounding to 16
// bits, but not for fp32 results: there the leading planes' products and the
// others (2^-8 of them and less) go to accumulators of their own, and every
// kChunk stages (8 additions) both are added into fp32 registers of the
// epilogue warps.
//
// Planes.  16-bit factors are multiplied as they are (1 plane).  fp32 factors
// arrive as three bf16 planes x = x0 + x1 + x2 of 8 significant bits each
// (exact) and six products x0w0 + x0w1 + x1w0 + x1w1 + x0w2 + x2w0, which
// drops 2^-24 of each product; 16-bit products are exact in the tensor core
// and summed in fp32.  The Newton-Schulz iterates are two fp16 planes of
// value * 4096 (|value| < 16 by the check on the coefficients; the second
// plane then keeps its 11 bits down to values of 2^-26) and three products,
// 22 bits; where the result is rounded to bf16 one plane is enough.
#include "experts_tc.cuh"
#include "tc_ptx.cuh"

#include <algorithm>

namespace gmmxx {
namespace experts {

using namespace ptx;

__device__ int g_status = 0;  // sticky: 1 when a bounded wait ran out (gmmxx_products_status)

namespace {

constexpr int kBM = 128;
constexpr int kGatherWarp0 = 12, kGatherThreads = 128;
constexpr int kEpiWarp0 = 4, kEpiWarps = 8;
constexpr int kABytes = kBM * 128;  // one plane of A per stage
constexpr int kMaxStages = 8;
constexpr int kChunk = 2;  // stages per accumulation where there are several planes
constexpr int kSmemLimit = 232448 - 1024;

struct Bars {
  uint64_t full[kMaxStages], ready[kMaxStages], empty[kMaxStages];  // ready: full, and the proxies fenced
  uint64_t accfull[2], accempty[2];
  uint32_t tmem_base;
  int abort;
};

// 16 bytes to shared memory, or zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
// arrives on the barrier when this thread's copies so far have landed
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void mma_16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  mma_bf16(d, a, b, idesc, acc);  // kind::f16: the types are the descriptor's
}

// a bounded wait ran out: every warp of the block stops at its next wait
__device__ __forceinline__ void give_up(Bars* bars, int lane) {
  if (lane == 0) {
    *(volatile int*)&bars->abort = 1;
    atomicOr(&g_status, 1);
  }
}

// one poll, without waiting
__device__ __forceinline__ bool mbar_test(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(b)), "r"(parity)
      : "memory");
  return ok != 0;
}

// position in the ring of stages (or of the two accumulators): index and phase, counted without divisions
struct Ring {
  int i = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void step(int n) {
    if (++i == n) {
      i = 0;
      phase ^= 1;
    }
  }
};

// one output tile
struct Tile {
  int g;       // group / matrix
  int pos;     // first position (routed)
  int rows;    // kRows: rows of the tile; kWeights: rows of the segment; kBatch: rows of the tile
  int m0, n0;
  int slot;    // kWeights: partial slot or -1
  int kb;      // contraction stages; 0: the result is zero
};

template <int KIND>
__device__ __forceinline__ int64_t tile_count(const ProductArgs& a) {
  const int64_t items = KIND == kBatch ? a.items : (int64_t)__ldg(a.table);
  return items * a.mt * a.nt;
}

template <int KIND>
__device__ __forceinline__ Tile decode(const ProductArgs& a, int64_t it) {
  Tile t;
  t.n0 = (int)(it % a.nt) * a.bn;
  it /= a.nt;
  if (KIND == kRows) {
    const int32_t* e = a.table + kTileHeader + it * kTileInts;
    t.g = __ldg(e);
    t.pos = __ldg(e + 1);
    t.rows = __ldg(e + 2);
    t.m0 = 0;
    t.slot = -1;
    t.kb = t.g < a.groups ? (a.k + kBlockK - 1) / kBlockK : 0;
    return t;
  }
  t.m0 = (int)(it % a.mt) * kBM;
  it /= a.mt;
  if (KIND == kWeights) {
    const int32_t* e = a.table + kSegHeader + it * kSegInts;
    t.g = __ldg(e);
    t.pos = __ldg(e + 1);
    t.rows = __ldg(e + 2);
    t.slot = __ldg(e + 3);
    t.kb = (t.rows + kBlockK - 1) / kBlockK;
  } else {
    t.g = (int)it;
    t.pos = 0;
    t.rows = min(kBM, a.m - t.m0);
    t.slot = -1;
    t.kb = (a.k + kBlockK - 1) / kBlockK;
  }
  return t;
}

__device__ __forceinline__ uint4 pack8(const float* v, int dt) {
  uint4 q;
  uint32_t* p = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dt == GMMXX_BFLOAT16) {
      p[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
    } else {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      p[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return q;
}

// 32 values of one row to out[row0 + c], nv of them valid
__device__ __forceinline__ void store32(void* out, int dt, int64_t at, const float* v, int nv, int vec) {
  if (vec && nv >= 32) {
    if (dt == GMMXX_FLOAT32) {
      float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
      uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = pack8(v + 8 * i, dt);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i < nv) store_y(out, at + i, dt, v[i]);
}

// kBatch: 32 values of one row: combine with the planes e and write planes or the result
template <int PLANES>
__device__ __forceinline__ void batch32(const ProductArgs& a, const Tile& t, int row, int c, float* v, int nv) {
  const int64_t at = t.g * a.p_stride + (int64_t)row * a.ldp + c;
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] *= a.alpha;
  if (a.e[0] != nullptr) {
#pragma unroll
    for (int i0 = 0; i0 < 32; i0 += 8) {  // ldp is a multiple of 8: whole 16-byte pieces (their tail is never used)
      if (i0 >= nv) break;
#pragma unroll
      for (int p = PLANES - 1; p >= 0; --p) {
        const uint4 q = *reinterpret_cast<const uint4*>(a.e[p] + at + i0);
        const __half2* h = reinterpret_cast<const __half2*>(&q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __half22float2(h[i]);
          v[i0 + 2 * i] = fmaf(a.beta, f.x, v[i0 + 2 * i]);
          v[i0 + 2 * i + 1] = fmaf(a.beta, f.y, v[i0 + 2 * i + 1]);
        }
      }
    }
  }
  if (a.out != nullptr) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= 1.f / kPlaneScale;
    store32(a.out, a.out_dt, t.g * a.out_stride + (int64_t)row * a.ldo + c, v, nv, a.vec);
    return;
  }
#pragma unroll
  for (int i0 = 0; i0 < 32; i0 += 8) {
    if (i0 >= nv) break;
    uint4 q[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = v[i0 + 2 * i], y = v[i0 + 2 * i + 1];
      const __half2 hi = __floats2half2_rn(x, y);
      reinterpret_cast<__half2*>(&q[0])[i] = hi;
      if (PLANES > 1) {
        const float2 f = __half22float2(hi);
        reinterpret_cast<__half2*>(&q[1])[i] = __floats2half2_rn(x - f.x, y - f.y);
      }
    }
#pragma unroll
    for (int p = 0; p < PLANES; ++p) *reinterpret_cast<uint4*>(a.o[p] + at + i0) = q[p];
  }
}

template <int KIND, int PLANES>
struct Roles {
  static constexpr bool kGather = KIND != kBatch && PLANES == 1;      // rows by cp.async
  static constexpr bool kTma = !(KIND == kWeights && PLANES == 1);    // something by TMA
  static constexpr int kThreads = kGather ? 512 : 384;
  static constexpr int kFullCount = (kGather ? kGatherThreads : 0) + (kTma ? 1 : 0);
};

template <int KIND, int PLANES>
__global__ void __launch_bounds__(Roles<KIND, PLANES>::kThreads, 1)
    product_kernel(const __grid_constant__ ProductMaps maps, const ProductArgs a) {
  using R = Roles<KIND, PLANES>;
  extern __shared__ __align__(1024) char smem_raw[];
  __shared__ Bars bars;
  char* sm = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bbytes = a.bn * 128;  // one plane of B per stage
  const int stage_bytes = PLANES * (kABytes + bbytes);
  volatile int* abort = &bars.abort;
  // two buffers of one accumulator, or of two (leading products, others)
  constexpr int kAccs = PLANES > 1 ? 2 : 1;
  const uint32_t tmem_cols = 2 * kAccs * a.bn;  // a power of two of at least 32

  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(&bars.full[i], R::kFullCount);
      mbar_init(&bars.ready[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.accfull[i], 1);
      mbar_init(&bars.accempty[i], kEpiWarps);
    }
    bars.abort = 0;
    fence_barrier_init();
  }
  if (warp == 2) tmem_alloc(&bars.tmem_base, tmem_cols);
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = bars.tmem_base;
  const int64_t total = tile_count<KIND>(a);

  if (R::kTma && warp == 0) {
    // ---- tiled loads: kRows' matrices, sorted planes, stacks ----
    if (lane < PLANES) {
      if (!R::kGather) prefetch_tmap(&maps.a[lane]);
      prefetch_tmap(&maps.b[lane]);
    }
    Ring ring;
    int64_t filled = 0;
    bool ok = true;
    const uint32_t bytes = (uint32_t)(R::kGather ? bbytes : stage_bytes);
    for (int64_t it = blockIdx.x; ok && it < total; it += gridDim.x) {
      const Tile t = decode<KIND>(a, it);
      for (int kb = 0; kb < t.kb; ++kb, ring.step(a.stages), ++filled) {
        const int s = ring.i;
        ok = mbar_wait_warp(&bars.empty[s], ring.phase ^ 1, abort);
        if (!ok) break;
        char* sa = sm + s * stage_bytes;
        char* sb = sa + PLANES * kABytes;
        uint64_t* bar = &bars.full[s];
        if (lane == 0) mbar_expect_tx(bar, bytes);
        __syncwarp();
        const int k0 = kb * kBlockK;
#pragma unroll
        for (int p = 0; p < PLANES; ++p) {
          char* pa = sa + p * kABytes;
          char* pb = sb + p * bbytes;
          if (KIND == kWeights) {  // 64 sorted rows x 64 columns per box
            if (lane < 2) tma_load_3d(pa + lane * 8192, &maps.a[p], t.m0 + lane * 64, t.pos + k0, 0, bar);
            if (lane < a.bn / 64) tma_load_3d(pb + lane * 8192, &maps.b[p], t.n0 + lane * 64, t.pos + k0, 0, bar);
            continue;
          }
          if (KIND == kRows) {
            if (!R::kGather && lane == 0) tma_load_3d(pa, &maps.a[p], k0, t.pos, 0, bar);
          } else if (a.a_mn) {
            if (lane < 2) tma_load_3d(pa + lane * 8192, &maps.a[p], t.m0 + lane * 64, k0, t.g, bar);
          } else {
            if (lane == 0) tma_load_3d(pa, &maps.a[p], k0, t.m0, t.g, bar);
          }
          if (a.b_mn) {
            if (lane < a.bn / 64) tma_load_3d(pb + lane * 8192, &maps.b[p], t.n0 + lane * 64, k0, t.g, bar);
          } else {
            if (lane == 0) tma_load_3d(pb, &maps.b[p], k0, t.n0, t.g, bar);
          }
        }
      }
    }
    if (!ok) {  // the copies in flight still write shared memory: wait for them before the block ends
      give_up(&bars, lane);
      const int64_t first = filled > a.stages ? filled - a.stages : 0;
      for (int64_t f = first; f < filled; ++f) mbar_wait_warp(&bars.full[f % a.stages], (uint32_t)((f / a.stages) & 1), nullptr);
    }
  } else if (PLANES == 1 && warp == 1) {
    // ---- products of one plane: one thread ----
    if (lane == 0) {
      Ring ring, sums;
      int64_t use = 0;
      bool ok = true, peeked = false;  // peeked: the stage at `ring` is known to be there
      const uint32_t step_a = (a.a_mn ? 2048 : 32) >> 4, step_b = (a.b_mn ? 2048 : 32) >> 4;
      const uint64_t desc_a = a.a_mn ? desc_mnmajor(smem_u32(sm), 8192) : desc_kmajor(smem_u32(sm));
      const uint32_t sb0 = smem_u32(sm) + kABytes;
      const uint64_t desc_b = a.b_mn ? desc_mnmajor(sb0, 8192) : desc_kmajor(sb0);
      const uint32_t stage_units = (uint32_t)stage_bytes >> 4;
      const uint32_t idesc = a.idesc;
      uint64_t* there = R::kGather ? bars.ready : bars.full;
      Tile t{};
      if (blockIdx.x < total) t = decode<KIND>(a, blockIdx.x);
      for (int64_t it = blockIdx.x; ok && it < total; it += gridDim.x) {
        const int64_t ahead = it + gridDim.x < total ? it + gridDim.x : it;
        if (t.kb == 0) {
          t = decode<KIND>(a, ahead);
          continue;
        }
        ok = mbar_wait(&bars.accempty[sums.i], sums.phase ^ 1, abort);
        if (!ok) break;
        tmem_fence_after();
        const uint32_t d = tmem + sums.i * a.bn;
        Tile u = t;
        for (int kb = 0; kb < t.kb; ++kb, ++use) {
          if (!peeked) ok = mbar_wait(&there[ring.i], ring.phase, abort);
          if (!ok) break;
          tmem_fence_after();
          const uint64_t da = desc_a + (uint32_t)ring.i * stage_units, db = desc_b + (uint32_t)ring.i * stage_units;
          uint64_t* done = &bars.empty[ring.i];
          const bool last = kb == t.kb - 1;
          const int steps = KIND == kWeights && last ? min(4, (t.rows - kb * kBlockK + 15) >> 4) : 4;
          ring.step(a.stages);
          if (steps == 4) {
            mma_16(d, da, db, idesc, kb != 0);
            mma_16(d, da + step_a, db + step_b, idesc, 1);
            // While these run: whether the next stage is there, or what comes after this tile.  The
            // tensor core takes few products ahead, so what stands between two stages' products is idle time.
            if (last) u = decode<KIND>(a, ahead);
            peeked = mbar_test(&there[ring.i], ring.phase);
            mma_16(d, da + 2 * step_a, db + 2 * step_b, idesc, 1);
            mma_16(d, da + 3 * step_a, db + 3 * step_b, idesc, 1);
          } else {
            for (int k = 0; k < steps; ++k) mma_16(d, da + k * step_a, db + k * step_b, idesc, (kb | k) != 0);
            u = decode<KIND>(a, ahead);
            peeked = false;
          }
          mma_commit(done);
          if (last) mma_commit(&bars.accfull[sums.i]);
        }
        sums.step(2);
        t = u;
      }
      if (!ok) {  // products in flight still read shared and write tensor memory
        give_up(&bars, 0);
        const int64_t first = use > a.stages ? use - a.stages : 0;
        for (int64_t f = first; f < use; ++f) mbar_wait(&bars.empty[f % a.stages], (uint32_t)((f / a.stages) & 1), nullptr);
      }
    }
  } else if (R::kGather && warp == 3) {
    // ---- stages whose copies have landed: fence the proxies (cp.async wrote through the generic one) ----
    Ring ring;
    bool ok = true;
    for (int64_t it = blockIdx.x; ok && it < total; it += gridDim.x) {
      const int n = decode<KIND>(a, it).kb;
      for (int kb = 0; kb < n; ++kb, ring.step(a.stages)) {
        ok = mbar_wait_warp(&bars.full[ring.i], ring.phase, abort);
        if (!ok) break;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.ready[ring.i]);
      }
    }
    if (!ok) give_up(&bars, lane);
  } else if (PLANES > 1 && warp == 1) {
    // ---- products ----
    Ring ring, sums;
    int64_t use = 0;
    bool ok = true;
    // descriptor units (16 bytes) per 16 contraction elements
    const uint32_t step_a = (a.a_mn ? 2048 : 32) >> 4, step_b = (a.b_mn ? 2048 : 32) >> 4;
    const uint64_t desc_a = a.a_mn ? desc_mnmajor(smem_u32(sm), 8192) : desc_kmajor(smem_u32(sm));
    const uint32_t sb0 = smem_u32(sm) + PLANES * kABytes;
    const uint64_t desc_b = a.b_mn ? desc_mnmajor(sb0, 8192) : desc_kmajor(sb0);
    const uint32_t stage_units = (uint32_t)stage_bytes >> 4, b_units = (uint32_t)bbytes >> 4;
    const uint32_t idesc = a.idesc;
    for (int64_t it = blockIdx.x; ok && it < total; it += gridDim.x) {
      const Tile t = decode<KIND>(a, it);
      int buf = 0;
      uint32_t d = 0;
      for (int kb = 0; kb < t.kb; ++kb, ring.step(a.stages), ++use) {
        const int in_sum = PLANES > 1 ? kb % kChunk : kb;  // stages already in this accumulator
        if (in_sum == 0) {
          buf = sums.i;
          ok = mbar_wait_warp(&bars.accempty[buf], sums.phase ^ 1, abort);
          if (!ok) break;
          tmem_fence_after();
          d = tmem + buf * kAccs * a.bn;
          sums.step(2);
        }
        const int s = ring.i;
        ok = mbar_wait_warp(&bars.full[s], ring.phase, abort);
        if (!ok) break;
        int steps = 4;
        if (KIND == kWeights) {
          const int left = t.rows - kb * kBlockK;
          if (left < kBlockK) steps = (left + 15) >> 4;
          if (left < kBlockK) {
            const int zero = steps * 16 - left;  // rows to clear, of 128 bytes in each 64-column group
            if (zero > 0) {
              char* sa = sm + s * stage_bytes;
              char* sb = sa + PLANES * kABytes;
              const int groups = PLANES * (2 + a.bn / 64);
              for (int i = lane; i < groups * zero * 8; i += 32) {
                const int grp = i / (zero * 8), r = left + (i % (zero * 8)) / 8, q = i % 8;
                char* g = grp < 2 * PLANES ? sa + grp * 8192 : sb + (grp - 2 * PLANES) * 8192;
                *reinterpret_cast<uint4*>(g + r * 128 + q * 16) = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async();
              __syncwarp();
            }
          }
        }
        if (lane == 0) {
          tmem_fence_after();
          constexpr int kPairs = PLANES == 1 ? 1 : PLANES == 2 ? 3 : 6;
#pragma unroll
          for (int c = 0; c < kPairs; ++c) {
            constexpr int pa[6] = {0, 0, 1, 1, 0, 2}, pb[6] = {0, 1, 0, 1, 2, 0};
            const uint64_t da = desc_a + (uint32_t)s * stage_units + pa[c] * (kABytes >> 4);
            const uint64_t db = desc_b + (uint32_t)s * stage_units + pb[c] * b_units;
            const uint32_t dc = c == 0 ? d : d + a.bn;
            const bool add = in_sum != 0 || c > 1;
            if (steps == 4) {
#pragma unroll
              for (int k = 0; k < 4; ++k) mma_16(dc, da + k * step_a, db + k * step_b, idesc, k != 0 || add);
            } else {
              for (int k = 0; k < steps; ++k) mma_16(dc, da + k * step_a, db + k * step_b, idesc, k != 0 || add);
            }
          }
          mma_commit(&bars.empty[s]);
          if (kb == t.kb - 1 || (PLANES > 1 && in_sum == kChunk - 1)) mma_commit(&bars.accfull[buf]);
        }
        __syncwarp();
      }
    }
    if (!ok) {  // products in flight still read shared and write tensor memory
      give_up(&bars, lane);
      const int64_t first = use > a.stages ? use - a.stages : 0;
      for (int64_t u = first; u < use; ++u) mbar_wait_warp(&bars.empty[u % a.stages], (uint32_t)((u / a.stages) & 1), nullptr);
    }
  } else if (warp >= kEpiWarp0 && warp < kEpiWarp0 + kEpiWarps) {
    // ---- results ----
    const int w = warp - kEpiWarp0;
    const int row = (w & 3) * 32 + lane;            // row of the tile: the accumulator's lane
    const int c_lo = (w >> 2) * (a.bn / 2), c_hi = c_lo + a.bn / 2;
    Ring sums;
    bool ok = true;
    for (int64_t it = blockIdx.x; ok && it < total; it += gridDim.x) {
      const Tile t = decode<KIND>(a, it);
      float held[PLANES > 1 ? 64 : 1];  // sums of the finished accumulations (bn <= 128: 64 columns at most)
      if (PLANES > 1) {
#pragma unroll
        for (int i = 0; i < 64; ++i) held[i] = 0.f;
        for (int kb = 0; kb < t.kb; kb += kChunk, sums.step(2)) {
          const int buf = sums.i;
          ok = mbar_wait_warp(&bars.accfull[buf], sums.phase, abort);
          if (!ok) break;
          tmem_fence_after();
          const uint32_t acc = tmem + buf * 2 * a.bn + c_lo + ((uint32_t)((w & 3) * 32) << 16);
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (c_lo + 32 * j < c_hi) {
              float lead[32], rest[32];
              tmem_ld32(acc + 32 * j, lead);
              tmem_ld32(acc + a.bn + 32 * j, rest);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) held[32 * j + i] += lead[i] + rest[i];
            }
          tmem_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.accempty[buf]);
        }
      } else if (t.kb > 0) {
        ok = mbar_wait_warp(&bars.accfull[sums.i], sums.phase, abort);
        tmem_fence_after();
      }
      if (!ok) {
        give_up(&bars, lane);
        break;
      }
      const int buf = sums.i;
      if (PLANES == 1 && t.kb > 0) sums.step(2);
      // where this thread's row goes
      const int valid_rows = KIND == kWeights ? min(kBM, a.m - t.m0) : t.rows;
      const bool live = row < valid_rows;
      void* out = a.out;
      int dt = a.out_dt, vec = a.vec;
      int64_t at = 0;
      if (KIND == kRows && live) {
        at = (int64_t)__ldg(a.order + t.pos + row) * a.ldo;
      } else if (KIND == kWeights) {
        if (t.slot >= 0) {
          out = a.part;
          dt = GMMXX_FLOAT32;
          vec = (a.n & 3) == 0;
          at = ((int64_t)t.slot * a.m + t.m0 + row) * a.n;
        } else {
          at = t.g * a.out_stride + (int64_t)(t.m0 + row) * a.ldo;
        }
      }
      const int n_left = a.n - t.n0;
#pragma unroll
      for (int j = 0; j < (PLANES > 1 ? 2 : 4); ++j) {
        const int c = c_lo + 32 * j;
        if (c >= c_hi) break;
        float v[32];
        __syncwarp();
        if (PLANES > 1) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = held[(32 * j + i) % (PLANES > 1 ? 64 : 1)];
        } else if (t.kb > 0) {
          tmem_ld32(tmem + buf * a.bn + c + ((uint32_t)((w & 3) * 32) << 16), v);
          tmem_wait_ld();
          if (c + 32 == c_hi) {  // the accumulator is in registers: free it for the tile after next
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.accempty[buf]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.f;
        }
        const int nv = n_left - c;
        if (!live || nv <= 0) continue;
        if (KIND == kBatch) {
          batch32<PLANES>(a, t, t.m0 + row, t.n0 + c, v, nv);
        } else {
          if (KIND == kRows && a.bias != nullptr && t.kb > 0) {
            const int64_t b0 = (int64_t)t.g * a.n + t.n0 + c;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < nv) v[i] += load_x(a.bias, b0 + i, a.bias_dt);
          }
          store32(out, dt, at + t.n0 + c, v, nv, vec);
        }
      }
    }
  }
  if (R::kGather && warp >= kGatherWarp0) {
    // ---- gathered rows: thread = 16-byte piece `q` of every 16th row ----
    const int tid = threadIdx.x - kGatherWarp0 * 32, q = tid & 7, r0 = tid >> 3;
    const uint32_t at = (uint32_t)(r0 * 128 + ((q ^ (r0 & 7)) << 4));  // 128-byte swizzle; rows r0 + 16 i: + 2048 i
    Ring ring;
    bool ok = true;
    constexpr int kR = KIND == kRows ? 8 : 4;  // rows of a stage per thread
    // The next tile's place and rows are fetched while this tile's stages are
    // in flight: each of these loads waits for the one before.
    Tile t{};
    if (blockIdx.x < total) t = decode<KIND>(a, blockIdx.x);
    int next[kR];
    auto first_rows = [&](const Tile& u) {
#pragma unroll
      for (int i = 0; i < kR; ++i) {
        const int r = r0 + 16 * i;
        if (u.kb > 0) next[i] = __ldg(a.order + u.pos + (r < u.rows ? r : 0));
      }
    };
    first_rows(t);
    for (int64_t it = blockIdx.x; ok && it < total; it += gridDim.x) {
      const int64_t ahead = it + gridDim.x < total ? it + gridDim.x : it;
      Tile u = t;
      if (t.kb == 0) {
        t = decode<KIND>(a, ahead);
        first_rows(t);
        continue;
      }
      const char* src[8];
      if (KIND == kRows) {
#pragma unroll
        for (int i = 0; i < kR; ++i) src[i] = a.src_a + ((int64_t)(next[i] / a.div_a) * a.ld_a + q * 8) * 2;
      }
      for (int kb = 0; kb < t.kb; ++kb, ring.step(a.stages)) {
        const bool last = kb == t.kb - 1;
        const int s = ring.i;
        if (KIND == kWeights) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            src[i] = a.src_a + ((int64_t)(next[i] / a.div_a) * a.ld_a + q * 8 + t.m0) * 2;
            src[4 + i] = a.src_b + ((int64_t)(next[i] / a.div_b) * a.ld_b + q * 8 + t.n0) * 2;
            if (!last) next[i] = __ldg(a.order + t.pos + min((kb + 1) * kBlockK + r0 + 16 * i, t.rows - 1));
          }
        }
        ok = mbar_wait_warp(&bars.empty[s], ring.phase ^ 1, abort);
        if (!ok) break;
        const uint32_t sa = smem_u32(sm) + s * stage_bytes + at;
        if (KIND == kRows) {
          const bool live = kb * kBlockK + q * 8 < a.k;
          const int64_t k0 = live ? (int64_t)kb * (kBlockK * 2) : 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) copy16(sa + 2048 * i, src[i] + k0, live);
        } else {
          const uint32_t sb = sa + kABytes;
          const int left = t.rows - kb * kBlockK - r0;  // rows r0 + 16 i < left are the segment's
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const bool in = t.m0 + g * 64 + q * 8 < a.m;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool live = in && 16 * i < left;
              copy16(sa + g * 8192 + 2048 * i, live ? src[i] + g * 128 : a.src_a, live);
            }
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (g >= a.bn / 64) break;
            const bool in = t.n0 + g * 64 + q * 8 < a.n;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool live = in && 16 * i < left;
              copy16(sb + g * 8192 + 2048 * i, live ? src[4 + i] + g * 128 : a.src_b, live);
            }
          }
        }
        copies_arrive(&bars.full[s]);
        if (kb == 0) u = decode<KIND>(a, ahead);
        if (last) first_rows(u);
      }
      t = u;
    }
    if (!ok && lane == 0) give_up(&bars, lane);
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, tmem_cols);
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode(CUtensorMap* map, const void* base, int fp16, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box) {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<EncodeFn>(p) : nullptr;
  }();
  if (fn == nullptr) return set_error(GMMXX_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult rc = fn(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
                         const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return set_error(GMMXX_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)rc);
  return GMMXX_OK;
}

template <int KIND, int PLANES>
int launch_one(const ProductMaps& maps, const ProductArgs& a, unsigned grid, cudaStream_t st) {
  const int smem = a.stages * PLANES * (kABytes + a.bn * 128) + 1024;
  if (int rc = allow_smem((const void*)product_kernel<KIND, PLANES>, smem)) return rc;
  product_kernel<KIND, PLANES><<<grid, Roles<KIND, PLANES>::kThreads, smem, st>>>(maps, a);
  return check_launch("product_kernel");
}

}  // namespace

// a stack of matrices: boxes of 64 elements x box_rows rows of one matrix; what lies beyond a matrix reads as zero
int encode_stack(CUtensorMap* map, const void* base, int fp16, int64_t cols, int64_t rows, int64_t ld, int64_t stack,
                 int64_t stride, int box_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)stack};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)stride * 2};
  const cuuint32_t box[3] = {kBlockK, (cuuint32_t)box_rows, 1};
  return encode(map, base, fp16, 3, dims, strides, box);
}

uint32_t product_idesc(int fp16, int bn, int a_mn, int b_mn) {
  uint32_t d = idesc_bf16(kBM, bn, a_mn, b_mn);
  if (fp16) d &= ~((1u << 7) | (1u << 10));  // A and B types: 0 = fp16, 1 = bf16
  return d;
}

int product_stages(int planes, int bn) {
  return std::min(kMaxStages, (kSmemLimit - 2048) / (planes * (kABytes + bn * 128)));
}

int device_sms(int* sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return set_error(GMMXX_ERR_CUDA, "device query: %s", cudaGetErrorString(e));
  return GMMXX_OK;
}

int launch_product(Kind kind, int planes, const ProductMaps& maps, const ProductArgs& a, int64_t max_items,
                   cudaStream_t st) {
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(sms, max_items * a.mt * a.nt));
  if (kind == kRows) return planes == 1 ? launch_one<kRows, 1>(maps, a, grid, st) : launch_one<kRows, 3>(maps, a, grid, st);
  if (kind == kWeights)
    return planes == 1 ? launch_one<kWeights, 1>(maps, a, grid, st) : launch_one<kWeights, 3>(maps, a, grid, st);
  return planes == 1 ? launch_one<kBatch, 1>(maps, a, grid, st) : launch_one<kBatch, 2>(maps, a, grid, st);
}

int read_status(int* out, cudaStream_t st) {
  int v = 0;
  const int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && v != 0) e = cudaMemcpyToSymbolAsync(g_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
  if (e == cudaSuccess && v != 0) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return set_error(GMMXX_ERR_CUDA, "status read: %s", cudaGetErrorString(e));
  *out = v != 0 ? GMMXX_ERR_TIMEOUT : GMMXX_OK;
  return GMMXX_OK;
}

}  // namespace experts
}  // namespace gmmxx
