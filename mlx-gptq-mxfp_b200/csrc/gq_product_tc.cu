// Grouped and dense products on the 5th-generation tensor cores: Y[s] = X[rows[s]] W_e^T,
// optionally with SwiGLU, for bf16 / f16 rows (tcgen05 kind::f16, fp32 sums) and 8-bit
// codes (kind::i8, exact s32 sums, scales per row and channel in the epilogue).
//
// The weights are the M operand and the rows the N operand: D^T[channel][row]. A tile is
// then 256 channels of one expert by 16 .. 256 of its rows (a multiple of 16, of 32 for
// s8), so an expert's rows are cut into equal tiles and a ragged expert costs at most 15
// (31) idle rows instead of most of a 128-row tile; and a row of D^T is one channel, so
// SwiGLU needs no exchange: gate and up are two accumulators with the same lanes and
// columns, combined by the thread that drains them.
//
// A cluster of two CTAs shares a tile (cta_group::2, M = 256): each loads 128 channels of
// the weights and half of the rows per 128-byte k-step. Persistent: pair p takes tiles p,
// p + pairs, ... of a list that every role derives from the offsets on the device (tiles
// per expert, scanned once into shared memory): nothing is read back to the host.
//   warp 0       TMA: weights [expert, channel, k] and, without a row list, X (32-row boxes)
//   warp 1       MMA issuer (even CTA), one of two TMEM accumulator sets per tile
//   warps 2-9    drain the other set, scale / bias / SwiGLU, round once, store
//   warps 10-13  with a row list: cp.async gathers of X rows into the swizzled stage
// Every wait is bounded (gq_common.cuh); a wait that gives up records GQ_ERR_TIMEOUT.
#include <algorithm>
#include <atomic>

#include "gq_product.cuh"

namespace gq {
namespace prod {
namespace {

constexpr int EPI_WARPS = 8, GATHER_WARPS = 4;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t A_BYTES = 128 * 128;  // 128 channels x 128 bytes of k
constexpr int BOX_ROWS = 32;             // rows of one TMA box of X
constexpr uint32_t BOX_BYTES = BOX_ROWS * 128;
constexpr int GATHER_LAG = 3;            // stages whose copies a gather warp has in flight
constexpr uint32_t kEvenCta = 0xFEFFFFFFu;  // shared::cluster address -> even CTA of the pair

template <bool GLU>
struct Shape {
  static constexpr int NMAX = GLU ? 128 : 256;  // rows per tile
  static constexpr int ACCS = GLU ? 2 : 1;      // accumulators (gate, up)
  static constexpr uint32_t B_BYTES = uint32_t(NMAX / 2) * 128;
  static constexpr uint32_t STAGE_BYTES = ACCS * A_BYTES + B_BYTES;
  static constexpr int STAGES = GLU ? 5 : 6;
  static constexpr size_t SMEM_BYTES =
      size_t(STAGES) * STAGE_BYTES + 1024 /*align*/ + 256 /*barriers*/ + 8 * (kMaxExperts + 1) /*tiles, rows*/;
};
static_assert(Shape<false>::SMEM_BYTES <= 227 * 1024 && Shape<true>::SMEM_BYTES <= 227 * 1024, "shared memory");

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t even_cta(const void* p) { return smem_u32(p) & kEvenCta; }

// Arrive on a barrier of the even CTA, releasing this thread's writes to the cluster.
__device__ __forceinline__ void arrive_even(uint64_t* bar) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(bar)));
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(r) : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// mbar_wait for barriers that the other CTA of the pair arrives on.
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                             int32_t* status) {
  if (!mbar_wait(bar, parity, abort_flag, status)) return false;
  return try_wait_cluster(bar, parity);  // complete already: acquires the other CTA's writes
}

__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(even_cta(bar))
      : "memory");
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
      "%4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(even_cta(bar))
      : "memory");
}

template <bool I8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (I8)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives on the barrier at this offset in both CTAs once the issued MMAs complete.
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(uint16_t(3))
      : "memory");
}

// 16 bytes global -> shared, zeros where on is false (nothing is read then).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

// Instruction descriptor: M = 256, N rows, both operands K-major.
__device__ __forceinline__ uint32_t instruction_desc(Kind kind, int n) {
  const uint32_t types = kind == S8 ? (2u << 4) | (1u << 7) | (1u << 10)     // s32 sums, s8 x s8
                                    : (1u << 4) | (kind == BF16 ? (1u << 7) | (1u << 10) : 0u);  // f32 sums
  return types | (uint32_t(n >> 3) << 17) | (uint32_t(256 >> 4) << 24);
}

struct Tile {
  int64_t row0;  // first product row
  int rows;      // rows that are written
  int n;         // rows of the MMA (a multiple of the kind's step)
  int expert, channel0;
};

// Tile q of the list: expert by expert, row tile by row tile, its 256-channel tiles.
__device__ __forceinline__ Tile tile_of(int64_t q, const int32_t* first_tile, int E, int ct,
                                        int nmax, int step, const Args& a) {
  int lo = 0, hi = E;  // last expert whose tiles begin at or before q / ct
  const int32_t r = int32_t(q / ct);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_tile[mid] <= r) lo = mid; else hi = mid;
  }
  int64_t begin, end;
  segment(a, lo, begin, end);
  const int64_t n = end - begin;
  const int tiles = int((n + nmax - 1) / nmax);
  const int per = int(((n + tiles - 1) / tiles + step - 1) / step) * step;  // <= nmax: nmax is a multiple of step
  Tile t;
  t.expert = lo;
  t.channel0 = int(q % ct) * 256;
  const int64_t r0 = int64_t(r - first_tile[lo]) * per;
  t.row0 = begin + r0;
  t.rows = int(n - r0 < per ? (n - r0 > 0 ? n - r0 : 0) : per);
  t.n = per;
  return t;
}

template <bool I8, bool GLU, bool GATHER>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(64 + 32 * EPI_WARPS + (GATHER ? 32 * GATHER_WARPS : 0), 1)
    tc_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Args a,
              const Kind kind) {
  typedef Shape<GLU> Sh;
  constexpr int STAGES = Sh::STAGES, NMAX = Sh::NMAX, STEP = I8 ? 32 : 16;
  constexpr int KSTEP = I8 ? 128 : 64;  // elements per stage
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * Sh::STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;  // [2] accumulator set complete (both CTAs)
  uint64_t* tempty = tfull + 2;      // [2] accumulator set drained by both CTAs (used in the even CTA)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int32_t* first_tile = reinterpret_cast<int32_t*>(smem + STAGES * Sh::STAGE_BYTES + 256);  // [E + 1]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  const int E = int(a.E), pairs = int(gridDim.x >> 1), pair = int(blockIdx.x >> 1);
  const int64_t I = GLU ? a.N / 2 : a.N;
  const int ct = int((I + 255) / 256);
  const int KT = int((a.K + KSTEP - 1) / KSTEP);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1 + (GATHER ? 2 * GATHER_WARPS : 0));
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * EPI_WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  if (warp == 2) {  // exclusive scan of the experts' row tiles
    int32_t carry = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      int64_t begin = 0, end = 0;
      if (e < E) segment(a, e, begin, end);
      const int32_t mine = int32_t((end - begin + NMAX - 1) / NMAX);
      int32_t incl = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int32_t o = __shfl_up_sync(~0u, incl, d);
        if (lane >= d) incl += o;
      }
      if (e < E) first_tile[e] = carry + incl - mine;
      carry += __shfl_sync(~0u, incl, 31);
    }
    if (lane == 0) first_tile[E] = carry;
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t tiles = int64_t(first_tile[E]) * ct;

  if (warp == 0) {
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&wmap)) : "memory");
      if (!GATHER) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&xmap)) : "memory");
      int64_t it = 0;
      bool ok = true;
      for (int64_t q = pair; q < tiles && ok; q += pairs) {
        const Tile t = tile_of(q, first_tile, E, ct, NMAX, STEP, a);
        const int half = t.n / 2, boxes = GATHER ? 0 : (half + BOX_ROWS - 1) / BOX_ROWS;
        const uint32_t bytes = Sh::ACCS * A_BYTES + uint32_t(boxes) * BOX_BYTES;
        const int ch = t.channel0 + int(rank) * 128, y = int(t.row0) + int(rank) * half;
        for (int kt = 0; kt < KT; ++kt, ++it) {
          const int s = int(it % STAGES);
          if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * bytes);  // both CTAs' bytes
          uint8_t* st = smem + s * Sh::STAGE_BYTES;
          tma_3d(st, &wmap, kt * KSTEP, ch, t.expert, &full[s]);
          if (GLU) tma_3d(st + A_BYTES, &wmap, kt * KSTEP, int(I) + ch, t.expert, &full[s]);
          for (int b = 0; b < boxes; ++b)
            tma_2d(st + Sh::ACCS * A_BYTES + b * BOX_BYTES, &xmap, kt * KSTEP, y + b * BOX_ROWS, &full[s]);
        }
      }
      if (*abort_flag && rank == 0) {  // let copies already in flight land before the CTA exits
        volatile int never = 0;
        for (int64_t i = it > STAGES ? it - STAGES : 0; i < it; ++i)
          mbar_wait(&full[i % STAGES], (i / STAGES) & 1, &never, nullptr);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int64_t it = 0;
      int n_tile = 0;
      bool ok = true;
      for (int64_t q = pair; q < tiles && ok; q += pairs, ++n_tile) {
        const Tile t = tile_of(q, first_tile, E, ct, NMAX, STEP, a);
        const uint32_t idesc = instruction_desc(kind, t.n);
        const int buf = n_tile & 1;
        if (!wait_cluster(&tempty[buf], ((n_tile >> 1) & 1) ^ 1, abort_flag, a.status)) break;
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(buf * 256);
        for (int kt = 0; kt < KT; ++kt, ++it) {
          const int s = int(it % STAGES);
          if (!wait_cluster(&full[s], (it / STAGES) & 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + s * Sh::STAGE_BYTES), b0 = a0 + Sh::ACCS * A_BYTES;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {  // 32 bytes of k each, inside the 128-byte swizzle atom
            const uint64_t bd = umma_desc_sw128(b0 + kk * 32, 16, 1024);
            mma<I8>(d, umma_desc_sw128(a0 + kk * 32, 16, 1024), bd, idesc, kt != 0 || kk != 0);
            if (GLU) mma<I8>(d + 128, umma_desc_sw128(a0 + A_BYTES + kk * 32, 16, 1024), bd, idesc, kt != 0 || kk != 0);
          }
          commit(&empty[s]);  // frees the stage once these MMAs have read it
        }
        if (ok) commit(&tfull[buf]);
      }
    }
  } else if (warp < 2 + EPI_WARPS) {
    // TMEM lane quarter warp % 4 (channels), half of the tile's columns (rows)
    const int qw = warp & 3, part = (warp - 2) >> 2;
    const uint32_t lane_base = uint32_t(qw * 32) << 16;
    int n_tile = 0;
    for (int64_t q = pair; q < tiles; q += pairs, ++n_tile) {
      const Tile t = tile_of(q, first_tile, E, ct, NMAX, STEP, a);
      const int buf = n_tile & 1;
      if (!mbar_wait(&tfull[buf], (n_tile >> 1) & 1, abort_flag, a.status)) break;
      tc_fence_after();
      const int64_t ch = t.channel0 + int(rank) * 128 + qw * 32 + lane;
      const bool live = ch < I;
      float ws = 1.0f, ws_up = 1.0f, bias = 0.0f;
      if (live && I8) {
        ws = a.ws[t.expert * a.N + ch];
        if (GLU) ws_up = a.ws[t.expert * a.N + I + ch];
      }
      if (live && a.bias) bias = load_as_f32(a.bias, ch, a.bias_dtype);
      for (int c = part * 32; c < t.rows; c += 64) {
        uint32_t r[32], u[GLU ? 32 : 1];
        tmem_ld32(tmem + lane_base + uint32_t(buf * 256 + c), r);
        if constexpr (GLU) tmem_ld32(tmem + lane_base + uint32_t(buf * 256 + 128 + c), u);
        float xs_lane = 0.0f;
        if (I8 && c + lane < t.rows) {
          const int64_t src = source_row(a, t.row0 + c + lane);
          xs_lane = src >= 0 ? a.xs[src] : 0.0f;
        }
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          float v, up = 0.0f;
          if (I8) {
            const float xs = __shfl_sync(~0u, xs_lane, j);
            v = float(int32_t(r[j])) * xs * ws;
            if constexpr (GLU) up = float(int32_t(u[j])) * xs * ws_up;
          } else {
            v = __uint_as_float(r[j]);
            if constexpr (GLU) up = __uint_as_float(u[j]);
          }
          v = v + bias;
          if (GLU) v = swiglu(v, up);
          if (live && c + j < t.rows) store_from_f32(a.Y, (t.row0 + c + j) * a.ldy + ch, v, a.out_dtype);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_even(&tempty[buf]);
    }
    if (a.zero_behind) {
      const int64_t first = rows_end(a), count = (a.S - first) * I;
      for (int64_t i = int64_t(blockIdx.x) * (32 * EPI_WARPS) + threadIdx.x - 64; i < count;
           i += int64_t(gridDim.x) * (32 * EPI_WARPS))
        store_from_f32(a.Y, (first + i / I) * a.ldy + i % I, 0.0f, a.out_dtype);
    }
  } else if (GATHER) {
    const int tid = threadIdx.x - (64 + 32 * EPI_WARPS), chunk = tid & 7, r_base = tid >> 3;
    constexpr int RPT = NMAX / 2 / 16;  // rows per thread
    const int64_t kbytes = a.K * (I8 ? 1 : 2);
    int64_t it = 0, arrived = 0;
    bool ok = true;
    for (int64_t q = pair; q < tiles && ok; q += pairs) {
      const Tile t = tile_of(q, first_tile, E, ct, NMAX, STEP, a);
      const int half = t.n / 2;
      const uint8_t* src[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int r = int(rank) * half + r_base + 16 * i;  // row of the tile
        const int64_t x = r_base + 16 * i < half && r < t.rows ? source_row(a, t.row0 + r) : -1;
        src[i] = x >= 0 ? a.X + x * a.ldx + chunk * 16 : nullptr;
      }
      for (int kt = 0; kt < KT; ++kt, ++it) {
        const int s = int(it % STAGES);
        if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1, abort_flag, a.status)) {
          ok = false;
          break;
        }
        const uint32_t dst = smem_u32(smem + s * Sh::STAGE_BYTES + Sh::ACCS * A_BYTES);
        const bool in = kt * 128 + chunk * 16 < kbytes;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const int r = r_base + 16 * i;
          if (r < half) {
            const bool on = in && src[i] != nullptr;
            cp_async16(dst + r * 128 + ((chunk ^ (r & 7)) << 4), on ? src[i] + kt * 128 : a.X, on);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (it >= GATHER_LAG) {
          asm volatile("cp.async.wait_group %0;" ::"n"(GATHER_LAG) : "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) arrive_even(&full[arrived % STAGES]);
          ++arrived;
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    for (; arrived < it; ++arrived)
      if (lane == 0) arrive_even(&full[arrived % STAGES]);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
  }
}

int encode(CUtensorMap* map, const void* base, Kind kind, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (!enc) {
    set_last_error("cuTensorMapEncodeTiled unavailable");
    return GQ_ERR_CUDA;
  }
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType type = kind == S8     ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : kind == BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = enc(map, type, cuuint32_t(rank), const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("cuTensorMapEncodeTiled failed (%d)", int(r));
    return GQ_ERR_CUDA;
  }
  return GQ_OK;
}

template <bool I8, bool GLU, bool GATHER>
int launch(const CUtensorMap& wmap, const CUtensorMap& xmap, const Args& a, Kind kind, unsigned grid, cudaStream_t s) {
  auto* k = tc_kernel<I8, GLU, GATHER>;
  GQ_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Shape<GLU>::SMEM_BYTES)));
  const int threads = 64 + 32 * EPI_WARPS + (GATHER ? 32 * GATHER_WARPS : 0);
  k<<<grid, threads, Shape<GLU>::SMEM_BYTES, s>>>(wmap, xmap, a, kind);
  return check_launch("tc_kernel");
}

template <bool I8, bool GLU>
int launch_gather(const CUtensorMap& wmap, const CUtensorMap& xmap, const Args& a, Kind kind, unsigned grid,
                  cudaStream_t s) {
  return a.rows ? launch<I8, GLU, true>(wmap, xmap, a, kind, grid, s)
                : launch<I8, GLU, false>(wmap, xmap, a, kind, grid, s);
}

}  // namespace

int launch_tc(const Args& a, Kind kind, bool glu, cudaStream_t s) {
  const cuuint64_t es = kind == S8 ? 1 : 2;
  const cuuint32_t kbox = cuuint32_t(128 / es);
  CUtensorMap wmap, xmap;
  const cuuint64_t wdims[3] = {cuuint64_t(a.K), cuuint64_t(a.N), cuuint64_t(a.E)};
  const cuuint64_t wstrides[2] = {cuuint64_t(a.ldw), cuuint64_t(a.stride_w)};
  const cuuint32_t wbox[3] = {kbox, 128, 1};
  int st = encode(&wmap, a.W, kind, 3, wdims, wstrides, wbox);
  if (st != GQ_OK) return st;
  xmap = wmap;
  if (!a.rows) {
    const cuuint64_t xdims[2] = {cuuint64_t(a.K), cuuint64_t(a.n_src)};
    const cuuint64_t xstrides[1] = {cuuint64_t(a.ldx)};
    const cuuint32_t xbox[2] = {kbox, cuuint32_t(BOX_ROWS)};
    st = encode(&xmap, a.X, kind, 2, xdims, xstrides, xbox);
    if (st != GQ_OK) return st;
  }
  int dev = 0, sms = 0;
  GQ_CUDA_TRY(cudaGetDevice(&dev));
  GQ_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const int64_t I = glu ? a.N / 2 : a.N, nmax = glu ? 128 : 256;
  const int64_t most = ((I + 255) / 256) * (a.S / nmax + std::min(a.S, a.E));  // at least the number of tiles
  const unsigned grid = unsigned(2 * std::min<int64_t>(std::max(sms / 2, 1), std::max<int64_t>(most, 1)));
  if (kind == S8)
    return glu ? launch_gather<true, true>(wmap, xmap, a, kind, grid, s)
               : launch_gather<true, false>(wmap, xmap, a, kind, grid, s);
  return glu ? launch_gather<false, true>(wmap, xmap, a, kind, grid, s)
             : launch_gather<false, false>(wmap, xmap, a, kind, grid, s);
}

}  // namespace prod
}  // namespace gq
