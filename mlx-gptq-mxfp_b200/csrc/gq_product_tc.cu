// Grouped and dense products on the 5th-generation tensor cores: Y[s] = X[rows[s]] W_e^T,
// optionally with SwiGLU, for bf16 / f16 rows (tcgen05 kind::f16, fp32 sums) and 8-bit
// codes (kind::i8, exact s32 sums, scales per row and channel in the epilogue).
//
// The weights are the M operand and the rows the N operand: D^T[channel][row]. A tile is
// then 256 channels of one expert by 16 .. 256 of its rows (a multiple of 16, of 32 for
// s8), so an expert's rows are cut into equal tiles and a ragged expert costs at most 15
// (31) idle rows instead of most of a 128-row tile. With SwiGLU the 256 channels are 128
// gate channels and their up channels, interleaved by the order of the tensor map's
// dimensions: a channel's two sums sit in neighbouring lanes, and SwiGLU is one shuffle.
//
// A cluster of two CTAs shares a tile (cta_group::2, M = 256): each loads 128 channels of
// the weights and half of the rows per 128-byte k-step. Persistent: pair p takes tiles p,
// p + pairs, ... of a list that every role derives from the offsets on the device (tiles
// per expert, scanned once into shared memory): nothing is read back to the host.
//   warps 0, 2   TMA: weights [expert, channel, k]; rows of X
//   warp 1       MMA issuer (even CTA) into one of two TMEM accumulator sets
//   warps 4-11   drain the other set into registers; scale / bias / SwiGLU, round once, store
// A row list is applied by a copy before the launch (gather_kernel): 8192 x 4096 x 4096 bf16
// takes 186 us without and 205 us with it. Gathering inside the kernel was built and measured
// on the same product: 262 us with cp.async by six warps into the stages, 284 us with gather4
// loads issued by six threads (20 ns each, 32 per stage).
//
// What bounds it, on the same product (7 tiles of 64 k-steps per pair): the loads alone take
// 135 us (32 KB per step, 109 GB/s per SM). The MMAs are 512 cycles per step by arithmetic,
// 146 us at the 1.58 GHz that the SMs hold here, and the tensor pipes read active for 76% of
// the kernel's time (188 us under ncu). Loads and MMAs share shared memory's bandwidth. The
// library's product takes 180 us. Grouped batches stay further from it (65536 rows of 128
// experts of [1536, 2048], SwiGLU: 422 us, pipes active 47%): uneven experts account for 47
// us, SwiGLU with its shorter accumulations for 32. Weights from HBM cost at most 39: experts
// that overlap in memory, and so stay in L2, take 383 us, and equal experts gain nothing by it.
//
// Precision: a tensor-core step loses up to a float32 step of the partial sum, always
// toward zero, so one accumulator over K = 2048 drifts by 5e-6 of |y| (8 x a float32 FMA
// chain). The 16-bit kinds therefore leave TMEM every kChunk k-steps and add the chunks in
// registers, rounding to nearest (the same remedy as in gq_hessian.cu): 1024 products, which
// keeps the drift 30 times below an f16 output's rounding and costs 2 to 3%. Before SwiGLU,
// whose rows are operands again, sums stay as near as an FMA chain's: with L k-steps per
// chunk the drift is proportional to L |y|, the chain's rounding grows with sqrt(K) at most,
// so L is 7 at K = 2048, grows with sqrt(K) above and shrinks with K below. Measured there:
// the rows' error, once rounded to bf16, is 1.2 x that of a float32 product's rows, 3.0 x
// with one accumulation (this goes with the root of the float32 error: 1.5 x and 9 x of it);
// 430 us against 397 with one for 16384 x 2048 x 8192, 450 against 420 for 65536 rows of 128
// experts of [1536, 2048]. s32 sums are exact: one accumulation per tile.
// Every wait is bounded (gq_common.cuh); a wait that gives up records GQ_ERR_TIMEOUT.
#include <algorithm>
#include <type_traits>

#include "gq_product.cuh"

namespace gq {
namespace prod {
namespace {

constexpr int EPI_WARP0 = 4, EPI_WARPS = 8;
// k-steps (64 elements each) per TMEM accumulation of the 16-bit kinds, see above
constexpr int kChunk = 16;
__device__ __forceinline__ int chunk_glu(int steps) {
  return steps > 32 ? __float2int_rn(sqrtf(1.5f * float(steps))) : max(2, (7 * steps + 16) / 32);
}
// Registers: the drain holds a warp's 32 x 128 sums, so the other warps give it some of
// theirs: (88 + 2 * 208) * 128 = 384 threads * 168.
constexpr int THREADS = 32 * (EPI_WARP0 + EPI_WARPS), REGS_FEW = 88, REGS_DRAIN = 208;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t A_BYTES = 128 * 128;  // 128 channels x 128 bytes of k
constexpr int X_MAPS = 4;                // TMA boxes of X: 128, 64, 32 and 16 rows
constexpr uint32_t kEvenCta = 0xFEFFFFFFu;  // shared::cluster address -> even CTA of the pair

// Two tile widths. 256 rows for throughput. 64 rows where experts have few (decoding
// batches): the time is then that of streaming the weights, a tile's loads are nearly all
// weights, and 10 stages of 20 KB keep more of them in flight than 6 of 32 KB. 128 experts
// of [1536, 2048] and [2048, 768], 64 tokens x 8: 112 against 118 us for both products; 256
// tokens: 171 against 165.
template <int NMAX>
struct Shape {
  static constexpr uint32_t B_BYTES = uint32_t(NMAX / 2) * 128;
  static constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = NMAX == 256 ? 6 : 10;
  static constexpr size_t SMEM_BYTES = size_t(STAGES) * STAGE_BYTES + 1024 /*align*/ + 256 /*barriers*/ +
                                       12 * (kMaxExperts + 1) /*tiles and rows of every expert*/;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
  static_assert((2 * STAGES + 4) * 8 + 8 <= 256, "barriers");
};

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Arrive on a barrier of the even CTA, releasing this thread's writes to the cluster.
__device__ __forceinline__ void arrive_even(uint64_t* bar) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(bar)));
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(r) : "memory");
}
// Waits on a barrier given by its address; the first try is inline, the bounded loop is not.
// CLUSTER: the other CTA of the pair arrives on it, and its writes are acquired.
__device__ __noinline__ bool wait_slowly(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status) {
  return mbar_wait(reinterpret_cast<uint64_t*>(__cvta_shared_to_generic(bar)), parity, abort_flag, status);
}
template <bool CLUSTER>
__device__ __forceinline__ bool wait_at(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status) {
  uint32_t ok;
  if constexpr (CLUSTER)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
  if (ok) return true;
  if (!wait_slowly(bar, parity, abort_flag, status)) return false;
  if (CLUSTER) asm volatile("fence.acq_rel.cluster;" ::: "memory");
  return true;
}

__device__ __forceinline__ void expect_tx_at(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// TMA loads into dst, announced on bar of the even CTA (shared-memory addresses).
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar & kEvenCta)
      : "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
      "%4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar & kEvenCta)
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
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          bar),
      "h"(uint16_t(3))
      : "memory");
}

// Instruction descriptor: M = 256, N rows, both operands K-major.
__device__ __forceinline__ uint32_t instruction_desc(Kind kind, int n) {
  const uint32_t types = kind == S8 ? (2u << 4) | (1u << 7) | (1u << 10)     // s32 sums, s8 x s8
                                    : (1u << 4) | (kind == BF16 ? (1u << 7) | (1u << 10) : 0u);  // f32 sums
  return types | (uint32_t(n >> 3) << 17) | (uint32_t(256 >> 4) << 24);
}

// Position in the stage ring, as the shared-memory addresses of the stage and its barriers.
// The loops over it run on one thread each and bound the kernel when they are long: no
// division, no address arithmetic beyond a step (64-bit remainders cost 15% here, one
// thread for both operands' loads 5%).
template <int STAGES, uint32_t STAGE_BYTES>
struct Ring {
  uint32_t data, bar, phase = 0;  // stage s: data + s * STAGE_BYTES; bar: its full, bar + 8 * STAGES: its empty barrier
  uint32_t data0, end;
  __device__ __forceinline__ Ring(const uint8_t* smem, const uint64_t* full)
      : data(smem_u32(smem)), bar(smem_u32(full)), data0(data), end(data + STAGES * STAGE_BYTES) {}
  __device__ __forceinline__ void step() {
    data += STAGE_BYTES, bar += 8;
    if (data == end) data = data0, bar -= 8 * STAGES, phase ^= 1;
  }
  __device__ __forceinline__ uint32_t full() const { return bar; }
  __device__ __forceinline__ uint32_t empty() const { return bar + 8 * STAGES; }
};

struct XMaps {
  CUtensorMap box[X_MAPS];  // box[i]: 128 >> i rows
};

struct Tile {
  int64_t row0;  // first product row
  int rows;      // rows that are written
  int n;         // rows of the MMA (a multiple of the kind's step)
  int expert, block;  // block: of the 256 channels, in the order the tile holds them
};

// The experts' rows [begin, end) and the first of each one's row tiles, in shared memory.
struct Experts {
  int32_t *first_tile, *begin, *end;
};

// Tile q of the list: expert by expert, row tile by row tile, its channel blocks.
__device__ __forceinline__ Tile tile_of(int q, const Experts& x, int E, int ct, int step, int most) {
  int lo = 0, hi = E;  // last expert whose tiles begin at or before q / ct
  const int r = q / ct;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (x.first_tile[mid] <= r) lo = mid; else hi = mid;
  }
  const int n = x.end[lo] - x.begin[lo];
  const int tiles = (n + most - 1) / most;
  const int per = ((n + tiles - 1) / tiles + step - 1) / step * step;  // <= most, a multiple of step
  Tile t;
  t.expert = lo;
  t.block = q - r * ct;
  const int r0 = (r - x.first_tile[lo]) * per;
  t.row0 = int64_t(x.begin[lo]) + r0;
  t.rows = n - r0 < per ? (n - r0 > 0 ? n - r0 : 0) : per;
  t.n = per;
  return t;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (DT == GQ_BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two rows of one channel (packed, row j low) in this lane and of the neighbouring channel in
// lane ^ d -> two channels of one row: row j in the lane with bit d clear, row j + 1 in the
// other. One shuffle and one byte permutation per two elements.
__device__ __forceinline__ uint32_t swap_rows(uint32_t w, int d, bool upper) {
  const uint32_t got = __shfl_xor_sync(~0u, w, d);
  return __byte_perm(w, got, upper ? 0x3276u : 0x5410u);
}

// Store v[j] = Y[row0 + j][ch], j < 32, where row0 + j < end; lanes hold consecutive
// channels ch, those below I are real. 16-bit types: neighbouring lanes swap every other
// row and write two channels of one row as 4 bytes (pairs: I and ldy even, Y 4-byte
// aligned); this code runs once per tile on two warps per scheduler, so it counts
// instructions: convert, shuffle, permute, store and a pointer step per two elements.
template <int DT>
__device__ __forceinline__ void store_block(const Args& a, int64_t row0, int64_t end, int64_t ch, int64_t I, bool pairs,
                                            const float (&v)[32]) {
  const int rows = end - row0 < 32 ? int(end - row0) : 32;
  if (DT != GQ_F32 && pairs) {
    const int odd = threadIdx.x & 1;  // tiles begin at even channels
    uint8_t* p = reinterpret_cast<uint8_t*>(a.Y) + ((row0 + odd) * a.ldy + (ch - odd)) * 2;
    const int64_t step = 4 * a.ldy;
    const int left = ch < I ? rows - odd : 0;  // I is even: a pair's channels go together
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      const uint32_t w = swap_rows(pack2<DT>(v[j], v[j + 1]), 1, odd);
      if (j < left) *reinterpret_cast<uint32_t*>(p) = w;
      p += step;
    }
  } else if (DT == GQ_F32) {
    float* p = reinterpret_cast<float*>(a.Y) + row0 * a.ldy + ch;
    const int left = ch < I ? rows : 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      if (j < left) *p = v[j];
      p += a.ldy;
    }
  } else if (ch < I) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < rows) store_from_f32(a.Y, (row0 + j) * a.ldy + ch, v[j], DT);
  }
}

// The same after SwiGLU: even lanes hold gate, odd lanes up sums of the channel ch that
// lane / 2 stands for. Lanes swap every other row: the even lane finishes row j, the odd
// lane row j + 1 of each pair; then lanes 2 apart swap rows as above.
template <int DT>
__device__ __forceinline__ void store_block_glu(const Args& a, int64_t row0, int64_t end, int64_t ch, int64_t I,
                                                bool pairs, const float (&v)[32]) {
  const int lane = threadIdx.x & 31, odd = lane & 1, odd2 = (lane >> 1) & 1;
  const int rows = end - row0 < 32 ? int(end - row0) : 32;
  float y[16];  // rows 2 j + odd
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float got = __shfl_xor_sync(~0u, odd ? v[2 * j] : v[2 * j + 1], 1);
    y[j] = swiglu(odd ? got : v[2 * j], odd ? v[2 * j + 1] : got);
  }
  if (DT != GQ_F32 && pairs) {
    const int first = odd + 2 * odd2;  // rows first + 4 i
    uint8_t* p = reinterpret_cast<uint8_t*>(a.Y) + ((row0 + first) * a.ldy + (ch - odd2)) * 2;
    const int64_t step = 8 * a.ldy;
    const int left = ch < I ? rows - first : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = swap_rows(pack2<DT>(y[2 * i], y[2 * i + 1]), 2, odd2);
      if (4 * i < left) *reinterpret_cast<uint32_t*>(p) = w;
      p += step;
    }
  } else if (ch < I) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (2 * j + odd < rows) store_from_f32(a.Y, (row0 + 2 * j + odd) * a.ldy + ch, y[j], DT);
  }
}

template <bool GLU>
__device__ __forceinline__ void store_any_block(const Args& a, int64_t row0, int64_t end, int64_t ch, int64_t I,
                                                bool pairs, const float (&v)[32]) {
  if constexpr (GLU) {
    if (a.out_dtype == GQ_BF16) store_block_glu<GQ_BF16>(a, row0, end, ch, I, pairs, v);
    else if (a.out_dtype == GQ_F16) store_block_glu<GQ_F16>(a, row0, end, ch, I, pairs, v);
    else store_block_glu<GQ_F32>(a, row0, end, ch, I, pairs, v);
  } else {
    if (a.out_dtype == GQ_BF16) store_block<GQ_BF16>(a, row0, end, ch, I, pairs, v);
    else if (a.out_dtype == GQ_F16) store_block<GQ_F16>(a, row0, end, ch, I, pairs, v);
    else store_block<GQ_F32>(a, row0, end, ch, I, pairs, v);
  }
}

template <bool I8, bool GLU, int NMAX>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    tc_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ XMaps xmaps, const Args a,
              const Kind kind, const int most) {  // most: rows per tile, a multiple of 32 up to NMAX
  constexpr int STEP = I8 ? 32 : 16, STAGES = Shape<NMAX>::STAGES, BLOCKS = NMAX / 64;
  constexpr uint32_t STAGE_BYTES = Shape<NMAX>::STAGE_BYTES;
  constexpr int KSTEP = I8 ? 128 : 64;  // elements per stage
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;  // [2] accumulator set complete (both CTAs)
  uint64_t* tempty = tfull + 2;      // [2] accumulator set drained by both CTAs (used in the even CTA)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  Experts ex;
  ex.first_tile = reinterpret_cast<int32_t*>(smem + STAGES * STAGE_BYTES + 256);  // [E + 1]
  ex.begin = ex.first_tile + kMaxExperts + 1;
  ex.end = ex.begin + kMaxExperts + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  const int E = int(a.E), pairs = int(gridDim.x >> 1), pair = int(blockIdx.x >> 1);
  const int64_t I = GLU ? a.N / 2 : a.N;
  const int ct = int((I + (GLU ? 127 : 255)) / (GLU ? 128 : 256));  // channel blocks
  const int KT = int((a.K + KSTEP - 1) / KSTEP);
  const int chunk = I8 ? KT : (GLU ? chunk_glu(KT) : kChunk);  // k-steps per accumulation

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
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
  if (!a.early) grid_wait();  // the barriers and TMEM above were set up while the kernel before ended
  if (warp == 2) {
    // Rows of every expert and the exclusive scan of their tiles. Offsets that run backwards
    // are raised to the largest before them, so that the tiles stay within S rows whatever
    // the offsets hold.
    int32_t carry = 0, reached = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      int64_t begin = 0, end = 0;
      if (e < E) segment(a, e, begin, end);
      int32_t stop = int32_t(end);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int32_t o = __shfl_up_sync(~0u, stop, d);
        if (lane >= d) stop = max(stop, o);
      }
      stop = max(stop, reached);
      int32_t start = __shfl_up_sync(~0u, stop, 1);
      start = max(int32_t(begin), lane ? start : reached);
      if (start > stop) start = stop;
      const int32_t mine = (stop - start + most - 1) / most;
      int32_t incl = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int32_t o = __shfl_up_sync(~0u, incl, d);
        if (lane >= d) incl += o;
      }
      if (e < E) ex.first_tile[e] = carry + incl - mine, ex.begin[e] = start, ex.end[e] = stop;
      carry += __shfl_sync(~0u, incl, 31);
      reached = __shfl_sync(~0u, stop, 31);
    }
    if (lane == 0) ex.first_tile[E] = carry;
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  if (warp != 0) {  // the weights' thread goes ahead
    if (a.early) grid_wait();
    grid_release();
  }
  const uint32_t tmem = *tmem_slot;
  const int tiles = ex.first_tile[E] * ct;  // below 2^31: checked by the host for any offsets

  if (warp >= EPI_WARP0) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_DRAIN));
    // TMEM lane quarter warp % 4 (channels); every other 32 of the tile's columns (rows)
    typedef typename std::conditional<I8, int32_t, float>::type Sum;
    const int qw = warp & 3, part = (warp - EPI_WARP0) >> 2;
    const uint32_t lane_base = uint32_t(qw * 32) << 16;
    const bool in_pairs = a.out_dtype != GQ_F32 && I % 2 == 0 && a.ldy % 2 == 0 &&
                          (reinterpret_cast<uintptr_t>(a.Y) & 3u) == 0;
    int n_chunk = 0;
    bool ok = true;
    for (int q = pair; q < tiles && ok; q += pairs) {
      const Tile t = tile_of(q, ex, E, ct, STEP, most);
      Sum acc[BLOCKS][32];
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[b][j] = Sum(0);
      for (int k0 = 0; k0 < KT; k0 += chunk, ++n_chunk) {
        const int buf = n_chunk & 1;
        if (!mbar_wait(&tfull[buf], (n_chunk >> 1) & 1, abort_flag, a.status)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
          const int c = part * 32 + 64 * b;
          if (c < t.rows) {
            uint32_t r[32];
            tmem_ld32(tmem + lane_base + uint32_t(buf * 256 + c), r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if constexpr (I8)
                acc[b][j] = int32_t(r[j]);  // one chunk
              else
                acc[b][j] = acc[b][j] + __uint_as_float(r[j]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_even(&tempty[buf]);
      }
      if (!ok) break;
      const int row128 = int(rank) * 128 + qw * 32 + lane;  // of the tile's 256 channels
      const int64_t ch = GLU ? t.block * 128 + row128 / 2 : t.block * 256 + row128;
      float ws = 1.0f, bias = 0.0f;
      if (I8 && ch < I) {
        ws = a.ws[t.expert * a.N + ch + (GLU && lane & 1 ? I : 0)];
        if (a.bias) bias = load_as_f32(a.bias, ch, a.bias_dtype);
      }
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const int c = part * 32 + 64 * b;
        if (c < t.rows) {
          float xs_lane = 0.0f;
          if (I8 && c + lane < t.rows) {
            const int64_t src = source_row(a, t.row0 + c + lane);
            xs_lane = src >= 0 ? a.xs[src] : 0.0f;
          }
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if constexpr (I8)
              v[j] = float(acc[b][j]) * __shfl_sync(~0u, xs_lane, j) * ws + bias;
            else
              v[j] = acc[b][j];
          }
          store_any_block<GLU>(a, t.row0 + c, t.row0 + t.rows, ch, I, in_pairs, v);
        }
      }
    }
    if (a.zero_behind) {
      const int64_t first = rows_end(a), count = (a.S - first) * I;
      for (int64_t i = int64_t(blockIdx.x) * (32 * EPI_WARPS) + threadIdx.x - 32 * EPI_WARP0; i < count;
           i += int64_t(gridDim.x) * (32 * EPI_WARPS))
        store_from_f32(a.Y, (first + i / I) * a.ldy + i % I, 0.0f, a.out_dtype);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEW));
    if (warp == 0 && lane == 0) {
      // The weights, and the announcement of both CTAs' bytes. Never waits for the rows: with
      // early the stages fill with weights while the kernel before ends.
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&wmap)) : "memory");
      Ring<STAGES, STAGE_BYTES> ring(smem, full);
      int64_t loads = 0;
      bool ok = true;
      for (int q = pair; q < tiles && ok; q += pairs) {
        const Tile t = tile_of(q, ex, E, ct, STEP, most);
        const uint32_t bytes = 2 * (A_BYTES + uint32_t((t.n / 2 + 15) / 16 * 16) * 128);
        const int ch = (t.block * 2 + int(rank)) * (GLU ? 64 : 128);
        for (int kt = 0; kt < KT; ++kt) {
          if (!wait_at<false>(ring.empty(), ring.phase ^ 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          if (rank == 0) expect_tx_at(ring.full(), bytes);
          tma_4d(ring.data, &wmap, kt * KSTEP, 0, ch, t.expert, ring.full());  // (k, gate / up, channel, expert)
          ring.step();
          ++loads;
        }
      }
      if (*abort_flag && rank == 0) {  // let copies already in flight land before the CTA exits
        volatile int never = 0;
        for (int64_t i = loads > STAGES ? loads - STAGES : 0; i < loads; ++i)
          mbar_wait(&full[i % STAGES], (i / STAGES) & 1, &never, nullptr);
      }
    } else if (warp == 2 && lane == 0) {
      // The rows, by a thread of their own: issuing both loads from one costs 5%.
      for (int b = 0; b < X_MAPS; ++b)
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&xmaps.box[b])) : "memory");
      Ring<STAGES, STAGE_BYTES> ring(smem, full);
      bool ok = true;
      for (int q = pair; q < tiles && ok; q += pairs) {
        const Tile t = tile_of(q, ex, E, ct, STEP, most);
        const int half = t.n / 2, x_rows = (half + 15) / 16 * 16;  // <= 128
        const int y = int(t.row0) + int(rank) * half;
        // few large boxes: the largest that fits, and what is left
        int first = 0;
        while (x_rows < (128 >> first)) ++first;
        const CUtensorMap* map = &xmaps.box[first];
        const int left = x_rows - (128 >> first);
        for (int kt = 0; kt < KT; ++kt) {
          if (!wait_at<false>(ring.empty(), ring.phase ^ 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          tma_2d(ring.data + A_BYTES, map, kt * KSTEP, y, ring.full());
          if (left)
            for (int b = first + 1, r = 128 >> first; b < X_MAPS; ++b)
              if (left & (128 >> b)) {
                tma_2d(ring.data + A_BYTES + r * 128, &xmaps.box[b], kt * KSTEP, y + r, ring.full());
                r += 128 >> b;
              }
          ring.step();
        }
      }
    } else if (warp == 1 && lane == 0 && rank == 0) {
      Ring<STAGES, STAGE_BYTES> ring(smem, full);
      int n_chunk = 0;
      bool ok = true;
      const uint64_t desc = umma_desc_sw128(0, 16, 1024);  // + (address >> 4)
      for (int q = pair; q < tiles && ok; q += pairs) {
        const Tile t = tile_of(q, ex, E, ct, STEP, most);
        const uint32_t idesc = instruction_desc(kind, t.n);
        for (int k0 = 0; k0 < KT && ok; k0 += chunk, ++n_chunk) {
          const int buf = n_chunk & 1, k1 = k0 + chunk < KT ? k0 + chunk : KT;
          if (!wait_at<true>(smem_u32(&tempty[buf]), ((n_chunk >> 1) & 1) ^ 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          const uint32_t d = tmem + uint32_t(buf * 256);
          for (int kt = k0; kt < k1; ++kt) {
            if (!wait_at<true>(ring.full(), ring.phase, abort_flag, a.status)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t ad = desc + (ring.data >> 4), bd = ad + (A_BYTES >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // 32 bytes of k each, inside the 128-byte swizzle atom
              mma<I8>(d, ad + 2 * kk, bd + 2 * kk, idesc, kk != 0 || kt != k0);
            commit(ring.empty());  // frees the stage once these MMAs have read it
            ring.step();
          }
          if (ok) commit(smem_u32(&tfull[buf]));
        }
      }
    }
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
  const cuuint32_t estr[4] = {1, 1, 1, 1};
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

template <int NMAX>
int launch(const CUtensorMap& wmap, const XMaps& xmaps, const Args& a, Kind kind, bool glu, int most, unsigned grid,
           cudaStream_t s) {
  const bool i8 = kind == S8;
  auto* k = i8 ? (glu ? tc_kernel<true, true, NMAX> : tc_kernel<true, false, NMAX>)
               : (glu ? tc_kernel<false, true, NMAX> : tc_kernel<false, false, NMAX>);
  constexpr size_t smem = Shape<NMAX>::SMEM_BYTES;
  GQ_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  return launch_dependent("tc_kernel", k, dim3(grid), THREADS, smem, s, wmap, xmaps, a, kind, most);
}

// dst[s] = X[rows[s]] for the rows of every expert (a row of zeros where there is none).
// HBM-bound copy: a warp per row, four 16-byte loads per lane in flight.
__global__ void __launch_bounds__(256) gather_kernel(const Args a, uint4* __restrict__ dst, int64_t vecs) {
  grid_wait();
  grid_release();
  const int lane = threadIdx.x & 31;
  const int64_t last = rows_end(a), stride = int64_t(gridDim.x) * (blockDim.x >> 5);
  for (int64_t s = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); s < last; s += stride) {
    const int64_t src = source_row(a, s);
    const uint4* x = reinterpret_cast<const uint4*>(a.X + (src >= 0 ? src : 0) * a.ldx);
    for (int64_t v0 = lane; v0 < vecs; v0 += 128) {
      uint4 r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r[i] = make_uint4(0, 0, 0, 0);
        if (src >= 0 && v0 + 32 * i < vecs) r[i] = x[v0 + 32 * i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v0 + 32 * i < vecs) dst[s * vecs + v0 + 32 * i] = r[i];
    }
  }
}

// Rows per tile. Grouped: 256, the counts are on the device. Dense: the number of row tiles
// whose rounds over the CTA pairs cost least, a round of tiles of n rows being taken as the
// bytes that a k-step of such a tile loads per SM, 128 channels and n / 2 rows of 128 bytes.
// 1357 rows x 4096 channels: 96 tiles of 240 rows on 74 pairs are two rounds, 144 tiles of
// 160 rows two shorter ones (K = 11008, s8: 78 against 91 us).
int rows_per_tile(const Args& a, int64_t pairs, int64_t blocks) {
  if (a.offsets) return 256;
  int best = 256;
  double best_time = 1e300;
  for (int rows = 256; rows >= 64; rows -= 32) {
    const int64_t tiles = (a.S + rows - 1) / rows, n = ((a.S + tiles - 1) / tiles + 31) / 32 * 32;
    const int64_t rounds = (tiles * blocks + pairs - 1) / pairs;
    const double time = double(rounds) * (16384.0 + 64.0 * double(n));
    if (time < best_time) best_time = time, best = rows;
  }
  return best;
}

}  // namespace

int launch_tc(const Args& args, Kind kind, bool glu, void* gathered, cudaStream_t s) {
  Args a = args;
  int dev = 0, sms = 0;
  GQ_CUDA_TRY(cudaGetDevice(&dev));
  GQ_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const cuuint64_t es = kind == S8 ? 1 : 2;
  const cuuint32_t kbox = cuuint32_t(128 / es);
  CUtensorMap wmap;
  XMaps xmaps;
  // (k, gate / up, channel, expert): gate and up channels interleaved; plain: a dimension of 1
  const cuuint64_t I = cuuint64_t(glu ? a.N / 2 : a.N), halves = glu ? 2 : 1;
  const cuuint64_t wdims[4] = {cuuint64_t(a.K), halves, I, cuuint64_t(a.E)};
  const cuuint64_t wstrides[3] = {glu ? I * cuuint64_t(a.ldw) : cuuint64_t(a.ldw), cuuint64_t(a.ldw),
                                  cuuint64_t(a.stride_w)};
  const cuuint32_t wbox[4] = {kbox, cuuint32_t(halves), cuuint32_t(128 / halves), 1};
  int st = encode(&wmap, a.W, kind, 4, wdims, wstrides, wbox);
  if (st != GQ_OK) return st;
  const int64_t row_bytes = a.K * int64_t(es);
  if (a.rows) {
    const int64_t warps = std::min<int64_t>(a.S, int64_t(sms) * 64);
    st = launch_dependent("gather_kernel", gather_kernel, dim3(unsigned((warps + 7) / 8)), 256, 0, s, a,
                          reinterpret_cast<uint4*>(gathered), row_bytes / 16);
    if (st != GQ_OK) return st;
    a.early = 1;  // W and offsets are older than the copy
  }
  for (int b = 0; b < X_MAPS; ++b) {
    const cuuint64_t xdims[2] = {cuuint64_t(a.K), cuuint64_t(a.rows ? a.S : a.n_src)};
    const cuuint64_t xstrides[1] = {cuuint64_t(a.rows ? row_bytes : a.ldx)};
    const cuuint32_t xbox[2] = {kbox, cuuint32_t(128 >> b)};
    st = encode(&xmaps.box[b], a.rows ? gathered : (const void*)a.X, kind, 2, xdims, xstrides, xbox);
    if (st != GQ_OK) return st;
  }
  const int64_t pairs = std::max(sms / 2, 1), blocks = (a.N + 255) / 256;
  const bool narrow = a.S <= (a.offsets ? 8 : 32) * a.E;
  const int most = narrow ? 64 : rows_per_tile(a, pairs, blocks);
  const int64_t count = blocks * (a.S / most + std::min(a.S, a.E));  // at least the number of tiles
  GQ_REQUIRE(count < (int64_t(1) << 31) - 65536, "product: too many tiles");
  const unsigned grid = unsigned(2 * std::min(pairs, std::max<int64_t>(count, 1)));
  return narrow ? launch<64>(wmap, xmaps, a, kind, glu, most, grid, s)
                : launch<256>(wmap, xmaps, a, kind, glu, most, grid, s);
}

}  // namespace prod
}  // namespace gq
