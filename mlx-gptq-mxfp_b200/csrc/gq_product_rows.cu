// Products with few rows per expert (decoding): Y[s] = X[rows[s]] W_e^T, optionally with
// SwiGLU, for bf16 / f16 rows (fp32 sums) and 8-bit codes (exact s32 sums, scales per row
// and channel).
//
// With few rows the time is that of reading the weights once from HBM, so nothing is
// staged: every weight byte goes from global memory straight into the register fragment
// of an mma.sync (m16n8k16, or m16n8k32 for s8) that uses it. A lane loads 16 consecutive
// bytes of channel g (and g + 8) and of row g; the contraction order inside a 64-byte
// block is permuted the same way for both operands, so the fragments need no shuffle:
//   lane (g, t) holds bytes [16 t, 16 t + 16) of the block = registers r0..r3;
//   mma 1 takes (r0, r1), mma 2 (r2, r3) as its two k-halves, for A and B alike.
// One CTA takes 16 channels (with SwiGLU 8 gate and the matching 8 up channels, which land
// in the same thread's accumulators); its 8 warps split the contraction and are summed in
// warp order through shared memory. Rows are taken 8 * NT at a time.
#include "gq_product.cuh"

namespace gq {
namespace prod {
namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int UNROLL = 4;  // 64-byte blocks of each channel in flight per warp

__device__ __forceinline__ uint4 load16(const uint8_t* p, bool on) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (on)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}

template <int KIND>
struct Acc {
  typedef float T;
};
template <>
struct Acc<S8> {
  typedef int32_t T;
};

template <int KIND, typename T>
__device__ __forceinline__ void mma(T (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if constexpr (KIND == S8)
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else if constexpr (KIND == F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// blockIdx.y: the expert, or with by_row (fewer rows than experts) a product row, which
// stands for the expert that begins there; one more y, where there is one, writes the rows
// behind. The weights wait for the expert, so it is found in one step of memory latency:
// every lane of a warp counts the offsets at or before the row.
template <int KIND, bool GLU, int NT>
__global__ void __launch_bounds__(THREADS) rows_kernel(const Args a, const int by_row, const int experts_y) {
  typedef typename Acc<KIND>::T T;
  __shared__ T part[WARPS][NT][4][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t I = GLU ? a.N / 2 : a.N;  // output channels
  constexpr int CH = GLU ? 8 : 16;        // of them per CTA
  const int64_t c0 = int64_t(blockIdx.x) * CH;

  if (!a.early || int(blockIdx.y) == experts_y) grid_wait();
  if (int(blockIdx.y) == experts_y) {
    for (int64_t s = rows_end(a) + threadIdx.x / CH; s < a.S; s += THREADS / CH) {
      const int64_t c = c0 + threadIdx.x % CH;
      if (c < I) store_from_f32(a.Y, s * a.ldy + c, 0.0f, a.out_dtype);
    }
    return;
  }
  int64_t e = blockIdx.y, begin, end;
  if (by_row) {
    int before = 0;  // offsets[0 .. E - 1] at or before the row: the last of them begins its expert
    for (int64_t i = lane; i < a.E; i += 32) before += a.offsets[i] <= int64_t(blockIdx.y);
    e = __reduce_add_sync(~0u, before) - 1;
  }
  begin = end = 0;
  if (e >= 0) segment(a, e, begin, end);
  if (begin >= end || (by_row && begin != int64_t(blockIdx.y))) {
    grid_wait();  // a grid that ends has waited for the one before it, in every CTA
    return;
  }

  constexpr int64_t ES = KIND == S8 ? 1 : 2;
  const int64_t kbytes = a.K * ES, blocks = (kbytes + 63) / 64;
  // channels of the two fragment halves: g and g + 8, or gate g and up g
  const int64_t ca = c0 + g, cb = GLU ? I + c0 + g : c0 + g + 8;
  const bool oka = ca < I, okb = GLU ? ca < I : cb < I;
  const uint8_t* wa = a.W + e * a.stride_w + (oka ? ca : 0) * a.ldw + t * 16;
  const uint8_t* wb = a.W + e * a.stride_w + (okb ? cb : 0) * a.ldw + t * 16;

  uint4 A[UNROLL], B[UNROLL];
  auto load_weights = [&](int64_t b) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const bool in = (b + u) * 64 + t * 16 < kbytes;
      A[u] = load16(wa + (b + u) * 64, in && oka);
      B[u] = load16(wb + (b + u) * 64, in && okb);
    }
  };
  load_weights(warp * UNROLL);  // in flight while the kernel before (the rows' producer) ends
  if (a.early) grid_wait();
  grid_release();

  for (int64_t r0 = begin; r0 < end; r0 += 8 * NT) {
    const uint8_t* xp[NT];
    bool okx[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int64_t s = r0 + n * 8 + g, src = s < end ? source_row(a, s) : -1;
      okx[n] = src >= 0;
      xp[n] = a.X + (okx[n] ? src : 0) * a.ldx + t * 16;
    }
    T acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = T(0);
    if (r0 != begin) load_weights(warp * UNROLL);
    for (int64_t b = warp * UNROLL; b < blocks; b += WARPS * UNROLL) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          const bool in = (b + u) * 64 + t * 16 < kbytes;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (in && okx[n]) x = *reinterpret_cast<const uint4*>(xp[n] + (b + u) * 64);
          mma<KIND>(acc[n], A[u].x, B[u].x, A[u].y, B[u].y, x.x, x.y);
          mma<KIND>(acc[n], A[u].z, B[u].z, A[u].w, B[u].w, x.z, x.w);
        }
      }
      if (b + WARPS * UNROLL < blocks) load_weights(b + WARPS * UNROLL);
    }
    __syncthreads();  // the sums of the previous rows have been read
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[warp][n][i][lane] = acc[n][i];
    __syncthreads();
    // accumulator i of lane (g, t): channel half i / 2, row 2 t + i % 2
    for (int o = threadIdx.x; o < NT * 8 * CH; o += THREADS) {
      const int c = o % CH, row = o / CH, n = row >> 3, j = row & 7;
      const int64_t s = r0 + row, ch = c0 + c;
      if (s >= end || ch >= I) continue;
      const int src_lane = (c & 7) * 4 + (j >> 1), odd = j & 1;
      T v0 = T(0), v1 = T(0);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        v0 += part[w][n][GLU ? odd : (c >> 3) * 2 + odd][src_lane];
        if (GLU) v1 += part[w][n][2 + odd][src_lane];
      }
      float y = float(v0), up = float(v1);
      if (KIND == S8) {
        const int64_t src = source_row(a, s);
        const float xs = src >= 0 ? a.xs[src] : 0.0f;
        y = y * xs * a.ws[e * a.N + ch];
        if (GLU) up = up * xs * a.ws[e * a.N + I + ch];
      }
      if (a.bias) y = y + load_as_f32(a.bias, ch, a.bias_dtype);
      if (GLU) y = swiglu(y, up);
      store_from_f32(a.Y, s * a.ldy + ch, y, a.out_dtype);
    }
  }
}

template <int KIND, bool GLU>
int launch_nt(const Args& a, cudaStream_t s) {
  const int64_t I = GLU ? a.N / 2 : a.N, CH = GLU ? 8 : 16;
  const int by_row = a.offsets && a.S < a.E;
  const int64_t gx = (I + CH - 1) / CH, experts = by_row ? a.S : a.E;
  const dim3 grid{unsigned(gx), unsigned(experts + (a.zero_behind && a.offsets ? 1 : 0))};
  const int64_t most = a.offsets ? (a.S + a.E - 1) / a.E * 2 : a.S;  // rows of a busy expert
  if (most <= 8)
    return launch_dependent("rows_kernel", rows_kernel<KIND, GLU, 1>, grid, THREADS, 0, s, a, by_row, int(experts));
  if (most <= 16)
    return launch_dependent("rows_kernel", rows_kernel<KIND, GLU, 2>, grid, THREADS, 0, s, a, by_row, int(experts));
  return launch_dependent("rows_kernel", rows_kernel<KIND, GLU, 4>, grid, THREADS, 0, s, a, by_row, int(experts));
}

}  // namespace

int launch_rows(const Args& a, Kind kind, bool glu, cudaStream_t s) {
  if (kind == S8) return glu ? launch_nt<S8, true>(a, s) : launch_nt<S8, false>(a, s);
  if (kind == F16) return glu ? launch_nt<F16, true>(a, s) : launch_nt<F16, false>(a, s);
  return glu ? launch_nt<BF16, true>(a, s) : launch_nt<BF16, false>(a, s);
}

}  // namespace prod
}  // namespace gq
