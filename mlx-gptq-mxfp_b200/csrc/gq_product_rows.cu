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
__global__ void __launch_bounds__(THREADS, NT == 1 ? 4 : (NT == 2 ? 3 : 2)) rows_kernel(const Args a, const int by_row, const int experts_y) {
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

// ---------------------------------------------------------------------------
// One token. Its k slots are found in the index itself (no route launch) and summed inside
// a cluster (no combine launch): two launches for the expert MLP of a decoding step, whose
// time is that of reading k experts' weights and of what comes before the first load.
// ---------------------------------------------------------------------------

// 16 channels (glu: 8 gate, 8 up) times one row: v0 = channel c0 + threadIdx.x (up: v1), in
// threads below CH. x: the row, in global memory, valid after wait().
template <int KIND, bool GLU, int U, typename Wait>
__device__ __forceinline__ void one_row(const uint8_t* W, int64_t ldw, int64_t c0, int64_t I, int64_t kbytes,
                                        const uint8_t* x, bool live, Wait wait, float& v0, float& v1) {
  __shared__ float part[WARPS][2][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t ca = c0 + g, cb = GLU ? I + c0 + g : c0 + g + 8, blocks = (kbytes + 63) / 64;
  const bool oka = live && ca < I, okb = live && (GLU ? ca < I : cb < I);
  const uint8_t *wa = W + (oka ? ca : 0) * ldw + t * 16, *wb = W + (okb ? cb : 0) * ldw + t * 16;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t b = warp * U; b == warp * U || b < blocks; b += WARPS * U) {
    uint4 A[U], B[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = (b + u) * 64 + t * 16 < kbytes;
      A[u] = load16(wa + (b + u) * 64, in && oka);
      B[u] = load16(wb + (b + u) * 64, in && okb);
    }
    if (b == warp * U) wait();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint4 v = make_uint4(0, 0, 0, 0);  // column 0 of the mma is the row, the others are zeros
      if (live && g == 0 && (b + u) * 64 + t * 16 < kbytes) v = *reinterpret_cast<const uint4*>(x + (b + u) * 64 + t * 16);
      mma<KIND>(acc, A[u].x, B[u].x, A[u].y, B[u].y, v.x, v.y);
      mma<KIND>(acc, A[u].z, B[u].z, A[u].w, B[u].w, v.z, v.w);
    }
  }
  if (t == 0) part[warp][0][g] = acc[0], part[warp][1][g] = acc[2];  // column 0: channels g and g + 8
  __syncthreads();
  v0 = v1 = 0.0f;
  if (threadIdx.x < (GLU ? 8 : 16)) {
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      v0 += part[w][GLU ? 0 : threadIdx.x >> 3][threadIdx.x & 7];
      if (GLU) v1 += part[w][1][threadIdx.x & 7];
    }
  }
}

struct Token {
  const void* index;  // [k] of index_bits
  int index_bits, k, E;
};

// The expert of slot j (-1: dropped) and its place among the token's slots by (expert, position).
__device__ __forceinline__ int token_slot(const Token& k, int j, int& place) {
  const int lane = threadIdx.x & 31;
  int64_t e = -1;
  if (lane < k.k)
    e = k.index_bits == 64 ? reinterpret_cast<const int64_t*>(k.index)[lane]
                           : int64_t(reinterpret_cast<const int32_t*>(k.index)[lane]);
  if (e < 0 || e >= k.E) e = -1;
  const int mine = __shfl_sync(~0u, int(e), j);
  place = __popc(__ballot_sync(~0u, e >= 0 && (e < mine || (e == mine && lane < j))));
  return mine;
}

// acts[place] = silu(gate_e x) * (up_e x); blockIdx.y: the position. Y = acts.
// Three CTAs per SM, though four would fit: what is left takes the CTAs of the second
// kernel, whose weights are then under way before this one ends (18.4 -> 16.8 us for both,
// 8 experts of [1536, 2048] and [2048, 768]: 4.5 TB/s).
template <int KIND>
__global__ void __launch_bounds__(THREADS, 3) token_glu_kernel(const Args a, const Token k) {
  grid_wait();
  grid_release();
  int place;
  const int e = token_slot(k, blockIdx.y, place);
  if (e < 0) return;
  const int64_t I = a.N / 2, c0 = int64_t(blockIdx.x) * 8, ch = c0 + threadIdx.x;
  float gate, up;
  one_row<KIND, true, UNROLL>(a.W + e * a.stride_w, a.ldw, c0, I, a.K * 2, a.X, true, [] {}, gate, up);
  if (threadIdx.x < 8 && ch < I) store_from_f32(a.Y, place * a.ldy + ch, swiglu(gate, up), a.out_dtype);
}

// out = sum over positions j, in order, of weights[j] * (down_e acts[place]): a cluster is
// the k positions of one block of 16 channels. X = acts, Y = out.
// U: blocks of the contraction a warp has in flight, all of them where that is at most 4.
template <int KIND, int U>
__global__ void __launch_bounds__(THREADS, 4) token_down_kernel(const Args a, const Token k, const float* weights) {
  __shared__ float term[16];
  int place;
  const int e = token_slot(k, blockIdx.y, place);  // the index is older than the kernel before this one
  const int64_t c0 = int64_t(blockIdx.x) * 16;
  float v, unused;
  one_row<KIND, false, U>(a.W + (e < 0 ? 0 : e) * a.stride_w, a.ldw, c0, a.N, a.K * 2, a.X + place * a.ldx, e >= 0,
                       [] { grid_wait(); }, v, unused);
  grid_release();
  if (threadIdx.x < 16) term[threadIdx.x] = e < 0 ? 0.0f : weights[blockIdx.y] * v;
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (blockIdx.y == 0 && threadIdx.x < 16 && c0 + threadIdx.x < a.N) {
    float sum = 0.0f;
    for (int j = 0; j < k.k; ++j) {  // the cluster's rank is the position
      uint32_t addr;
      float y;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(&term[threadIdx.x])), "r"(j));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y) : "r"(addr) : "memory");
      sum += y;
    }
    store_from_f32(a.Y, c0 + threadIdx.x, sum, a.out_dtype);
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int KIND>
int launch_token_kind(const Args& up, const Args& down, const Token& k, const float* weights, cudaStream_t s) {
  const int64_t I = up.N / 2;
  const int st = launch_dependent("token_glu_kernel", token_glu_kernel<KIND>, dim3(unsigned((I + 7) / 8), unsigned(k.k)),
                                  THREADS, 0, s, up, k);
  if (st != GQ_OK) return st;
  const int64_t turns = ((down.K * 2 + 63) / 64 + WARPS - 1) / WARPS;  // blocks per warp
  auto* kernel = turns <= 2 ? token_down_kernel<KIND, 2> : turns == 3 ? token_down_kernel<KIND, 3> : token_down_kernel<KIND, 4>;
  return launch_dependent_in<Args, Token, const float*>("token_down_kernel", kernel,
                                                        dim3(unsigned((down.N + 15) / 16), unsigned(k.k)), THREADS, 0,
                                                        s, Cluster{1, unsigned(k.k)}, down, k, weights);
}

// ---------------------------------------------------------------------------
// One or two rows through an 8-bit layer: every CTA quantizes the rows itself (they are a
// few KB in L2, and the weights are on their way meanwhile) instead of waiting for a launch
// that does. The codes are those of gq_rtn_int8: the same IEEE operations.
// ---------------------------------------------------------------------------
template <typename T, int M>
__global__ void __launch_bounds__(THREADS)
    linear_rows_kernel(const T* X, const int64_t ldx, const Args a) {
  extern __shared__ __align__(16) int8_t codes[];  // [M][K]
  __shared__ uint32_t max_bits[M][WARPS];
  __shared__ int32_t part[WARPS][4][32];
  grid_wait();
  grid_release();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t c0 = int64_t(blockIdx.x) * 16, ca = c0 + g, cb = ca + 8, blocks = (a.K + 63) / 64;
  const bool oka = ca < a.N, okb = cb < a.N;
  const uint8_t *wa = a.W + (oka ? ca : 0) * a.ldw + t * 16, *wb = a.W + (okb ? cb : 0) * a.ldw + t * 16;
  uint4 A[UNROLL], B[UNROLL];
  auto load_weights = [&](int64_t b) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const bool in = (b + u) * 64 + t * 16 < a.K;
      A[u] = load16(wa + (b + u) * 64, in && oka);
      B[u] = load16(wb + (b + u) * 64, in && okb);
    }
  };
  load_weights(warp * UNROLL);
  constexpr int V = 16 / int(sizeof(T));  // elements per load
  float scale[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    uint32_t bits = 0;
    for (int64_t c = threadIdx.x * V; c < a.K; c += THREADS * V) {
      T v[V];
      *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(X + m * ldx + c);
#pragma unroll
      for (int i = 0; i < V; ++i) bits = max(bits, __float_as_uint(to_f32<T>(v[i])) & 0x7FFFFFFFu);
    }
    bits = __reduce_max_sync(~0u, bits);
    if (lane == 0) max_bits[m][warp] = bits;
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < M; ++m) {
    uint32_t bits = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) bits = max(bits, max_bits[m][w]);
    scale[m] = __uint_as_float(bits) / 127.0f;
    for (int64_t c = threadIdx.x * V; c < a.K; c += THREADS * V) {
      T v[V];
      *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(X + m * ldx + c);
      float f[V];
      uint32_t word[V / 4];
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = to_f32<T>(v[i]);
      int8_codes<V>(f, scale[m], word);
#pragma unroll
      for (int i = 0; i < V / 4; ++i) reinterpret_cast<uint32_t*>(codes + m * a.K + c)[i] = word[i];
    }
  }
  __syncthreads();
  int32_t acc[4] = {0, 0, 0, 0};
  for (int64_t b = warp * UNROLL; b < blocks; b += WARPS * UNROLL) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (g < M && (b + u) * 64 + t * 16 < a.K)
        x = *reinterpret_cast<const uint4*>(codes + g * a.K + (b + u) * 64 + t * 16);
      mma<S8>(acc, A[u].x, B[u].x, A[u].y, B[u].y, x.x, x.y);
      mma<S8>(acc, A[u].z, B[u].z, A[u].w, B[u].w, x.z, x.w);
    }
    if (b + WARPS * UNROLL < blocks) load_weights(b + WARPS * UNROLL);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[warp][i][lane] = acc[i];
  __syncthreads();
  // accumulator i of lane (g, t): channel g + 8 (i / 2), row 2 t + i % 2
  if (threadIdx.x < 16 * M) {
    const int c = threadIdx.x & 15, m = threadIdx.x >> 4;
    const int64_t ch = c0 + c;
    if (ch < a.N) {
      int32_t sum = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) sum += part[w][(c >> 3) * 2 + m][(c & 7) * 4];
      float y = float(sum) * (m == 0 ? scale[0] : scale[M - 1]) * a.ws[ch];
      if (a.bias) y = y + load_as_f32(a.bias, ch, a.bias_dtype);
      store_from_f32(a.Y, m * a.ldy + ch, y, a.out_dtype);
    }
  }
}

template <typename T>
int linear_rows(const void* X, int64_t ldx, const Args& a, cudaStream_t s) {
  const dim3 grid(unsigned((a.N + 15) / 16));
  const size_t smem = size_t(a.S) * size_t(a.K);
  return launch_dependent("linear_rows_kernel", a.S == 1 ? linear_rows_kernel<T, 1> : linear_rows_kernel<T, 2>, grid,
                          THREADS, smem, s, reinterpret_cast<const T*>(X), ldx, a);
}

}  // namespace

bool token_fits(int64_t T, int64_t k, int64_t E) { return T == 1 && k <= 8 && E < (int64_t(1) << 31); }

int launch_token(const Args& up, const Args& down, Kind kind, const void* index, int index_bits, int64_t k,
                 const float* weights, cudaStream_t s) {
  const Token t = {index, index_bits, int(k), int(up.E)};
  return kind == F16 ? launch_token_kind<F16>(up, down, t, weights, s)
                     : launch_token_kind<BF16>(up, down, t, weights, s);
}

bool linear_rows_fit(const void* X, int dtype, int64_t M, int64_t K, int64_t ldx) {
  const int64_t es = dtype == GQ_F32 ? 4 : 2;
  return M <= 2 && K % 16 == 0 && M * K <= 32768 && aligned16(X) && (M == 1 || ldx * es % 16 == 0);
}

int launch_linear_rows(const void* X, int dtype, int64_t ldx, const Args& a, cudaStream_t s) {
  if (dtype == GQ_BF16) return linear_rows<__nv_bfloat16>(X, ldx, a, s);
  if (dtype == GQ_F16) return linear_rows<__half>(X, ldx, a, s);
  return linear_rows<float>(X, ldx, a, s);
}

int launch_rows(const Args& a, Kind kind, bool glu, cudaStream_t s) {
  if (kind == S8) return glu ? launch_nt<S8, true>(a, s) : launch_nt<S8, false>(a, s);
  if (kind == F16) return glu ? launch_nt<F16, true>(a, s) : launch_nt<F16, false>(a, s);
  return glu ? launch_nt<BF16, true>(a, s) : launch_nt<BF16, false>(a, s);
}

}  // namespace prod
}  // namespace gq
