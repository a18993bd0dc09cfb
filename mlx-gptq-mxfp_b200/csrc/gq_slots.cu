// The slots of a top-k routing: their order by expert (route) and the weighted sum of
// their rows per token (combine). The sort-based expert forward of the Python package
// needs both (mlx_gptq/capture.py:192-207 is the reference's per-expert interception).
//
// Route is a stable counting sort with one digit, the expert. Slots are taken in
// (position, token) order, i = position * T + token, cut into chunks of one CTA each:
//   count_kernel   how many slots of each expert a chunk has;
//   place_kernel   first slot of every expert (a scan over experts of the chunk sums),
//                  this chunk's share of it, then 1024 slots at a time: a slot's rank
//                  among its warp's (match), the warps before it, the chunk before them.
// With one chunk (decoding) place_kernel counts itself and is the only launch. Indices
// outside [0, E) go to bin E, behind every expert. Integers only: the result does not
// depend on the order in which anything runs.
#include <algorithm>

#include "gq_product.cuh"

namespace gq {
namespace slots {

constexpr int THREADS = 1024, WARPS = THREADS / 32;
constexpr int64_t kMaxExperts = 1024;
constexpr int64_t kMaxChunks = 128;    // place_kernel reads every earlier chunk's counts
constexpr int64_t kOneChunk = 1024;    // up to here one CTA sorts everything in one launch (2048 slots: 9.1 us against 7.8)

__host__ __device__ inline int64_t chunk_size(int64_t slots) {
  if (slots <= kOneChunk) return kOneChunk;
  const int64_t c = (slots + kMaxChunks - 1) / kMaxChunks;
  return c < 1024 ? 1024 : (c + 1023) / 1024 * 1024;
}
__host__ __device__ inline int64_t chunks_of(int64_t slots) {
  return (slots + chunk_size(slots) - 1) / chunk_size(slots);
}

// Bin of slot i (position-major): its expert, or E.
template <typename I>
__device__ __forceinline__ int bin_of(const I* __restrict__ index, int64_t i, int64_t T, int64_t k, int E) {
  const int64_t e = int64_t(index[(i % T) * k + i / T]);
  return e >= 0 && e < E ? int(e) : E;
}

template <typename I>
__global__ void __launch_bounds__(THREADS)
    count_kernel(const I* __restrict__ index, int64_t T, int64_t k, int E, int64_t chunk, int32_t* __restrict__ counts) {
  __shared__ int32_t h[kMaxExperts + 1];
  grid_wait();
  grid_release();
  for (int e = threadIdx.x; e <= E; e += THREADS) h[e] = 0;
  __syncthreads();
  const int64_t i0 = int64_t(blockIdx.x) * chunk, i1 = i0 + chunk < T * k ? i0 + chunk : T * k;
  for (int64_t i = i0 + threadIdx.x; i < i1; i += THREADS) atomicAdd(&h[bin_of(index, i, T, k, E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += THREADS) counts[int64_t(blockIdx.x) * (E + 1) + e] = h[e];
}

// counts: [gridDim.x, E + 1] from count_kernel; not read with a single chunk.
template <typename I>
__global__ void __launch_bounds__(THREADS)
    place_kernel(const I* __restrict__ index, int64_t T, int64_t k, int E, int64_t chunk,
                 const int32_t* __restrict__ counts, int32_t* __restrict__ tok, int32_t* __restrict__ slot,
                 int64_t* __restrict__ offsets) {
  extern __shared__ uint16_t before[];  // [WARPS][E + 1]: slots of the bin in the warp, then in the warps before it
  __shared__ int32_t next[kMaxExperts + 1];  // where the bin's next slot goes
  __shared__ int32_t total[kMaxExperts + 1], warp_sum[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, bins = E + 1;
  grid_wait();
  grid_release();
  const int64_t slots = T * k, i0 = int64_t(blockIdx.x) * chunk, i1 = i0 + chunk < slots ? i0 + chunk : slots;

  // slots of every bin: all of them (total) and those of the chunks before this one (next)
  for (int e = tid; e < bins; e += THREADS) {
    int32_t all = 0, earlier = 0;
    if (gridDim.x > 1)
      for (int b = 0; b < int(gridDim.x); ++b) {
        const int32_t c = counts[int64_t(b) * bins + e];
        all += c;
        if (b < int(blockIdx.x)) earlier += c;
      }
    total[e] = all;
    next[e] = earlier;
  }
  __syncthreads();
  if (gridDim.x == 1) {
    for (int64_t i = tid; i < slots; i += THREADS) atomicAdd(&total[bin_of(index, i, T, k, E)], 1);
    __syncthreads();
  }
  // exclusive scan over the experts (E <= 1024: one per thread); bin E follows the last
  const int32_t mine = tid < E ? total[tid] : 0;
  int32_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int32_t o = __shfl_up_sync(~0u, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int32_t base = 0;
  for (int w = 0; w < warp; ++w) base += warp_sum[w];
  const int32_t first = base + incl - mine;
  if (tid < E) next[tid] += first;
  if (tid == E - 1) next[E] += first + mine;
  if (blockIdx.x == 0) {
    if (tid < E) offsets[tid] = first;
    if (tid == E - 1) offsets[E] = first + mine;
  }
  __syncthreads();

  for (int64_t s0 = i0; s0 < i1; s0 += THREADS) {
    for (int j = tid; j < WARPS * bins; j += THREADS) before[j] = 0;
    __syncthreads();
    const int64_t i = s0 + tid;
    const bool on = i < i1;
    const int e = on ? bin_of(index, i, T, k, E) : -1;
    const uint32_t same = __match_any_sync(~0u, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    if (on && rank == 0) before[warp * bins + e] = uint16_t(__popc(same));
    __syncthreads();
    for (int b = tid; b < bins; b += THREADS) {
      int32_t sum = 0;
      for (int w = 0; w < WARPS; ++w) {
        const int32_t c = before[w * bins + b];
        before[w * bins + b] = uint16_t(sum);
        sum += c;
      }
      total[b] = sum;
    }
    __syncthreads();
    if (on) {
      const int32_t p = next[e] + before[warp * bins + e] + rank;
      const int64_t t = i % T;
      tok[p] = e < E ? int32_t(t) : -1;
      slot[t * k + i / T] = e < E ? p : -1;
    }
    __syncthreads();
    for (int b = tid; b < bins; b += THREADS) next[b] += total[b];
    __syncthreads();
  }
}

// out[t, c .. c + V) = sum over positions j of weights[t, j] * y[slot[t, j], c .. c + V),
// in position order in fp32, rounded once. HBM-bound: k rows in, one out. A thread takes
// the V channels of one token that 16 bytes of a row hold (V = 1 where sizes or alignment do
// not allow that) and has up to eight rows in flight. Y: T, or float for rows that the sum
// takes unrounded.
template <typename Y, typename T, int V>
__global__ void __launch_bounds__(256)
    combine_kernel(const Y* __restrict__ y, int64_t S, int64_t ldy, const int32_t* __restrict__ slot,
                   const float* __restrict__ weights, int64_t tokens, int64_t k, int64_t N, T* __restrict__ out,
                   int64_t ldo) {
  grid_wait();
  grid_release();
  const int64_t per = N / V, i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= tokens * per) return;
  const int64_t t = i / per, c = (i % per) * V;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  for (int64_t j0 = 0; j0 < k; j0 += 8) {
    Y rows[8][V];
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int32_t s = j0 + j < k ? slot[t * k + j0 + j] : -1;
      const bool on = s >= 0 && s < S;
      w[j] = on ? weights[t * k + j0 + j] : 0.0f;
      if (V > 1) {  // one 16-byte load of the row
        uint4 r = make_uint4(0, 0, 0, 0);
        if (on) r = *reinterpret_cast<const uint4*>(y + int64_t(s) * ldy + c);
        *reinterpret_cast<uint4*>(rows[j]) = r;
      } else {
        rows[j][0] = on ? y[int64_t(s) * ldy + c] : from_f32<Y>(0.0f);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(w[j], to_f32<Y>(rows[j][v]), acc[v]);
  }
  T r[V];
#pragma unroll
  for (int v = 0; v < V; ++v) r[v] = from_f32<T>(acc[v]);
  if (V == 8)
    *reinterpret_cast<uint4*>(out + t * ldo + c) = *reinterpret_cast<const uint4*>(r);
  else if (V == 4)
    *reinterpret_cast<uint2*>(out + t * ldo + c) = *reinterpret_cast<const uint2*>(r);
  else
    out[t * ldo + c] = r[0];
}

template <typename I>
int route(const I* index, int64_t T, int64_t k, int64_t E, int32_t* tok, int32_t* slot, int64_t* offsets,
          int32_t* counts, cudaStream_t s) {
  const int64_t chunk = chunk_size(T * k), n = chunks_of(T * k);
  if (n > 1) {
    const int st = launch_dependent("count_kernel", count_kernel<I>, dim3(unsigned(n)), THREADS, 0, s, index, T, k,
                                    int(E), chunk, counts);
    if (st != GQ_OK) return st;
  }
  // The limit is one value per function and device, shared by every host thread: always the
  // largest, whatever this call needs of it.
  constexpr size_t most = size_t(WARPS) * size_t(kMaxExperts + 1) * 2;  // 64 KB + 64
  const size_t smem = size_t(WARPS) * size_t(E + 1) * 2;
  GQ_CUDA_TRY(cudaFuncSetAttribute(place_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(most)));
  return launch_dependent("place_kernel", place_kernel<I>, dim3(unsigned(n)), THREADS, smem, s, index, T, k, int(E),
                          chunk, counts, tok, slot, offsets);
}

template <typename Y, typename T>
int combine(const void* y, int64_t S, int64_t ldy, const int32_t* slot, const float* weights, int64_t tokens,
            int64_t k, int64_t N, void* out, int64_t ldo, cudaStream_t s) {
  constexpr int V = 16 / int(sizeof(Y));
  const bool wide = N % V == 0 && ldy % V == 0 && ldo % V == 0 && aligned16(y) &&
                    (reinterpret_cast<uintptr_t>(out) & (V * sizeof(T) - 1)) == 0;
  const int64_t threads = tokens * (wide ? N / V : N);
  const unsigned grid = unsigned((threads + 255) / 256);
  return launch_dependent("combine_kernel", wide ? combine_kernel<Y, T, V> : combine_kernel<Y, T, 1>, dim3(grid), 256,
                          0, s, (const Y*)y, S, ldy, slot, weights, tokens, k, N, (T*)out, ldo);
}

// The weighted sum of rows of y_dtype (float32 or dtype) into rows of dtype.
int combine_rows(const void* y, int y_dtype, int dtype, int64_t S, int64_t ldy, const int32_t* slot,
                 const float* weights, int64_t T, int64_t k, int64_t N, void* out, int64_t ldo, cudaStream_t s) {
  GQ_REQUIRE(S >= 0 && T >= 0 && k >= 1 && N >= 1 && T <= INT32_MAX / k && ldy >= N && ldo >= N,
             "gq_combine_slots: sizes");
  GQ_REQUIRE(N <= (int64_t(1) << 38) / (T + 1), "gq_combine_slots: %lld tokens x %lld channels", (long long)T,
             (long long)N);
  if (T == 0) return GQ_OK;
  GQ_REQUIRE(slot && weights && out && (y || S == 0), "gq_combine_slots: null pointer");
  if (y_dtype == GQ_F32)
    return dtype == GQ_BF16 ? combine<float, __nv_bfloat16>(y, S, ldy, slot, weights, T, k, N, out, ldo, s)
                            : combine<float, __half>(y, S, ldy, slot, weights, T, k, N, out, ldo, s);
  return dtype == GQ_BF16 ? combine<__nv_bfloat16, __nv_bfloat16>(y, S, ldy, slot, weights, T, k, N, out, ldo, s)
                          : combine<__half, __half>(y, S, ldy, slot, weights, T, k, N, out, ldo, s);
}

}  // namespace slots
}  // namespace gq

using namespace gq;

extern "C" size_t gq_route_slots_workspace_size(int64_t T, int64_t k, int64_t E) {
  if (T <= 0 || k <= 0 || E <= 0 || E > slots::kMaxExperts || T > INT32_MAX / k) return 0;
  const int64_t n = slots::chunks_of(T * k);
  return n > 1 ? size_t(n) * size_t(E + 1) * 4 : 0;
}

extern "C" int gq_route_slots(const void* index, int index_bits, int64_t T, int64_t k, int64_t E, int32_t* tok,
                              int32_t* slot, int64_t* offsets, void* workspace, size_t workspace_bytes, void* stream) {
  GQ_REQUIRE(index_bits == 32 || index_bits == 64, "gq_route_slots: indices have 32 or 64 bits, not %d", index_bits);
  GQ_REQUIRE(T >= 0 && k >= 1 && T <= INT32_MAX / k, "gq_route_slots: %lld tokens x %lld positions", (long long)T,
             (long long)k);
  GQ_REQUIRE(E >= 1 && E <= slots::kMaxExperts, "gq_route_slots: %lld experts, at most %lld", (long long)E,
             (long long)slots::kMaxExperts);
  GQ_REQUIRE(offsets, "gq_route_slots: null pointer");
  cudaStream_t s = (cudaStream_t)stream;
  if (T == 0) {
    GQ_CUDA_TRY(cudaMemsetAsync(offsets, 0, size_t(E + 1) * 8, s));
    return GQ_OK;
  }
  GQ_REQUIRE(index && tok && slot, "gq_route_slots: null pointer");
  const size_t need = gq_route_slots_workspace_size(T, k, E);
  GQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "gq_route_slots: workspace too small (%zu < %zu)",
             workspace_bytes, need);
  int32_t* counts = reinterpret_cast<int32_t*>(workspace);
  return index_bits == 64 ? slots::route((const int64_t*)index, T, k, E, tok, slot, offsets, counts, s)
                          : slots::route((const int32_t*)index, T, k, E, tok, slot, offsets, counts, s);
}

extern "C" int gq_combine_slots(const void* y, int dtype, int64_t S, int64_t ldy, const int32_t* slot,
                                const float* weights, int64_t T, int64_t k, int64_t N, void* out, int64_t ldo,
                                void* stream) {
  GQ_REQUIRE(dtype == GQ_BF16 || dtype == GQ_F16, "gq_combine_slots: rows are bf16 or f16 (dtype %d)", dtype);
  return slots::combine_rows(y, dtype, dtype, S, ldy, slot, weights, T, k, N, out, ldo, (cudaStream_t)stream);
}
