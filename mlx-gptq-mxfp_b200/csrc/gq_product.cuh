// Products of activation rows with weights, grouped by expert (ragged) or dense:
// what the few-rows kernel (gq_product_rows.cu) and the tcgen05 kernel
// (gq_product_tc.cu) share.
#pragma once

#include "gq_common.cuh"

namespace gq {
namespace slots {
int combine_rows(const void* y, int y_dtype, int dtype, int64_t S, int64_t ldy, const int32_t* slot,
                 const float* weights, int64_t T, int64_t k, int64_t N, void* out, int64_t ldo, cudaStream_t s);
}

namespace prod {

// Element kinds of a product: both operands in the kind, sums in fp32 (s32 for S8, exact).
enum Kind : int { BF16 = 0, F16 = 1, S8 = 2 };

constexpr int64_t kMaxExperts = 1024;

// Y[s] = op(X[rows[s]] W_e^T) for the rows s of expert e = [offsets[e], offsets[e + 1]).
struct Args {
  const uint8_t* X;        // [n_src, K]
  int64_t n_src, ldx;      // ldx: bytes between rows, a multiple of 16
  const int32_t* rows;     // [S] row of X per product row (nullable: row s itself)
  const int64_t* offsets;  // [E + 1] on the device (nullable: one expert with all S rows)
  int64_t E, S;
  const uint8_t* W;        // [E, N, K]
  int64_t N, K;            // output channels (2 * I with glu), contracted size in elements
  int64_t ldw, stride_w;   // bytes between channels and between experts, multiples of 16
  const float* xs;         // S8: [n_src] scale per row of X
  const float* ws;         // S8: [E, N] scale per channel
  const void* bias;        // [N], nullable (dense only)
  int bias_dtype;
  void* Y;                 // [S, N] (glu: [S, N / 2]) of out_dtype
  int64_t ldy;             // elements
  int out_dtype;
  int zero_behind;         // rows behind the last expert's: 1 = written as zeros, 0 = left alone
  int32_t* status;         // nullable
  int early;               // W and offsets are not written by the kernel launched just before
};

int launch_rows(const Args& a, Kind kind, bool glu, cudaStream_t s);
// The expert MLP of one token (token_fits): up: X = the token, Y = acts (k rows); down: X =
// acts, Y = the output row.
bool token_fits(int64_t T, int64_t k, int64_t E);
int launch_token(const Args& up, const Args& down, Kind kind, const void* index, int index_bits, int64_t k,
                 const float* weights, cudaStream_t s);
// One or two rows X (a.S) of dtype, quantized and multiplied in one launch.
bool linear_rows_fit(const void* X, int dtype, int64_t M, int64_t K, int64_t ldx);
int launch_linear_rows(const void* X, int dtype, int64_t ldx, const Args& a, cudaStream_t s);
// gathered: with a row list, S * K elements, 16-byte aligned.
int launch_tc(const Args& a, Kind kind, bool glu, void* gathered, cudaStream_t s);

// Rows of expert e, whatever the offsets hold: 0 <= begin <= end <= S.
__device__ __forceinline__ void segment(const Args& a, int64_t e, int64_t& begin, int64_t& end) {
  if (!a.offsets) {
    begin = 0, end = a.S;
    return;
  }
  const int64_t b = a.offsets[e], f = a.offsets[e + 1];
  begin = b < 0 ? 0 : (b > a.S ? a.S : b);
  end = f < begin ? begin : (f > a.S ? a.S : f);
}

// First row behind the last expert's.
__device__ __forceinline__ int64_t rows_end(const Args& a) {
  if (!a.offsets) return a.S;
  const int64_t f = a.offsets[a.E];
  return f < 0 ? 0 : (f > a.S ? a.S : f);
}

// Row of X behind product row s, or -1 where there is none (its products are zero).
__device__ __forceinline__ int64_t source_row(const Args& a, int64_t s) {
  const int64_t r = a.rows ? int64_t(a.rows[s]) : s;
  return r >= 0 && r < a.n_src ? r : -1;
}

__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
  if (dtype == GQ_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == GQ_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_from_f32(void* p, int64_t i, float v, int dtype) {
  if (dtype == GQ_BF16)
    reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (dtype == GQ_F16)
    reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    reinterpret_cast<float*>(p)[i] = v;
}

// silu(g) * u in fp32: the one rounding to the output's type comes after it.
// With t = exp(-|g|) in [0, 1]: silu(g) = g * (g >= 0 ? 1 : t) / (1 + t), which neither
// overflows nor divides by more than 2. t = 2^(hi + lo) with hi + lo the product
// -|g| log2(e) carried to twice float32, so its error (3 float32 steps) does not grow with
// |g|; about 15 instructions, a third of expf and an IEEE division.
__device__ __forceinline__ float swiglu(float g, float u) {
  constexpr float kLog2e = 1.44269504f, kLog2eRest = 1.925963033500e-8f, kLn2 = 0.693147181f;
  const float x = -fabsf(g);
  const float hi = x * kLog2e, lo = fmaf(x, kLog2eRest, fmaf(x, kLog2e, -hi));
  float t, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(t) : "f"(hi));
  t = t == 0.0f ? 0.0f : fmaf(t, lo * kLn2, t);  // hi = -inf: lo is not a number
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + t));
  return g * (g >= 0.0f ? r : t * r) * u;
}

}  // namespace prod
}  // namespace gq
