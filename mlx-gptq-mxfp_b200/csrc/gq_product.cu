// C entry points of the products of activation rows with weights: argument checks and the
// choice between the few-rows kernel (gq_product_rows.cu) and the tcgen05 kernel
// (gq_product_tc.cu).
#include "gq_product.cuh"

namespace gq {
namespace prod {
namespace {

// The few-rows kernel reads the weights of an expert once per 8 .. 32 rows, the tcgen05
// kernel once per 128 .. 256: the first while a busy expert's rows fit one pass.
bool by_rows(int64_t S, int64_t E, int engine) { return engine == 0 || (engine < 0 && S <= 8 * E); }

int run(const char* what, const Args& a, Kind kind, bool glu, int engine, void* workspace, size_t workspace_bytes,
        cudaStream_t s) {
  const int64_t es = kind == S8 ? 1 : 2;
  const int64_t I = glu ? a.N / 2 : a.N;
  GQ_REQUIRE(a.S >= 0 && a.S < (int64_t(1) << 31) && a.n_src >= 0 && a.n_src < (int64_t(1) << 31),
             "%s: %lld rows of %lld", what, (long long)a.S, (long long)a.n_src);
  GQ_REQUIRE(a.E >= 1 && a.E <= kMaxExperts, "%s: %lld experts, at most %lld", what, (long long)a.E,
             (long long)kMaxExperts);
  GQ_REQUIRE(a.N >= 1 && a.N < (int64_t(1) << 31) && a.K >= 1 && a.K < (int64_t(1) << 31), "%s: sizes", what);
  GQ_REQUIRE(!glu || a.N % 2 == 0, "%s: glu needs an even number of channels, not %lld", what, (long long)a.N);
  GQ_REQUIRE(a.K * es % 16 == 0 && a.ldx >= a.K * es && a.ldw >= a.K * es && a.ldx % 16 == 0 && a.ldw % 16 == 0 &&
                 a.stride_w % 16 == 0 && (a.E == 1 || a.stride_w >= a.K * es),
             "%s: rows must be whole and 16-byte aligned", what);
  GQ_REQUIRE(a.ldx < (int64_t(1) << 40) && a.ldw < (int64_t(1) << 40) && a.stride_w < (int64_t(1) << 40),
             "%s: strides", what);
  GQ_REQUIRE(a.ldy >= I, "%s: ldy < channels", what);
  GQ_REQUIRE(a.offsets || a.E == 1, "%s: offsets", what);
  GQ_REQUIRE(a.rows || a.n_src >= a.S, "%s: X has fewer rows than the product", what);
  GQ_REQUIRE(engine >= -1 && engine <= 1, "%s: engine %d", what, engine);
  if (a.S == 0) return GQ_OK;
  GQ_REQUIRE(a.X && a.W && a.Y && a.n_src > 0, "%s: null pointer", what);
  GQ_REQUIRE(aligned16(a.X) && aligned16(a.W), "%s: X and W must be 16-byte aligned", what);
  if (by_rows(a.S, a.E, engine)) return launch_rows(a, kind, glu, s);
  const size_t need = a.rows ? size_t(a.S) * size_t(a.K * es) : 0;
  GQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
             "%s: workspace too small (%zu < %zu)", what, workspace_bytes, need);
  return launch_tc(a, kind, glu, workspace, s);
}

}  // namespace
}  // namespace prod
}  // namespace gq

using namespace gq;
using namespace gq::prod;

extern "C" size_t gq_matmul_workspace_size(int64_t S, int64_t E, int64_t K, int element_bytes, int engine) {
  if (S <= 0 || E <= 0 || K <= 0) return 0;
  return by_rows(S, E, engine) ? 0 : size_t(S) * size_t(K) * size_t(element_bytes);
}

extern "C" int gq_matmul_grouped(const void* X, int64_t n, int64_t ldx, const int32_t* rows, int64_t S,
                                 const int64_t* offsets, int64_t E, const void* W, int64_t N, int64_t K, int64_t ldw,
                                 int64_t stride_w, int dtype, int glu, void* Y, int64_t ldy, int zero_behind,
                                 int engine, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  GQ_REQUIRE(dtype == GQ_BF16 || dtype == GQ_F16, "gq_matmul_grouped: rows and weights are bf16 or f16 (dtype %d)",
             dtype);
  Args a = {};
  a.X = (const uint8_t*)X, a.n_src = n, a.ldx = 2 * ldx, a.rows = rows, a.offsets = offsets, a.E = E, a.S = S;
  a.W = (const uint8_t*)W, a.N = N, a.K = K, a.ldw = 2 * ldw, a.stride_w = 2 * stride_w;
  a.Y = Y, a.ldy = ldy, a.out_dtype = dtype, a.zero_behind = zero_behind, a.status = status;
  return run("gq_matmul_grouped", a, dtype == GQ_BF16 ? BF16 : F16, glu != 0, engine, workspace,
             workspace_bytes, (cudaStream_t)stream);
}

extern "C" int gq_matmul_int8(const int8_t* Xq, const float* xs, int64_t n, int64_t ldx, const int32_t* rows,
                              int64_t S, const int64_t* offsets, int64_t E, const int8_t* Wq, const float* ws,
                              int64_t N, int64_t K, int64_t ldw, int64_t stride_w, const void* bias, int bias_dtype,
                              int glu, void* Y, int out_dtype, int64_t ldy, int zero_behind, int engine,
                              void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  GQ_REQUIRE(out_dtype == GQ_BF16 || out_dtype == GQ_F16 || out_dtype == GQ_F32, "gq_matmul_int8: out dtype %d",
             out_dtype);
  GQ_REQUIRE(!bias || bias_dtype == GQ_BF16 || bias_dtype == GQ_F16 || bias_dtype == GQ_F32,
             "gq_matmul_int8: bias dtype %d", bias_dtype);
  GQ_REQUIRE(!bias || (!offsets && !glu), "gq_matmul_int8: a bias goes with the dense product only");
  // |sum| <= K * 128 * 128 has to fit 31 bits
  GQ_REQUIRE(K <= 131071, "gq_matmul_int8: K = %lld, at most 131071 (32-bit sums)", (long long)K);
  GQ_REQUIRE(S <= 0 || (xs && ws), "gq_matmul_int8: null pointer");
  Args a = {};
  a.X = (const uint8_t*)Xq, a.n_src = n, a.ldx = ldx, a.rows = rows, a.offsets = offsets, a.E = E, a.S = S;
  a.W = (const uint8_t*)Wq, a.N = N, a.K = K, a.ldw = ldw, a.stride_w = stride_w;
  a.xs = xs, a.ws = ws, a.bias = bias, a.bias_dtype = bias_dtype;
  a.Y = Y, a.ldy = ldy, a.out_dtype = out_dtype, a.zero_behind = zero_behind, a.status = status;
  return run("gq_matmul_int8", a, S8, glu != 0, engine, workspace,
             workspace_bytes, (cudaStream_t)stream);
}
