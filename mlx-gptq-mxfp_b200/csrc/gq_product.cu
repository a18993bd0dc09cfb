// C entry points of the products of activation rows with weights: argument checks and the
// choice between the few-rows kernel (gq_product_rows.cu) and the tcgen05 kernel
// (gq_product_tc.cu).
#include <algorithm>

#include "gq_product.cuh"

namespace gq {
namespace prod {
namespace {

// The few-rows kernel streams the weights with any number of channel blocks and reads them
// again (from L2) for every 8 .. 32 rows; the tcgen05 kernel reads them once per 64 .. 256
// rows but has only CTA pairs x 256 channels to spread them over. Measured, 128 experts of
// [1536, 2048] with SwiGLU and of [2048, 768], both: 64 rows 61 against 66 us, 128 rows 85
// against 78, 512 rows 191 against 112; dense s8 [4096, 4096], 64 rows 13 against 16 us,
// 128 rows 23 against 16. The rule fits 128 experts and one. Between them it goes to the
// tcgen05 kernel too early: evenly routed rows through E experts of [1536, 2048] with SwiGLU,
// weights from HBM, E = 2 and 8 rows 6 against 16 us, E = 8 and 16 rows 12 against 18, E = 32
// and 64 rows 29 against 35; the two meet near 128 rows (E = 2 to 8) and 256 (E = 16, 32).
bool by_rows(int64_t S, int64_t E, int engine) {
  return engine == 0 || (engine < 0 && S <= (E == 1 ? 64 : (E + 1) / 2));
}

int check(const char* what, const Args& a, Kind kind, bool glu, int engine) {
  const int64_t es = kind == S8 ? 1 : 2;
  const int64_t I = glu ? a.N / 2 : a.N;
  GQ_REQUIRE(a.S >= 0 && a.S <= (int64_t(1) << 30) && a.n_src >= 0 && a.n_src < (int64_t(1) << 31),
             "%s: %lld rows of %lld, at most 2^30 of 2^31 - 1", what, (long long)a.S, (long long)a.n_src);
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
  return GQ_OK;
}

int run(const char* what, const Args& a, Kind kind, bool glu, int engine, void* workspace, size_t workspace_bytes,
        cudaStream_t s) {
  const int st = check(what, a, kind, glu, engine);
  if (st != GQ_OK || a.S == 0) return st;
  const int64_t es = kind == S8 ? 1 : 2;
  if (by_rows(a.S, a.E, engine)) return launch_rows(a, kind, glu, s);
  const size_t need = a.rows ? size_t(a.S) * size_t(a.K * es) : 0;
  GQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
             "%s: workspace too small (%zu < %zu)", what, workspace_bytes, need);
  return launch_tc(a, kind, glu, workspace, s);
}

// early (see Args): only for launches that follow one of this library's own kernels.
int grouped(bool early, const void* X, int64_t n, int64_t ldx, const int32_t* rows, int64_t S, const int64_t* offsets,
            int64_t E, const void* W, int64_t N, int64_t K, int64_t ldw, int64_t stride_w, int dtype, int glu, void* Y,
            int out_dtype, int64_t ldy, int zero_behind, int engine, void* workspace, size_t workspace_bytes, int32_t* status,
            void* stream) {
  GQ_REQUIRE(dtype == GQ_BF16 || dtype == GQ_F16, "gq_matmul_grouped: rows and weights are bf16 or f16 (dtype %d)",
             dtype);
  Args a = {};
  a.X = (const uint8_t*)X, a.n_src = n, a.ldx = 2 * ldx, a.rows = rows, a.offsets = offsets, a.E = E, a.S = S;
  a.W = (const uint8_t*)W, a.N = N, a.K = K, a.ldw = 2 * ldw, a.stride_w = 2 * stride_w;
  a.Y = Y, a.ldy = ldy, a.out_dtype = out_dtype, a.zero_behind = zero_behind, a.status = status, a.early = early;
  return run("gq_matmul_grouped", a, dtype == GQ_BF16 ? BF16 : F16, glu != 0, engine, workspace, workspace_bytes,
             (cudaStream_t)stream);
}

int int8(bool early, const int8_t* Xq, const float* xs, int64_t n, int64_t ldx, const int32_t* rows, int64_t S,
         const int64_t* offsets, int64_t E, const int8_t* Wq, const float* ws, int64_t N, int64_t K, int64_t ldw,
         int64_t stride_w, const void* bias, int bias_dtype, int glu, void* Y, int out_dtype, int64_t ldy,
         int zero_behind, int engine, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  GQ_REQUIRE(out_dtype == GQ_BF16 || out_dtype == GQ_F16 || out_dtype == GQ_F32, "gq_matmul_int8: out dtype %d",
             out_dtype);
  GQ_REQUIRE(!bias || bias_dtype == GQ_BF16 || bias_dtype == GQ_F16 || bias_dtype == GQ_F32,
             "gq_matmul_int8: bias dtype %d", bias_dtype);
  GQ_REQUIRE(!bias || (!offsets && !glu), "gq_matmul_int8: a bias goes with the dense product only");
  // |sum| <= K * 128 * 128 has to fit 31 bits: the largest multiple of 16 below 2^31 / 2^14
  GQ_REQUIRE(K <= 131056, "gq_matmul_int8: K = %lld, at most 131056 (32-bit sums)", (long long)K);
  GQ_REQUIRE(S <= 0 || (xs && ws), "gq_matmul_int8: null pointer");
  Args a = {};
  a.X = (const uint8_t*)Xq, a.n_src = n, a.ldx = ldx, a.rows = rows, a.offsets = offsets, a.E = E, a.S = S;
  a.W = (const uint8_t*)Wq, a.N = N, a.K = K, a.ldw = ldw, a.stride_w = stride_w;
  a.xs = xs, a.ws = ws, a.bias = bias, a.bias_dtype = bias_dtype;
  a.Y = Y, a.ldy = ldy, a.out_dtype = out_dtype, a.zero_behind = zero_behind, a.status = status, a.early = early;
  return run("gq_matmul_int8", a, S8, glu != 0, engine, workspace, workspace_bytes, (cudaStream_t)stream);
}

}  // namespace
}  // namespace prod
}  // namespace gq

using namespace gq;

extern "C" size_t gq_matmul_workspace_size(int64_t S, int64_t E, int64_t K, int element_bytes, int engine) {
  if (S <= 0 || E <= 0 || K <= 0) return 0;
  return prod::by_rows(S, E, engine) ? 0 : size_t(S) * size_t(K) * size_t(element_bytes);
}

extern "C" int gq_matmul_grouped(const void* X, int64_t n, int64_t ldx, const int32_t* rows, int64_t S,
                                 const int64_t* offsets, int64_t E, const void* W, int64_t N, int64_t K, int64_t ldw,
                                 int64_t stride_w, int dtype, int glu, void* Y, int64_t ldy, int zero_behind,
                                 int engine, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  return prod::grouped(false, X, n, ldx, rows, S, offsets, E, W, N, K, ldw, stride_w, dtype, glu, Y, dtype, ldy,
                       zero_behind, engine, workspace, workspace_bytes, status, stream);
}

extern "C" int gq_matmul_int8(const int8_t* Xq, const float* xs, int64_t n, int64_t ldx, const int32_t* rows,
                              int64_t S, const int64_t* offsets, int64_t E, const int8_t* Wq, const float* ws,
                              int64_t N, int64_t K, int64_t ldw, int64_t stride_w, const void* bias, int bias_dtype,
                              int glu, void* Y, int out_dtype, int64_t ldy, int zero_behind, int engine,
                              void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  return prod::int8(false, Xq, xs, n, ldx, rows, S, offsets, E, Wq, ws, N, K, ldw, stride_w, bias, bias_dtype, glu, Y,
                    out_dtype, ldy, zero_behind, engine, workspace, workspace_bytes, status, stream);
}

// ---------------------------------------------------------------------------
// Runs of them in one call: what a decoding loop calls once per layer, where the host's
// time per call counts.
// ---------------------------------------------------------------------------
namespace {

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct MlpPlan {
  size_t tok, slot, offsets, route, acts, y, gathered, gathered_bytes, total;
};

MlpPlan mlp_plan(int64_t T, int64_t k, int64_t E, int64_t K, int64_t I, int64_t N, bool own_acts) {
  MlpPlan p;
  const size_t S = size_t(T) * size_t(k);
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  p.tok = take(S * 4);
  p.slot = take(S * 4);
  p.offsets = take(size_t(E + 1) * 8);
  p.route = take(gq_route_slots_workspace_size(T, k, E));
  p.acts = take(own_acts ? S * size_t(I) * 2 : 0);
  // The gathered rows and the second product's rows share their bytes: the first product has
  // read the one when the second writes the other, which it does behind grid_wait(). y is
  // float32: the weighted sum takes the products unrounded.
  p.gathered_bytes = gq_matmul_workspace_size(int64_t(S), E, K, 2, -1);
  p.gathered = p.y = take(std::max(S * size_t(N) * 4, p.gathered_bytes));
  p.total = at;
  return p;
}

}  // namespace

extern "C" size_t gq_expert_mlp_workspace_size(int64_t T, int64_t k, int64_t E, int64_t K, int64_t I, int64_t N,
                                               int own_acts) {
  if (T <= 0 || k <= 0 || T > INT32_MAX / k || E <= 0 || K <= 0 || I <= 0 || N <= 0) return 0;
  return mlp_plan(T, k, E, K, I, N, own_acts != 0).total;
}

extern "C" int gq_expert_mlp(const void* X, int dtype, int64_t T, int64_t ldx, const void* index, int index_bits,
                             const float* weights, int64_t k, const void* gate_up, int64_t ld_gate_up,
                             int64_t stride_gate_up, const void* down, int64_t ld_down, int64_t stride_down, int64_t E,
                             int64_t K, int64_t I, int64_t N, void* acts, int64_t ld_acts, void* out, int64_t ldo,
                             void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  GQ_REQUIRE(T >= 0 && k >= 1 && T <= INT32_MAX / k && E >= 1 && K >= 1 && I >= 1 && N >= 1, "gq_expert_mlp: sizes");
  if (T == 0) return GQ_OK;
  GQ_REQUIRE(index && weights && out, "gq_expert_mlp: null pointer");
  const int64_t Kd = (I + 7) / 8 * 8;  // what the second product contracts; columns [I, Kd) hold zeros
  GQ_REQUIRE(acts ? ld_acts % 8 == 0 && ld_acts >= Kd : I % 8 == 0,
             "gq_expert_mlp: activation rows must be 16-byte aligned and hold I rounded up to 8");
  const MlpPlan p = mlp_plan(T, k, E, K, I, N, acts == nullptr);
  if (prod::token_fits(T, k, E) && (acts || (workspace && workspace_bytes >= p.total && aligned16(workspace)))) {
    prod::Args up = {}, dn = {};
    if (!acts) acts = reinterpret_cast<uint8_t*>(workspace) + p.acts, ld_acts = I;
    up.X = (const uint8_t*)X, up.n_src = T, up.ldx = 2 * ldx, up.E = E, up.S = 1, up.offsets = (const int64_t*)index;
    up.W = (const uint8_t*)gate_up, up.N = 2 * I, up.K = K, up.ldw = 2 * ld_gate_up, up.stride_w = 2 * stride_gate_up;
    up.Y = acts, up.ldy = ld_acts, up.out_dtype = dtype;
    dn.X = (const uint8_t*)acts, dn.n_src = k, dn.ldx = 2 * ld_acts, dn.E = E, dn.S = 1, dn.offsets = up.offsets;
    dn.W = (const uint8_t*)down, dn.N = N, dn.K = Kd, dn.ldw = 2 * ld_down, dn.stride_w = 2 * stride_down;
    dn.Y = out, dn.ldy = N, dn.out_dtype = dtype;  // offsets: only checked for being there
    GQ_REQUIRE(dtype == GQ_BF16 || dtype == GQ_F16, "gq_expert_mlp: rows and weights are bf16 or f16 (dtype %d)", dtype);
    GQ_REQUIRE(index_bits == 32 || index_bits == 64, "gq_expert_mlp: indices have 32 or 64 bits, not %d", index_bits);
    const prod::Kind kind = dtype == GQ_BF16 ? prod::BF16 : prod::F16;
    int bad = prod::check("gq_expert_mlp", up, kind, true, -1);
    if (bad == GQ_OK) bad = prod::check("gq_expert_mlp", dn, kind, false, -1);
    return bad != GQ_OK ? bad : prod::launch_token(up, dn, kind, index, index_bits, k, weights, (cudaStream_t)stream);
  }
  GQ_REQUIRE(workspace && workspace_bytes >= p.total && aligned16(workspace),
             "gq_expert_mlp: workspace too small (%zu < %zu)", workspace_bytes, p.total);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  int32_t *tok = reinterpret_cast<int32_t*>(ws + p.tok), *slot = reinterpret_cast<int32_t*>(ws + p.slot);
  int64_t* offsets = reinterpret_cast<int64_t*>(ws + p.offsets);
  const int64_t S = T * k;
  if (!acts) acts = ws + p.acts, ld_acts = I;
  int st = gq_route_slots(index, index_bits, T, k, E, tok, slot, offsets, ws + p.route, p.acts - p.route, stream);
  if (st != GQ_OK) return st;
  st = gq_matmul_grouped(X, T, ldx, tok, S, offsets, E, gate_up, 2 * I, K, ld_gate_up, stride_gate_up, dtype, 1, acts,
                         ld_acts, 0, -1, ws + p.gathered, p.gathered_bytes, status, stream);
  if (st != GQ_OK) return st;
  st = prod::grouped(true, acts, S, ld_acts, nullptr, S, offsets, E, down, N, Kd, ld_down, stride_down, dtype, 0,
                     ws + p.y, GQ_F32, N, 0, -1, nullptr, 0, status, stream);
  if (st != GQ_OK) return st;
  return slots::combine_rows(ws + p.y, GQ_F32, dtype, S, N, slot, weights, T, k, N, out, ldo, (cudaStream_t)stream);
}

extern "C" size_t gq_linear_int8_workspace_size(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0) return 0;
  return align256(size_t(M) * 4) + size_t(M) * size_t((K + 15) / 16 * 16);
}

extern "C" int gq_linear_int8(const void* X, int dtype, int64_t M, int64_t K, int64_t ldx, const int8_t* Wq,
                              const float* ws, int64_t N, int64_t ldw, const void* bias, int bias_dtype, void* Y,
                              int out_dtype, int64_t ldy, void* workspace, size_t workspace_bytes, int32_t* status,
                              void* stream) {
  if (M == 0) return GQ_OK;
  GQ_REQUIRE(K <= 131056, "gq_linear_int8: K = %lld, at most 131056 (32-bit sums)", (long long)K);
  const size_t need = gq_linear_int8_workspace_size(M, K);
  GQ_REQUIRE(need && workspace && workspace_bytes >= need && aligned16(workspace),
             "gq_linear_int8: workspace too small (%zu < %zu)", workspace_bytes, need);
  const int64_t Kp = (K + 15) / 16 * 16;
  if (X && Wq && ws && prod::linear_rows_fit(X, dtype, M, K, ldx)) {
    prod::Args a = {};
    a.X = (const uint8_t*)Wq, a.n_src = M, a.ldx = Kp, a.E = 1, a.S = M;  // X itself is not read as codes
    a.W = (const uint8_t*)Wq, a.N = N, a.K = K, a.ldw = ldw, a.stride_w = N * ldw, a.ws = ws;
    a.bias = bias, a.bias_dtype = bias_dtype, a.Y = Y, a.ldy = ldy, a.out_dtype = out_dtype;
    GQ_REQUIRE(dtype == GQ_BF16 || dtype == GQ_F16 || dtype == GQ_F32, "gq_linear_int8: dtype %d", dtype);
    GQ_REQUIRE(out_dtype == GQ_BF16 || out_dtype == GQ_F16 || out_dtype == GQ_F32, "gq_linear_int8: out dtype %d",
               out_dtype);
    GQ_REQUIRE(!bias || bias_dtype == GQ_BF16 || bias_dtype == GQ_F16 || bias_dtype == GQ_F32,
               "gq_linear_int8: bias dtype %d", bias_dtype);
    GQ_REQUIRE(ldx >= K, "gq_linear_int8: ldx < K");
    const int st = prod::check("gq_linear_int8", a, prod::S8, false, -1);
    return st != GQ_OK ? st : prod::launch_linear_rows(X, dtype, ldx, a, (cudaStream_t)stream);
  }
  float* xs = reinterpret_cast<float*>(workspace);
  int8_t* q = reinterpret_cast<int8_t*>(workspace) + align256(size_t(M) * 4);
  const int st = gq_rtn_int8(X, dtype, M, K, ldx, q, Kp, Kp, xs, stream);
  if (st != GQ_OK) return st;
  return prod::int8(true, q, xs, M, Kp, nullptr, M, nullptr, 1, Wq, ws, N, Kp, ldw, N * ldw, bias, bias_dtype, 0, Y,
                        out_dtype, ldy, 0, -1, nullptr, 0, status, stream);
}
