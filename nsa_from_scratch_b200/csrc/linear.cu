// Projections and the gated feed-forward block: argument checks, workspaces, and the order of the matrix products.
#include "gemm.cuh"

namespace nsa {

// ---------------------------------------------------------------- gradient through the activation, bias gradient
// dz = dy * act'(z) (ACT: an activation stands between) and the column sums of dz (part: a row of partial sums per
// block row).  A thread owns 8 columns and walks the rows of its block row; bound by HBM.
template <typename T>
__global__ void __launch_bounds__(128) act_bwd_kernel(const void* __restrict__ dy, const void* __restrict__ z, void* __restrict__ dz,
                                                      float* __restrict__ part, int M, int N, int rows, int act, int vec) {
  const int c = (blockIdx.x * 128 + threadIdx.x) * 8, n = N - c;
  if (n <= 0) return;
  const int r0 = blockIdx.y * rows, r1 = min(M, r0 + rows);
  float sum[8] = {};
  for (int r = r0; r < r1; ++r) {
    const long long at = (long long)r * N + c;
    float d[8];
    load8<T>(dy, at, n, vec, d);
    if (act != ACT_NONE) {
      float v[8];
      load8<T>(z, at, n, vec, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float p, s;
        act_both(v[i], act, p, s);
        d[i] *= s;
      }
      store8<T>(dz, at, n, vec, d);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += d[i];
  }
  if (part != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) part[(long long)blockIdx.y * N + c + i] = sum[i];
  }
}

struct ActBwdPlan { int strips, groups, rows; };
static ActBwdPlan act_bwd_plan(int M, int N) {
  ActBwdPlan p;
  p.strips = (N + 1023) / 1024;
  const int want = (4 * sm_count() + p.strips - 1) / p.strips;                  // four blocks an SM
  p.rows = (M + want - 1) / want;
  if (p.rows < 1) p.rows = 1;
  p.groups = (M + p.rows - 1) / p.rows;
  return p;
}

static int act_bwd(const void* dy, const void* z, void* dz, float* part, int M, int N, int act, int dtype, cudaStream_t st) {
  const ActBwdPlan p = act_bwd_plan(M, N);
  const int vec = N % 8 == 0 && aligned16(dy) && aligned16(z) && aligned16(dz);
  const dim3 grid(p.strips, p.groups);
  if (dtype == NSA_BF16) act_bwd_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(dy, z, dz, part, M, N, p.rows, act, vec);
  else act_bwd_kernel<__half><<<grid, 128, 0, st>>>(dy, z, dz, part, M, N, p.rows, act, vec);
  return launch_status("act_bwd");
}

// ---------------------------------------------------------------- workspaces
// Hands out 256-byte aligned pieces; with base 0 it only counts.
struct Arena {
  unsigned char* base;
  long long at = 0;
  void* take(long long bytes) {
    void* p = base == nullptr ? nullptr : base + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  }
};

static int gemm(const GemmProblem& p, cudaStream_t st) {
  if (p.M == 0 || p.N == 0) return NSA_OK;
  return gemm_generic(p, st);
}

static GemmProblem problem(const void* A, int a_mn, long long lda, const void* B, int b_mn, long long ldb, int M, int N, int K, int dtype) {
  GemmProblem p = {};
  p.A[0] = A; p.B[0] = B;
  p.segments = 1;
  p.a_mn = a_mn; p.b_mn = b_mn;
  p.M = M; p.N = N; p.K = K;
  p.lda = lda; p.ldb = ldb;
  p.dtype = p.out_dtype = dtype;
  p.e.M = M; p.e.N = N;
  return p;
}
// EPI_LINEAR without anything around the sums
static int product(GemmProblem p, void* out, cudaStream_t st) {
  if (out == nullptr) return NSA_OK;
  p.e.mode = EPI_LINEAR;
  p.e.y = out;
  p.e.vec = p.N % 8 == 0 && aligned16(out);
  return gemm(p, st);
}

static bool is16(int dt) { return dt == NSA_BF16 || dt == NSA_FP16; }
static bool is8(int dt) { return dt == NSA_FP8_E4M3 || dt == NSA_FP8_E5M2; }

// ---------------------------------------------------------------- linear
static int check_linear(const nsa_linear_args& a) {
  NSA_REQUIRE(a.M >= 0 && a.N > 0 && a.K > 0, NSA_ERR_ARG, "linear: bad sizes M=%d N=%d K=%d", a.M, a.N, a.K);
  NSA_REQUIRE(is16(a.dtype) || is8(a.dtype), NSA_ERR_UNSUPPORTED, "linear: operand dtype %d", a.dtype);
  NSA_REQUIRE(is16(a.y_dtype) && (is8(a.dtype) || a.y_dtype == a.dtype), NSA_ERR_UNSUPPORTED, "linear: result dtype %d of operands %d", a.y_dtype, a.dtype);
  NSA_REQUIRE(a.act >= NSA_ACT_NONE && a.act <= NSA_ACT_RELU, NSA_ERR_ARG, "linear: activation %d", a.act);
  return NSA_OK;
}

int linear(const nsa_linear_args& a, cudaStream_t st) {
  int rc = check_linear(a);
  if (rc != NSA_OK) return rc;
  if (a.M == 0) return NSA_OK;
  NSA_REQUIRE(a.x && a.w && a.y, NSA_ERR_ARG, "linear: NULL pointer");
  NSA_REQUIRE(is8(a.dtype) == (a.x_scale != nullptr) && is8(a.dtype) == (a.w_scale != nullptr), NSA_ERR_ARG, "linear: fp8 operands, and only they, have scales");
  NSA_REQUIRE(a.z == nullptr || is16(a.dtype), NSA_ERR_UNSUPPORTED, "linear: fp8 operands keep nothing for a backward");
  GemmProblem p = problem(a.x, 0, a.K, a.w, 0, a.K, a.M, a.N, a.K, a.dtype);
  p.out_dtype = a.y_dtype;
  p.e.mode = EPI_LINEAR;
  p.e.act = a.act;
  p.e.bias = a.bias; p.e.residual = a.residual; p.e.xs = a.x_scale; p.e.ws = a.w_scale;
  p.e.y = a.y; p.e.o1 = a.z;
  p.e.vec = a.N % 8 == 0 && aligned16(a.bias) && aligned16(a.residual) && aligned16(a.y) && aligned16(a.z);
  return gemm(p, st);
}

static long long linear_bwd_ws(const nsa_linear_bwd_args& a, unsigned char* base, void** dz, float** part) {
  Arena w{base};
  *dz = a.act != NSA_ACT_NONE ? w.take((long long)a.M * a.N * 2) : nullptr;
  *part = reinterpret_cast<float*>(w.take((long long)act_bwd_plan(a.M, a.N).groups * a.N * 4));
  return w.at;
}

static int check_linear_bwd(const nsa_linear_bwd_args& a) {
  NSA_REQUIRE(a.M >= 0 && a.N > 0 && a.K > 0, NSA_ERR_ARG, "linear backward: bad sizes M=%d N=%d K=%d", a.M, a.N, a.K);
  NSA_REQUIRE(is16(a.dtype), NSA_ERR_UNSUPPORTED, "linear backward: dtype %d", a.dtype);
  NSA_REQUIRE(a.act >= NSA_ACT_NONE && a.act <= NSA_ACT_RELU, NSA_ERR_ARG, "linear backward: activation %d", a.act);
  return NSA_OK;
}

static int zero(void* p, long long bytes, cudaStream_t st) {
  if (p != nullptr) NSA_CUDA_OK(cudaMemsetAsync(p, 0, (size_t)bytes, st));
  return NSA_OK;
}

int linear_bwd(const nsa_linear_bwd_args& a, cudaStream_t st) {
  int rc = check_linear_bwd(a);
  if (rc != NSA_OK) return rc;
  if (a.M == 0) {                                             // sums over no rows
    if ((rc = zero(a.dw, (long long)a.N * a.K * 2, st)) != NSA_OK) return rc;
    return zero(a.dbias, (long long)a.N * 2, st);
  }
  NSA_REQUIRE(a.dy && a.x && a.w && a.ws && (a.z || a.act == NSA_ACT_NONE), NSA_ERR_ARG, "linear backward: NULL pointer");
  void* dz;
  float* part;
  const long long need = linear_bwd_ws(a, reinterpret_cast<unsigned char*>(a.ws), &dz, &part);
  NSA_REQUIRE(a.ws_bytes >= need, NSA_ERR_ARG, "linear backward: workspace of %lld bytes, %lld needed", (long long)a.ws_bytes, need);
  const void* g = a.dy;
  if (a.act != NSA_ACT_NONE || a.dbias != nullptr) {
    if ((rc = act_bwd(a.dy, a.z, dz, a.dbias ? part : nullptr, a.M, a.N, a.act, a.dtype, st)) != NSA_OK) return rc;
    if (a.act != NSA_ACT_NONE) g = dz;
    if (a.dbias != nullptr && (rc = column_sum(part, a.dbias, act_bwd_plan(a.M, a.N).groups, a.N, a.dtype, st)) != NSA_OK) return rc;
  }
  if ((rc = product(problem(g, 0, a.N, a.w, 1, a.K, a.M, a.K, a.N, a.dtype), a.dx, st)) != NSA_OK) return rc;
  return product(problem(g, 1, a.N, a.x, 1, a.K, a.N, a.K, a.M, a.dtype), a.dw, st);
}

// ---------------------------------------------------------------- gated feed-forward block
static int check_mlp(int M, int N, int F, int dtype, int act) {
  NSA_REQUIRE(M >= 0 && N > 0 && F > 0, NSA_ERR_ARG, "gated_mlp: bad sizes M=%d N=%d F=%d", M, N, F);
  NSA_REQUIRE(is16(dtype), NSA_ERR_UNSUPPORTED, "gated_mlp: dtype %d", dtype);
  NSA_REQUIRE(act >= NSA_ACT_NONE && act <= NSA_ACT_RELU, NSA_ERR_ARG, "gated_mlp: activation %d", act);
  return NSA_OK;
}
static long long mlp_ws(const nsa_gated_mlp_args& a, unsigned char* base, void** h) {
  Arena w{base};
  *h = w.take((long long)a.M * a.F * 2);
  return w.at;
}

int gated_mlp(const nsa_gated_mlp_args& a, cudaStream_t st) {
  int rc = check_mlp(a.M, a.N, a.F, a.dtype, a.act);
  if (rc != NSA_OK) return rc;
  if (a.M == 0) return NSA_OK;
  NSA_REQUIRE(a.x && a.wg && a.wu && a.wd && a.y && a.ws, NSA_ERR_ARG, "gated_mlp: NULL pointer");
  NSA_REQUIRE((a.g == nullptr) == (a.u == nullptr), NSA_ERR_ARG, "gated_mlp: give both g and u or neither");
  void* h;
  const long long need = mlp_ws(a, reinterpret_cast<unsigned char*>(a.ws), &h);
  NSA_REQUIRE(a.ws_bytes >= need, NSA_ERR_ARG, "gated_mlp: workspace of %lld bytes, %lld needed", (long long)a.ws_bytes, need);
  GemmProblem p = problem(a.x, 0, a.N, a.wg, 0, a.N, a.M, a.F, a.N, a.dtype);
  p.B[1] = a.wu;
  p.e.mode = EPI_GLU;
  p.e.act = a.act;
  p.e.y = h; p.e.o1 = a.g; p.e.o2 = a.u;
  p.e.vec = a.F % 8 == 0 && aligned16(h) && aligned16(a.g) && aligned16(a.u);
  if ((rc = gemm(p, st)) != NSA_OK) return rc;
  GemmProblem d = problem(h, 0, a.F, a.wd, 0, a.F, a.M, a.N, a.F, a.dtype);
  d.e.mode = EPI_LINEAR;
  d.e.residual = a.residual;
  d.e.y = a.y;
  d.e.vec = a.N % 8 == 0 && aligned16(a.residual) && aligned16(a.y);
  return gemm(d, st);
}

static long long mlp_bwd_ws(const nsa_gated_mlp_bwd_args& a, unsigned char* base, void** dg, void** du, void** h) {
  Arena w{base};
  *dg = w.take((long long)a.M * a.F * 2);
  *du = w.take((long long)a.M * a.F * 2);
  *h = w.take((long long)a.M * a.F * 2);
  return w.at;
}

int gated_mlp_bwd(const nsa_gated_mlp_bwd_args& a, cudaStream_t st) {
  int rc = check_mlp(a.M, a.N, a.F, a.dtype, a.act);
  if (rc != NSA_OK) return rc;
  if (a.M == 0) {
    const long long bytes = (long long)a.N * a.F * 2;
    if ((rc = zero(a.dwg, bytes, st)) != NSA_OK || (rc = zero(a.dwu, bytes, st)) != NSA_OK) return rc;
    return zero(a.dwd, bytes, st);
  }
  NSA_REQUIRE(a.dy && a.x && a.wg && a.wu && a.wd && a.g && a.u && a.ws, NSA_ERR_ARG, "gated_mlp backward: NULL pointer");
  void *dg, *du, *h;
  const long long need = mlp_bwd_ws(a, reinterpret_cast<unsigned char*>(a.ws), &dg, &du, &h);
  NSA_REQUIRE(a.ws_bytes >= need, NSA_ERR_ARG, "gated_mlp backward: workspace of %lld bytes, %lld needed", (long long)a.ws_bytes, need);
  GemmProblem p = problem(a.dy, 0, a.N, a.wd, 1, a.F, a.M, a.F, a.N, a.dtype);             // dh = dy wd
  p.e.mode = EPI_GLU_BWD;
  p.e.act = a.act;
  p.e.i0 = a.g; p.e.i1 = a.u;
  p.e.y = dg; p.e.o1 = du; p.e.o2 = h;
  p.e.vec = a.F % 8 == 0 && aligned16(a.g) && aligned16(a.u);
  if ((rc = gemm(p, st)) != NSA_OK) return rc;
  GemmProblem x = problem(dg, 0, a.F, a.wg, 1, a.N, a.M, a.N, a.F, a.dtype);               // dx = dg wg + du wu
  x.A[1] = du; x.B[1] = a.wu;
  x.segments = 2;
  if ((rc = product(x, a.dx, st)) != NSA_OK) return rc;
  if ((rc = product(problem(dg, 1, a.F, a.x, 1, a.N, a.F, a.N, a.M, a.dtype), a.dwg, st)) != NSA_OK) return rc;
  if ((rc = product(problem(du, 1, a.F, a.x, 1, a.N, a.F, a.N, a.M, a.dtype), a.dwu, st)) != NSA_OK) return rc;
  return product(problem(a.dy, 1, a.N, h, 1, a.F, a.N, a.F, a.M, a.dtype), a.dwd, st);
}

int rms_norm(const nsa_norm_args&, cudaStream_t);
int rms_norm_bwd(const nsa_norm_bwd_args&, cudaStream_t);
long long rms_norm_bwd_ws_bytes(long long, int);
int quantize_rows(const void*, void*, float*, long long, int, int, int, cudaStream_t);
int rope_axes(const nsa_rope_axes_args&, cudaStream_t);

static bool is_real(int dt) { return is16(dt) || dt == NSA_FP32; }

}  // namespace nsa

using namespace nsa;

extern "C" {

int nsa_rms_norm(const nsa_norm_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "rms_norm: NULL argument block");
  NSA_REQUIRE(a->rows >= 0 && a->rows < 2147483648LL && a->hidden > 0, NSA_ERR_ARG, "rms_norm: bad sizes rows=%lld hidden=%d", (long long)a->rows, a->hidden);
  NSA_REQUIRE(is_real(a->x_dtype), NSA_ERR_UNSUPPORTED, "rms_norm: x dtype %d", a->x_dtype);
  NSA_REQUIRE(a->w_dtype == a->x_dtype || a->w_dtype == NSA_FP32, NSA_ERR_UNSUPPORTED, "rms_norm: weight dtype %d beside x %d", a->w_dtype, a->x_dtype);
  NSA_REQUIRE(a->y_dtype == a->x_dtype || is8(a->y_dtype), NSA_ERR_UNSUPPORTED, "rms_norm: result dtype %d of x %d", a->y_dtype, a->x_dtype);
  NSA_REQUIRE(a->eps >= 0.f, NSA_ERR_ARG, "rms_norm: eps must not be negative");
  NSA_REQUIRE((a->residual == nullptr) == (a->h == nullptr), NSA_ERR_ARG, "rms_norm: residual and h must both be given or both be NULL");
  NSA_REQUIRE(a->residual == nullptr || a->res_dtype == a->x_dtype || a->res_dtype == NSA_FP32, NSA_ERR_UNSUPPORTED, "rms_norm: residual dtype %d beside x %d",
              a->res_dtype, a->x_dtype);
  if (a->rows == 0) return NSA_OK;
  NSA_REQUIRE(a->x && a->weight && a->y && (a->scale != nullptr || !is8(a->y_dtype)), NSA_ERR_ARG, "rms_norm: NULL pointer");
  return rms_norm(*a, (cudaStream_t)stream);
}

int64_t nsa_rms_norm_bwd_ws_bytes(int64_t rows, int hidden) {
  NSA_REQUIRE(rows >= 0 && hidden > 0, NSA_ERR_ARG, "rms_norm backward: bad sizes rows=%lld hidden=%d", (long long)rows, hidden);
  return rms_norm_bwd_ws_bytes(rows, hidden);
}

int nsa_rms_norm_bwd(const nsa_norm_bwd_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "rms_norm backward: NULL argument block");
  NSA_REQUIRE(a->rows >= 0 && a->hidden > 0, NSA_ERR_ARG, "rms_norm backward: bad sizes rows=%lld hidden=%d", (long long)a->rows, a->hidden);
  NSA_REQUIRE(is_real(a->x_dtype) && (a->w_dtype == a->x_dtype || a->w_dtype == NSA_FP32) && (a->res_dtype == a->x_dtype || a->res_dtype == NSA_FP32),
              NSA_ERR_UNSUPPORTED, "rms_norm backward: dtypes %d/%d/%d", a->x_dtype, a->res_dtype, a->w_dtype);
  if (a->rows == 0) return zero(a->dweight, (long long)a->hidden * (a->w_dtype == NSA_FP32 ? 4 : 2), (cudaStream_t)stream);
  NSA_REQUIRE(a->dy && a->h && a->weight && a->rstd && a->dx && a->ws, NSA_ERR_ARG, "rms_norm backward: NULL pointer");
  const long long need = rms_norm_bwd_ws_bytes(a->rows, a->hidden);
  NSA_REQUIRE(a->ws_bytes >= need, NSA_ERR_ARG, "rms_norm backward: workspace of %lld bytes, %lld needed", (long long)a->ws_bytes, need);
  return rms_norm_bwd(*a, (cudaStream_t)stream);
}

int nsa_quantize_rows_fp8(const void* x, void* q, float* scale, int64_t rows, int n, int x_dtype, int fmt, nsa_stream_t stream) {
  NSA_REQUIRE(rows >= 0 && rows < 2147483648LL && n > 0, NSA_ERR_ARG, "quantize_rows: bad sizes rows=%lld n=%d", (long long)rows, n);
  NSA_REQUIRE(is_real(x_dtype), NSA_ERR_UNSUPPORTED, "quantize_rows: dtype %d", x_dtype);
  NSA_REQUIRE(is8(fmt), NSA_ERR_ARG, "quantize_rows: format %d", fmt);
  if (rows == 0) return NSA_OK;
  NSA_REQUIRE(x && q && scale, NSA_ERR_ARG, "quantize_rows: NULL pointer");
  return quantize_rows(x, q, scale, rows, n, x_dtype, fmt, (cudaStream_t)stream);
}

int nsa_rope_axes(const nsa_rope_axes_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "rope_axes: NULL argument block");
  NSA_REQUIRE(a->B >= 0 && a->T >= 0 && a->H > 0 && a->Hkv > 0 && a->H + 2LL * a->Hkv < 65536, NSA_ERR_ARG, "rope_axes: bad sizes B=%d T=%d H=%d Hkv=%d", a->B, a->T,
              a->H, a->Hkv);
  NSA_REQUIRE(a->D > 0 && a->D % 2 == 0 && a->D <= 1024, NSA_ERR_UNSUPPORTED, "rope_axes: D=%d must be even and at most 1024", a->D);
  NSA_REQUIRE(a->n_axes >= 1 && a->n_axes <= 8, NSA_ERR_ARG, "rope_axes: %d axes (1 to 8 are taken)", a->n_axes);
  long long sum = 0;
  for (int i = 0; i < a->n_axes; ++i) {
    NSA_REQUIRE(a->sections[i] >= 0, NSA_ERR_ARG, "rope_axes: section %d is negative", i);
    sum += a->sections[i];
  }
  NSA_REQUIRE(sum == a->D / 2, NSA_ERR_ARG, "rope_axes: the sections add up to %lld, not to D/2 = %d", sum, a->D / 2);
  NSA_REQUIRE(is_real(a->x_dtype), NSA_ERR_UNSUPPORTED, "rope_axes: x dtype %d", a->x_dtype);
  NSA_REQUIRE(is16(a->y_dtype), NSA_ERR_UNSUPPORTED, "rope_axes: y dtype %d must be 16-bit", a->y_dtype);
  if (a->B == 0 || a->T == 0) return NSA_OK;
  NSA_REQUIRE(a->q && a->k && a->v && a->q_out && a->k_out && a->v_out && a->positions && a->inv_freq, NSA_ERR_ARG, "rope_axes: NULL pointer");
  NSA_REQUIRE(a->q_batch >= 0 && a->q_token >= 0 && a->k_batch >= 0 && a->k_token >= 0 && a->v_batch >= 0 && a->v_token >= 0, NSA_ERR_ARG,
              "rope_axes: negative pitch");
  return rope_axes(*a, (cudaStream_t)stream);
}

int64_t nsa_linear_ws_bytes(const nsa_linear_args* a) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "linear: NULL argument block");
  const int rc = check_linear(*a);
  return rc != NSA_OK ? rc : 0;
}
int nsa_linear(const nsa_linear_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "linear: NULL argument block");
  return linear(*a, (cudaStream_t)stream);
}
int64_t nsa_linear_bwd_ws_bytes(const nsa_linear_bwd_args* a) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "linear backward: NULL argument block");
  const int rc = check_linear_bwd(*a);
  void* dz;
  float* part;
  return rc != NSA_OK ? rc : linear_bwd_ws(*a, nullptr, &dz, &part);
}
int nsa_linear_bwd(const nsa_linear_bwd_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "linear backward: NULL argument block");
  return linear_bwd(*a, (cudaStream_t)stream);
}
int64_t nsa_gated_mlp_ws_bytes(const nsa_gated_mlp_args* a) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "gated_mlp: NULL argument block");
  const int rc = check_mlp(a->M, a->N, a->F, a->dtype, a->act);
  void* h;
  return rc != NSA_OK ? rc : mlp_ws(*a, nullptr, &h);
}
int nsa_gated_mlp(const nsa_gated_mlp_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "gated_mlp: NULL argument block");
  return gated_mlp(*a, (cudaStream_t)stream);
}
int64_t nsa_gated_mlp_bwd_ws_bytes(const nsa_gated_mlp_bwd_args* a) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "gated_mlp backward: NULL argument block");
  const int rc = check_mlp(a->M, a->N, a->F, a->dtype, a->act);
  void *dg, *du, *h;
  return rc != NSA_OK ? rc : mlp_bwd_ws(*a, nullptr, &dg, &du, &h);
}
int nsa_gated_mlp_bwd(const nsa_gated_mlp_bwd_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "gated_mlp backward: NULL argument block");
  return gated_mlp_bwd(*a, (cudaStream_t)stream);
}

}  // extern "C"
