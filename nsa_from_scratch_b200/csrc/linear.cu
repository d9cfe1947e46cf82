// Projections and the gated feed-forward block: argument checks, workspaces, and the order of the matrix products.
#include "gemm.cuh"

namespace nsa {

int sm_count() {
  static int known[64];              // 0: not asked yet; every thread finds the same number
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && known[dev] > 0) return known[dev];
  int sms = 148;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (dev >= 0 && dev < 64) known[dev] = sms;
  return sms;
}

// ---------------------------------------------------------------- gradient through the activation, bias gradient
// dz = dy * act' (slope: coded by the forward; NULL: no activation, nothing is written) and the column sums of dz
// (part: a row of partial sums per block row; NULL: not wanted).  A thread owns 8 columns and walks the rows of its
// block row, four under way at a time; bound by HBM: 22 us at 4001 x 4096 = 4.5 TB/s.
template <typename T>
__global__ void __launch_bounds__(128) act_bwd_kernel(const void* __restrict__ dy, const uint16_t* __restrict__ slope, void* __restrict__ dz,
                                                      float* __restrict__ part, int M, int N, long long lddz, int rows, int vec, int vecz) {
  const int c = (blockIdx.x * 128 + threadIdx.x) * 8, n = N - c;
  if (n <= 0) return;
  const int r0 = blockIdx.y * rows, r1 = r0 + min(rows, M - r0);
  float sum[8] = {};
  constexpr int U = 4;
  for (int r = r0; r < r1; r += U) {
    float d[U][8];
    uint32_t v[U][4];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      if (r + q >= r1) break;
      const long long at = (long long)(r + q) * N + c;
      load8<T>(dy, at, n, vec, d[q]);
      if (slope != nullptr) {
        if (vec) {
          const uint4 w = *reinterpret_cast<const uint4*>(slope + at);
          v[q][0] = w.x; v[q][1] = w.y; v[q][2] = w.z; v[q][3] = w.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[q][i] = (2 * i < n ? slope[at + 2 * i] : 0u) | ((2 * i + 1 < n ? (uint32_t)slope[at + 2 * i + 1] : 0u) << 16);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      if (r + q >= r1) break;
      if (slope != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[q][i] *= slope_value(v[q][i >> 1] >> (16 * (i & 1)));
        store8<T>(dz, (long long)(r + q) * lddz + c, n, vecz, d[q]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += d[q][i];
    }
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
  const int want = (8 * sm_count() + p.strips - 1) / p.strips;                  // eight blocks an SM
  p.rows = (M - 1) / want + 1;                                                  // M > 0; M + rows may pass 32 bits
  p.groups = (M - 1) / p.rows + 1;
  return p;
}

static int act_bwd(const void* dy, const void* slope, void* dz, long long lddz, float* part, int M, int N, int dtype, cudaStream_t st) {
  const ActBwdPlan p = act_bwd_plan(M, N);
  const int vec = N % 8 == 0 && aligned16(dy) && aligned16(slope), vecz = lddz % 8 == 0;
  const dim3 grid(p.strips, p.groups);
  if (dtype == NSA_BF16) act_bwd_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(dy, (const uint16_t*)slope, dz, part, M, N, lddz, p.rows, vec, vecz);
  else act_bwd_kernel<__half><<<grid, 128, 0, st>>>(dy, (const uint16_t*)slope, dz, part, M, N, lddz, p.rows, vec, vecz);
  return launch_status("act_bwd");
}

// ---------------------------------------------------------------- workspaces
// The workspace of a call: 256-byte aligned pieces, then one scratch area that its matrix products use in turn.  Each call
// goes through its steps twice, dry (counting, nothing is launched) and in earnest.
struct Arena {
  unsigned char* base;               // NULL: dry
  long long scratch_at;              // where the scratch starts (from the dry pass)
  cudaStream_t st;
  long long at = 0, scratch = 0;
  bool dry() const { return base == nullptr; }
  void* take(long long bytes) {
    void* p = dry() ? nullptr : base + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  }
  long long bytes() const { return at + scratch; }
};

template <typename Args>
static long long ws_bytes(const Args& a, int (*steps)(const Args&, Arena&)) {
  Arena w{nullptr, 0, nullptr};
  const int rc = steps(a, w);
  return rc != NSA_OK ? rc : w.bytes();
}
template <typename Args>
static int run_steps(const char* what, const Args& a, int (*steps)(const Args&, Arena&), cudaStream_t st) {
  Arena count{nullptr, 0, st};
  int rc = steps(a, count);
  if (rc != NSA_OK) return rc;
  const long long need = count.bytes();
  NSA_REQUIRE(a.ws_bytes >= need && (a.ws != nullptr || need == 0), NSA_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what, (long long)a.ws_bytes, need);
  NSA_REQUIRE(need == 0 || (reinterpret_cast<uintptr_t>(a.ws) & 255) == 0, NSA_ERR_ARG, "%s: the workspace is not 256-byte aligned", what);
  static unsigned char none[16];     // stands for a workspace of no bytes
  Arena w{a.ws != nullptr ? reinterpret_cast<unsigned char*>(a.ws) : none, count.at, st};
  return steps(a, w);
}

// Every pointer given lies on a multiple of `size`: what no kernel can do without, whichever path it takes
template <typename... P> static bool on(int size, const P*... p) { return ((reinterpret_cast<uintptr_t>(p) % size == 0) && ...); }
static bool is16(int dt) { return dt == NSA_BF16 || dt == NSA_FP16; }
static bool is8(int dt) { return dt == NSA_FP8_E4M3 || dt == NSA_FP8_E5M2; }
static int elem(int dt) { return is16(dt) ? 2 : 1; }
static long long padded(long long cols, int dt) { const int per = 16 / elem(dt); return (cols + per - 1) / per * per; }

// dst [rows][ldd] = src [rows][cols], zeros behind: 16 bytes a thread
template <typename E>
__global__ void __launch_bounds__(256) pad_rows_kernel(const E* __restrict__ src, E* __restrict__ dst, long long rows, int cols, int ldd) {
  constexpr int PER = 16 / sizeof(E);
  const int groups = ldd / PER;
  const long long total = rows * groups;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i / groups;
    const int c = (int)(i % groups) * PER;
    __align__(16) E v[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) v[e] = c + e < cols ? src[r * cols + c + e] : E(0);
    *reinterpret_cast<uint4*>(dst + r * ldd + c) = *reinterpret_cast<const uint4*>(v);
  }
}

// A size that the kernels' 32-bit counts hold with room to step past its end
static bool sized(int n) { return n > 0 && n <= NSA_MAX_SIZE; }

// An operand whose rows start on 16-byte boundaries: the caller's own, or a padded copy.
struct Mat { const void* p; long long ld; };
static int operand(Arena& w, const void* p, long long rows, int cols, int dtype, Mat* m) {
  const long long ld = padded(cols, dtype);
  *m = Mat{p, cols};
  if (ld == cols && aligned16(p)) return NSA_OK;
  void* q = w.take(rows * ld * elem(dtype));
  *m = Mat{q, ld};
  if (w.dry()) return NSA_OK;
  const long long want = (rows * (ld * elem(dtype) / 16) + 255) / 256, cap = 16LL * sm_count();
  const int grid = (int)(want < cap ? want : cap);
  if (is16(dtype)) pad_rows_kernel<<<grid, 256, 0, w.st>>>((const uint16_t*)p, (uint16_t*)q, rows, cols, (int)ld);
  else pad_rows_kernel<<<grid, 256, 0, w.st>>>((const uint8_t*)p, (uint8_t*)q, rows, cols, (int)ld);
  return launch_status("pad_rows");
}

static int gemm(Arena& w, const GemmProblem& p) {
  if (!w.dry()) return gemm_tc5(p, w.base + w.scratch_at, w.st);
  const long long need = gemm_tc5_ws_bytes(p);
  if (need > w.scratch) w.scratch = need;
  return NSA_OK;
}

static GemmProblem problem(Mat A, int a_mn, Mat B, int b_mn, int M, int N, int K, int dtype) {
  GemmProblem p = {};
  p.A[0] = A.p; p.B[0] = B.p;
  p.segments = 1;
  p.a_mn = a_mn; p.b_mn = b_mn;
  p.M = M; p.N = N; p.K = K;
  p.lda = A.ld; p.ldb = B.ld;
  p.dtype = p.out_dtype = dtype;
  p.e.M = M; p.e.N = N; p.e.ldy = N;
  return p;
}
// Plain products that are independent of each other, gathered for one launch.
struct Products {
  GemmProblem p[4];
  int count = 0;
  void add(GemmProblem q, void* out) {
    q.e.mode = EPI_LINEAR;
    q.e.y = out;
    q.e.vec = q.e.vecy = q.N % 8 == 0 && aligned16(out);
    p[count++] = q;
  }
  int run(Arena& w) const {
    if (count == 0) return NSA_OK;
    if (!w.dry()) return gemm_tc5_group(p, count, w.base + w.scratch_at, w.st);
    const long long need = gemm_tc5_group_ws_bytes(p, count);
    if (need > w.scratch) w.scratch = need;
    return NSA_OK;
  }
};

static int zero(void* p, long long bytes, cudaStream_t st) {
  if (p != nullptr) NSA_CUDA_OK(cudaMemsetAsync(p, 0, (size_t)bytes, st));
  return NSA_OK;
}
#define NSA_TRY(expr) do { const int rc__ = (expr); if (rc__ != NSA_OK) return rc__; } while (0)

// ---------------------------------------------------------------- linear
static int check_linear(const nsa_linear_args& a) {
  NSA_REQUIRE((a.M == 0 || sized(a.M)) && sized(a.N) && sized(a.K), NSA_ERR_ARG, "linear: bad sizes M=%d N=%d K=%d", a.M, a.N, a.K);
  NSA_REQUIRE(is16(a.dtype) || is8(a.dtype), NSA_ERR_UNSUPPORTED, "linear: operand dtype %d", a.dtype);
  NSA_REQUIRE(is16(a.y_dtype) && (is8(a.dtype) || a.y_dtype == a.dtype), NSA_ERR_UNSUPPORTED, "linear: result dtype %d of operands %d", a.y_dtype, a.dtype);
  NSA_REQUIRE(a.act >= NSA_ACT_NONE && a.act <= NSA_ACT_RELU, NSA_ERR_ARG, "linear: activation %d", a.act);
  return NSA_OK;
}

static int linear_steps(const nsa_linear_args& a, Arena& w) {
  const bool few = gemm_skinny_takes(a.M, a.N, a.K, EPI_LINEAR);
  Mat x{a.x, a.K}, wt{a.w, a.K};
  if (!few) {
    NSA_TRY(operand(w, a.x, a.M, a.K, a.dtype, &x));
    NSA_TRY(operand(w, a.w, a.N, a.K, a.dtype, &wt));
  }
  GemmProblem p = problem(x, 0, wt, 0, a.M, a.N, a.K, a.dtype);
  p.out_dtype = a.y_dtype;
  p.e.mode = EPI_LINEAR;
  p.e.act = a.act;
  p.e.bias = a.bias; p.e.residual = a.residual; p.e.xs = a.x_scale; p.e.ws = a.w_scale;
  p.e.y = a.y; p.e.o1 = a.slope;
  p.e.vec = a.N % 8 == 0 && aligned16(a.bias) && aligned16(a.residual) && aligned16(a.slope) && aligned16(a.w_scale);
  p.e.vecy = a.N % 8 == 0 && aligned16(a.y);
  if (few) return w.dry() ? NSA_OK : gemm_skinny(p, false, w.st);
  return gemm(w, p);
}

int linear(const nsa_linear_args& a, cudaStream_t st) {
  NSA_TRY(check_linear(a));
  if (a.M == 0) return NSA_OK;
  NSA_REQUIRE(a.x && a.w && a.y, NSA_ERR_ARG, "linear: NULL pointer");
  NSA_REQUIRE(is8(a.dtype) == (a.x_scale != nullptr) && is8(a.dtype) == (a.w_scale != nullptr), NSA_ERR_ARG, "linear: fp8 operands, and only they, have scales");
  NSA_REQUIRE(a.slope == nullptr || (is16(a.dtype) && a.act != NSA_ACT_NONE), NSA_ERR_ARG, "linear: only an activation of 16-bit operands leaves a slope");
  NSA_REQUIRE(on(elem(a.dtype), a.x, a.w) && on(2, a.bias, a.residual, a.y, a.slope) && on(4, a.x_scale, a.w_scale), NSA_ERR_ARG, "linear: a pointer is not aligned to its elements");
  return run_steps("linear", a, linear_steps, st);
}

static int check_linear_bwd(const nsa_linear_bwd_args& a) {
  NSA_REQUIRE((a.M == 0 || sized(a.M)) && sized(a.N) && sized(a.K), NSA_ERR_ARG, "linear backward: bad sizes M=%d N=%d K=%d", a.M, a.N, a.K);
  NSA_REQUIRE(is16(a.dtype), NSA_ERR_UNSUPPORTED, "linear backward: dtype %d", a.dtype);
  return NSA_OK;
}

static int linear_bwd_steps(const nsa_linear_bwd_args& a, Arena& w) {
  const bool run = !w.dry();
  Mat g, x, wt;
  float* part = reinterpret_cast<float*>(w.take((long long)act_bwd_plan(a.M, a.N).groups * a.N * 4));
  if (a.has_act) {
    const long long ld = padded(a.N, a.dtype);
    void* dz = w.take((long long)a.M * ld * 2);
    g = Mat{dz, ld};
    if (run) NSA_TRY(act_bwd(a.dy, a.slope, dz, ld, a.dbias ? part : nullptr, a.M, a.N, a.dtype, w.st));
  } else {
    if (run && a.dbias) NSA_TRY(act_bwd(a.dy, nullptr, nullptr, 0, part, a.M, a.N, a.dtype, w.st));
    if (a.dx || a.dw) NSA_TRY(operand(w, a.dy, a.M, a.N, a.dtype, &g));
  }
  if (run && a.dbias) NSA_TRY(column_sum(part, a.dbias, act_bwd_plan(a.M, a.N).groups, a.N, a.dtype, w.st));
  Products ps;
  if (a.dx) {
    NSA_TRY(operand(w, a.w, a.N, a.K, a.dtype, &wt));
    ps.add(problem(g, 0, wt, 1, a.M, a.K, a.N, a.dtype), a.dx);
  }
  if (a.dw) {
    NSA_TRY(operand(w, a.x, a.M, a.K, a.dtype, &x));
    ps.add(problem(g, 1, x, 1, a.N, a.K, a.M, a.dtype), a.dw);
  }
  return ps.run(w);
}

int linear_bwd(const nsa_linear_bwd_args& a, cudaStream_t st) {
  NSA_TRY(check_linear_bwd(a));
  if (a.M == 0) {                                             // sums over no rows
    NSA_TRY(zero(a.dw, (long long)a.N * a.K * 2, st));
    return zero(a.dbias, (long long)a.N * 2, st);
  }
  NSA_REQUIRE(a.dy && a.x && a.w && (a.slope != nullptr) == (a.has_act != 0), NSA_ERR_ARG, "linear backward: NULL pointer");
  NSA_REQUIRE(on(2, a.dy, a.x, a.w, a.slope, a.dx, a.dw, a.dbias), NSA_ERR_ARG, "linear backward: a pointer is not aligned to its elements");
  return run_steps("linear backward", a, linear_bwd_steps, st);
}

// ---------------------------------------------------------------- gated feed-forward block
static int check_mlp(int M, int N, int F, int dtype, int act) {
  NSA_REQUIRE((M == 0 || sized(M)) && sized(N) && sized(F), NSA_ERR_ARG, "gated_mlp: bad sizes M=%d N=%d F=%d", M, N, F);
  NSA_REQUIRE(is16(dtype), NSA_ERR_UNSUPPORTED, "gated_mlp: dtype %d", dtype);
  NSA_REQUIRE(act >= NSA_ACT_NONE && act <= NSA_ACT_RELU, NSA_ERR_ARG, "gated_mlp: activation %d", act);
  return NSA_OK;
}

static int mlp_steps(const nsa_gated_mlp_args& a, Arena& w) {
  const long long ldh = padded(a.F, a.dtype);
  void* h = a.h != nullptr ? a.h : w.take((long long)a.M * ldh * 2);
  const bool few = gemm_skinny_takes(a.M, a.F, a.N, EPI_GLU), few_down = gemm_skinny_takes(a.M, a.N, a.F, EPI_LINEAR);
  Mat x{a.x, a.N}, wg{a.wg, a.N}, wu{a.wu, a.N}, wd{a.wd, a.F};
  if (!few) {
    NSA_TRY(operand(w, a.x, a.M, a.N, a.dtype, &x));
    NSA_TRY(operand(w, a.wg, a.F, a.N, a.dtype, &wg));
    NSA_TRY(operand(w, a.wu, a.F, a.N, a.dtype, &wu));
  }
  GemmProblem p = problem(x, 0, wg, 0, a.M, a.F, a.N, a.dtype);
  p.B[1] = wu.p;
  p.e.mode = EPI_GLU;
  p.e.act = a.act;
  p.e.y = h; p.e.o1 = a.p; p.e.o2 = a.s; p.e.o3 = a.low;
  p.e.ldy = ldh; p.e.vec = p.e.vecy = 1;
  if (few) {
    if (!w.dry()) NSA_TRY(gemm_skinny(p, false, w.st));
  } else {
    NSA_TRY(gemm(w, p));
  }
  if (!few_down) NSA_TRY(operand(w, a.wd, a.N, a.F, a.dtype, &wd));
  GemmProblem d = problem(Mat{h, ldh}, 0, wd, 0, a.M, a.N, a.F, a.dtype);
  d.e.mode = EPI_LINEAR;
  d.e.residual = a.residual;
  d.e.y = a.y;
  d.e.vec = a.N % 8 == 0 && aligned16(a.residual);
  d.e.vecy = a.N % 8 == 0 && aligned16(a.y);
  if (few_down) return w.dry() ? NSA_OK : gemm_skinny(d, true, w.st);
  return gemm(w, d);
}

int gated_mlp(const nsa_gated_mlp_args& a, cudaStream_t st) {
  NSA_TRY(check_mlp(a.M, a.N, a.F, a.dtype, a.act));
  if (a.M == 0) return NSA_OK;
  NSA_REQUIRE(a.x && a.wg && a.wu && a.wd && a.y, NSA_ERR_ARG, "gated_mlp: NULL pointer");
  NSA_REQUIRE((a.p == nullptr) == (a.s == nullptr) && (a.p == nullptr) == (a.low == nullptr) && (a.p == nullptr) == (a.h == nullptr), NSA_ERR_ARG,
              "gated_mlp: give all of p, s, low and h or none");
  NSA_REQUIRE(aligned16(a.p) && aligned16(a.s) && aligned16(a.low) && aligned16(a.h), NSA_ERR_ARG, "gated_mlp: p, s, low and h must be 16-byte aligned");
  NSA_REQUIRE(on(2, a.x, a.wg, a.wu, a.wd, a.residual, a.y), NSA_ERR_ARG, "gated_mlp: a pointer is not aligned to its elements");
  return run_steps("gated_mlp", a, mlp_steps, st);
}

static int mlp_bwd_steps(const nsa_gated_mlp_bwd_args& a, Arena& w) {
  const long long ldh = padded(a.F, a.dtype);
  void *dg = w.take((long long)a.M * ldh * 2), *du = w.take((long long)a.M * ldh * 2);
  Mat dy, x, wg, wu, wd;
  NSA_TRY(operand(w, a.dy, a.M, a.N, a.dtype, &dy));
  NSA_TRY(operand(w, a.wd, a.N, a.F, a.dtype, &wd));
  GemmProblem p = problem(dy, 0, wd, 1, a.M, a.F, a.N, a.dtype);                            // dh = dy wd
  p.e.mode = EPI_GLU_BWD;
  p.e.i0 = a.p; p.e.i1 = a.s; p.e.i2 = a.low;
  p.e.y = dg; p.e.o1 = du;
  p.e.ldy = ldh; p.e.vec = p.e.vecy = 1;
  NSA_TRY(gemm(w, p));
  Products ps;
  if (a.dwg || a.dwu) NSA_TRY(operand(w, a.x, a.M, a.N, a.dtype, &x));
  if (a.dwg) ps.add(problem(Mat{dg, ldh}, 1, x, 1, a.F, a.N, a.M, a.dtype), a.dwg);
  if (a.dwu) ps.add(problem(Mat{du, ldh}, 1, x, 1, a.F, a.N, a.M, a.dtype), a.dwu);
  if (a.dwd) ps.add(problem(dy, 1, Mat{a.h, ldh}, 1, a.N, a.F, a.M, a.dtype), a.dwd);
  if (a.dx) {                                                                               // dx = dg wg + du wu
    NSA_TRY(operand(w, a.wg, a.F, a.N, a.dtype, &wg));
    NSA_TRY(operand(w, a.wu, a.F, a.N, a.dtype, &wu));
    GemmProblem q = problem(Mat{dg, ldh}, 0, wg, 1, a.M, a.N, a.F, a.dtype);
    q.A[1] = du; q.B[1] = wu.p;
    q.segments = 2;
    ps.add(q, a.dx);
  }
  return ps.run(w);
}

int gated_mlp_bwd(const nsa_gated_mlp_bwd_args& a, cudaStream_t st) {
  NSA_TRY(check_mlp(a.M, a.N, a.F, a.dtype, 0));
  if (a.M == 0) {
    const long long bytes = (long long)a.N * a.F * 2;
    NSA_TRY(zero(a.dwg, bytes, st));
    NSA_TRY(zero(a.dwu, bytes, st));
    return zero(a.dwd, bytes, st);
  }
  NSA_REQUIRE(a.dy && a.x && a.wg && a.wu && a.wd && a.p && a.s && a.low && a.h, NSA_ERR_ARG, "gated_mlp backward: NULL pointer");
  NSA_REQUIRE(aligned16(a.p) && aligned16(a.s) && aligned16(a.low) && aligned16(a.h), NSA_ERR_ARG, "gated_mlp backward: p, s, low and h must be 16-byte aligned");
  NSA_REQUIRE(on(2, a.dy, a.x, a.wg, a.wu, a.wd, a.dx, a.dwg, a.dwu, a.dwd), NSA_ERR_ARG, "gated_mlp backward: a pointer is not aligned to its elements");
  return run_steps("gated_mlp backward", a, mlp_bwd_steps, st);
}

int rms_norm(const nsa_norm_args&, cudaStream_t);
int rms_norm_bwd(const nsa_norm_bwd_args&, cudaStream_t);
long long rms_norm_bwd_ws_bytes(long long, int);
int quantize_rows(const void*, void*, float*, long long, int, int, int, cudaStream_t);
int rope_axes(const nsa_rope_axes_args&, cudaStream_t);

static bool is_real(int dt) { return is16(dt) || dt == NSA_FP32; }
static int bytes_of(int dt) { return dt == NSA_FP32 ? 4 : elem(dt); }

}  // namespace nsa

using namespace nsa;

extern "C" {

int nsa_rms_norm(const nsa_norm_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "rms_norm: NULL argument block");
  NSA_REQUIRE(a->rows >= 0 && a->rows < 2147483648LL && sized(a->hidden), NSA_ERR_ARG, "rms_norm: bad sizes rows=%lld hidden=%d", (long long)a->rows, a->hidden);
  NSA_REQUIRE(is_real(a->x_dtype), NSA_ERR_UNSUPPORTED, "rms_norm: x dtype %d", a->x_dtype);
  NSA_REQUIRE(a->w_dtype == a->x_dtype || a->w_dtype == NSA_FP32, NSA_ERR_UNSUPPORTED, "rms_norm: weight dtype %d beside x %d", a->w_dtype, a->x_dtype);
  NSA_REQUIRE(a->y_dtype == a->x_dtype || is8(a->y_dtype), NSA_ERR_UNSUPPORTED, "rms_norm: result dtype %d of x %d", a->y_dtype, a->x_dtype);
  NSA_REQUIRE(a->eps >= 0.f, NSA_ERR_ARG, "rms_norm: eps must not be negative");
  NSA_REQUIRE((a->residual == nullptr) == (a->h == nullptr), NSA_ERR_ARG, "rms_norm: residual and h must both be given or both be NULL");
  NSA_REQUIRE(a->residual == nullptr || a->res_dtype == a->x_dtype || a->res_dtype == NSA_FP32, NSA_ERR_UNSUPPORTED, "rms_norm: residual dtype %d beside x %d",
              a->res_dtype, a->x_dtype);
  if (a->rows == 0) return NSA_OK;
  NSA_REQUIRE(a->x && a->weight && a->y && (a->scale != nullptr || !is8(a->y_dtype)), NSA_ERR_ARG, "rms_norm: NULL pointer");
  NSA_REQUIRE(on(bytes_of(a->x_dtype), a->x) && on(bytes_of(a->y_dtype), a->y) && on(bytes_of(a->w_dtype), a->weight) &&
                  (a->residual == nullptr || on(bytes_of(a->res_dtype), a->residual, a->h)) && on(4, a->scale, a->rstd),
              NSA_ERR_ARG, "rms_norm: a pointer is not aligned to its elements");
  return rms_norm(*a, (cudaStream_t)stream);
}

int64_t nsa_rms_norm_bwd_ws_bytes(int64_t rows, int hidden) {
  NSA_REQUIRE(rows >= 0 && sized(hidden), NSA_ERR_ARG, "rms_norm backward: bad sizes rows=%lld hidden=%d", (long long)rows, hidden);
  return rms_norm_bwd_ws_bytes(rows, hidden);
}

int nsa_rms_norm_bwd(const nsa_norm_bwd_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "rms_norm backward: NULL argument block");
  NSA_REQUIRE(a->rows >= 0 && sized(a->hidden), NSA_ERR_ARG, "rms_norm backward: bad sizes rows=%lld hidden=%d", (long long)a->rows, a->hidden);
  NSA_REQUIRE(is_real(a->x_dtype) && (a->w_dtype == a->x_dtype || a->w_dtype == NSA_FP32) && (a->res_dtype == a->x_dtype || a->res_dtype == NSA_FP32),
              NSA_ERR_UNSUPPORTED, "rms_norm backward: dtypes %d/%d/%d", a->x_dtype, a->res_dtype, a->w_dtype);
  if (a->rows == 0) return zero(a->dweight, (long long)a->hidden * (a->w_dtype == NSA_FP32 ? 4 : 2), (cudaStream_t)stream);
  NSA_REQUIRE(a->dy && a->h && a->weight && a->rstd && a->dx && a->ws, NSA_ERR_ARG, "rms_norm backward: NULL pointer");
  const long long need = rms_norm_bwd_ws_bytes(a->rows, a->hidden);
  NSA_REQUIRE(a->ws_bytes >= need, NSA_ERR_ARG, "rms_norm backward: workspace of %lld bytes, %lld needed", (long long)a->ws_bytes, need);
  NSA_REQUIRE((reinterpret_cast<uintptr_t>(a->ws) & 255) == 0, NSA_ERR_ARG, "rms_norm backward: the workspace is not 256-byte aligned");
  NSA_REQUIRE(on(bytes_of(a->x_dtype), a->dy, a->dx) && on(bytes_of(a->res_dtype), a->dh, a->h, a->dres) && on(bytes_of(a->w_dtype), a->weight, a->dweight) && on(4, a->rstd),
              NSA_ERR_ARG, "rms_norm backward: a pointer is not aligned to its elements");
  return rms_norm_bwd(*a, (cudaStream_t)stream);
}

int nsa_quantize_rows_fp8(const void* x, void* q, float* scale, int64_t rows, int n, int x_dtype, int fmt, nsa_stream_t stream) {
  NSA_REQUIRE(rows >= 0 && rows < 2147483648LL && sized(n), NSA_ERR_ARG, "quantize_rows: bad sizes rows=%lld n=%d", (long long)rows, n);
  NSA_REQUIRE(is_real(x_dtype), NSA_ERR_UNSUPPORTED, "quantize_rows: dtype %d", x_dtype);
  NSA_REQUIRE(is8(fmt), NSA_ERR_ARG, "quantize_rows: format %d", fmt);
  if (rows == 0) return NSA_OK;
  NSA_REQUIRE(x && q && scale, NSA_ERR_ARG, "quantize_rows: NULL pointer");
  NSA_REQUIRE(on(bytes_of(x_dtype), x) && on(4, scale), NSA_ERR_ARG, "quantize_rows: a pointer is not aligned to its elements");
  return quantize_rows(x, q, scale, rows, n, x_dtype, fmt, (cudaStream_t)stream);
}

int nsa_rope_axes(const nsa_rope_axes_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "rope_axes: NULL argument block");
  NSA_REQUIRE(a->B >= 0 && (a->T == 0 || sized(a->T)) && a->H > 0 && a->Hkv > 0 && a->H + 2LL * a->Hkv < 65536, NSA_ERR_ARG, "rope_axes: bad sizes B=%d T=%d H=%d Hkv=%d", a->B, a->T,
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
  const int in = bytes_of(a->backward ? a->y_dtype : a->x_dtype), out = bytes_of(a->backward ? a->x_dtype : a->y_dtype);
  NSA_REQUIRE(on(in, a->q, a->k, a->v) && on(out, a->q_out, a->k_out, a->v_out) && on(a->pos64 ? 8 : 4, a->positions) && on(8, a->inv_freq), NSA_ERR_ARG,
              "rope_axes: a pointer is not aligned to its elements");
  return rope_axes(*a, (cudaStream_t)stream);
}

int64_t nsa_linear_ws_bytes(const nsa_linear_args* a) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "linear: NULL argument block");
  const int rc = check_linear(*a);
  return rc != NSA_OK ? rc : a->M == 0 ? 0 : ws_bytes(*a, linear_steps);
}
int nsa_linear(const nsa_linear_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "linear: NULL argument block");
  return linear(*a, (cudaStream_t)stream);
}
int64_t nsa_linear_bwd_ws_bytes(const nsa_linear_bwd_args* a) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "linear backward: NULL argument block");
  const int rc = check_linear_bwd(*a);
  return rc != NSA_OK ? rc : a->M == 0 ? 0 : ws_bytes(*a, linear_bwd_steps);
}
int nsa_linear_bwd(const nsa_linear_bwd_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "linear backward: NULL argument block");
  return linear_bwd(*a, (cudaStream_t)stream);
}
int64_t nsa_gated_mlp_ws_bytes(const nsa_gated_mlp_args* a) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "gated_mlp: NULL argument block");
  const int rc = check_mlp(a->M, a->N, a->F, a->dtype, a->act);
  return rc != NSA_OK ? rc : a->M == 0 ? 0 : ws_bytes(*a, mlp_steps);
}
int nsa_gated_mlp(const nsa_gated_mlp_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "gated_mlp: NULL argument block");
  return gated_mlp(*a, (cudaStream_t)stream);
}
int64_t nsa_gated_mlp_bwd_ws_bytes(const nsa_gated_mlp_bwd_args* a) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "gated_mlp backward: NULL argument block");
  const int rc = check_mlp(a->M, a->N, a->F, a->dtype, 0);
  return rc != NSA_OK ? rc : a->M == 0 ? 0 : ws_bytes(*a, mlp_bwd_steps);
}
int nsa_gated_mlp_bwd(const nsa_gated_mlp_bwd_args* a, nsa_stream_t stream) {
  NSA_REQUIRE(a, NSA_ERR_ARG, "gated_mlp backward: NULL argument block");
  return gated_mlp_bwd(*a, (cudaStream_t)stream);
}

}  // extern "C"
