// Matrix product for a few rows (decoding): y [M,N] = epilogue(x [M,K] w [N,K]^T), M <= 32, operands of any alignment:
// 5.9 TB/s at 8 x 8192 x 8192 (23 us), 5.4 at a gated block of 4 x 4096 x 11008 (49 us for its two products).
//
// Bound by the weights' bytes: each is read once, 16 bytes a load, straight into the registers of mma.sync, whose 16-row
// operand is the weights and whose 8-column operand is the tokens (the 128 rows of a tcgen05 tile would be empty but for
// a few, and a tile's way through shared memory buys nothing where nothing is used twice).  A lane's 16 bytes are 8
// consecutive k of one row; the products take k in the order in which the lanes hold it, the same for both operands.
// A block owns 16 rows of w (of each of a gated pair); its warps deal out k among themselves and join their sums in a fixed order.  All blocks
// are resident at once where that is possible, so that no last round runs half empty.
#include "gemm.cuh"

namespace nsa {

struct SkinnyParams {
  const void* x;
  const void* w[2];
  Epi e;
  long long ldx;            // elements between rows of x
  int K;
  int early;                // the kernel before this one in the stream is known not to write w: read it before that has ended
};

// 16 bytes of a row from element k on, zeros behind its end
template <typename S, bool VEC>
__device__ __forceinline__ uint4 row16(const S* row, int k, int K) {
  constexpr int PER = 16 / sizeof(S);
  if constexpr (VEC) {
    if (k < K) return *reinterpret_cast<const uint4*>(row + k);          // K is a multiple of 16 bytes
    return make_uint4(0, 0, 0, 0);
  } else {
    __align__(16) S v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (k + i < K) v[i] = row[k + i];
      else memset(&v[i], 0, sizeof(S));
    }
    return *reinterpret_cast<const uint4*>(v);
  }
}
template <typename S, bool VEC>
__device__ __forceinline__ uint4 weight16(const S* row, int k, int K) {  // read once: not kept in L1
  if constexpr (VEC) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k < K) asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(row + k));
    return v;
  } else return row16<S, false>(row, k, K);
}
// the pair of k that product j of a 16-byte piece takes as half h (0: k, 1: k + 8 of the instruction), as 16-bit values
template <typename S>
__device__ __forceinline__ uint32_t pair_of(const uint4& v, int j, int h) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(S) == 2) return w[2 * j + h];
  else {
    const __nv_fp8x2_storage_t two = (__nv_fp8x2_storage_t)(w[j] >> (16 * h));
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(two, sizeof(S) == 1 && __is_same(S, __nv_fp8_e5m2) ? __NV_E5M2 : __NV_E4M3);
    return *reinterpret_cast<const uint32_t*>(&r);                       // exact
  }
}

// S: stored type, T: what is multiplied, O: result type; MT: tokens / 8; U: steps whose weights are under way together
template <typename S, typename T, typename O, int MODE, int MT, int WARPS, int U, bool VEC>
__global__ void __launch_bounds__(WARPS * 32) gemm_skinny_kernel(const SkinnyParams p) {
  constexpr int NB = MODE == EPI_GLU ? 2 : 1;
  constexpr int PER = 16 / sizeof(S), STEP = 4 * PER;                    // k of a lane, of a quad
  constexpr int MM = PER / 4;                                            // products per step
  __shared__ __align__(16) float part[WARPS][NB * 16][MT * 8 + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int n0 = blockIdx.x * 16;
  const S* wr[NB][2];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h) wr[b][h] = reinterpret_cast<const S*>(p.w[b]) + (long long)min(n0 + h * 8 + g, p.e.N - 1) * p.K + q * PER;
  const S* xr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xr[m] = reinterpret_cast<const S*>(p.x) + (long long)min(m * 8 + g, p.e.M - 1) * p.ldx + q * PER;
  float acc[NB][MT][4] = {};
  uint4 w[U][NB][2];
  auto fetch = [&](int k) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) w[u][b][h] = weight16<S, VEC>(wr[b][h], k + u * STEP, p.K - q * PER);
  };
  const int stride = WARPS * U * STEP;
  int k = warp * U * STEP;
  if (p.early) fetch(k);
  grid_dep_wait();
  grid_dep_launch();
  if (!p.early) fetch(k);
  for (; k < p.K; k += stride) {
    uint4 xv[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MT; ++m) xv[u][m] = row16<S, VEC>(xr[m], k + u * STEP, p.K - q * PER);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < MM; ++j) {
        uint32_t b0[MT], b1[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) { b0[m] = pair_of<S>(xv[u][m], j, 0); b1[m] = pair_of<S>(xv[u][m], j, 1); }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t a[4] = {pair_of<S>(w[u][b][0], j, 0), pair_of<S>(w[u][b][1], j, 0), pair_of<S>(w[u][b][0], j, 1), pair_of<S>(w[u][b][1], j, 1)};
#pragma unroll
          for (int m = 0; m < MT; ++m) mma16816<T>(acc[b][m], a, b0[m], b1[m]);
        }
      }
    if (k + stride < p.K) fetch(k + stride);
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[warp][b * 16 + g + (i >> 1) * 8][m * 8 + q * 2 + (i & 1)] = acc[b][m][i];
  __syncthreads();
  // 8 columns of one token a thread
  for (int i = threadIdx.x; i < MT * 16; i += WARPS * 32) {
    const int m = i / 2, c = (i % 2) * 8;
    if (m >= p.e.M) continue;
    float s[NB][8] = {};
    for (int v = 0; v < WARPS; ++v)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[b][e] += part[v][b * 16 + c + e][m];
    epilogue8<O, MODE>(p.e, m, n0 + c, s[0], s[NB - 1]);
  }
}

template <typename S, typename T, typename O, int MODE, int MT, int WARPS, int U>
static int launch(const SkinnyParams& p, bool vec, cudaStream_t st) {
  const dim3 grid((unsigned)((p.e.N + 15) / 16));
  if (vec) return launch_pdl("gemm_skinny", gemm_skinny_kernel<S, T, O, MODE, MT, WARPS, U, true>, grid, WARPS * 32, 0, st, p);
  return launch_pdl("gemm_skinny", gemm_skinny_kernel<S, T, O, MODE, MT, WARPS, U, false>, grid, WARPS * 32, 0, st, p);
}
// Warps a block and steps under way, by whether there are three blocks an SM (measured, bf16, us):
//   4 tokens: 8192 x 8192 22.8 with 4 warps of 4 steps (28.3 with 16 of 4, 26.3 with 16 of 2);  4096 x 11008 17.7 with 16 of 2
//   (22.9 with 4 of 4);  gated 11008 x 4096 33.0 with 4 of 2 (33.1 with 8 of 2, 38.2 with 16 of 1), 2816 x 1024 3.6 with 8 of 2
//   16 tokens: 8192 x 8192 27.1 with 8 of 2 (30.1 with 4 of 4);  4096 x 11008 19.2 with 16 of 2;  gated 36.3 with 4 of 2
template <typename S, typename T, typename O, int MODE>
static int shape(const SkinnyParams& p, bool vec, cudaStream_t st) {
  const bool many = (p.e.N + 15) / 16 >= 3 * sm_count();
  if constexpr (MODE == EPI_GLU) {
    if (p.e.M <= 8) return many ? launch<S, T, O, MODE, 1, 4, 2>(p, vec, st) : launch<S, T, O, MODE, 1, 8, 2>(p, vec, st);
    if (p.e.M <= 16) return many ? launch<S, T, O, MODE, 2, 4, 2>(p, vec, st) : launch<S, T, O, MODE, 2, 8, 2>(p, vec, st);
    return launch<S, T, O, MODE, 4, 4, 4>(p, vec, st);
  } else {
    if (p.e.M <= 8) return many ? launch<S, T, O, MODE, 1, 4, 4>(p, vec, st) : launch<S, T, O, MODE, 1, 16, 2>(p, vec, st);
    if (p.e.M <= 16) return many ? launch<S, T, O, MODE, 2, 8, 2>(p, vec, st) : launch<S, T, O, MODE, 2, 16, 2>(p, vec, st);
    return launch<S, T, O, MODE, 4, 8, 2>(p, vec, st);
  }
}

// From 17 tokens on the tiled kernel is faster, but for small weights, whose time is its set-up (32 tokens: 8192 x 8192 36
// against 52 us, 4096 x 4096 13 against 20, 1024 x 2816 9 against 10, 1152 x 1024 7.4 against 4.5), and for gated pairs up
// to 32 (11008 x 4096 60 against 46).
bool gemm_skinny_takes(int M, int N, int K, int mode) { return M <= 16 || (M <= 32 && (mode == EPI_GLU || (long long)N * K <= 2 << 20)); }

int gemm_skinny(const GemmProblem& q, bool early, cudaStream_t st) {
  SkinnyParams p;
  p.x = q.A[0];
  p.w[0] = q.B[0]; p.w[1] = q.B[1];
  p.e = q.e;
  p.ldx = q.lda;
  p.K = q.K;
  p.early = early;
  const int size = q.dtype == NSA_BF16 || q.dtype == NSA_FP16 ? 2 : 1;
  const bool vec = (long long)q.K * size % 16 == 0 && q.lda * size % 16 == 0 && aligned16(p.x) && aligned16(p.w[0]) && (q.e.mode != EPI_GLU || aligned16(p.w[1]));
  if (q.e.mode == EPI_GLU) {
    if (q.dtype == NSA_BF16) return shape<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16, EPI_GLU>(p, vec, st);
    return shape<__half, __half, __half, EPI_GLU>(p, vec, st);
  }
  if (q.dtype == NSA_BF16) return shape<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16, EPI_LINEAR>(p, vec, st);
  if (q.dtype == NSA_FP16) return shape<__half, __half, __half, EPI_LINEAR>(p, vec, st);
  const bool bf = q.out_dtype == NSA_BF16;
  if (q.dtype == NSA_FP8_E4M3)
    return bf ? shape<__nv_fp8_e4m3, __half, __nv_bfloat16, EPI_LINEAR>(p, vec, st) : shape<__nv_fp8_e4m3, __half, __half, EPI_LINEAR>(p, vec, st);
  return bf ? shape<__nv_fp8_e5m2, __half, __nv_bfloat16, EPI_LINEAR>(p, vec, st) : shape<__nv_fp8_e5m2, __half, __half, EPI_LINEAR>(p, vec, st);
}

}  // namespace nsa
