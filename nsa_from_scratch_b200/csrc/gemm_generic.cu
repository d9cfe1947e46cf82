// Matrix product for every size, pitch and alignment: mma.sync on 64 x 64 tiles, operands staged element by element.
//
// The tiles' loads are scalar (an odd contraction length leaves every second row of a 16-bit matrix off the 4-byte
// grid), so the staging, not the tensor pipe, sets the pace.  The aligned shapes go to the kernels beside it.
#include "gemm.cuh"

namespace nsa {

template <typename S> __device__ __forceinline__ float raw_to_f(S v);
template <> __device__ __forceinline__ float raw_to_f(__nv_fp8_e4m3 v) { return (float)v; }
template <> __device__ __forceinline__ float raw_to_f(__nv_fp8_e5m2 v) { return (float)v; }

constexpr int GBM = 64, GBN = 64, GBK = 32, GPITCH = GBK + 8, CPITCH = GBN + 4;

// S: stored type; T: the type the tensor cores multiply (fp8 values are exact in fp16); O: result type
template <typename S, typename T>
__device__ __forceinline__ void stage(T (*dst)[GPITCH], const S* __restrict__ src, long long ld, int mn, int r0, int rows, int k0, int K) {
  for (int i = threadIdx.x; i < GBM * GBK; i += 128) {
    const int r = mn ? i % GBM : i / GBK, k = mn ? i / GBM : i % GBK;
    T v = T(0.f);
    if (r0 + r < rows && k0 + k < K) {
      const S raw = mn ? src[(long long)(k0 + k) * ld + r0 + r] : src[(long long)(r0 + r) * ld + k0 + k];
      if constexpr (sizeof(S) == 1) v = Elem<T>::from_f(raw_to_f(raw));
      else v = raw;
    }
    dst[r][k] = v;
  }
}

template <typename S, typename T, typename O, int MODE>
__global__ void __launch_bounds__(128) gemm_generic_kernel(const GemmProblem p) {
  constexpr int NB = MODE == EPI_GLU ? 2 : 1;
  // the sums pass through the tiles' memory once the products are done
  __shared__ __align__(16) unsigned char raw[NB * GBM * CPITCH * 4];
  T (*As)[GPITCH] = reinterpret_cast<T (*)[GPITCH]>(raw);
  T (*Bs)[GBN][GPITCH] = reinterpret_cast<T (*)[GBN][GPITCH]>(raw + GBM * GPITCH * sizeof(T));
  float (*Cs)[GBM][CPITCH] = reinterpret_cast<float (*)[GBM][CPITCH]>(raw);
  static_assert((1 + NB) * GBM * GPITCH * sizeof(T) <= sizeof(raw), "tiles");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tiles_n = (p.N + GBN - 1) / GBN;
  const int m0 = (int)(blockIdx.x / tiles_n) * GBM, n0 = (int)(blockIdx.x % tiles_n) * GBN;
  const int wm = (warp >> 1) * 32, wn = (warp & 1) * 32;
  float acc[NB][2][4][4] = {};
  for (int s = 0; s < p.segments; ++s) {
    for (int k0 = 0; k0 < p.K; k0 += GBK) {
      stage<S, T>(As, reinterpret_cast<const S*>(p.A[s]), p.lda, p.a_mn, m0, p.M, k0, p.K);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) stage<S, T>(Bs[nb], reinterpret_cast<const S*>(p.B[s + nb]), p.ldb, p.b_mn, n0, p.N, k0, p.K);
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < GBK; kk += 16) {
        uint32_t a[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) ldsm_x4(a[i][0], a[i][1], a[i][2], a[i][3], smem_u32(&As[wm + i * 16 + (lane & 15)][kk + (lane >> 4) * 8]));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int j = 0; j < 2; ++j) {                    // 16 columns: two n8 tiles
            uint32_t b0, b1, b2, b3;
            ldsm_x4(b0, b1, b2, b3, smem_u32(&Bs[nb][wn + j * 16 + (lane & 7) + (lane >> 4) * 8][kk + ((lane >> 3) & 1) * 8]));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              mma16816<T>(acc[nb][i][2 * j], a[i], b0, b1);
              mma16816<T>(acc[nb][i][2 * j + 1], a[i], b2, b3);
            }
          }
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<float2*>(&Cs[nb][wm + i * 16 + (lane >> 2) + h * 8][wn + j * 8 + (lane & 3) * 2]) =
              make_float2(acc[nb][i][j][2 * h], acc[nb][i][j][2 * h + 1]);
  __syncthreads();
  for (int i = tid; i < GBM * GBN / 8; i += 128) {
    const int r = i / (GBN / 8), c = (i % (GBN / 8)) * 8;
    float a[8], b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { a[e] = Cs[0][r][c + e]; b[e] = Cs[NB - 1][r][c + e]; }
    epilogue8<O, MODE>(p.e, m0 + r, n0 + c, a, b);
  }
}

template <typename S, typename T, typename O>
static int launch(const GemmProblem& p, cudaStream_t st) {
  const long long tiles = (long long)((p.M + GBM - 1) / GBM) * ((p.N + GBN - 1) / GBN);
  NSA_REQUIRE(tiles < 2147483647LL, NSA_ERR_ARG, "matrix product: %d x %d results do not fit a grid", p.M, p.N);
  const dim3 grid((unsigned)tiles);
  if (p.e.mode == EPI_LINEAR) gemm_generic_kernel<S, T, O, EPI_LINEAR><<<grid, 128, 0, st>>>(p);
  else if constexpr (sizeof(S) == 2) {
    if (p.e.mode == EPI_GLU) gemm_generic_kernel<S, T, O, EPI_GLU><<<grid, 128, 0, st>>>(p);
    else gemm_generic_kernel<S, T, O, EPI_GLU_BWD><<<grid, 128, 0, st>>>(p);
  } else return fail(NSA_ERR_UNSUPPORTED, "matrix product: gated epilogues take 16-bit operands");
  return launch_status("gemm_generic");
}

int gemm_generic(const GemmProblem& p, cudaStream_t st) {
  if (p.dtype == NSA_BF16) return launch<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16>(p, st);
  if (p.dtype == NSA_FP16) return launch<__half, __half, __half>(p, st);
  if (p.dtype == NSA_FP8_E4M3)
    return p.out_dtype == NSA_BF16 ? launch<__nv_fp8_e4m3, __half, __nv_bfloat16>(p, st) : launch<__nv_fp8_e4m3, __half, __half>(p, st);
  return p.out_dtype == NSA_BF16 ? launch<__nv_fp8_e5m2, __half, __nv_bfloat16>(p, st) : launch<__nv_fp8_e5m2, __half, __half>(p, st);
}

}  // namespace nsa
