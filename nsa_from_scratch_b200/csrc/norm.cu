// Root-mean-square norm behind the residual's addition, with a 16-bit, fp32 or fp8 result, and its backward pass.
//
//   h = round(x + residual)   (h = x without a residual; the stream is normed as it is stored)
//   r = 1 / sqrt(mean(h^2) + eps),  y = h * r * w
//   fp8 result: scale = max|y| / fmt_max per row (at least 1e-12 / fmt_max), q = round(y / scale)
//   backward:  n = h * r,  u = dy * w,  dx = r * (u - n * mean(u * n)) + dh,  dw = sum over rows of dy * n
//
// Bound by HBM.  A block owns a row: every element is read once, 16 bytes a load, and stays in registers (fp32) between
// the sum and the result.  V = vectors of 8 elements per thread.  Sums are fp32, formed in a fixed order.
// 16384 x 8192 bf16 with the residual and an fp8 result: 172 us = 5.5 TB/s (a plain copy reaches 6.5); 250 with one vector
// a thread, 173 with four, 178 with streaming loads and stores.  8189 x 4096 fp16: 46 us = 5.8 TB/s.
#include "gemm.cuh"
#include "tc5_ptx.cuh"

namespace nsa {

struct NormParams {
  const void *x, *res, *w;
  void *y, *h;
  float *scale, *rstd;
  long long rows;
  int N, wdt;               // wdt: the weight's type
  int fmt;                  // fp8 result: NSA_FP8_*
  float eps;
};

__device__ __forceinline__ float f8max(int fmt) { return fmt == NSA_FP8_E5M2 ? 57344.f : 448.f; }

template <typename T> __device__ __forceinline__ float get1(const T* p, long long i) {
  if constexpr (sizeof(T) == 4) return p[i];
  else return Elem<T>::to_f(p[i]);
}
template <typename T> __device__ __forceinline__ void put1(T* p, long long i, float v) {
  if constexpr (sizeof(T) == 4) p[i] = v;
  else p[i] = Elem<T>::from_f(v);
}
template <typename T> __device__ __forceinline__ float round_as(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else return Elem<T>::to_f(Elem<T>::from_f(v));
}
template <typename T> __device__ __forceinline__ void get8(const T* p, long long i, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p + i), b = *reinterpret_cast<const float4*>(p + i + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    load8<T>(p, i, 8, 1, v);
  }
}
template <typename T> __device__ __forceinline__ void put8(T* p, long long i, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p + i) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    store8<T>(p, i, 8, 1, v);
  }
}
__device__ __forceinline__ void weight8(const void* w, int dt, int i, float (&v)[8]) {
  if (dt == NSA_FP32) get8(reinterpret_cast<const float*>(w), i, v);
  else if (dt == NSA_FP16) get8(reinterpret_cast<const __half*>(w), i, v);
  else get8(reinterpret_cast<const __nv_bfloat16*>(w), i, v);
}
__device__ __forceinline__ float weight1(const void* w, int dt, int i) {
  if (dt == NSA_FP32) return reinterpret_cast<const float*>(w)[i];
  if (dt == NSA_FP16) return __half2float(reinterpret_cast<const __half*>(w)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
}

// Sum over the block in a fixed order, known to every thread.  `part` has a slot per warp and is not used again before
// the next __syncthreads.
__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < warps; ++i) s += part[i];
  return s;
}
// Largest magnitude over the block.  Magnitudes are compared as integers, where NaN is the largest: a row that holds one
// gets a NaN scale.
__device__ __forceinline__ float block_amax(uint32_t m, uint32_t* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const int warps = blockDim.x >> 5;
  if (warps > 1) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int i = 0; i < warps; ++i) m = max(m, part[i]);
  }
  return __uint_as_float(m);
}
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float row_scale(float amax, int fmt) { return (amax < 1e-12f ? 1e-12f : amax) / f8max(fmt); }
__device__ __forceinline__ uint8_t to_f8(float v, int fmt) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, fmt == NSA_FP8_E5M2 ? __NV_E5M2 : __NV_E4M3);
}
// v / s as it is rounded to fp8: the quotient, not a product with a rounded reciprocal, by which a y between two fp8 numbers to
// the last bit (the scale times a midpoint) would fall to either side.  1 / s is held in two numbers, its upper 24 bits cut off
// and what they leave: v / s = v inv + v rest, one rounding, off by 2^-47 (2^-30 for scales above 10^23, where rest is
// subnormal).  rest >= 0 keeps the sign of zeros.  Two at a time, since the instructions count: rows of 8192 bf16 quantised,
// 16384 of them, 72 us so and by the rounded reciprocal, 78 one at a time, 97 by __fdiv_rn.
struct Quotient {
  tc5::f32x2 inv, rest;
  __device__ __forceinline__ explicit Quotient(float s) {
    const float a = __frcp_rd(s), b = isinf(s) ? 0.f : fmaf(-s, a, 1.f) * a;     // over infinity: 0, and NaN for an infinite v
    inv = tc5::mk2(a, a);
    rest = tc5::mk2(b, b);
  }
  __device__ __forceinline__ float2 operator()(float v0, float v1) const {
    const tc5::f32x2 v = tc5::mk2(v0, v1);
    float2 q;
    tc5::un2(tc5::fma2(v, inv, tc5::mul2(v, rest)), q.x, q.y);
    return q;
  }
};
__device__ __forceinline__ uint32_t to_f8x4(const float* v, const Quotient& by, int fmt) {
  const __nv_fp8_interpretation_t k = fmt == NSA_FP8_E5M2 ? __NV_E5M2 : __NV_E4M3;
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(by(v[0], v[1]), __NV_SATFINITE, k);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(by(v[2], v[3]), __NV_SATFINITE, k);
  return lo | (hi << 16);
}

// X: type of x (and of a 16-bit or fp32 result); R: type of the residual stream; NORM 0: quantise the rows of x as they are
template <typename X, typename R, int V, bool OUT8, bool NORM>
__global__ void __launch_bounds__(V == 1 ? 128 : 512) rms_norm_kernel(const NormParams p) {
  __shared__ float part[32];
  __shared__ uint32_t mpart[32];
  const long long row = blockIdx.x;
  const long long base = row * p.N;
  const int vecs = p.N / 8, T = blockDim.x;
  float h[V][8];
  float ss = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = threadIdx.x + v * T;
    if (c < vecs) get8(reinterpret_cast<const X*>(p.x), base + c * 8, h[v]);
    else {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[v][i] = 0.f;
    }
  }
  if constexpr (NORM) {
    if (p.res != nullptr) {
      float r[V][8];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = threadIdx.x + v * T;
        if (c < vecs) get8(reinterpret_cast<const R*>(p.res), base + c * 8, r[v]);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = threadIdx.x + v * T;
        if (c < vecs) {
#pragma unroll
          for (int i = 0; i < 8; ++i) h[v][i] = round_as<R>(h[v][i] + r[v][i]);
          put8(reinterpret_cast<R*>(p.h), base + c * 8, h[v]);
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(h[v][i], h[v][i], ss);
    ss = block_sum(ss, part);
    const float r = rsqrtf(ss / (float)p.N + p.eps);
    if (p.rstd != nullptr && threadIdx.x == 0) p.rstd[row] = r;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = threadIdx.x + v * T;
      if (c < vecs) {
        float w[8];
        weight8(p.w, p.wdt, c * 8, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[v][i] = h[v][i] * r * w[i];
      }
    }
  }
  if constexpr (!OUT8) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = threadIdx.x + v * T;
      if (c < vecs) put8(reinterpret_cast<X*>(p.y), base + c * 8, h[v]);
    }
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, mag(h[v][i]));
    const float s = row_scale(block_amax(m, mpart), p.fmt);
    if (threadIdx.x == 0) p.scale[row] = s;
    const Quotient by(s);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = threadIdx.x + v * T;
      if (c < vecs)
        *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(p.y) + base + c * 8) = make_uint2(to_f8x4(h[v], by, p.fmt), to_f8x4(h[v] + 4, by, p.fmt));
    }
  }
}

// Any N and any alignment: the row is read again (from L2) instead of kept.
template <typename X, typename R, bool OUT8, bool NORM>
__global__ void __launch_bounds__(256) rms_norm_any_kernel(const NormParams p) {
  __shared__ float part[32];
  __shared__ uint32_t mpart[32];
  const long long row = blockIdx.x;
  const long long base = row * p.N;
  const X* x = reinterpret_cast<const X*>(p.x) + base;
  const bool stream = NORM && p.res != nullptr;
  float r = 1.f;
  if constexpr (NORM) {
    float ss = 0.f;
    for (int c = threadIdx.x; c < p.N; c += 256) {
      float v = get1(x, c);
      if (stream) {
        v = round_as<R>(v + get1(reinterpret_cast<const R*>(p.res), base + c));
        put1(reinterpret_cast<R*>(p.h), base + c, v);
      }
      ss = fmaf(v, v, ss);
    }
    ss = block_sum(ss, part);
    r = rsqrtf(ss / (float)p.N + p.eps);
    if (p.rstd != nullptr && threadIdx.x == 0) p.rstd[row] = r;
  }
  // every thread reads back what it wrote itself
  auto value = [&](int c) {
    const float v = stream ? get1(reinterpret_cast<const R*>(p.h), base + c) : get1(x, c);
    return NORM ? v * r * weight1(p.w, p.wdt, c) : v;
  };
  if constexpr (!OUT8) {
    for (int c = threadIdx.x; c < p.N; c += 256) put1(reinterpret_cast<X*>(p.y), base + c, value(c));
  } else {
    uint32_t m = 0;
    for (int c = threadIdx.x; c < p.N; c += 256) m = max(m, mag(value(c)));
    const float s = row_scale(block_amax(m, mpart), p.fmt);
    if (threadIdx.x == 0) p.scale[row] = s;
    const Quotient by(s);
    for (int c = threadIdx.x; c < p.N; c += 256) reinterpret_cast<uint8_t*>(p.y)[base + c] = to_f8(by(value(c), 0.f).x, p.fmt);
  }
}

// Threads of a row and vectors per thread: 1 vector up to 1024 columns (a short row still spreads over several warps),
// 2 up to 8192, else 4; more than 16384 columns go to the kernel that re-reads the row.
static int vectors_for(int N) { return N <= 1024 ? 1 : N <= 8192 ? 2 : 4; }
static int threads_for(int N, int V) { return N < 8 ? 32 : ((N / 8 + V - 1) / V + 31) / 32 * 32; }

template <typename X, typename R, bool OUT8, bool NORM>
static int norm_launch(const NormParams& p, cudaStream_t st) {
  const bool vec = p.N % 8 == 0 && p.N <= 16384 && aligned16(p.x) && aligned16(p.y) && aligned16(p.w) && aligned16(p.res) && aligned16(p.h);
  const unsigned grid = (unsigned)p.rows;
  if (!vec) rms_norm_any_kernel<X, R, OUT8, NORM><<<grid, 256, 0, st>>>(p);
  else {
    const int V = vectors_for(p.N), T = threads_for(p.N, V);
    if (V == 1) rms_norm_kernel<X, R, 1, OUT8, NORM><<<grid, T, 0, st>>>(p);
    else if (V == 2) rms_norm_kernel<X, R, 2, OUT8, NORM><<<grid, T, 0, st>>>(p);
    else rms_norm_kernel<X, R, 4, OUT8, NORM><<<grid, T, 0, st>>>(p);
  }
  return launch_status("rms_norm");
}
template <bool OUT8, bool NORM>
static int norm_types(const NormParams& p, int xdt, int rdt, cudaStream_t st) {
  const bool wide = NORM && p.res != nullptr && rdt == NSA_FP32;
  if (xdt == NSA_FP32) return norm_launch<float, float, OUT8, NORM>(p, st);
  if (xdt == NSA_FP16) {
    if constexpr (NORM) if (wide) return norm_launch<__half, float, OUT8, NORM>(p, st);
    return norm_launch<__half, __half, OUT8, NORM>(p, st);
  }
  if constexpr (NORM) if (wide) return norm_launch<__nv_bfloat16, float, OUT8, NORM>(p, st);
  return norm_launch<__nv_bfloat16, __nv_bfloat16, OUT8, NORM>(p, st);
}

int rms_norm(const nsa_norm_args& a, cudaStream_t st) {
  const bool out8 = a.y_dtype == NSA_FP8_E4M3 || a.y_dtype == NSA_FP8_E5M2;
  NormParams p{a.x, a.residual, a.weight, a.y, a.h, a.scale, a.rstd, a.rows, a.hidden, a.w_dtype, a.y_dtype, a.eps};
  return out8 ? norm_types<true, true>(p, a.x_dtype, a.res_dtype, st) : norm_types<false, true>(p, a.x_dtype, a.res_dtype, st);
}

int quantize_rows(const void* x, void* q, float* scale, long long rows, int N, int xdt, int fmt, cudaStream_t st) {
  NormParams p{x, nullptr, nullptr, q, nullptr, scale, nullptr, rows, N, NSA_FP32, fmt, 0.f};
  return norm_types<true, false>(p, xdt, xdt, st);
}

// ------------------------------------------------------------------ backward
struct NormBwdParams {
  const void *dy, *dh, *h, *w;
  const float* rstd;
  void *dx, *dres;          // dres: the same values in the residual's type, NULL where that is x's
  float* part;              // [blocks][N] partial sums of dw
  long long rows;
  int N, wdt;
};

// 8 elements as they are stored
template <typename T> struct Raw {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (sizeof(T) == 4) {
      const float* q = reinterpret_cast<const float*>(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = q[i];
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
#pragma unroll
      for (int i = 0; i < 4; ++i) { const float2 t = Elem<T>::unpack(w[i]); f[2 * i] = t.x; f[2 * i + 1] = t.y; }
    }
  }
};

// A block walks the rows b, b + grid, ...; its share of dw stays in registers and is written once.  A row stays as it was
// stored (raw) across the barrier of its sum and is unpacked twice: with 64 registers a thread, 1024 threads an SM, so
// that some rows are on their way while others are summed.  8189 x 4096 fp16 with dh: 49 us = 5.5 TB/s; 60 with the next row
// held in registers, 62 with a cp.async ring, 65 with two rows at a time.
template <typename X, typename R, int V, bool DH, int T_MAX>
__global__ void __launch_bounds__(T_MAX, 1024 / T_MAX) rms_norm_bwd_kernel(const NormBwdParams p) {
  __shared__ float part[2][32];
  const int vecs = p.N / 8, T = blockDim.x;
  float dw[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[v][i] = 0.f;
  const float inv_n = 1.f / (float)p.N;
  int turn = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const long long base = row * p.N;
    Raw<X> ry[V];
    Raw<R> rh[V], rd[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = threadIdx.x + v * T;
      if (c < vecs) {
        ry[v].load(reinterpret_cast<const X*>(p.dy) + base + c * 8);
        rh[v].load(reinterpret_cast<const R*>(p.h) + base + c * 8);
        if constexpr (DH) rd[v].load(reinterpret_cast<const R*>(p.dh) + base + c * 8);
      }
    }
    const float r = p.rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = threadIdx.x + v * T;
      if (c < vecs) {
        float u[8], n[8], w[8];
        weight8(p.w, p.wdt, c * 8, w);
        ry[v].get(u);
        rh[v].get(n);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          n[i] *= r;
          dw[v][i] = fmaf(u[i], n[i], dw[v][i]);
          dot = fmaf(u[i] * w[i], n[i], dot);
        }
      }
    }
    dot = block_sum(dot, part[turn]) * inv_n;               // two sets of slots: a row's are read while the next one's are written
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = threadIdx.x + v * T;
      if (c < vecs) {
        float u[8], n[8], w[8];
        weight8(p.w, p.wdt, c * 8, w);
        ry[v].get(u);
        rh[v].get(n);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = r * (u[i] * w[i] - n[i] * r * dot);
        if constexpr (DH) {
          rd[v].get(n);
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] += n[i];
        }
        put8(reinterpret_cast<X*>(p.dx), base + c * 8, u);
        if (p.dres != nullptr) put8(reinterpret_cast<R*>(p.dres), base + c * 8, u);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = threadIdx.x + v * T;
    if (c < vecs) put8(p.part, (long long)blockIdx.x * p.N + c * 8, dw[v]);
  }
}

// Any N and any alignment: dw accumulates in the block's own row of `part`.
template <typename X, typename R>
__global__ void __launch_bounds__(256) rms_norm_bwd_any_kernel(const NormBwdParams p) {
  __shared__ float part[2][32];
  float* dw = p.part + (long long)blockIdx.x * p.N;
  for (int c = threadIdx.x; c < p.N; c += 256) dw[c] = 0.f;
  int turn = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const long long base = row * p.N;
    const float r = p.rstd[row];
    const X* dy = reinterpret_cast<const X*>(p.dy) + base;
    const R* h = reinterpret_cast<const R*>(p.h) + base;
    float dot = 0.f;
    for (int c = threadIdx.x; c < p.N; c += 256) {
      const float d = get1(dy, c), n = get1(h, c) * r;
      dw[c] = fmaf(d, n, dw[c]);
      dot = fmaf(d * weight1(p.w, p.wdt, c), n, dot);
    }
    dot = block_sum(dot, part[turn]) / (float)p.N;
    for (int c = threadIdx.x; c < p.N; c += 256) {
      float g = r * (get1(dy, c) * weight1(p.w, p.wdt, c) - get1(h, c) * r * dot);
      if (p.dh != nullptr) g += get1(reinterpret_cast<const R*>(p.dh), base + c);
      put1(reinterpret_cast<X*>(p.dx), base + c, g);
      if (p.dres != nullptr) put1(reinterpret_cast<R*>(p.dres), base + c, g);
    }
  }
}

// out[c] = sum over `parts` rows of part[.][c]: 32 columns a block, 32 rows at a time, joined in a fixed order
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part, void* __restrict__ out, int parts, int N, int dt) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, g = threadIdx.x >> 5;
  float a[4] = {};
  if (c < N) {
    int r = g;
    for (; r + 96 < parts; r += 128)
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] += part[(long long)(r + 32 * i) * N + c];
    for (; r < parts; r += 32) a[0] += part[(long long)r * N + c];
  }
  s[g][lane] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  float v = s[lane][g];                                     // warp g: column g, a row group a lane
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int col = blockIdx.x * 32 + g;
  if (lane == 0 && col < N) {
    if (dt == NSA_FP32) reinterpret_cast<float*>(out)[col] = v;
    else if (dt == NSA_FP16) reinterpret_cast<__half*>(out)[col] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(out)[col] = __float2bfloat16_rn(v);
  }
}
int column_sum(const float* part, void* out, int parts, int N, int dt, cudaStream_t st) {
  column_sum_kernel<<<(N + 31) / 32, 1024, 0, st>>>(part, out, parts, N, dt);
  return launch_status("column_sum");
}

// Backward: 2 vectors a thread from 2048 columns on, 4 from 8200 on; blocks for 1024 threads an SM, and no more, since each
// leaves a row of partial sums.
static int bwd_vectors_for(int N) { return N < 2048 ? 1 : N <= 8192 ? 2 : 4; }
static int norm_bwd_blocks(long long rows, int N) {
  const int T = threads_for(N, bwd_vectors_for(N));
  const long long want = (long long)sm_count() * (T >= 512 ? 2 : 1024 / T);
  return (int)(rows < want ? rows : want);
}
long long rms_norm_bwd_ws_bytes(long long rows, int N) { return (long long)norm_bwd_blocks(rows, N) * N * 4; }

template <typename X, typename R, bool DH>
static int norm_bwd_launch(const NormBwdParams& p, int blocks, cudaStream_t st) {
  const bool vec = p.N % 8 == 0 && p.N <= 16384 && aligned16(p.dy) && aligned16(p.dh) && aligned16(p.h) && aligned16(p.w) && aligned16(p.dx) && aligned16(p.dres);
  if (!vec) rms_norm_bwd_any_kernel<X, R><<<blocks, 256, 0, st>>>(p);
  else {
    const int V = bwd_vectors_for(p.N), T = threads_for(p.N, V);
    if (V == 1) rms_norm_bwd_kernel<X, R, 1, DH, 256><<<blocks, T, 0, st>>>(p);
    else if (V == 2 && T <= 256) rms_norm_bwd_kernel<X, R, 2, DH, 256><<<blocks, T, 0, st>>>(p);
    else if (V == 2) rms_norm_bwd_kernel<X, R, 2, DH, 512><<<blocks, T, 0, st>>>(p);
    else rms_norm_bwd_kernel<X, R, 4, DH, 512><<<blocks, T, 0, st>>>(p);
  }
  return launch_status("rms_norm_bwd");
}
template <typename X, typename R>
static int norm_bwd_stream(const NormBwdParams& p, int blocks, cudaStream_t st) {
  return p.dh != nullptr ? norm_bwd_launch<X, R, true>(p, blocks, st) : norm_bwd_launch<X, R, false>(p, blocks, st);
}

int rms_norm_bwd(const nsa_norm_bwd_args& a, cudaStream_t st) {
  const int blocks = norm_bwd_blocks(a.rows, a.hidden);
  const bool wide = a.res_dtype == NSA_FP32;
  NormBwdParams p{a.dy, a.dh, a.h, a.weight, a.rstd, a.dx, a.dres, reinterpret_cast<float*>(a.ws), a.rows, a.hidden, a.w_dtype};
  int rc;
  if (a.x_dtype == NSA_FP32) rc = norm_bwd_stream<float, float>(p, blocks, st);
  else if (a.x_dtype == NSA_FP16) rc = wide ? norm_bwd_stream<__half, float>(p, blocks, st) : norm_bwd_stream<__half, __half>(p, blocks, st);
  else rc = wide ? norm_bwd_stream<__nv_bfloat16, float>(p, blocks, st) : norm_bwd_stream<__nv_bfloat16, __nv_bfloat16>(p, blocks, st);
  if (rc != NSA_OK || a.dweight == nullptr) return rc;
  return column_sum(p.part, a.dweight, blocks, a.hidden, a.w_dtype, st);
}

}  // namespace nsa
