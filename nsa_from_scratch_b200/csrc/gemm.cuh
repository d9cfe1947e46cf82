// What the matrix-product kernels of the layer share: the problem they are given, the activations, and the epilogue that
// turns fp32 sums into results, eight consecutive columns of a row at a time.
//
//   out[m,n] = epilogue( sum_k A[m,k] * B[n,k] )
//
// A and B are 16-bit (fp32 sums) or fp8 (e4m3 / e5m2, fp32 sums); each is stored with the contraction k along its rows
// ("k-major", [rows][k]) or down its columns ("mn-major", [k][rows]): x W^T, dy W and dy^T x are the same kernel.
// A contraction may come in two segments (A0 B0^T + A1 B1^T: the gradient that reaches x through gate and up).
#pragma once
#include "common.cuh"

namespace nsa {

enum { ACT_NONE = 0, ACT_SILU = 1, ACT_GELU_TANH = 2, ACT_RELU = 3 };
enum {
  EPI_LINEAR = 0,   // v = acc * xs[m] * ws[n] + bias[n]; o1 = act'(v) (optional, coded); y = act(v) + residual
  EPI_GLU = 1,      // two products g, u of the same A: y = act(g) * u; optional o1, o2, o3: act(g) and act'(g) * u in 24 bits
  EPI_GLU_BWD = 2   // acc = dh: y = dg = dh * act'(g) u, o1 = du = dh * act(g), from what the forward left (i0, i1, i2)
};

// p = act(z), d = act'(z).  Both activations go through s = 1 / (1 + 2^e), e negative multiples of their argument; 2^e
// overflows to infinity for large negative z, and s is then 0, as it should be.
//   silu: s = sigmoid(z), p = z s, d = s + p (1 - s)
//   gelu in its tanh form: 0.5 (1 + tanh(u)) = sigmoid(2 u), u = sqrt(2/pi) (z + 0.044715 z^3), so
//         s = sigmoid(2 u), p = z s, d = s + p (1 - s) 2 u'(z):  10 operations (through tanh: about 40)
__device__ __forceinline__ float rcp_f(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
constexpr float kGelu1 = 1.5957691216057308f;                 // 2 sqrt(2 / pi)
constexpr float kGelu3 = kGelu1 * 0.044715f;
template <int ACT> __device__ __forceinline__ float act_one(float z) {
  if (ACT == ACT_SILU) return z * rcp_f(1.f + ex2(z * -kLog2e));
  if (ACT == ACT_GELU_TANH) return z * rcp_f(1.f + ex2(z * fmaf(z * z, -kGelu3 * kLog2e, -kGelu1 * kLog2e)));
  if (ACT == ACT_RELU) return z < 0.f ? 0.f : z;              // a comparison that NaN fails keeps NaN
  return z;
}
template <int ACT> __device__ __forceinline__ void act_one_both(float z, float& p, float& d) {
  if (ACT == ACT_SILU) {
    const float s = rcp_f(1.f + ex2(z * -kLog2e));
    p = z * s;
    d = s + fmaf(-p, s, p);
  } else if (ACT == ACT_GELU_TANH) {
    const float q = fminf(z * z, 1e30f);                      // finite: times (1 - s) = 0 it has to vanish
    const float s = rcp_f(1.f + ex2(z * fmaf(q, -kGelu3 * kLog2e, -kGelu1 * kLog2e)));
    p = z * s;
    d = fmaf(fmaf(-p, s, p), fmaf(q, 3.f * kGelu3, kGelu1), s);
  } else if (ACT == ACT_RELU) {
    p = z < 0.f ? 0.f : z;
    d = z > 0.f ? 1.f : 0.f;
  } else {
    p = z;
    d = 1.f;
  }
}
// act' as the backward gets it: a signed 16-bit q with act' = q |q| 2^-28 (it lies in [-0.13, 1.13]).  Half a step of q is 2^-15,
// so act' is off by 2^-14 sqrt(|act'|): a quarter of an fp16 rounding where it is large, and still 2 % at 10^-5.  Rounded to
// x's own type it would add as much error to the gradients as the roundings that cannot be had without.  -32768, which no
// act' of a number needs, is NaN (a NaN argument; silu and gelu at infinite ones).
__device__ __forceinline__ uint32_t slope_code(float d) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(fabsf(d) * 268435456.f));
  return d != d ? 0x8000u : (uint32_t)(uint16_t)(int16_t)__float2int_rn(copysignf(r, d));
}
__device__ __forceinline__ float slope_value(uint32_t code) {
  const uint32_t c = code & 0xffffu;
  const float q = (float)(int16_t)(uint16_t)c;
  return c == 0x8000u ? __uint_as_float(0x7fc00000u) : q * fabsf(q) * 3.7252902984619140625e-9f;             // 2^-28
}

// What a gated pair leaves for the backward, p = act(g) and s = act'(g) u: fp32 rounded to its upper 24 bits (2^-16), the upper
// 16 in an array each, the next 8 of both in a third (p's in the lower byte).  Rounded to 16 bits they would add as much
// error to the gradients as the roundings that cannot be had without; in fp32 they would take 8 bytes instead of 6.
// Infinities stay what they are; NaN is set apart, because half a step on top of the NaN that the arithmetic yields, 0x7fffffff,
// would make it -0.
__device__ __forceinline__ uint32_t cut24(float v) { return v != v ? 0x7fc00000u : __float_as_uint(v) + 0x80u; }
__device__ __forceinline__ uint32_t low_bytes(uint32_t p, uint32_t s) { return ((p >> 8) & 0xffu) | (s & 0xff00u); }
__device__ __forceinline__ float join24_p(uint32_t hi, uint32_t low) { return __uint_as_float((hi << 16) | ((low & 0xffu) << 8)); }
__device__ __forceinline__ float join24_s(uint32_t hi, uint32_t low) { return __uint_as_float((hi << 16) | (low & 0xff00u)); }

// Several at a time: the choice is made once, so that their chains of exp and division run side by side (chosen element by
// element they ran one after the other: 111 against 93 us for the gated product of 8191 x 2816 x 1024).
template <int ACT, int R> __device__ __forceinline__ void act_as(float (&a)[R]) {
#pragma unroll
  for (int i = 0; i < R; ++i) a[i] = act_one<ACT>(a[i]);
}
template <int ACT, int R> __device__ __forceinline__ void act_both_as(float (&a)[R], float (&d)[R]) {
#pragma unroll
  for (int i = 0; i < R; ++i) act_one_both<ACT>(a[i], a[i], d[i]);
}
template <int R> __device__ __forceinline__ void act_all(float (&a)[R], int act) {
  if (act == ACT_SILU) act_as<ACT_SILU>(a);
  else if (act == ACT_GELU_TANH) act_as<ACT_GELU_TANH>(a);
  else if (act == ACT_RELU) act_as<ACT_RELU>(a);
}
// a = act(a), d = act'(a)
template <int R> __device__ __forceinline__ void act_all_both(float (&a)[R], float (&d)[R], int act) {
  if (act == ACT_SILU) act_both_as<ACT_SILU>(a, d);
  else if (act == ACT_GELU_TANH) act_both_as<ACT_GELU_TANH>(a, d);
  else if (act == ACT_RELU) act_both_as<ACT_RELU>(a, d);
  else act_both_as<ACT_NONE>(a, d);
}

struct Epi {
  int mode, act;
  int M, N;                      // results are [M][N]
  long long ldy;                 // elements between rows of y; in the gated modes of the o's and i's too.  The rest is dense
  int vec;                       // 1: N % 8 == 0 and every 16-bit pointer to a dense matrix is 16-byte aligned
  int vecy;                      // 1: the same of ldy and what it goes with; columns N..ldy-1 of a padded row are then written
  const void *bias, *residual;   // EPI_LINEAR; out type; NULL: none
  const float *xs, *ws;          // EPI_LINEAR: scales per row and per column of the sums; NULL: none
  const void *i0, *i1, *i2;      // EPI_GLU_BWD
  void *y, *o1, *o2, *o3;        // o1 (LINEAR), o1 to o3 (GLU): NULL: not wanted
};

// One product.  gemm_tc5: rows of A and B start on 16-byte boundaries.
struct GemmProblem {
  const void *A[2], *B[2];       // EPI_GLU: B[0], B[1] are the two weights (one segment)
  int segments;                  // 1 or 2
  int a_mn, b_mn;                // 1: stored [K][M] / [K][N]
  int M, N, K;                   // K: contraction length of each segment
  long long lda, ldb;            // elements between stored rows
  int dtype;                     // NSA_BF16, NSA_FP16, or an fp8 type of both operands
  int out_dtype;                 // NSA_BF16 or NSA_FP16
  Epi e;
};

template <typename T>
__device__ __forceinline__ void load8(const void* p, long long i, int n, int vec, float (&v)[8]) {
  const T* q = reinterpret_cast<const T*>(p) + i;
  if (vec) {
    const uint4 a = *reinterpret_cast<const uint4*>(q);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) { const float2 f = Elem<T>::unpack(w[e]); v[2 * e] = f.x; v[2 * e + 1] = f.y; }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? Elem<T>::to_f(q[e]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(void* p, long long i, int n, int vec, const float (&v)[8]) {
  T* q = reinterpret_cast<T*>(p) + i;
  if (vec) {
    *reinterpret_cast<uint4*>(q) = make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]), Elem<T>::pack(v[6], v[7]));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) q[e] = Elem<T>::from_f(v[e]);
  }
}

// Columns col..col+7 (those below N) of row `row`: a = fp32 sums, b = the second product's (EPI_GLU).  Everything is
// formed in fp32 and rounded once where it is stored.
template <typename T, int MODE>
__device__ __forceinline__ void epilogue8(const Epi& e, long long row, int col, float (&a)[8], const float (&b)[8]) {
  const int n = e.N - col;
  if (row >= e.M || n <= 0) return;
  const long long at = row * e.N + col, ay = row * e.ldy + col;
  float v[8];
  if constexpr (MODE == EPI_LINEAR) {
    if (e.xs != nullptr) {
      const float s = e.xs[row];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] *= i < n ? s * e.ws[col + i] : 0.f;
    }
    if (e.bias != nullptr) {
      load8<T>(e.bias, col, n, e.vec, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] += v[i];
    }
    if (e.o1 != nullptr) {
      act_all_both(a, v, e.act);
      uint16_t* q = reinterpret_cast<uint16_t*>(e.o1) + at;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = (uint16_t)slope_code(v[i]);
    } else {
      act_all(a, e.act);
    }
    if (e.residual != nullptr) {
      load8<T>(e.residual, at, n, e.vec, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] += v[i];
    }
  } else if constexpr (MODE == EPI_GLU) {
    if (e.o1 != nullptr) {
      act_all_both(a, v, e.act);
      uint16_t *op = reinterpret_cast<uint16_t*>(e.o1) + ay, *os = reinterpret_cast<uint16_t*>(e.o2) + ay, *ol = reinterpret_cast<uint16_t*>(e.o3) + ay;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) {
          const uint32_t cp = cut24(a[i]), cs = cut24(v[i] * b[i]);
          op[i] = (uint16_t)(cp >> 16);
          os[i] = (uint16_t)(cs >> 16);
          ol[i] = (uint16_t)low_bytes(cp, cs);
        }
    } else {
      act_all(a, e.act);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] *= b[i];
  } else {
    const uint16_t *ip = reinterpret_cast<const uint16_t*>(e.i0) + ay, *is = reinterpret_cast<const uint16_t*>(e.i1) + ay,
                   *il = reinterpret_cast<const uint16_t*>(e.i2) + ay;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = i < n ? a[i] * join24_p(ip[i], il[i]) : 0.f;
      a[i] = i < n ? a[i] * join24_s(is[i], il[i]) : 0.f;
    }
    store8<T>(e.o1, ay, n, e.vecy, v);
  }
  store8<T>(e.y, ay, n, e.vecy, a);
}

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int sm_count();                                                            // of the current device (linear.cu)
long long gemm_tc5_ws_bytes(const GemmProblem& p);                       // gemm_tc5.cu
int gemm_tc5(const GemmProblem& p, void* ws, cudaStream_t st);
bool gemm_skinny_takes(int M, int N, int K, int mode);                     // gemm_skinny.cu: k-major operands of any alignment
int gemm_skinny(const GemmProblem& p, bool early, cudaStream_t st);        // early: what runs before it in the stream does not write the weights
long long gemm_tc5_group_ws_bytes(const GemmProblem* p, int count);
int gemm_tc5_group(const GemmProblem* p, int count, void* ws, cudaStream_t st);
int column_sum(const float* part, void* out, int parts, int N, int dt, cudaStream_t st);   // norm.cu

}  // namespace nsa
