// Rotary embedding with several position axes, q, k and v in one launch:
//
//   frequency j of D/2 takes its position from axis a(j) (axis a owns sections[a] consecutive frequencies)
//   angle = positions[a(j), b, t] * inv_freq[j]
//   out[d] = x[d] cos - x[d + D/2] sin,  out[d + D/2] = x[d + D/2] cos + x[d] sin        (fp32, one rounding)
//
// forward: x [B,T,heads,D] (any batch and token pitch) -> [B,heads,T,D];  backward: the same with -angle, from
// [B,heads,T,D] to [B,T,heads,D].  v is only re-laid out.
//
// Bound by HBM: each element is read and written once.  The angle of a far position does not fit fp32 (position 10^6
// leaves 0.06 rad), so it is formed in fp64 as a number of turns and only its fraction goes on to fp32: one fp64
// product per (token, frequency), shared by all heads through shared memory.  32768 tokens, 72 heads of 128, bf16: 210 us =
// 5.75 TB/s (a plain copy reaches 6.5); one token of eight sequences: 4.1 us, a launch's latency.
#include "gemm.cuh"

namespace nsa {

constexpr int ROPE_THREADS = 256;

struct RopeParams {
  const void* x[3];
  void* y[3];
  long long xb[3], xt[3];             // pitch of batch and token on the token-major side (elements); heads are D apart
  const void* pos;
  const double* inv_freq;
  int B, T, D, heads[3];
  int n_axes, sec_end[8], pos64, vec;
  int tt;                             // tokens of a block: their rows of one head are a contiguous run of the head-major side
  int per_block;                      // heads of a block
};

template <typename T> __device__ __forceinline__ float r_get(const T* p) {
  if constexpr (sizeof(T) == 4) return *p;
  else return Elem<T>::to_f(*p);
}
template <typename T> __device__ __forceinline__ void r_put(T* p, float v) {
  if constexpr (sizeof(T) == 4) *p = v;
  else *p = Elem<T>::from_f(v);
}
template <typename T> __device__ __forceinline__ void r_get8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else load8<T>(p, 0, 8, 1, v);
}
template <typename T> __device__ __forceinline__ void r_put8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else store8<T>(p, 0, 8, 1, v);
}

// X: type read, Y: type written; BACK: head-major to token-major with the angle reversed; VEC: 16-byte rows.
// VEC: a thread owns 8 columns and their 8 partners of one token, keeps the 8 (cos, sin) in registers and walks the heads.
template <typename X, typename Y, bool BACK, bool VEC>
__global__ void __launch_bounds__(ROPE_THREADS) rope_axes_kernel(const RopeParams p) {
  extern __shared__ float2 cs[];                                   // [tt][D/2] (cos, sin)
  const int half = p.D / 2;
  const int tiles = (p.T + p.tt - 1) / p.tt;
  const int b = (int)(blockIdx.x / tiles), t0 = (int)(blockIdx.x % tiles) * p.tt;
  const int tn = min(p.tt, p.T - t0);
  const int all = p.heads[0] + p.heads[1] + p.heads[2], rotated = p.heads[0] + p.heads[1];
  const int h0 = blockIdx.y * p.per_block, h1 = min(all, h0 + p.per_block);
  auto angles = [&] {
    for (int i = threadIdx.x; i < tn * half; i += ROPE_THREADS) {
      const int t = i / half, j = i % half;
      int axis = 0;
      while (j >= p.sec_end[axis]) ++axis;                            // sec_end[n_axes - 1] == half
      const long long at = ((long long)axis * p.B + b) * p.T + t0 + t;
      const double pos = p.pos64 ? (double)reinterpret_cast<const long long*>(p.pos)[at] : (double)reinterpret_cast<const int*>(p.pos)[at];
      const double turns = pos * (p.inv_freq[j] * 0.15915494309189535);      // 1 / (2 pi)
      float s, c;
      sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
      cs[i] = make_float2(c, BACK ? -s : s);
    }
  };
  // where head h (of q, k and v in a row) and token t start on either side
  auto rows = [&](int h, int t, const X*& src, Y*& dst) {
    const int which = h < p.heads[0] ? 0 : (h < rotated ? 1 : 2);
    if (which > 0) h -= p.heads[0];
    if (which > 1) h -= p.heads[1];
    const long long tok = (long long)b * p.xb[which] + (long long)(t0 + t) * p.xt[which] + (long long)h * p.D;
    const long long hm = (((long long)b * p.heads[which] + h) * p.T + t0 + t) * p.D;
    src = reinterpret_cast<const X*>(p.x[which]) + (BACK ? hm : tok);
    dst = reinterpret_cast<Y*>(p.y[which]) + (BACK ? tok : hm);
  };
  if constexpr (VEC) {
    const int chunks = p.D / 16;
    const int ch = threadIdx.x % chunks, rest = threadIdx.x / chunks, t = rest % p.tt;
    const int step = ROPE_THREADS / chunks / p.tt;                    // heads side by side
    const bool mine = t < tn && rest / p.tt < step;
    float2 w[8];
    float lo[8], hi[8];
    const X* src;
    Y* dst;
    auto fetch = [&](int h) {
      if (!mine || h >= h1) return;
      rows(h, t, src, dst);
      r_get8(src + ch * 8, lo);
      r_get8(src + half + ch * 8, hi);
    };
    int h = h0 + rest / p.tt;
    fetch(h);                                                         // on its way while the angles are formed
    if (h0 < rotated) { angles(); __syncthreads(); }
    if (h0 < rotated && mine) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = cs[t * half + ch * 8 + e];
    }
    for (; mine && h < h1; h += step) {
      if (h < rotated) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = lo[e], c = hi[e];
          lo[e] = fmaf(a, w[e].x, -c * w[e].y);
          hi[e] = fmaf(c, w[e].x, a * w[e].y);
        }
      }
      r_put8(dst + ch * 8, lo);
      r_put8(dst + half + ch * 8, hi);
      fetch(h + step);
    }
  } else {
    if (h0 < rotated) { angles(); __syncthreads(); }
    const int per_head = tn * half;
    for (int i = threadIdx.x; i < (h1 - h0) * per_head; i += ROPE_THREADS) {
      const int h = h0 + i / per_head, r = i % per_head, t = r / half, ch = r % half;
      const X* src;
      Y* dst;
      rows(h, t, src, dst);
      const float a = r_get(src + ch), c = r_get(src + half + ch);
      const bool turn = h < rotated;
      const float2 w = turn ? cs[t * half + ch] : make_float2(1.f, 0.f);
      r_put(dst + ch, turn ? fmaf(a, w.x, -c * w.y) : a);
      r_put(dst + half + ch, turn ? fmaf(c, w.x, a * w.y) : c);
    }
  }
}

template <typename X, typename Y, bool BACK>
static int rope_launch(RopeParams& p, cudaStream_t st) {
  // Tokens of a block: a quarter of what its threads cover side by side, so that four heads are under way at a time (a power
  // of two, no more than there are).  Measured at 32768 tokens, 72 heads of 128: 214 us with 8 tokens, 222 with 32 (one
  // head), 246 with 2;  2 x 4001 tokens, 14 heads of 64: 13.0 with 16, 16.2 with 32.
  const int side = p.vec ? ROPE_THREADS / 4 / (p.D / 16) : 4;
  p.tt = 1;
  while (p.tt * 2 <= side && p.tt < p.T) p.tt *= 2;
  const long long tiles = (long long)p.B * ((p.T + p.tt - 1) / p.tt);
  NSA_REQUIRE(tiles < 2147483647LL, NSA_ERR_ARG, "rope_axes: %d x %d tokens do not fit a grid", p.B, p.T);
  const int all = p.heads[0] + p.heads[1] + p.heads[2];
  // few tokens: the heads are spread over blocks until every SM has two; a block's angles are formed anew in each
  long long ways = (2LL * sm_count() + tiles - 1) / tiles;
  if (ways > (all + 3) / 4) ways = (all + 3) / 4;
  p.per_block = (int)((all + ways - 1) / ways);
  const dim3 grid((unsigned)tiles, (unsigned)((all + p.per_block - 1) / p.per_block));
  const size_t smem = (size_t)p.tt * (p.D / 2) * sizeof(float2);
  if (p.vec) rope_axes_kernel<X, Y, BACK, true><<<grid, ROPE_THREADS, smem, st>>>(p);
  else rope_axes_kernel<X, Y, BACK, false><<<grid, ROPE_THREADS, smem, st>>>(p);
  return launch_status("rope_axes");
}

int rope_axes(const nsa_rope_axes_args& a, cudaStream_t st) {
  RopeParams p = {};
  const int xs = a.x_dtype == NSA_FP32 ? 4 : 2;
  const void* x[3] = {a.q, a.k, a.v};
  void* y[3] = {a.q_out, a.k_out, a.v_out};
  const long long xb[3] = {a.q_batch, a.k_batch, a.v_batch}, xt[3] = {a.q_token, a.k_token, a.v_token};
  p.heads[0] = a.H; p.heads[1] = p.heads[2] = a.Hkv;
  bool vec = a.D % 16 == 0;
  for (int i = 0; i < 3; ++i) {
    p.x[i] = x[i]; p.y[i] = y[i];
    if (a.backward) { p.xt[i] = (long long)p.heads[i] * a.D; p.xb[i] = p.xt[i] * a.T; }      // gradients are written dense
    else { p.xt[i] = xt[i]; p.xb[i] = xb[i]; }
    vec = vec && aligned16(x[i]) && aligned16(y[i]) && p.xt[i] * xs % 16 == 0 && p.xb[i] * xs % 16 == 0;
  }
  p.pos = a.positions; p.inv_freq = a.inv_freq;
  p.B = a.B; p.T = a.T; p.D = a.D; p.n_axes = a.n_axes; p.pos64 = a.pos64; p.vec = vec;
  int end = 0;
  for (int i = 0; i < a.n_axes; ++i) p.sec_end[i] = end += a.sections[i];
  if (!a.backward) {
    if (a.y_dtype == NSA_BF16) {
      if (a.x_dtype == NSA_FP32) return rope_launch<float, __nv_bfloat16, false>(p, st);
      if (a.x_dtype == NSA_FP16) return rope_launch<__half, __nv_bfloat16, false>(p, st);
      return rope_launch<__nv_bfloat16, __nv_bfloat16, false>(p, st);
    }
    if (a.x_dtype == NSA_FP32) return rope_launch<float, __half, false>(p, st);
    if (a.x_dtype == NSA_FP16) return rope_launch<__half, __half, false>(p, st);
    return rope_launch<__nv_bfloat16, __half, false>(p, st);
  }
  if (a.y_dtype == NSA_BF16) {
    if (a.x_dtype == NSA_FP32) return rope_launch<__nv_bfloat16, float, true>(p, st);
    if (a.x_dtype == NSA_FP16) return rope_launch<__nv_bfloat16, __half, true>(p, st);
    return rope_launch<__nv_bfloat16, __nv_bfloat16, true>(p, st);
  }
  if (a.x_dtype == NSA_FP32) return rope_launch<__half, float, true>(p, st);
  if (a.x_dtype == NSA_FP16) return rope_launch<__half, __half, true>(p, st);
  return rope_launch<__half, __nv_bfloat16, true>(p, st);
}

}  // namespace nsa
