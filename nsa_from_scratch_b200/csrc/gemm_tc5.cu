// Matrix product on the 5th-generation tensor cores; operand rows start on 16-byte boundaries (linear.cu pads others).
//
// Persistent and warp-specialised: warp 0 brings operand tiles with TMA (128-byte swizzle, zeros outside), warp 1 issues
// tcgen05.mma, warps 4-11 take the finished sums from TMEM, a thread to a row, and run the epilogue.  The sums are double
// buffered in TMEM, so a tile's epilogue runs under the next tile's products.  What the epilogue reads (residual, stored
// factors) and writes passes through shared memory by TMA, whole boxes at a time, read and overwritten in place: with loads
// and stores of its own and their bounds and alignment cases in the loop, a step of 32 x 32 results took 2000 clk, most of
// it fetching instructions.  Results whose rows are not 16-byte aligned leave as fp32 sums for gemm_join_kernel.
//
//   CG = 2: a pair of CTAs computes 256 x 256 results; each brings 128 rows of A and half of B's 256 rows, and the pair's
//           tensor cores read both halves: 32 KB a CTA and 64-deep step.  An SM receives 64 bytes a clk from L2, so that is
//           512 clk, where the products take 405 (measured: 405 while the ring is full, 510 in the long run).
//   CG = 1: one CTA computes 128 x 128 results: up to 128 rows.  The same 32 KB for half of the pair's share, so larger
//           problems stay on pairs however few tiles that leaves.
//
// A launch takes up to four products of the same kind (a layer's gradients): their tiles share the SMs' rounds.
//
// EPI_GLU computes both products in one tile: the B rows of a tile are BN/2 rows of each weight, so that g and u of a
// column stand BN/2 columns apart in the same TMEM lane.
//
// Measured: 8192 x 9216 x 8192 e4m3 404 us = 3.06 PFLOP/s (tensor pipe busy 90 %); the gated pair of 2048 x 11008 x 4096 bf16 235 us =
// 1.57 PFLOP/s (85 %) and of 8192 x 22016 x 8192 at the board's power limit, 1.39 PFLOP/s for the whole block; both gradients of
// 4001 x 4096 x 4096 in one launch 171 us = 1.57 PFLOP/s (86 %).  With a contraction of only 16 steps the results' way out shows: the
// gated pair of 8191 x 2816 x 1024 takes 64 us, and 88 (55 %) when it keeps its factors, the product that forms their gradients
// 64 (35 %).  Their epilogues end in time, but 128 KB of results (and 192 of factors) an SM and tile share L2 with 512 KB of
// operands, whose loads then stall; boxes of 64 instead of 32 columns and stores by the threads instead of TMA measure the same.
//
// Every wait is bounded; a wait that gives up raises the CTA's abort flag and the device status word, and the CTA still
// frees its TMEM.
#include "gemm.cuh"
#include "tc5_ptx.cuh"

#include <cudaTypedefs.h>

namespace nsa {

using namespace tc5;

__device__ int g_gemm_status;

// ---------------------------------------------------------------- CTA pairs
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// relaxed: what it announces is that TMEM was read, which the tcgen05 fences order
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_addr) : "memory");
}
// shared memory -> global, tracked by the issuing thread's bulk groups; what lies outside the tensor is not written
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\n" ::"l"(map), "r"(src), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];\n" ::"l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void group_sync(int id) { asm volatile("bar.sync %0, 128;\n" ::"r"(id) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// `bar` is a shared::cluster address: with CG = 2 the pair's first CTA counts the bytes of both
template <int CG>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  if constexpr (CG == 2)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
template <int CG> __device__ __forceinline__ void tm_alloc(uint32_t smem_dst, uint32_t ncols) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_dst), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  } else {
    tmem_alloc(smem_dst, ncols);
    tmem_relinquish();
  }
}
template <int CG> __device__ __forceinline__ void tm_dealloc(uint32_t taddr, uint32_t ncols) {
  if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(ncols) : "memory");
  else tmem_dealloc(taddr, ncols);
}
// one arrival on `bar` (of both CTAs of a pair: `first` is the rank of its first) when every product issued so far is done
template <int CG> __device__ __forceinline__ void commit(uint32_t bar, uint32_t first = 0) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar), "h"((uint16_t)(3u << first)) : "memory");
  else tc_commit(bar);
}
template <int CG, bool F8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define NSA_MMA(G, K)                                                                                                        \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::" G ".kind::" K " [%0], %1, %2, %3, p;\n\t}\n" \
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory")
  if constexpr (CG == 2) { if constexpr (F8) NSA_MMA("2", "f8f6f4"); else NSA_MMA("2", "f16"); }
  else { if constexpr (F8) NSA_MMA("1", "f8f6f4"); else NSA_MMA("1", "f16"); }
#undef NSA_MMA
}

// ---------------------------------------------------------------- 16 columns of a row
// Until here the loads behind v (and u) may still be under way: naming the registers keeps their uses behind the wait.
__device__ __forceinline__ void wait_loaded(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
                 "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :: "memory");
}
template <typename T> __device__ __forceinline__ void put16(uint32_t p0, uint32_t p1, const float (&a)[16]) {
  sts128(p0, make_uint4(Elem<T>::pack(a[0], a[1]), Elem<T>::pack(a[2], a[3]), Elem<T>::pack(a[4], a[5]), Elem<T>::pack(a[6], a[7])));
  sts128(p1, make_uint4(Elem<T>::pack(a[8], a[9]), Elem<T>::pack(a[10], a[11]), Elem<T>::pack(a[12], a[13]), Elem<T>::pack(a[14], a[15])));
}
template <typename T> __device__ __forceinline__ void add8(float* a, const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) { const float2 f = Elem<T>::unpack(w[j]); a[2 * j] += f.x; a[2 * j + 1] += f.y; }
}

// ---------------------------------------------------------------- kernel
struct TcProduct {
  CUtensorMap tmA[2], tmB[2], tmY;
  int M, N;
  int tiles_m, tiles_n, first;                  // first: number of its first tile
  int ksteps, segments;                         // 128-byte steps of one segment
  int a_mn, b_mn;
};
constexpr int TC_PRODUCTS = 4;
struct GemmTcParams {
  TcProduct pr[TC_PRODUCTS];
  CUtensorMap tmO1, tmO2, tmO3, tmI0, tmI1, tmI2;   // further results and inputs of the epilogue (I0: residual in EPI_LINEAR); one product
  Epi e;
  CUtensorMap tmPart;                           // PARTIAL: [splits][products of a pair][M][N] fp32 sums; one product
  int products, tiles;                          // tiles: of all products and splits
  int splits, per_split;                        // the steps of all segments, dealt out to `splits` tiles
};

// EPI_SLOPE: EPI_LINEAR that also writes act', coded (e.o1).  EPI_PARTIAL, EPI_PARTIAL2: raw sums of one product, of a gated pair,
// for the joining kernel.
constexpr int EPI_SLOPE = 3, EPI_PARTIAL = 4, EPI_PARTIAL2 = 5;

template <int MODE, int CG, int BN> struct TcShape {
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BN / CG * 128;
  // bytes of each of the two epilogue groups (EPI_GLU_BWD: two stages of three boxes), and stages of the operands' ring
  static constexpr int EPI_BYTES = MODE == EPI_GLU_BWD ? 49152 : 32768, STAGES = (229376 - 2 * EPI_BYTES) / (A_BYTES + B_BYTES);
  static constexpr int SMEM = STAGES * (A_BYTES + B_BYTES) + 2 * EPI_BYTES + 1024;
};

// F: 0 fp16, 1 bf16, 2 e4m3, 3 e5m2;  T: result type
template <int F, typename T, int MODE, int CG, int BN>
__global__ void __launch_bounds__(384, 1) gemm_tc5_kernel(const __grid_constant__ GemmTcParams p) {
  using S = TcShape<MODE, CG, BN>;
  constexpr bool F8 = F >= 2;
  constexpr int KE = F8 ? 128 : 64;                                  // elements of a 128-byte step
  constexpr bool PAIR = MODE == EPI_GLU || MODE == EPI_PARTIAL2;     // two products a tile
  constexpr int NW = PAIR ? BN / 2 : BN;                             // result columns of a tile
  constexpr int BROWS = BN / CG;                                     // B rows that this CTA brings
  constexpr uint32_t IDESC = idesc_f16(F8 ? F - 2 : F, 128 * CG, BN, 0, 0);

  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s_tiles = smem_u32(smem);
  __shared__ __align__(8) uint64_t full[S::STAGES], empty[S::STAGES], tfull[2], tempty[2], loaded[2][2];
  __shared__ uint32_t tmem_s;
  __shared__ int abort_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const int unit = blockIdx.x / CG, units = gridDim.x / CG;

  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < S::STAGES; ++i) { mbar_init(smem_u32(&full[i]), 1); mbar_init(smem_u32(&empty[i]), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&tfull[i]), 1); mbar_init(smem_u32(&tempty[i]), 8 * CG); }
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&loaded[i >> 1][i & 1]), 1);
    fence_barrier_init();
  }
  if (warp == 2) tm_alloc<CG>(smem_u32(&tmem_s), 2 * BN);
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  int fail_id = 0;
  grid_dep_launch();                                                     // the next product's CTAs may set themselves up as these leave
  grid_dep_wait();

  // tile t: whose it is, which split of the contraction, which rows and columns (8 tile rows walk the columns together: their
  // B tiles meet in L2)
  struct Place { const TcProduct* pr; int m0, n0, k0, k1, split; };
  auto place = [&](int t) {
    Place w;
    int i = 0;
    while (i + 1 < p.products && t >= p.pr[i + 1].first) ++i;
    w.pr = &p.pr[i];
    t -= w.pr->first;
    const int mn = w.pr->tiles_m * w.pr->tiles_n;
    w.split = t / mn;
    t -= w.split * mn;
    const int group = 8 * w.pr->tiles_n, g = t / group, first = g * 8, rows = min(8, w.pr->tiles_m - first);
    t -= g * group;
    w.m0 = (first + t % rows) * 128 * CG;
    w.n0 = t / rows * NW;
    const int steps = w.pr->ksteps * w.pr->segments;
    w.k0 = w.split * p.per_split;
    w.k1 = p.splits == 1 ? steps : min(steps, w.k0 + p.per_split);
    return w;
  };

  if (warp == 0) {
    // =============================== TMA producer ===============================
    const bool leader = elect_one();
    if (leader) {
      for (int i = 0; i < p.products; ++i) {
        tma_prefetch_desc(&p.pr[i].tmA[0]);
        tma_prefetch_desc(&p.pr[i].tmB[0]);
        if (p.pr[i].segments == 2) { tma_prefetch_desc(&p.pr[i].tmA[1]); tma_prefetch_desc(&p.pr[i].tmB[1]); }
      }
      if constexpr (PAIR) tma_prefetch_desc(&p.pr[0].tmB[1]);
    }
    __syncwarp();
    int it = 0;
    bool ok = true;
    for (int t = unit; t < p.tiles && ok; t += units) {
      const Place w = place(t);
      const int a_mn = w.pr->a_mn, b_mn = w.pr->b_mn, ksteps = w.pr->ksteps, ma = w.m0 + (int)rank * 128, nb = w.n0 + (int)rank * BROWS;
      for (int k = w.k0; k < w.k1; ++k, ++it) {
        const int s = it % S::STAGES, ph = (it / S::STAGES) & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[s]), ph ^ 1, &abort_flag));
        if (!ok) { fail_id = 1; break; }
        if (leader) {
          uint32_t bar = smem_u32(&full[s]);
          if (rank == 0) mbar_expect_tx(bar, CG * (S::A_BYTES + S::B_BYTES));
          if constexpr (CG == 2) bar = map_to_rank(bar, 0);
          const int seg = k >= ksteps, kc = (k - seg * ksteps) * KE;
          const uint32_t da = s_tiles + s * (S::A_BYTES + S::B_BYTES), db = da + S::A_BYTES;
          const CUtensorMap *ta = &w.pr->tmA[seg], *tb = &w.pr->tmB[seg];
          if (!F8 && a_mn) {
            tma_load_2d<CG>(da, ta, bar, ma, kc);
            tma_load_2d<CG>(da + 8192, ta, bar, ma + 64, kc);
          } else {
            tma_load_2d<CG>(da, ta, bar, kc, ma);
          }
          if constexpr (PAIR) {
            if constexpr (CG == 2) tma_load_2d<CG>(db, &w.pr->tmB[rank], bar, kc, w.n0);
            else { tma_load_2d<CG>(db, &w.pr->tmB[0], bar, kc, w.n0); tma_load_2d<CG>(db + S::B_BYTES / 2, &w.pr->tmB[1], bar, kc, w.n0); }
          } else if (!F8 && b_mn) {
#pragma unroll
            for (int c = 0; c < BROWS / 64; ++c) tma_load_2d<CG>(db + c * 8192, tb, bar, nb + c * 64, kc);
          } else {
            tma_load_2d<CG>(db, tb, bar, kc, nb);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // =============================== MMA issuer (the pair's first CTA) ===============================
    if (rank == 0) {
      const bool leader = elect_one();
      int it = 0, n = 0;
      bool ok = true;
      for (int t = unit; t < p.tiles && ok; t += units, ++n) {
        const Place w = place(t);
        const int a_mn = F8 ? 0 : w.pr->a_mn, b_mn = F8 ? 0 : w.pr->b_mn;
        const uint32_t idesc = IDESC | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16);
        const int sa = a_mn ? 128 : 2, sb = b_mn ? 128 : 2;               // from one 32-byte (or 16-row) slice of a step to the next
        const int buf = n & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&tempty[buf]), ((n >> 1) & 1) ^ 1, &abort_flag));
        if (!ok) { fail_id = 2; break; }
        tc_fence_after();
        const uint32_t acc = tmem + buf * BN;
        for (int k = w.k0; k < w.k1; ++k, ++it) {
          const int s = it % S::STAGES, ph = (it / S::STAGES) & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[s]), ph, &abort_flag));
          if (!ok) { fail_id = 3; break; }
          tc_fence_after();
          if (leader) {
            const uint32_t da = s_tiles + s * (S::A_BYTES + S::B_BYTES);
            const uint64_t a = smem_desc_sw128(da, a_mn ? 8192 : 16, 1024), b = smem_desc_sw128(da + S::A_BYTES, b_mn ? 8192 : 16, 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i) mma<CG, F8>(acc, a + i * sa, b + i * sb, idesc, (k > w.k0 || i > 0) ? 1u : 0u);
            commit<CG>(smem_u32(&empty[s]));
          }
          __syncwarp();
        }
        if (!ok) break;
        if (leader) commit<CG>(smem_u32(&tfull[buf]));
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    // =============================== epilogue ===============================
    // Two groups of four warps, each with half of the tile's columns; a thread owns a row (a TMEM lane).  A group works in
    // chunks of CW columns, 16 columns of sums at a time.  Its 32 KB of shared memory hold, per chunk and stage, a box of
    // 128 rows of each tensor that is read or written; inputs are requested a chunk or two ahead, results overwrite them.
    // A wait that gave up ends the work but not the barriers that the group's warps share.
    const int quarter = warp & 3, group = (warp - 4) >> 2;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const bool lead = quarter == 0 && lane == 0;
    constexpr bool RAW = MODE == EPI_PARTIAL || MODE == EPI_PARTIAL2;
    constexpr int GW = NW / 2;                                           // columns of the group
    constexpr int CW = MODE == EPI_LINEAR ? 64 : 32;                     // columns of a chunk
    constexpr int NC = GW / CW;
    constexpr int BOX = 128 * CW * (RAW ? 4 : 2);                        // bytes of a box: 128 rows of CW columns
    constexpr int STAGE = MODE == EPI_GLU ? 0 : S::EPI_BYTES / 2;        // between the two stages (EPI_GLU: one stage of four boxes)
    const uint32_t stage0 = s_tiles + S::STAGES * (S::A_BYTES + S::B_BYTES) + group * S::EPI_BYTES;
    constexpr bool LIN = MODE == EPI_LINEAR || MODE == EPI_SLOPE;
    const bool inputs = MODE == EPI_GLU_BWD || (LIN && p.e.residual != nullptr);
    // 16-byte piece j of this thread's row in a box
    auto piece = [&](uint32_t box, int j) { return CW == 64 ? box + row * 128 + ((j ^ (row & 7)) << 4) : box + row * 64 + ((j ^ ((row >> 1) & 3)) << 4); };
    int n = 0, cnt = 0;                                                  // tiles and chunks so far
    bool ok = true;
    for (int t = unit; t < p.tiles; t += units, ++n) {
      const Place w = place(t);
      const int buf = n & 1;
      const int M = w.pr->M, N = w.pr->N;
      const int mr = w.m0 + (int)rank * 128, nc0 = w.n0 + group * GW;
      auto request = [&](int c, int count) {                             // lead only: the inputs of chunk c of this tile
        const int st = count & 1;
        const uint32_t bar = smem_u32(&loaded[group][st]), box = stage0 + st * STAGE;
        mbar_expect_tx(bar, MODE == EPI_GLU_BWD ? 3 * BOX : BOX);
        tma_load_2d<1>(box, &p.tmI0, bar, nc0 + c * CW, mr);
        if constexpr (MODE == EPI_GLU_BWD) {
          tma_load_2d<1>(box + BOX, &p.tmI1, bar, nc0 + c * CW, mr);
          tma_load_2d<1>(box + 2 * BOX, &p.tmI2, bar, nc0 + c * CW, mr);
        }
      };
      if (inputs && lead) {
        bulk_wait_read<0>();
        request(0, cnt);
        if (NC > 1) request(1, cnt + 1);
      }
      if (ok) ok = mbar_wait(smem_u32(&tfull[buf]), (n >> 1) & 1, &abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) fail_id = 4;
      tc_fence_after();
      const uint32_t acc = tmem + lanes + buf * BN + group * GW;
      const int grow = mr + row;
      float xs = 1.f;
      if constexpr (LIN) { if (p.e.xs != nullptr && grow < M) xs = p.e.xs[grow]; }
      auto drained = [&] {                                               // the last sums are in registers: the buffer may be filled again
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2) arrive_remote(map_to_rank(smem_u32(&tempty[buf]), 0));
          else mbar_arrive(smem_u32(&tempty[buf]));
        }
      };
      if constexpr (RAW) {
        constexpr int PR = PAIR ? 2 : 1;
#pragma unroll 1
        for (int c = 0; c < NC * PR; ++c, ++cnt) {
          const uint32_t box = stage0 + (cnt & 1) * STAGE;
          const int q = PAIR ? c / NC : 0, col = (PAIR ? c % NC : c) * CW;
          if (lead) bulk_wait_read<1>();
          group_sync(1 + group);
          uint32_t v[32];
          tmem_ld32(acc + q * NW + col, v);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) sts128(box + row * 128 + ((i ^ (row & 7)) << 4), make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
          if (c == NC * PR - 1) drained();
          fence_proxy_async();
          group_sync(1 + group);
          if (lead && ok) {
            tma_store_3d(&p.tmPart, box, nc0 + col, mr, w.split * PR + q);
            bulk_commit();
          }
        }
      } else {
        // the next 16 columns leave TMEM while these are worked on
        uint32_t v[16], u[MODE == EPI_GLU ? 16 : 1];
        auto load = [&](int col) {
          tmem_ld16(acc + col, v);
          if constexpr (MODE == EPI_GLU) tmem_ld16(acc + NW + col, u);
        };
        load(0);
#pragma unroll 1
        for (int c = 0; c < NC; ++c, ++cnt) {
          const int st = cnt & 1;
          const uint32_t box = stage0 + st * STAGE;
          if (inputs) {
            if (ok) ok = mbar_wait(smem_u32(&loaded[group][st]), (cnt >> 1) & 1, &abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) fail_id = 5;
          } else {
            if (lead) { if constexpr (MODE == EPI_GLU) bulk_wait_read<0>(); else bulk_wait_read<1>(); }
            group_sync(1 + group);                                       // the boxes that are about to be written have left
          }
#pragma unroll 1
          for (int h = 0; h < CW / 16; ++h) {
            const int col = c * CW + h * 16;
            float a[16], b[MODE == EPI_GLU ? 16 : 1];
            const uint32_t p0 = piece(box, 2 * h), p1 = piece(box, 2 * h + 1);
            const int gc = nc0 + col;                                    // columns come in eights: N is a multiple of 8
            uint4 bias[2] = {}, res[2] = {};                             // asked for ahead of the sums
            if constexpr (LIN) {
              if (p.e.bias != nullptr) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                  if (gc + 8 * i < N) bias[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.e.bias) + gc + 8 * i);
              }
              if (p.e.residual != nullptr) { res[0] = lds128(p0); res[1] = lds128(p1); }
            }
            wait_loaded(v);
            if constexpr (MODE == EPI_GLU) wait_loaded(u);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              a[i] = __uint_as_float(v[i]);
              if constexpr (MODE == EPI_GLU) b[i] = __uint_as_float(u[i]);
            }
            if (col + 16 < GW) load(col + 16);
            if constexpr (MODE == EPI_GLU) {
              if (p.e.o1 != nullptr) {
                float d[16];
                act_all_both(a, d, p.e.act);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  uint32_t hp[4], hs[4], lo[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const int k = 8 * j + 2 * i;
                    const uint32_t p0 = cut24(a[k]), p1 = cut24(a[k + 1]), s0 = cut24(d[k] * b[k]), s1 = cut24(d[k + 1] * b[k + 1]);
                    hp[i] = __byte_perm(p0, p1, 0x7632);
                    hs[i] = __byte_perm(s0, s1, 0x7632);
                    lo[i] = __byte_perm(__byte_perm(p0, s0, 0x0051), __byte_perm(p1, s1, 0x0051), 0x5410);
                  }
                  sts128(piece(box + BOX, 2 * h + j), make_uint4(hp[0], hp[1], hp[2], hp[3]));
                  sts128(piece(box + 2 * BOX, 2 * h + j), make_uint4(hs[0], hs[1], hs[2], hs[3]));
                  sts128(piece(box + 3 * BOX, 2 * h + j), make_uint4(lo[0], lo[1], lo[2], lo[3]));
                }
              } else {
                act_all(a, p.e.act);
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) a[i] *= b[i];
            }
            if constexpr (LIN) {
              if (p.e.xs != nullptr) {
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                  if (gc + i < N) {
                    const float4 f = *reinterpret_cast<const float4*>(p.e.ws + gc + i);
                    a[i] *= xs * f.x; a[i + 1] *= xs * f.y; a[i + 2] *= xs * f.z; a[i + 3] *= xs * f.w;
                  }
              }
              if (p.e.bias != nullptr) { add8<T>(a, bias[0]); add8<T>(a + 8, bias[1]); }
              if constexpr (MODE == EPI_SLOPE) {
                float d[16];
                act_all_both(a, d, p.e.act);
                uint32_t q[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = slope_code(d[2 * i]) | (slope_code(d[2 * i + 1]) << 16);
                sts128(piece(box + BOX, 2 * h), make_uint4(q[0], q[1], q[2], q[3]));
                sts128(piece(box + BOX, 2 * h + 1), make_uint4(q[4], q[5], q[6], q[7]));
              } else {
                act_all(a, p.e.act);
              }
              if (p.e.residual != nullptr) { add8<T>(a, res[0]); add8<T>(a + 8, res[1]); }
            } else if constexpr (MODE == EPI_GLU_BWD) {
              float d[16];
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const uint4 hp = lds128(piece(box, 2 * h + j)), hs = lds128(piece(box + BOX, 2 * h + j)), lo = lds128(piece(box + 2 * BOX, 2 * h + j));
                const uint32_t wp[4] = {hp.x, hp.y, hp.z, hp.w}, ws[4] = {hs.x, hs.y, hs.z, hs.w}, wl[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int k = 8 * j + 2 * i;                           // an fp32's bytes: upper 16 bits, the low byte, nothing
                  auto join = [](uint32_t hi, uint32_t low, uint32_t bytes) { return __uint_as_float(__byte_perm(hi, low, bytes) & 0xffffff00u); };
                  d[k] = a[k] * join(wp[i], wl[i], 0x1044);
                  d[k + 1] = a[k + 1] * join(wp[i], wl[i], 0x3266);
                  a[k] *= join(ws[i], wl[i], 0x1055);
                  a[k + 1] *= join(ws[i], wl[i], 0x3277);
                }
              }
              put16<T>(p0, p1, d);                                       // du, over p
              put16<T>(piece(box + BOX, 2 * h), piece(box + BOX, 2 * h + 1), a);      // dg, over s
            }
            if constexpr (MODE != EPI_GLU_BWD) put16<T>(p0, p1, a);
          }
          if (c == NC - 1) drained();
          fence_proxy_async();
          group_sync(1 + group);
          if (lead && ok) {
            const int gc = nc0 + c * CW;
            if constexpr (MODE == EPI_GLU_BWD) {
              tma_store_2d(&p.tmO1, box, gc, mr);
              tma_store_2d(&w.pr->tmY, box + BOX, gc, mr);
            } else {
              tma_store_2d(&w.pr->tmY, box, gc, mr);
              if constexpr (MODE == EPI_SLOPE) tma_store_2d(&p.tmO1, box + BOX, gc, mr);
              if constexpr (MODE == EPI_GLU) {
                if (p.e.o1 != nullptr) {
                  tma_store_2d(&p.tmO1, box + BOX, gc, mr);
                  tma_store_2d(&p.tmO2, box + 2 * BOX, gc, mr);
                  tma_store_2d(&p.tmO3, box + 3 * BOX, gc, mr);
                }
              }
            }
            bulk_commit();
            if (inputs && c + 2 < NC) {
              bulk_wait_read<0>();                                       // the request overwrites what was just sent
              request(c + 2, cnt + 2);
            }
          }
        }
      }
    }
    if (lead) bulk_wait_read<0>();                                       // shared memory has been read; the kernel's end sees to the rest
  }

  if (fail_id != 0) atomicCAS(&g_gemm_status, 0, fail_id);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (abort_flag) __nanosleep(1000000);                                  // copies still under way land long before this
  if constexpr (CG == 2) cluster_sync();                                 // no CTA of a pair leaves while the other may signal it
  if (warp == 2) { tc_fence_after(); tm_dealloc<CG>(tmem, 2 * BN); }
}

// ---------------------------------------------------------------- few tiles: a cluster shares a tile's contraction
// The S = p.splits pairs of a cluster each take a part of the contraction of one tile of 256 x 128, and hand the sums round
// through distributed shared memory: part q writes what it has of the columns of part s, 1/S of the tile's, into s's shared
// memory; s adds the parts in their order and runs the epilogue on its columns.  One launch, and no sums through L2: 256 x 4096 x
// 4096 bf16 15.1 us (17.8 through the joining kernel), 256 x 1024 x 1024 7.7 (9.3), 1024 x 1024 x 1024 8.8 (9.8 whole), 300 x 2048 x
// 2048 11.1 (12.4).
struct GemmClusterParams {
  TcProduct pr;
  Epi e;
  int splits, per_split;
};
// Tiles of 256 columns would leave room for three stages of the ring, and twice as much to exchange: slower in every case.
// Single CTAs, for up to 128 rows: 0 to 1 us faster than joining at 4096 x 4096, slower at 1024 x 1024; they keep to that.
// Sums: 16-byte pieces of 4 columns, a column of 128 rows each (a warp writes 512 bytes in a row), 16 bytes apart for the reading.
constexpr int CLUSTER_BN = 128;
struct ClusterShape {
  static constexpr int A_BYTES = 128 * 128, B_BYTES = CLUSTER_BN / 2 * 128, PIECE = 128 * 16 + 16, SUMS = CLUSTER_BN / 4 * PIECE;
  static constexpr int STAGES = (229376 - SUMS) / (A_BYTES + B_BYTES), SMEM = STAGES * (A_BYTES + B_BYTES) + SUMS + 1024;
};
__device__ __forceinline__ void sts128_cluster(uint32_t a, uint4 v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

template <int F, typename T, int MODE>
__global__ void __launch_bounds__(384, 1) gemm_cluster_kernel(const __grid_constant__ GemmClusterParams p) {
  using S = ClusterShape;
  constexpr int CG = 2, BN = CLUSTER_BN;
  constexpr bool F8 = F >= 2, PAIR = MODE == EPI_GLU;
  constexpr int KE = F8 ? 128 : 64, NW = PAIR ? BN / 2 : BN, BROWS = BN / CG;
  constexpr uint32_t IDESC = idesc_f16(F8 ? F - 2 : F, 128 * CG, BN, 0, 0);
  extern __shared__ unsigned char smem_raw[];
  const uint32_t s_tiles = (smem_u32(smem_raw) + 1023) & ~1023u, s_sums = s_tiles + S::STAGES * (S::A_BYTES + S::B_BYTES);
  __shared__ __align__(8) uint64_t full[S::STAGES], empty[S::STAGES], tfull;
  __shared__ uint32_t tmem_s;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t at = cluster_rank(), rank = at & 1, first = at - rank;     // of the pair
  const int split = (int)at / CG, tile = blockIdx.x / (CG * p.splits);
  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < S::STAGES; ++i) { mbar_init(smem_u32(&full[i]), 1); mbar_init(smem_u32(&empty[i]), 1); }
    mbar_init(smem_u32(&tfull), 1);
    fence_barrier_init();
  }
  if (warp == 2) tm_alloc<CG>(smem_u32(&tmem_s), BN);
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                                        // every CTA's barriers and sums may be written from here on
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  int fail_id = 0;
  grid_dep_launch();
  grid_dep_wait();

  const int m0 = tile % p.pr.tiles_m * 128 * CG, n0 = tile / p.pr.tiles_m * NW;
  const int k0 = split * p.per_split, k1 = min(p.pr.ksteps * p.pr.segments, k0 + p.per_split);
  const int a_mn = F8 ? 0 : p.pr.a_mn, b_mn = F8 ? 0 : p.pr.b_mn;
  bool ok = true;
  if (warp == 0) {
    // =============================== TMA producer ===============================
    const bool leader = elect_one();
    const int ma = m0 + (int)rank * 128, nb = n0 + (int)rank * BROWS;
    for (int k = k0, it = 0; k < k1; ++k, ++it) {
      const int s = it % S::STAGES, ph = (it / S::STAGES) & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[s]), ph ^ 1, &abort_flag));
      if (!ok) { fail_id = 1; break; }
      if (leader) {
        if (rank == 0) mbar_expect_tx(smem_u32(&full[s]), CG * (S::A_BYTES + S::B_BYTES));
        const uint32_t bar = map_to_rank(smem_u32(&full[s]), first);
        const int seg = k >= p.pr.ksteps, kc = (k - seg * p.pr.ksteps) * KE;
        const uint32_t da = s_tiles + s * (S::A_BYTES + S::B_BYTES), db = da + S::A_BYTES;
        const CUtensorMap *ta = &p.pr.tmA[seg], *tb = &p.pr.tmB[seg];
        if (a_mn) {
          tma_load_2d<CG>(da, ta, bar, ma, kc);
          tma_load_2d<CG>(da + 8192, ta, bar, ma + 64, kc);
        } else {
          tma_load_2d<CG>(da, ta, bar, kc, ma);
        }
        if constexpr (PAIR) {
          tma_load_2d<CG>(db, &p.pr.tmB[rank], bar, kc, n0);
        } else if (b_mn) {
          tma_load_2d<CG>(db, tb, bar, nb, kc);                          // 64 columns
        } else {
          tma_load_2d<CG>(db, tb, bar, kc, nb);
        }
      }
      __syncwarp();
    }
  } else if (warp == 1 && rank == 0) {
    // =============================== MMA issuer ===============================
    const bool leader = elect_one();
    const uint32_t idesc = IDESC | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16);
    const int sa = a_mn ? 128 : 2, sb = b_mn ? 128 : 2;
    for (int k = k0, it = 0; k < k1; ++k, ++it) {
      const int s = it % S::STAGES, ph = (it / S::STAGES) & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[s]), ph, &abort_flag));
      if (!ok) { fail_id = 3; break; }
      tc_fence_after();
      if (leader) {
        const uint32_t da = s_tiles + s * (S::A_BYTES + S::B_BYTES);
        const uint64_t a = smem_desc_sw128(da, a_mn ? 8192 : 16, 1024), b = smem_desc_sw128(da + S::A_BYTES, b_mn ? 8192 : 16, 1024);
#pragma unroll
        for (int i = 0; i < 4; ++i) mma<CG, F8>(tmem, a + i * sa, b + i * sb, idesc, (it > 0 || i > 0) ? 1u : 0u);
        commit<CG>(smem_u32(&empty[s]), first);
      }
      __syncwarp();
    }
    if (ok && leader) commit<CG>(smem_u32(&tfull), first);
    __syncwarp();
  }

  // =============================== the sums go round ===============================
  const int own = NW / p.splits, pieces = BN / p.splits / 4;             // result columns of a part; pieces of a row of its sums
  auto slot = [&](int from, int piece, int row) { return s_sums + (from * pieces + piece) * S::PIECE + row * 16; };
  if (warp >= 4) {
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&tfull), 0, &abort_flag));
    if (!ok) fail_id = 4;
    tc_fence_after();
#pragma unroll 1
    for (int i = (warp - 4) >> 2; ok && i < BN / 16; i += 2) {
      const int half = PAIR ? i / (NW / 16) : 0, col = i * 16 - half * NW, to = col / own;
      uint32_t v[16];
      tmem_ld16(acc + i * 16, v);
      tc_wait_ld();
      const uint32_t base = map_to_rank(slot(split, (half * own + col - to * own) / 4, row), (uint32_t)(to * CG) + rank);
#pragma unroll
      for (int j = 0; j < 4; ++j) sts128_cluster(base + j * S::PIECE, make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
    }
  }
  __syncwarp();
  cluster_sync();
  if (warp >= 4 && ok) {
    const int groups = own / 8;                                          // of 8 columns: neighbouring threads share a row
#pragma unroll 1
    for (int i = tid - 128; i < 128 * groups; i += 256) {
      const int row = i / groups, g = i % groups;
      float a[8] = {}, b[8] = {};
      auto add = [&](float (&sum)[8], int q, int piece) {
        const uint4 lo = lds128(slot(q, piece, row)), hi = lds128(slot(q, piece + 1, row));
        sum[0] += __uint_as_float(lo.x); sum[1] += __uint_as_float(lo.y); sum[2] += __uint_as_float(lo.z); sum[3] += __uint_as_float(lo.w);
        sum[4] += __uint_as_float(hi.x); sum[5] += __uint_as_float(hi.y); sum[6] += __uint_as_float(hi.z); sum[7] += __uint_as_float(hi.w);
      };
      for (int q = 0; q < p.splits; ++q) {
        add(a, q, 2 * g);
        if constexpr (PAIR) add(b, q, own / 4 + 2 * g);
      }
      epilogue8<T, MODE>(p.e, m0 + (int)rank * 128 + row, n0 + split * own + 8 * g, a, b);
    }
  }

  if (fail_id != 0) atomicCAS(&g_gemm_status, 0, fail_id);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (abort_flag) __nanosleep(1000000);                                  // copies still under way land long before this
  cluster_sync();
  if (warp == 2) { tc_fence_after(); tm_dealloc<CG>(tmem, BN); }
}

// Joins the partial sums of a split contraction, in split order, and runs the epilogue: 8 columns a thread.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) gemm_join_kernel(const float* __restrict__ part, const Epi e, int splits, int ldp) {
  constexpr int PR = MODE == EPI_GLU ? 2 : 1;
  const int groups = ldp / 8;
  const long long total = (long long)e.M * groups;
  const long long mn = (long long)e.M * ldp;
  grid_dep_wait();
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long row = i / groups;
    const int col = (int)(i % groups) * 8;
    float a[PR][8] = {};
    for (int s = 0; s < splits; ++s) {
#pragma unroll
      for (int q = 0; q < PR; ++q) {
        const float4* src = reinterpret_cast<const float4*>(part + (s * PR + q) * mn + row * ldp + col);
        const float4 lo = src[0], hi = src[1];
        a[q][0] += lo.x; a[q][1] += lo.y; a[q][2] += lo.z; a[q][3] += lo.w;
        a[q][4] += hi.x; a[q][5] += hi.y; a[q][6] += hi.z; a[q][7] += hi.w;
      }
    }
    epilogue8<T, MODE>(e, row, col, a[0], a[PR - 1]);
  }
}

// ---------------------------------------------------------------- host side
static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return fn;
}

// [rows][cols] matrix with `ld` elements between rows; boxes of box_cols x box_rows with the swizzle of their 64 or 128
// bytes; zeros outside
static int map_2d(CUtensorMap* m, const void* ptr, long long rows, long long cols, long long ld, int box_cols, int box_rows, int dtype) {
  auto enc = tensor_map_encoder();
  NSA_REQUIRE(enc != nullptr, NSA_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const int size = dtype == NSA_BF16 || dtype == NSA_FP16 ? 2 : 1;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * size};
  cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  cuuint32_t es[2] = {1, 1};
  const CUtensorMapSwizzle swizzle = box_cols * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  const CUtensorMapDataType dt = dtype == NSA_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : dtype == NSA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  auto encode = [&] { return enc(m, dt, 2, const_cast<void*>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE); };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {     // a thread that has not used the runtime yet (autograd's): bind the device's context to it
    int dev = 0;
    NSA_CUDA_OK(cudaGetDevice(&dev));
    NSA_CUDA_OK(cudaSetDevice(dev));
    r = encode();
  }
  NSA_REQUIRE(r == CUDA_SUCCESS, NSA_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return NSA_OK;
}

static int pitch(int N) { return (N + 7) / 8 * 8; }                     // of partial sums
// [slabs][M][N] fp32 partial sums, rows `pitch` apart; boxes of 128 rows x 32 columns
static int map_part(CUtensorMap* m, void* ptr, int slabs, int M, int N) {
  auto enc = tensor_map_encoder();
  NSA_REQUIRE(enc != nullptr, NSA_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[3] = {(cuuint64_t)N, (cuuint64_t)M, (cuuint64_t)slabs};
  cuuint64_t strides[2] = {(cuuint64_t)pitch(N) * 4, (cuuint64_t)M * pitch(N) * 4};
  cuuint32_t box[3] = {32, 128, 1};
  cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, ptr, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  NSA_REQUIRE(r == CUDA_SUCCESS, NSA_ERR_CUDA, "cuTensorMapEncodeTiled (partial sums) failed with %d", (int)r);
  return NSA_OK;
}

static int esize(int dtype) { return dtype == NSA_BF16 || dtype == NSA_FP16 ? 2 : 1; }

// Which kernel, how many ways the contraction is split, and whether the sums leave raw: where they are split, or where
// the results' rows do not start on 16-byte boundaries (TMA writes them).
struct TcPlan { int cg, bn, tiles_m, tiles_n, ksteps, splits, per_split; bool raw, cluster; };

// Most steps of a contraction that one tile takes (16.8 M of 16 bits: 70 ms).  The waits for a finished tile are bounded to about a
// second, and an fp32 sum of more terms would stop growing; longer contractions (a weight's gradient over that many tokens) are split.
constexpr int MOST_STEPS = 1 << 18;

// How many clusters of `size` CTAs the device holds at a time, a CTA to an SM
static int cluster_room(int size) {
  static int known[64][2];                      // clusters of 4 and of 8; 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  int* slot = dev < 64 ? &known[dev][size == 8] : nullptr;
  if (slot != nullptr && *slot != 0) return *slot > 0 ? *slot : 0;
  auto fn = gemm_cluster_kernel<1, __nv_bfloat16, EPI_LINEAR>;
  const int smem = ClusterShape::SMEM;
  int n = 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size * 64);
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = size; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) {
    cudaGetLastError();                         // no device here, or none that takes them: the other forms remain
    n = 0;
  }
  if (slot != nullptr) *slot = n > 0 ? n : -1;
  return n;
}
static TcPlan tc_plan(const GemmProblem& p, bool whole = false) {     // whole: pairs on 256 columns, unsplit
  TcPlan t;
  const int pair = p.e.mode == EPI_GLU ? 2 : 1;
  const bool raw = !p.e.vec || !p.e.vecy;
  const int ksteps = (int)(((long long)p.K * esize(p.dtype) + 127) / 128), steps = ksteps * p.segments;     // at most 2^26
  const int least = (steps + MOST_STEPS - 1) / MOST_STEPS;
  // In clk: rounds of tiles at what a step brings through L2 and shared memory (512 for 256 columns on pairs and for 128 on
  // one CTA, 384 for 128 on pairs), and the epilogue that no other tile hides; splitting adds the sums' way out and back
  // (64 bytes a clk and SM) and the joining kernel.  The cheapest of both widths and up to 16 ways
  // (the fewest possible where those are more).
  double best = -1;
  for (int bn = 256; bn >= 128; bn -= 128) {
    const int cg = !whole && p.M <= 128 ? 1 : 2;
    if ((cg == 1 && bn == 256) || (whole && bn == 128)) continue;
    const int tm = (p.M + 128 * cg - 1) / (128 * cg), tn = (p.N + bn / pair - 1) / (bn / pair);
    const long long n = (long long)tm * tn, units = sm_count() / cg;
    const int step = cg == 2 && bn == 128 ? 384 : 512;
    for (int s = whole ? 1 : least; s <= (least > 16 ? least : 16) && s * 4 <= (steps > 4 ? steps : 4); ++s) {
      if (whole && s > 1) break;
      const int per = (steps + s - 1) / s, ways = (steps + per - 1) / per;
      double cost = (double)((n * ways + units - 1) / units) * per * step + 16 * bn;
      if (ways > 1 || raw) cost += 5000 + 8.0 * ways * pair * p.M * p.N / (64.0 * sm_count());
      if (best < 0 || cost < best) {
        best = cost;
        t.cg = cg; t.bn = bn;
        t.tiles_m = tm; t.tiles_n = tn;
        t.splits = ways; t.per_split = per;
      }
    }
  }
  t.cluster = false;
  // A cluster's parts exchange their sums on chip (5000 clk: from the times above the kernel); all clusters have to be
  // resident at once, and a part without work would have no sums.
  if (!whole && p.M > 128) {
    const int tm = (p.M + 255) / 256, tn = (p.N + CLUSTER_BN / pair - 1) / (CLUSTER_BN / pair);
    for (int s = 2; s <= 4; s *= 2) {
      const int per = (steps + s - 1) / s;
      if (per > MOST_STEPS || (s - 1) * per >= steps || (long long)tm * tn > cluster_room(2 * s)) continue;
      const double cost = (double)per * 384 + 5000;
      if (cost < best) {
        best = cost;
        t.cluster = true;
        t.cg = 2; t.bn = CLUSTER_BN;
        t.tiles_m = tm; t.tiles_n = tn;
        t.splits = s; t.per_split = per;
      }
    }
  }
  t.ksteps = ksteps;
  t.raw = !t.cluster && (raw || t.splits > 1);
  return t;
}

long long gemm_tc5_ws_bytes(const GemmProblem& p) {
  const TcPlan t = tc_plan(p);
  return t.raw ? (long long)t.splits * (p.e.mode == EPI_GLU ? 2 : 1) * p.M * pitch(p.N) * 4 : 0;
}

template <int F, typename T, int MODE, int CG, int BN>
static int tc_launch(const GemmTcParams& g, cudaStream_t st) {
  using S = TcShape<MODE, CG, BN>;
  auto fn = gemm_tc5_kernel<F, T, MODE, CG, BN>;
  static bool prepared[64];                   // per device: the attribute outlasts the call, and setting it twice is harmless
  int dev = 0;
  NSA_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64 || !prepared[dev]) {
    NSA_CUDA_OK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    if (dev < 64) prepared[dev] = true;
  }
  const int units = sm_count() / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((g.tiles < units ? g.tiles : units) * CG));
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = CG; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, g);
  if (e != cudaSuccess) return fail(NSA_ERR_CUDA, "gemm_tc5 launch failed: %s", cudaGetErrorString(e));
  return NSA_OK;
}

template <int F, typename T, int MODE>
static int cluster_launch(const GemmClusterParams& g, cudaStream_t st) {
  auto fn = gemm_cluster_kernel<F, T, MODE>;
  constexpr int smem = ClusterShape::SMEM;
  static bool prepared[64];
  int dev = 0;
  NSA_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64 || !prepared[dev]) {
    NSA_CUDA_OK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev < 64) prepared[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(g.pr.tiles_m * g.pr.tiles_n * 2 * g.splits));
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2 * g.splits; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, g);
  if (e != cudaSuccess) return fail(NSA_ERR_CUDA, "gemm_cluster launch failed: %s", cudaGetErrorString(e));
  return NSA_OK;
}
template <int F, typename T>
static int cluster_mode(const GemmClusterParams& g, cudaStream_t st) {
  if constexpr (F < 2) {
    if (g.e.mode == EPI_GLU) return cluster_launch<F, T, EPI_GLU>(g, st);
    if (g.e.mode == EPI_GLU_BWD) return cluster_launch<F, T, EPI_GLU_BWD>(g, st);
  }
  return cluster_launch<F, T, EPI_LINEAR>(g, st);
}
static int cluster_types(const GemmClusterParams& g, int dtype, bool bf, cudaStream_t st) {
  if (dtype == NSA_BF16) return cluster_mode<1, __nv_bfloat16>(g, st);
  if (dtype == NSA_FP16) return cluster_mode<0, __half>(g, st);
  if (dtype == NSA_FP8_E4M3) return bf ? cluster_mode<2, __nv_bfloat16>(g, st) : cluster_mode<2, __half>(g, st);
  return bf ? cluster_mode<3, __nv_bfloat16>(g, st) : cluster_mode<3, __half>(g, st);
}

template <int F, typename T, int MODE>
static int tc_shape(const GemmTcParams& g, const TcPlan& t, cudaStream_t st) {
  if (t.cg == 1) return tc_launch<F, T, MODE, 1, 128>(g, st);
  return t.bn == 256 ? tc_launch<F, T, MODE, 2, 256>(g, st) : tc_launch<F, T, MODE, 2, 128>(g, st);
}

// mode: EPI_*, as the kernel has it
template <int F, typename T>
static int tc_mode(const GemmTcParams& g, const TcPlan& t, int mode, cudaStream_t st) {
  if (mode == EPI_PARTIAL) return tc_shape<F, T, EPI_PARTIAL>(g, t, st);
  if constexpr (F < 2) {
    if (mode == EPI_PARTIAL2) return tc_shape<F, T, EPI_PARTIAL2>(g, t, st);
    if (mode == EPI_GLU) return tc_shape<F, T, EPI_GLU>(g, t, st);
    if (mode == EPI_GLU_BWD) return tc_shape<F, T, EPI_GLU_BWD>(g, t, st);
    if (mode == EPI_SLOPE) return tc_shape<F, T, EPI_SLOPE>(g, t, st);
  }
  return tc_shape<F, T, EPI_LINEAR>(g, t, st);
}
static int tc_types(const GemmTcParams& g, const TcPlan& t, int mode, int dtype, bool bf, cudaStream_t st) {
  if (dtype == NSA_BF16) return tc_mode<1, __nv_bfloat16>(g, t, mode, st);
  if (dtype == NSA_FP16) return tc_mode<0, __half>(g, t, mode, st);
  if (dtype == NSA_FP8_E4M3) return bf ? tc_mode<2, __nv_bfloat16>(g, t, mode, st) : tc_mode<2, __half>(g, t, mode, st);
  return bf ? tc_mode<3, __nv_bfloat16>(g, t, mode, st) : tc_mode<3, __half>(g, t, mode, st);
}

template <typename T>
static int join(const float* part, const GemmProblem& p, int splits, cudaStream_t st) {
  const long long want = ((long long)p.M * ((p.N + 7) / 8) + 255) / 256, cap = 8LL * sm_count();
  const dim3 grid((unsigned)(want < cap ? want : cap));
  if (p.e.mode == EPI_GLU) return launch_pdl("gemm_join", gemm_join_kernel<T, EPI_GLU>, grid, 256, 0, st, part, p.e, splits, pitch(p.N));
  if (p.e.mode == EPI_GLU_BWD) return launch_pdl("gemm_join", gemm_join_kernel<T, EPI_GLU_BWD>, grid, 256, 0, st, part, p.e, splits, pitch(p.N));
  return launch_pdl("gemm_join", gemm_join_kernel<T, EPI_LINEAR>, grid, 256, 0, st, part, p.e, splits, pitch(p.N));
}

// The maps and sizes of one product
static int tc_product(TcProduct* r, const GemmProblem& p, const TcPlan& t) {
  int rc;
  const int ke = 128 / esize(p.dtype);
  const int pair = p.e.mode == EPI_GLU;
  const int brows = pair ? t.bn / 2 : t.bn / t.cg;                     // rows of a box of B
  for (int i = 0; i < p.segments; ++i) {
    rc = p.a_mn ? map_2d(&r->tmA[i], p.A[i], p.K, p.M, p.lda, ke, ke, p.dtype) : map_2d(&r->tmA[i], p.A[i], p.M, p.K, p.lda, ke, 128, p.dtype);
    if (rc != NSA_OK) return rc;
    rc = p.b_mn ? map_2d(&r->tmB[i], p.B[i], p.K, p.N, p.ldb, ke, ke, p.dtype) : map_2d(&r->tmB[i], p.B[i], p.N, p.K, p.ldb, ke, brows, p.dtype);
    if (rc != NSA_OK) return rc;
  }
  if (pair && (rc = map_2d(&r->tmB[1], p.B[1], p.N, p.K, p.ldb, ke, brows, p.dtype)) != NSA_OK) return rc;
  r->M = p.M; r->N = p.N;
  r->tiles_m = t.tiles_m; r->tiles_n = t.tiles_n; r->first = 0;
  r->ksteps = t.ksteps; r->segments = p.segments;
  r->a_mn = p.a_mn; r->b_mn = p.b_mn;
  return NSA_OK;
}

int gemm_tc5(const GemmProblem& p, void* ws, cudaStream_t st) {
  const TcPlan t = tc_plan(p);
  const long long tiles = (long long)t.tiles_m * t.tiles_n * t.splits;
  NSA_REQUIRE(tiles < 2147483647LL - 65536, NSA_ERR_ARG, "matrix product: %d x %d results are too many tiles", p.M, p.N);
  int rc;
  const bool bf = p.out_dtype == NSA_BF16;
  if (t.cluster) {
    GemmClusterParams c;
    if ((rc = tc_product(&c.pr, p, t)) != NSA_OK) return rc;
    c.e = p.e;
    c.splits = t.splits; c.per_split = t.per_split;
    return cluster_types(c, p.dtype, bf, st);
  }
  GemmTcParams g;
  if ((rc = tc_product(&g.pr[0], p, t)) != NSA_OK) return rc;
  const bool gated = p.e.mode != EPI_LINEAR, slope = !gated && p.e.o1 != nullptr;
  if (t.raw) {
    if ((rc = map_part(&g.tmPart, ws, (p.e.mode == EPI_GLU ? 2 : 1) * t.splits, p.M, p.N)) != NSA_OK) return rc;
  } else {
    const int cw = gated || slope ? 32 : 64;
    auto box = [&](CUtensorMap* m, const void* ptr, long long ld) { return ptr == nullptr ? NSA_OK : map_2d(m, ptr, p.M, p.N, ld, cw, 128, p.out_dtype); };
    if ((rc = box(&g.pr[0].tmY, p.e.y, p.e.ldy)) != NSA_OK) return rc;
    if ((rc = box(&g.tmO1, p.e.o1, gated ? p.e.ldy : p.N)) != NSA_OK) return rc;
    if ((rc = box(&g.tmO2, p.e.o2, p.e.ldy)) != NSA_OK) return rc;
    if ((rc = box(&g.tmO3, p.e.o3, p.e.ldy)) != NSA_OK) return rc;
    if ((rc = box(&g.tmI0, gated ? p.e.i0 : p.e.residual, gated ? p.e.ldy : p.N)) != NSA_OK) return rc;
    if ((rc = box(&g.tmI1, p.e.i1, p.e.ldy)) != NSA_OK) return rc;
    if ((rc = box(&g.tmI2, p.e.i2, p.e.ldy)) != NSA_OK) return rc;
  }
  g.e = p.e;
  g.products = 1; g.tiles = (int)tiles;
  g.splits = t.splits; g.per_split = t.per_split;
  const int mode = t.raw ? (p.e.mode == EPI_GLU ? EPI_PARTIAL2 : EPI_PARTIAL) : slope ? EPI_SLOPE : p.e.mode;
  rc = tc_types(g, t, mode, p.dtype, bf, st);
  if (rc != NSA_OK || !t.raw) return rc;
  return bf ? join<__nv_bfloat16>((const float*)ws, p, t.splits, st) : join<__half>((const float*)ws, p, t.splits, st);
}

// Several plain products (EPI_LINEAR with nothing around the sums) of one 16-bit type.  One launch of whole tiles where
// together they fill at least half of the SMs; else one by one.
static bool groups(const GemmProblem* p, int count) {
  if (count < 2 || count > TC_PRODUCTS) return false;
  long long tiles = 0;
  for (int i = 0; i < count; ++i) {
    if (p[i].M <= 128 || !p[i].e.vec || !p[i].e.vecy) return false;
    const TcPlan t = tc_plan(p[i], true);
    if (t.ksteps * p[i].segments > MOST_STEPS) return false;
    tiles += (long long)t.tiles_m * t.tiles_n;
  }
  return tiles < 2147483647LL - 65536 && tiles * 4 >= sm_count();
}

long long gemm_tc5_group_ws_bytes(const GemmProblem* p, int count) {
  long long most = 0;
  if (!groups(p, count))
    for (int i = 0; i < count; ++i) {
      const long long n = gemm_tc5_ws_bytes(p[i]);
      if (n > most) most = n;
    }
  return most;
}

int gemm_tc5_group(const GemmProblem* p, int count, void* ws, cudaStream_t st) {
  if (!groups(p, count)) {
    for (int i = 0; i < count; ++i) {
      const int rc = gemm_tc5(p[i], ws, st);
      if (rc != NSA_OK) return rc;
    }
    return NSA_OK;
  }
  GemmTcParams g;
  g.e = p[0].e;
  g.products = count;
  g.splits = 1; g.per_split = 0;
  // the longest tiles first: the last round is then of the shortest
  int order[TC_PRODUCTS];
  for (int i = 0; i < count; ++i) {
    int j = i;
    for (; j > 0 && (long long)p[order[j - 1]].K * p[order[j - 1]].segments < (long long)p[i].K * p[i].segments; --j) order[j] = order[j - 1];
    order[j] = i;
  }
  int tiles = 0;
  TcPlan t = {};
  for (int i = 0; i < count; ++i) {
    const GemmProblem& q = p[order[i]];
    t = tc_plan(q, true);
    int rc = tc_product(&g.pr[i], q, t);
    if (rc == NSA_OK) rc = map_2d(&g.pr[i].tmY, q.e.y, q.M, q.N, q.e.ldy, 64, 128, q.out_dtype);
    if (rc != NSA_OK) return rc;
    g.pr[i].first = tiles;
    tiles += t.tiles_m * t.tiles_n;
  }
  g.tiles = tiles;
  return tc_types(g, t, EPI_LINEAR, p[0].dtype, p[0].out_dtype == NSA_BF16, st);
}

int gemm_take_status(int* status) {
  int v = 0, zero = 0;
  NSA_CUDA_OK(cudaMemcpyFromSymbol(&v, g_gemm_status, sizeof(int)));
  if (v != 0) NSA_CUDA_OK(cudaMemcpyToSymbol(g_gemm_status, &zero, sizeof(int)));
  *status = v;
  return NSA_OK;
}
int gemm_set_status(int v) {
  NSA_CUDA_OK(cudaMemcpyToSymbol(g_gemm_status, &v, sizeof(int)));
  return NSA_OK;
}

}  // namespace nsa
