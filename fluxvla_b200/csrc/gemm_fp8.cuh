// e4m3 product with block scales on tcgen05:
//   C[t, f] = sum_g sa[t, g] * sb[f / 128, g] * (sum_{k in group g} a[t,k] b[f,k])
// with one f32 scale per 128 columns of a token row and one per 128 x 128
// block of the weights.  The scales differ from group to group, so each
// group's product (128 columns, four MMAs of K = 32) goes to an accumulator of
// its own in TMEM and is scaled into f32 registers while the next groups'
// products run into the others.
//
// Token rows are the M side, so a TMEM lane holds one token's sums and the
// factor sa * sb of a group is one register for all its columns.  (With the
// features there, few tokens would not waste rows of the tensor core, but the
// factor would vary along the columns and come from shared memory for every
// product: 13.7 us against 12.6 us on 64 x 2048 x 16384.)
//
//   warp 0      TMA producer: ring of (tokens, weights) tiles of 128-byte rows
//   warp 1      tcgen05.mma issuer; the cluster kernel has a second one, warp 3,
//               for every other group: one takes longer over a group's waits,
//               MMAs and commits than a 128 x 128 product does (13.5 us
//               against 12.6 us on 64 x 2048 x 16384)
//   warp 2      factors, four groups at a time, two batches ahead
//   warps 4..11 read TMEM (warp w: lanes 32*(w%4)..+31, half of the columns),
//               multiply by the factors, accumulate
//
// Two kernels:
//   gemm_fp8_cluster  tiles of up to 128 tokens x 128 features, several to a CTA
//                     one after the other, or one to a cluster, whose CTAs
//                     split the groups: enough CTAs to fill the GPU however
//                     few the tiles are.  The partial tiles are
//                     exchanged through distributed shared memory and summed
//                     in the order of the groups, so a product is the same
//                     from call to call and needs no workspace.
//   gemm_fp8_pair     256 tokens x 256 features on two SMs (cta_group::2, each
//                     SM loads half of the features), persistent: for many
//                     tiles.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace fvb {
namespace g8 {

constexpr int GROUP = 128;
constexpr int BATCH = 4;  // groups of one batch of factors
constexpr int THREADS = 384;
constexpr int FACTOR_WARP = 2, FIRST_SUM_WARP = 4;

struct Dev {
  int m, n;          // tokens, features
  int groups;        // of 128 columns
  int f_tiles;       // feature tiles
  int t_tiles;       // token tiles
  int cl;            // CTAs of a cluster (gemm_fp8_cluster)
  int rows;          // tokens of a tile (gemm_fp8_cluster), a multiple of 8
  int stages;        // of the ring (gemm_fp8_cluster)
  const float* sa;   // [tokens, groups]
  long long ld_sa;
  const float* sb;   // [features / 128, groups]
  long long ld_sb;
  void* out;
  long long ldo;
  int vec_out;       // rows of out start and end on 16 bytes, n % 8 == 0
};

// kind::f8f6f4, e4m3 x e4m3 -> f32, both K-major
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
template <int CTAS>
__device__ __forceinline__ void mma_e4m3(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                         uint32_t idesc, uint32_t accumulate) {
  if (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// true in one lane of a converged warp.  The issuing warps run their loops
// with all lanes and only the MMAs and commits in this one: addresses and
// descriptors then stay warp-uniform (a loop of one lane measured 0.05 us more
// per group of the pair kernel).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t mapa(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}

// bounded wait with cluster-scope acquire (arrivals come from the peer too)
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  uint64_t t0 = 0;
  for (uint32_t n = 0;; ++n) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(addr), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((n & 63) == 0) {
      const uint64_t t = globaltimer_ns();
      if (!t0) t0 = t;
      if (t - t0 > FVB_WAIT_LIMIT_NS) {
        record_device_error(FVB_ERR_DEVICE_TIMEOUT);
        return false;
      }
    }
  }
}

// After a wait has run out: waits for the loads that are still under way into a
// ring, the last of `issued`, as the CTA may not end before them.
__device__ __forceinline__ void drain(uint64_t* full, int issued, int stages) {
  for (int i = max(issued - stages, 0); i < issued; ++i)
    mbar_wait_limit(&full[i % stages], (i / stages) & 1, FVB_WAIT_LIMIT_NS / 8);
}

// 32 TMEM lanes x 32 columns into registers; tmem_wait makes them valid
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  // the registers are read only after the wait
#pragma unroll
  for (int j = 0; j < N; ++j) asm volatile("" : "+r"(r[j]));
}

// acc[N] += r[N] * f
template <int N>
__device__ __forceinline__ void scale_add(float* acc, const uint32_t* r, float f) {
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = fmaf(__uint_as_float(r[j]), f, acc[j]);
}

// gelu(x) * up for two pairs, gelu in its tanh form as x / (1 + exp(-2u)): no
// cancellation where the tanh nears -1.  One reciprocal serves both; the
// exponents are capped at 2^60 so that the product of the two stays finite, and
// at the cap (x below -7.4) gelu is 0, which is closer than 2^-59 of x.  gelu
// is formed before its product with up, since x * up may be past the range
// where that is not.  (x t / (1 + t) with t = exp(2u) needs neither select, but
// a register that the pair kernel does not have: 78 us against 73.5 us on 816 x
// 32768 x 2048.)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void geglu2(float x0, float u0, float x1, float u1, float& y0,
                                       float& y1) {
  constexpr float C1 = -2.3022081985f, C3 = C1 * 0.044715f;  // -2 sqrt(2/pi) log2(e)
  const float d0 = 1.f + ex2(fminf(x0 * fmaf(C3, x0 * x0, C1), 60.f));
  const float d1 = 1.f + ex2(fminf(x1 * fmaf(C3, x1 * x1, C1), 60.f));
  const float r = __fdividef(1.f, d0 * d1);
  const float s0 = r * d1, s1 = r * d0;
  y0 = x0 * (s0 < 0x1p-59f ? 0.f : s0) * u0;
  y1 = x1 * (s1 < 0x1p-59f ? 0.f : s1) * u1;
}

// gelu(x) * up for one pair
__device__ __forceinline__ float geglu(float x, float up) {
  float y, unused;
  geglu2(x, up, 0.f, 0.f, y, unused);
  return y;
}

// Writes 8 consecutive features f.. of token t (for GEGLU features 2i, 2i+1
// are gate and up of output i) to rows that take 16-byte stores.
template <int EPI>
__device__ __forceinline__ void store8(const Dev& p, int t, int f, const float (&v)[8]) {
  if (EPI == FVB_EPI_F32_STORE) {
    float* o = static_cast<float*>(p.out) + (long long)t * p.ldo + f;
    *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else if (EPI == FVB_EPI_BF16) {
    *reinterpret_cast<uint4*>(static_cast<bf16*>(p.out) + (long long)t * p.ldo + f) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                   pack_bf16x2(v[6], v[7]));
  } else {
    float y[4];
    geglu2(v[0], v[1], v[2], v[3], y[0], y[1]);
    geglu2(v[4], v[5], v[6], v[7], y[2], y[3]);
    *reinterpret_cast<uint2*>(static_cast<bf16*>(p.out) + (long long)t * p.ldo + (f >> 1)) =
        make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
  }
}

// The factor warp: sa * sb of token rows t0..t0+127 and BLOCKS feature blocks
// for the groups g0..g1, a batch of four groups at a time into
// fac[slot][block][row][group].  Lanes run over the groups first: 16 bytes of a
// row are one access, where a load of one group for 32 rows would touch 32
// lines, and every summing warp would repeat it.  bt counts batches over a
// CTA's tiles.  (Ordinary loads: the kernel starts while the norm that writes sa
// may still run, and __ldg is for data that nothing writes meanwhile.)
template <int BLOCKS>
__device__ __forceinline__ bool write_factors(const Dev& p, int t0, int block, int g0, int g1,
                                              float* fac, uint64_t* ffull, uint64_t* fempty,
                                              int& bt, int lane) {
  const int e = lane & (BATCH - 1), r0 = lane / BATCH;
  const int last = (p.n - 1) / 128;
  for (int g = g0; g < g1; g += BATCH, ++bt) {
    const int ge = min(g + e, g1 - 1), slot = bt & 1;
    float a[16], b[BLOCKS];
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)
      b[i] = p.sb[(long long)min(block + i, last) * p.ld_sb + ge];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      a[i] = p.sa[(long long)min(t0 + i * 8 + r0, p.m - 1) * p.ld_sa + ge];
    // all lanes give up together, or none
    if (!__all_sync(0xffffffffu, mbar_wait(&fempty[slot], ((bt >> 1) & 1) ^ 1))) return false;
    float* f = fac + slot * (BATCH * 128 * BLOCKS);
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int j = 0; j < BLOCKS; ++j)
        f[(j * 128 + i * 8 + r0) * BATCH + e] = a[i] * b[j];
    __syncwarp();
    if (lane == 0) mbar_arrive(&ffull[slot]);
  }
  return true;
}
__device__ __forceinline__ float pick(const float4& v, int e) {
  return e == 0 ? v.x : (e == 1 ? v.y : (e == 2 ? v.z : v.w));
}

// ---------------------------------------------------------------------------
// tiles of one SM, or of a cluster that splits the groups
// ---------------------------------------------------------------------------
struct ClusterCfg {
  static constexpr int TILE = 128;                  // features (and most tokens)
  static constexpr int B_BYTES = TILE * GROUP;
  static constexpr int NB = 4;                      // accumulators
  static constexpr int COLS = TILE / 2;             // features of a warp
  static constexpr int PITCH = TILE + 4;            // floats of a partial row
  static constexpr int MAX_STAGES = 12;
  static constexpr int MAX_SMEM = 232448;           // of a CTA
  static constexpr int FAC = 2 * BATCH * TILE * 4;
  static constexpr int BARS = (2 * MAX_STAGES + 2 * NB + 5) * 8 + 16;
  // [ring][partials received: up to rows + 8 x PITCH f32][factors][barriers]
  __host__ __device__ static constexpr int stage_bytes(int rows) { return rows * GROUP + B_BYTES; }
  __host__ __device__ static constexpr int part_bytes(int rows) { return rows * PITCH * 4; }
  static constexpr int fixed_bytes(int rows) {
    return part_bytes(rows + 8) + FAC + BARS + 1024;
  }
  static int stages(int rows) {
    const int s = (MAX_SMEM - fixed_bytes(rows)) / stage_bytes(rows);
    return s < MAX_STAGES ? s : MAX_STAGES;
  }
  static int smem(int rows) { return fixed_bytes(rows) + stages(rows) * stage_bytes(rows); }
};

// Sums `cl` partials [per rows][PITCH] and writes them as token rows t0.. and
// features f0..; threads tid of n.
template <int EPI>
__device__ __forceinline__ void write_tile(const Dev& p, const float* part, int cl, int per, int t0,
                                           int f0, int tid, int n) {
  using C = ClusterCfg;
  const int lane = tid & 31;
  auto sum4 = [&](int r, int f) {
    float4 v = *reinterpret_cast<const float4*>(part + r * C::PITCH + f);
    for (int i = 1; i < cl; ++i) {
      const float4 w = *reinterpret_cast<const float4*>(part + (i * per + r) * C::PITCH + f);
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    return v;
  };
  if (p.vec_out) {
#pragma unroll 2
    for (int e = tid; e < per * (C::TILE / 8); e += n) {
      const int r = e / (C::TILE / 8), f = e % (C::TILE / 8) * 8;
      const float4 a = sum4(r, f), b = sum4(r, f + 4);
      const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      if (t0 + r < p.m && f0 + f < p.n) store8<EPI>(p, t0 + r, f0 + f, v);
    }
  } else {
    // rows that are not 16-byte aligned, or end inside the tile: consecutive
    // lanes write consecutive values
    constexpr int W = EPI == FVB_EPI_GEGLU ? 2 : 1;  // features of a value
    constexpr int N = C::TILE / W / 32;              // values of a lane in a row
    const int most = min(per, p.m - t0);
    for (int r = tid >> 5; r < most; r += n >> 5) {
      float v[N][W];
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) v[i][j] = part[r * C::PITCH + (i * 32 + lane) * W + j];
      for (int c = 1; c < cl; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int j = 0; j < W; ++j)
            v[i][j] += part[(c * per + r) * C::PITCH + (i * 32 + lane) * W + j];
      const long long at = (long long)(t0 + r) * p.ldo + f0 / W;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int f = i * 32 + lane;
        if (f0 + f * W >= p.n) continue;
        if (EPI == FVB_EPI_F32_STORE)
          static_cast<float*>(p.out)[at + f] = v[i][0];
        else
          static_cast<bf16*>(p.out)[at + f] =
              __float2bfloat16(EPI == FVB_EPI_GEGLU ? geglu(v[i][0], v[i][W - 1]) : v[i][0]);
      }
    }
  }
}

// MULTI: a CTA has every gridDim.x-th tile (cl = 1); else one tile, its own or
// its cluster's.  (One kernel for both starts 0.7 us later on the small
// products.)
template <int EPI, bool MULTI>
__global__ void __launch_bounds__(THREADS, 1)
    gemm_fp8_cluster(const __grid_constant__ CUtensorMap tmA,
                     const __grid_constant__ CUtensorMap tmB, const Dev p) {
  using C = ClusterCfg;
  constexpr int COLS = C::COLS, NB = C::NB;
  constexpr uint32_t IDESC = idesc_e4m3_f32(128, C::TILE);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int rows = p.rows, stages = p.stages;
  const int a_bytes = rows * GROUP, stage_bytes = a_bytes + C::B_BYTES;
  uint8_t* recv = smem + stages * stage_bytes;
  float* fac = reinterpret_cast<float*>(recv + C::part_bytes(rows + 8));
  uint64_t* full = reinterpret_cast<uint64_t*>(fac + C::FAC / 4);
  uint64_t* empty = full + C::MAX_STAGES;
  uint64_t* tfull = empty + C::MAX_STAGES;  // [NB]
  uint64_t* tempty = tfull + NB;            // [NB]
  uint64_t* ffull = tempty + NB;            // [2]
  uint64_t* fempty = ffull + 2;             // [2]
  uint64_t* recvd = fempty + 2;             // the cluster's partials are here
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(recvd + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cl = p.cl;
  const int rank = cl > 1 ? (int)cluster_rank() : 0;
  const int tile0 = blockIdx.x / cl, n_tiles = p.f_tiles * p.t_tiles;
  const int stride = gridDim.x;  // MULTI
  const int my_tiles = MULTI ? (n_tiles - tile0 + stride - 1) / stride : 1;
  const int f0 = tile0 % p.f_tiles * C::TILE, t0 = tile0 / p.f_tiles * rows;  // of the first
  const int g0 = (int)((long long)p.groups * rank / cl);
  const int g1 = (int)((long long)p.groups * (rank + 1) / cl);
  const int ng = g1 - g0;
  // token rows that this CTA sums
  const int my0 = rows * rank / cl, per = rows * (rank + 1) / cl - my0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < NB; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 8);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&ffull[a], 1);
      mbar_init(&fempty[a], 8);
    }
    mbar_init(recvd, 1);
    fence_barrier_init();
    mbar_arrive_expect_tx(recvd, cl * C::part_bytes(per));
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
  }
  if (warp == 1) tmem_alloc(tmem_slot, NB * C::TILE);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (cl > 1) cluster_arrive();  // waited for before the first remote copy
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  bool alive = true;  // no wait of this thread has run out
  int issued = 0;     // loads of the producer
  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t phase = 1;
      int w = tile0;
      do {
        const int f = w % p.f_tiles * C::TILE, t = w / p.f_tiles * rows;
        for (int g = g0; g < g1; ++g) {
          if (!mbar_wait_spin(&empty[s], phase)) { alive = false; break; }
          mbar_arrive_expect_tx(&full[s], stage_bytes);
          uint8_t* st = smem + s * stage_bytes;
          tma_load_2d(st + a_bytes, &tmB, g * GROUP, f, &full[s]);
          tma_load_2d(st, &tmA, g * GROUP, t, &full[s]);
          ++issued;
          if (++s == stages) {
            s = 0;
            phase ^= 1;
          }
        }
      } while (MULTI && alive && (w += stride) < n_tiles);
    }
    __syncwarp();
    if (cl > 1) cluster_wait();
  } else if (warp == 1 || warp == 3) {
    // a tile of fewer than 128 rows: the MMA reads on into the weights, which
    // makes sums in lanes that nobody reads
    const bool elected = elect_one();
    const int first = warp >> 1;
    int s = first % stages;
    uint32_t phase = (first / stages) & 1;
#pragma unroll 1
    for (int i = first; i < ng * my_tiles; i += 2) {
      const int b = i % NB;
      bool ready = mbar_wait_spin(&full[s], phase);
      ready = ready && mbar_wait_spin(&tempty[b], ((i / NB) & 1) ^ 1);
      alive = __all_sync(0xffffffffu, ready);
      if (!alive) break;
      tc_fence_after();
      if (elected) {
        const uint64_t da = smem_desc_sw128(smem_u32(smem + s * stage_bytes));
        const uint64_t db = smem_desc_sw128(smem_u32(smem + s * stage_bytes + a_bytes));
#pragma unroll
        for (int kk = 0; kk < GROUP / 32; ++kk)
          mma_e4m3<1>(tmem + b * C::TILE, da + kk * 2, db + kk * 2, IDESC, kk > 0);
        tc_commit(&tfull[b]);
        tc_commit(&empty[s]);
      }
      __syncwarp();
      s += 2;
      if (s >= stages) {
        s -= stages;
        phase ^= 1;
      }
    }
    if (cl > 1) cluster_wait();
  } else if (warp == FACTOR_WARP) {
    int bt = 0;
    int w = tile0;
    do {
      alive = write_factors<1>(p, w / p.f_tiles * rows, w % p.f_tiles, g0, g1, fac, ffull, fempty,
                               bt, lane);
    } while (MULTI && alive && (w += stride) < n_tiles);
    if (cl > 1) cluster_wait();
  } else {
    const int q = warp & 3, half = (warp - FIRST_SUM_WARP) >> 2;
    const bool used = q * 32 < rows;  // lanes past the last row are not read
    const uint32_t lane_base = tmem + ((uint32_t)(q * 32) << 16) + half * COLS;
    // the eight summing warps meet; true if none has given up a wait
    auto sum_barrier = [](bool fine) {
      uint32_t all;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.u32 p, %1, 0;\n\t"
          "bar.red.and.pred q, 1, 256, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(all)
          : "r"((uint32_t)fine)
          : "memory");
      return all != 0;
    };
    float acc[COLS];
    bool ok = true;
    int it = 0, bt = 0, w = tile0;
    do {
#pragma unroll
      for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
      for (int i0 = 0; i0 < ng && ok; i0 += BATCH) {
        const int batch = MULTI ? bt++ : i0 / BATCH, slot = batch & 1;
        ok = __all_sync(0xffffffffu, mbar_wait_spin(&ffull[slot], (batch >> 1) & 1));
        const float4 f4 = reinterpret_cast<const float4*>(fac)[slot * 128 + q * 32 + lane];
        __syncwarp();
        if (lane == 0) mbar_arrive(&fempty[slot]);
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
          if (i0 + e < ng && ok) {
            static_assert(NB == BATCH, "a batch starts at the first accumulator");
            const int b = MULTI ? it % NB : e;
            ok = mbar_wait_spin(&tfull[b], (MULTI ? it / NB : i0 / NB) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
              tc_fence_after();
              uint32_t r[COLS];
              if (used) {
#pragma unroll
                for (int j = 0; j < COLS; j += 32) tmem_ld32(lane_base + b * C::TILE + j, r + j);
                tmem_wait<COLS>(r);
              }
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&tempty[b]);
              if (used) scale_add<COLS>(acc, r, pick(f4, e));
              if (MULTI) ++it;
            }
          }
        }
      }
      if (!MULTI) break;  // written below
      // the tile goes through the space for received partials, while the next
      // tile's products are under way
      if (ok && q * 32 + lane < rows) {
        float* t = reinterpret_cast<float*>(recv) + (q * 32 + lane) * C::PITCH + half * COLS;
#pragma unroll
        for (int j = 0; j < COLS; j += 4)
          *reinterpret_cast<float4*>(t + j) =
              make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
      }
      ok = sum_barrier(ok);
      if (ok)
        write_tile<EPI>(p, reinterpret_cast<const float*>(recv), 1, rows, w / p.f_tiles * rows,
                        w % p.f_tiles * C::TILE, threadIdx.x - 32 * FIRST_SUM_WARP, 256);
      sum_barrier(ok);
    } while (ok && (w += stride) < n_tiles);
    if (!MULTI) {
      // every product has been read, so the ring is free: the partial tile goes
      // there, and each CTA's token rows in one copy to that CTA
      if (q * 32 + lane < rows) {
        float* t = reinterpret_cast<float*>(smem) + (q * 32 + lane) * C::PITCH + half * COLS;
#pragma unroll
        for (int j = 0; j < COLS; j += 4)
          *reinterpret_cast<float4*>(t + j) =
              make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
      }
      fence_proxy_async_smem();
      ok = sum_barrier(ok);
      if (cl > 1) cluster_wait();
      if (warp == FIRST_SUM_WARP && lane < cl && cl > 1 && ok) {
        const int to = rows * lane / cl;  // first row of the CTA that this lane serves
        const uint32_t bytes = C::part_bytes(rows * (lane + 1) / cl - to);
        asm volatile(
            "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes "
            "[%0], [%1], %2, [%3];" ::"r"(mapa(smem_u32(recv) + rank * bytes, lane)),
            "r"(smem_u32(smem) + C::part_bytes(to)), "r"(bytes), "r"(mapa(smem_u32(recvd), lane))
            : "memory");
      }
    }
    alive = ok;
  }
  tc_fence_before();
  if (__syncthreads_or(!alive) && threadIdx.x == 0) drain(full, issued, stages);
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, NB * C::TILE);
  }
  if (MULTI) return;
  // this CTA's tokens: the cluster's partials in the order of the groups
  if (cl > 1) mbar_wait_cluster(recvd, 0);
  write_tile<EPI>(p, reinterpret_cast<const float*>(cl > 1 ? recv : smem), cl, per, t0 + my0, f0,
                  threadIdx.x, THREADS);
  if (cl > 1) {
    // the copies out of this CTA have been received everywhere
    cluster_arrive();
    cluster_wait();
  }
}

// ---------------------------------------------------------------------------
// two-SM tiles, persistent
// ---------------------------------------------------------------------------
struct PairCfg {
  static constexpr int TILE = 256;                 // tokens and features of a tile
  static constexpr int HALF = 128 * GROUP;         // bytes of a CTA's half of either
  static constexpr int STAGE = 2 * HALF;
  static constexpr int STAGES = 5;
  static constexpr int SUM_WARPS = 8;
  static constexpr int COLS = TILE / 2;
  static constexpr int OFF_STG = STAGES * STAGE;   // [warps][32 rows][64 bytes]
  static constexpr int STG = 32 * 64;
  static constexpr int OFF_F = OFF_STG + SUM_WARPS * STG;  // [2][BATCH][2][128] f32
  static constexpr int OFF_BAR = OFF_F + 2 * BATCH * 2 * 128 * 4;
  static constexpr int SMEM = OFF_BAR + (2 * STAGES + 8) * 8 + 16 + 1024;
};

__device__ __forceinline__ void tma_load_2d_pair(void* smem_dst, const CUtensorMap* map, int32_t x,
                                                 int32_t y, uint32_t bar_cluster) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::"
      "complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar_cluster)
      : "memory");
}
__device__ __forceinline__ void commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster."
      "multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"((unsigned short)0x3)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar_cluster) {
  // relaxed: what it orders are TMEM reads, done before by tcgen05.wait::ld; a
  // cluster-scope release would wait for this thread's global stores as well
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster)
               : "memory");
}
// VEC: rows of out start and end on 16 bytes.  (A kernel of its own for the
// others, 87 us against 74 us on 816 x 32764 x 2048: with both in one the sums
// spill, and the aligned one took 86 us too.)
template <int EPI, bool VEC>
__global__ void __launch_bounds__(THREADS, 1)
    gemm_fp8_pair(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const Dev p) {
  using C = PairCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;  // [2]
  uint64_t* tempty = tfull + 2;         // [2] (leader: of both CTAs)
  uint64_t* ffull = tempty + 2;         // [2]
  uint64_t* fempty = ffull + 2;         // [2]
  float* fac = reinterpret_cast<float*>(smem + C::OFF_F);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fempty + 2);
  // {TMEM address, whether a wait of either CTA has run out, loads issued}
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int n_tiles = p.f_tiles * p.t_tiles;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * C::SUM_WARPS);
      mbar_init(&ffull[a], 1);
      mbar_init(&fempty[a], C::SUM_WARPS);
    }
    tmem_slot[1] = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncwarp();
  cluster_arrive();  // barriers of both CTAs initialised, TMEM allocated
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  // 384 threads start with 168 registers each; the eight summing warps take
  // 208 (128 sums and two TMEM reads of 32) and the first four keep 80:
  // 256 * 208 + 128 * 80 = 63488 <= 384 * 168.  (Sixteen summing warps of 64
  // columns measured 80 us against 71 us on 816 x 32768 x 2048.)
  // Token tiles vary fastest: the pairs at work share weight tiles.
  auto gave_up = [&]() {
    for (int c = 0; c < 2; ++c)
      asm volatile("st.shared::cluster.u32 [%0], 1;" ::"r"(mapa(smem_u32(tmem_slot + 1), c))
                   : "memory");
  };
  if (warp < FIRST_SUM_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    bool alive = true;
    if (warp == 0 && lane == 0) {
      int issued = 0;
      for (int w = pair; w < n_tiles && alive; w += n_pairs) {
        const int trow = (w % p.t_tiles) * C::TILE + (int)rank * 128;
        const int wrow = (w / p.t_tiles) * C::TILE + (int)rank * 128;
        for (int g = 0; g < p.groups; ++g, ++issued) {
          const int s = issued % C::STAGES;
          if (!mbar_wait(&empty[s], ((issued / C::STAGES) & 1) ^ 1)) { alive = false; break; }
          const uint32_t fb = mapa(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::STAGE);
          uint8_t* sa = smem + s * C::STAGE;
          tma_load_2d_pair(sa, &tmA, g * GROUP, trow, fb);
          tma_load_2d_pair(sa + C::HALF, &tmB, g * GROUP, wrow, fb);
        }
      }
      tmem_slot[2] = issued;
    } else if (warp == 1 && rank == 0) {
      constexpr uint32_t IDESC = idesc_e4m3_f32(256, C::TILE);
      const bool elected = elect_one();
      const int n_it = p.groups * ((n_tiles - pair + n_pairs - 1) / n_pairs);
      int s = 0;
      uint32_t phase = 0;
#pragma unroll 1
      for (int it = 0; it < n_it; ++it) {
        const int b = it & 1;
        bool ready = mbar_wait_spin(&full[s], phase);
        ready = ready && mbar_wait_cluster(&tempty[b], ((it >> 1) & 1) ^ 1);
        alive = __all_sync(0xffffffffu, ready);
        if (!alive) break;
        tc_fence_after();
        if (elected) {
          const uint64_t da = smem_desc_sw128(smem_u32(smem + s * C::STAGE));
          const uint64_t db = smem_desc_sw128(smem_u32(smem + s * C::STAGE + C::HALF));
#pragma unroll
          for (int kk = 0; kk < GROUP / 32; ++kk)
            mma_e4m3<2>(tmem + b * C::TILE, da + kk * 2, db + kk * 2, IDESC, kk > 0);
          commit_both(&tfull[b]);
          commit_both(&empty[s]);
        }
        __syncwarp();
        if (++s == C::STAGES) {
          s = 0;
          phase ^= 1;
        }
      }
    } else if (warp == FACTOR_WARP) {
      int bt = 0;
      for (int w = pair; w < n_tiles && alive; w += n_pairs)
        alive = write_factors<2>(p, (w % p.t_tiles) * C::TILE + (int)rank * 128,
                                 (w / p.t_tiles) * 2, 0, p.groups, fac, ffull, fempty, bt, lane);
    }
    if (!alive) gave_up();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int q = warp & 3, part = (warp - FIRST_SUM_WARP) >> 2;
    const uint32_t lane_base = tmem + ((uint32_t)(q * 32) << 16) + part * C::COLS;
    const uint32_t te[2] = {mapa(smem_u32(&tempty[0]), 0), mapa(smem_u32(&tempty[1]), 0)};
    const uint32_t stg = smem_u32(smem + C::OFF_STG) + (warp - FIRST_SUM_WARP) * C::STG;
    const float4* frow = reinterpret_cast<const float4*>(fac) + part * 128 + q * 32 + lane;
    int it = 0, bt = 0;
    bool ok = true;
    for (int w = pair; w < n_tiles && ok; w += n_pairs) {
      const int t0 = (w % p.t_tiles) * C::TILE + (int)rank * 128 + q * 32;
      const int f0 = (w / p.t_tiles) * C::TILE + part * C::COLS;
      float acc[C::COLS];
#pragma unroll
      for (int j = 0; j < C::COLS; ++j) acc[j] = 0.f;
      float4 f4;
#pragma unroll 1
      for (int g = 0; g < p.groups; ++g, ++it) {
        const int b = it & 1, e = g & (BATCH - 1), slot = bt & 1;
        if (e == 0) {
          ok = mbar_wait_spin(&ffull[slot], (bt >> 1) & 1);
          f4 = frow[slot * 256];
          __syncwarp();
          if (lane == 0) mbar_arrive(&fempty[slot]);
          ++bt;
        }
        const float f = pick(f4, e);
        ok = ok && mbar_wait_spin(&tfull[b], (it >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ta = lane_base + b * C::TILE;
        uint32_t r[2][32];
        tmem_ld32(ta, r[0]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          tmem_wait<32>(r[j & 1]);
          if (j < 3) {
            tmem_ld32(ta + 32 * j + 32, r[(j + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(te[b]);
          }
          scale_add<32>(acc + 32 * j, r[j & 1], f);
        }
      }
      if (!ok) {
        gave_up();
        break;
      }
      // A lane holds one token's features: 64 bytes of output a row at a time
      // go through shared memory (16-byte pieces swizzled by the row), so that
      // each store instruction writes 64 bytes of 8 rows.
      constexpr int FC = EPI == FVB_EPI_F32_STORE ? 16 : (EPI == FVB_EPI_BF16 ? 32 : 64);
      constexpr int eb = EPI == FVB_EPI_F32_STORE ? 4 : 2;
      const int nf_out = EPI == FVB_EPI_GEGLU ? p.n / 2 : p.n;
#pragma unroll
      for (int c = 0; c < C::COLS; c += FC) {
        uint32_t v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (EPI == FVB_EPI_F32_STORE) {
            v[j] = __float_as_uint(acc[c + j]);
          } else if (EPI == FVB_EPI_BF16) {
            v[j] = pack_bf16x2(acc[c + 2 * j], acc[c + 2 * j + 1]);
          } else {
            const float* a = acc + c + 4 * j;
            float y0, y1;
            geglu2(a[0], a[1], a[2], a[3], y0, y1);
            v[j] = pack_bf16x2(y0, y1);
          }
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                           stg + lane * 64 + ((j ^ (lane >> 1)) & 3) * 16),
                       "r"(v[4 * j]), "r"(v[4 * j + 1]), "r"(v[4 * j + 2]), "r"(v[4 * j + 3])
                       : "memory");
        __syncwarp();
        const int o0 = EPI == FVB_EPI_GEGLU ? (f0 + c) >> 1 : f0 + c;
        if (VEC) {
          const int col = o0 + (lane & 3) * (16 / eb);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2);
            uint32_t x[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                         : "r"(stg + row * 64 + (((lane & 3) ^ (row >> 1)) & 3) * 16));
            if (t0 + row < p.m && col < nf_out)
              *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) +
                                        ((long long)(t0 + row) * p.ldo + col) * eb) =
                  make_uint4(x[0], x[1], x[2], x[3]);
          }
        } else {
          // consecutive lanes write consecutive values
          constexpr int PER = EPI == FVB_EPI_F32_STORE ? 16 : 32;  // values of a row
          const int col = lane % PER;
#pragma unroll 2
          for (int i = 0; i < PER; ++i) {
            const int row = i * (32 / PER) + lane / PER, at = col * eb;
            const uint32_t src = stg + row * 64 + (((at >> 4) ^ (row >> 1)) & 3) * 16 + (at & 15);
            if (t0 + row >= p.m || o0 + col >= nf_out) continue;
            const long long to = (long long)(t0 + row) * p.ldo + o0 + col;
            if (EPI == FVB_EPI_F32_STORE) {
              uint32_t x;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(src));
              static_cast<uint32_t*>(p.out)[to] = x;
            } else {
              uint16_t x;
              asm volatile("ld.shared.b16 %0, [%1];" : "=h"(x) : "r"(src));
              static_cast<uint16_t*>(p.out)[to] = x;
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_arrive();  // every MMA, commit and remote arrival is done
  cluster_wait();
  if (tmem_slot[1]) {
    // the loads of both CTAs arrive at the leader's barriers; those that the
    // leader does not expect have the time of one wait
    if (threadIdx.x == 0) {
      if (rank == 0)
        drain(full, tmem_slot[2], C::STAGES);
      else
        mbar_wait_limit(&full[0], 0, FVB_WAIT_LIMIT_NS / 8);
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

}  // namespace g8
}  // namespace fvb
