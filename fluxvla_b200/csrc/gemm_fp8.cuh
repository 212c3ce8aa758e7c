// e4m3 product with block scales on tcgen05:
//   C[t, f] = sum_g sa[t, g] * sb[f / 128, g] * (sum_{k in group g} a[t,k] b[f,k])
// with one f32 scale per 128 columns of a token row and one per 128 x 128
// block of the weights.  The scales differ from group to group, so each
// group's product (128 columns, four MMAs of K = 32) goes to its own
// accumulator in TMEM and is scaled into f32 registers while the next
// group's product runs into the other accumulator.
//
//   warp 0     TMA producer: ring of (A, B) tiles of 128 bytes a row
//   warp 1     tcgen05.mma issuer, two TMEM accumulators of BN columns
//   warps 2..  read TMEM (warp w: lanes 32*(w%4)..+31), multiply by the
//              group's scales, accumulate
//
// Orientation: the M side (TMEM lanes) holds 128 token rows and the N side BN
// features; with SWAP (few tokens) the M side holds 128 features, so that the
// weights fill the 128 rows of the tensor core, and the N side BN tokens.
//
// CL CTAs of a cluster share a tile, each with a part of the groups; their f32
// partial tiles are summed through distributed shared memory in the order of
// the groups, so a product is the same from call to call and needs no
// workspace.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace fvb {
namespace g8 {

constexpr int GROUP = 128;

struct Dev {
  int m, n, k;       // tokens, features, columns
  int groups;        // of 128 columns
  int m_tiles;       // tiles along the M side
  int cl;            // CTAs of a cluster
  const float* sa;   // [tokens, groups]
  long long ld_sa;
  const float* sb;   // [features / 128, groups]
  long long ld_sb;
  void* out;
  long long ldo;
  int vec_out;       // rows of out take 16-byte (bf16: 8-byte) stores
};

// kind::f8f6f4, e4m3 x e4m3 -> f32, both K-major
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_e4m3(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                         uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// gelu(x) with the tanh form, as x / (1 + exp(-2u)): no cancellation where
// the tanh nears -1
__device__ __forceinline__ float gelu_sigmoid(float x) {
  const float u2 = 1.5957691216057308f * (x + 0.044715f * x * x * x);
  return x / (1.f + __expf(-u2));
}

template <int BN, bool SWAP>
struct Cfg {
  static constexpr int A_BYTES = 128 * GROUP;
  static constexpr int B_BYTES = BN * GROUP;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = (196 * 1024) / STAGE < 8 ? (196 * 1024) / STAGE : 8;
  static constexpr int PW = SWAP ? 4 : 8;            // scaling warps
  static constexpr int COLS = SWAP ? BN : BN / 2;    // accumulator columns of a warp
  static constexpr int THREADS = 64 + 32 * PW;
  // finished tile in shared memory: [tokens][features + 4] f32, over the ring
  static constexpr int T_ROWS = SWAP ? BN : 128;
  static constexpr int T_COLS = SWAP ? 128 : BN;
  static constexpr int PITCH = T_COLS + 4;
  static_assert(T_ROWS * PITCH * 4 <= STAGES * STAGE, "the finished tile reuses the ring");
  static constexpr int OFF_CS = STAGES * STAGE;      // SWAP: [PW][2][BN] column scales
  static constexpr int OFF_BAR = OFF_CS + (SWAP ? PW * 2 * BN * 4 : 0);
  static constexpr int SMEM = OFF_BAR + (2 * STAGES + 4) * 8 + 16 + 1024;
  static constexpr uint32_t TMEM_COLS =
      2 * BN <= 32 ? 32 : (2 * BN <= 64 ? 64 : (2 * BN <= 128 ? 128 : (2 * BN <= 256 ? 256 : 512)));
};

template <int BN, bool SWAP, int EPI>
__global__ void __launch_bounds__(Cfg<BN, SWAP>::THREADS, 1)
    gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmA,
                    const __grid_constant__ CUtensorMap tmB, const Dev p) {
  using C = Cfg<BN, SWAP>;
  constexpr int COLS = C::COLS;
  constexpr uint32_t IDESC = idesc_e4m3_f32(128, BN);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;  // [2]
  uint64_t* tempty = tfull + 2;         // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cl = p.cl;
  const uint32_t rank = cl > 1 ? cluster_rank() : 0;
  const int tile = blockIdx.x / cl;
  const int mt = tile % p.m_tiles, nt = tile / p.m_tiles;
  const int g0 = (int)((long long)p.groups * rank / cl);
  const int g1 = (int)((long long)p.groups * (rank + 1) / cl);
  const int ng = g1 - g0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], C::PW);
    }
    fence_barrier_init();
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
  }
  if (warp == 1) tmem_alloc(tmem_slot, C::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      const CUtensorMap* mw = SWAP ? &tmA : &tmB;
      const CUtensorMap* mx = SWAP ? &tmB : &tmA;
      constexpr int woff = SWAP ? 0 : C::A_BYTES, xoff = SWAP ? C::A_BYTES : 0;
      const int wrow = SWAP ? mt * 128 : nt * BN, xrow = SWAP ? nt * BN : mt * 128;
      griddep_wait();
      for (int i = 0; i < ng; ++i) {
        const int s = i % C::STAGES;
        if (!mbar_wait(&empty[s], ((i / C::STAGES) & 1) ^ 1)) break;
        mbar_arrive_expect_tx(&full[s], C::STAGE);
        tma_load_2d(smem + s * C::STAGE + woff, mw, (g0 + i) * GROUP, wrow, &full[s]);
        tma_load_2d(smem + s * C::STAGE + xoff, mx, (g0 + i) * GROUP, xrow, &full[s]);
      }
      griddep_launch_dependents();
    }
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < ng; ++i) {
        const int s = i % C::STAGES, b = i & 1;
        if (!mbar_wait(&tempty[b], ((i >> 1) & 1) ^ 1)) break;
        if (!mbar_wait(&full[s], (i / C::STAGES) & 1)) break;
        tc_fence_after();
        const uint64_t da = smem_desc_sw128(smem_u32(smem + s * C::STAGE));
        const uint64_t db = smem_desc_sw128(smem_u32(smem + s * C::STAGE + C::A_BYTES));
#pragma unroll
        for (int kk = 0; kk < GROUP / 32; ++kk)
          mma_e4m3(tmem + b * BN, da + kk * 2, db + kk * 2, IDESC, kk > 0);
        tc_commit(&empty[s]);
        tc_commit(&tfull[b]);
      }
    }
  } else {
    const int q = warp & 3, half = SWAP ? 0 : (warp - 2) >> 2;
    const int row = mt * 128 + q * 32 + lane;  // token (SWAP: feature) of this thread
    const int col0 = nt * BN + half * COLS;    // first feature (SWAP: token)
    griddep_wait();
    float acc[COLS];
#pragma unroll
    for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
    // scales are read one group ahead
    const float* sa_row = p.sa + (long long)min(row, p.m - 1) * p.ld_sa;
    const int sb_tile = SWAP ? mt : min(col0, p.n - 1) / GROUP;
    const float* sb_row = p.sb + (long long)sb_tile * p.ld_sb;
    float* cs = reinterpret_cast<float*>(smem + C::OFF_CS) + (SWAP ? (warp - 2) * 2 * BN : 0);
    constexpr int CPL = SWAP ? (BN + 31) / 32 : 1;  // column scales of a lane
    float sa_next[CPL], sb_next = 0.f;
    auto fetch = [&](int g) {
      sb_next = __ldg(sb_row + g);
      if (SWAP) {
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          const int t = min(col0 + c * 32 + lane, p.m - 1);
          sa_next[c] = __ldg(p.sa + (long long)t * p.ld_sa + g);
        }
      } else {
        sa_next[0] = __ldg(sa_row + g);
      }
    };
    if (ng > 0) fetch(g0);
    const uint32_t lane_base = tmem + ((uint32_t)(q * 32) << 16) + half * COLS;
    for (int i = 0; i < ng; ++i) {
      const int b = i & 1;
      float scale = sb_next;
      if (SWAP) {
#pragma unroll
        for (int c = 0; c < CPL; ++c)
          if (c * 32 + lane < BN) cs[b * BN + c * 32 + lane] = sa_next[c] * scale;
        __syncwarp();
      } else {
        scale *= sa_next[0];
      }
      if (i + 1 < ng) fetch(g0 + i + 1);
      ok = mbar_wait(&tfull[b], (i >> 1) & 1);
      __syncwarp();
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_fence_after();
      const uint32_t ta = lane_base + b * BN;
#pragma unroll
      for (int c = 0; c < COLS; c += 16) {
        uint32_t r[16];
        tmem_ld16_sync(ta + c, r);
        if (SWAP) {
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 s = *reinterpret_cast<const float4*>(cs + b * BN + c + j);
            acc[c + j] = fmaf(__uint_as_float(r[j]), s.x, acc[c + j]);
            acc[c + j + 1] = fmaf(__uint_as_float(r[j + 1]), s.y, acc[c + j + 1]);
            acc[c + j + 2] = fmaf(__uint_as_float(r[j + 2]), s.z, acc[c + j + 2]);
            acc[c + j + 3] = fmaf(__uint_as_float(r[j + 3]), s.w, acc[c + j + 3]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[c + j] = fmaf(__uint_as_float(r[j]), scale, acc[c + j]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[b]);
    }
    // every product has been read, so the ring is free for the finished tile
    float* ts = reinterpret_cast<float*>(smem);
    if (ok) {
      if (SWAP) {
#pragma unroll
        for (int j = 0; j < COLS; ++j) ts[j * C::PITCH + q * 32 + lane] = acc[j];
      } else {
#pragma unroll
        for (int j = 0; j < COLS; j += 4)
          *reinterpret_cast<float4*>(ts + (q * 32 + lane) * C::PITCH + half * COLS + j) =
              make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
  if (cl > 1) cluster_sync();

  // this CTA's share of the tile's token rows: sum over the cluster, epilogue
  const uint32_t ts = smem_u32(smem);
  const int t0 = SWAP ? nt * BN : mt * 128, f0 = SWAP ? mt * 128 : nt * BN;
  const int r0 = C::T_ROWS * rank / cl, r1 = C::T_ROWS * (rank + 1) / cl;
  constexpr int Q = C::T_COLS / 4;
  for (int e = threadIdx.x; e < (r1 - r0) * Q; e += C::THREADS) {
    const int r = r0 + e / Q, c = (e % Q) * 4;
    const int t = t0 + r, f = f0 + c;
    if (t >= p.m || f >= p.n) continue;
    const uint32_t at = ts + (r * C::PITCH + c) * 4;
    float4 v;
    if (cl > 1) {
      v = ld_cluster4(at, 0);
      for (int i = 1; i < cl; ++i) {
        const float4 w = ld_cluster4(at, i);
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
    } else {
      v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) +
                                           r * C::PITCH + c);
    }
    const int nf = min(4, p.n - f);
    if (EPI == FVB_EPI_F32_STORE) {
      float* o = static_cast<float*>(p.out) + (long long)t * p.ldo + f;
      if (p.vec_out && nf == 4) {
        *reinterpret_cast<float4*>(o) = v;
      } else {
        o[0] = v.x;
        if (nf > 1) o[1] = v.y;
        if (nf > 2) o[2] = v.z;
        if (nf > 3) o[3] = v.w;
      }
    } else if (EPI == FVB_EPI_BF16) {
      bf16* o = static_cast<bf16*>(p.out) + (long long)t * p.ldo + f;
      if (p.vec_out && nf == 4) {
        *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
      } else {
        o[0] = __float2bfloat16(v.x);
        if (nf > 1) o[1] = __float2bfloat16(v.y);
        if (nf > 2) o[2] = __float2bfloat16(v.z);
        if (nf > 3) o[3] = __float2bfloat16(v.w);
      }
    } else {  // FVB_EPI_GEGLU: features 2i, 2i+1 are gate and up of output i
      bf16* o = static_cast<bf16*>(p.out) + (long long)t * p.ldo + (f >> 1);
      const float y0 = gelu_sigmoid(v.x) * v.y, y1 = gelu_sigmoid(v.z) * v.w;
      if (p.vec_out && nf == 4) {
        *reinterpret_cast<uint32_t*>(o) = pack_bf16x2(y0, y1);
      } else {
        o[0] = __float2bfloat16(y0);
        if (nf > 3) o[1] = __float2bfloat16(y1);
      }
    }
  }
  if (cl > 1) cluster_sync();  // the others may still read this CTA's tile
}

}  // namespace g8
}  // namespace fvb
