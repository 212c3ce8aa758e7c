// A key-value cache in pages, [pages, page_size, kv_heads, dim] bf16 with any
// strides: rows are appended with the rotary positions applied on the way
// (append_kernel), and one new token of each sequence attends over the pages
// of its table row (attend_kernel).
#pragma once

#include "attention.cuh"
#include "common.cuh"

namespace fvb {
namespace paged {

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendDev {
  const bf16* q;
  long long q_rs, q_hs;
  const bf16* k;
  long long k_rs, k_hs;
  const bf16* v;
  long long v_rs, v_hs;
  bf16* q_out;
  long long qo_rs, qo_hs;
  bf16* k_cache;
  bf16* v_cache;
  long long kc_ps, kc_rs, kc_hs;  // strides of a page, a row, a head
  long long vc_ps, vc_rs, vc_hs;
  const int* slots;
  const int* positions;
  const float* rope_cs;
  int tokens, heads, kv_heads, dim;
  int page_size, max_pos, interleaved;
  long long n_slots;
};

// 8 rotary pairs of one head: the pairs' first halves in a, second in b
__device__ __forceinline__ void rotate8(float (&a)[8], float (&b)[8], const float* cs) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float4 t = __ldg(reinterpret_cast<const float4*>(cs + 2 * i));
    const float a0 = a[i], b0 = b[i], a1 = a[i + 1], b1 = b[i + 1];
    a[i] = a0 * t.x - b0 * t.y;
    b[i] = b0 * t.x + a0 * t.y;
    a[i + 1] = a1 * t.z - b1 * t.w;
    b[i + 1] = b1 * t.z + a1 * t.w;
  }
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __bfloat1622float2(h[j]);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                    pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// One thread moves 16 elements of one head of one token (8 rotary pairs) with
// 16-byte accesses (VEC), or 2 elements (one pair) where alignment or the
// head size rule those out.
template <bool VEC>
__global__ void __launch_bounds__(256) append_kernel(const AppendDev p) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int EL = VEC ? 16 : 2;
  const unsigned per_head = p.dim / EL;
  const unsigned per_token = per_head * (p.heads + 2 * p.kv_heads);
  const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long tok = idx / per_token;
  if (tok >= p.tokens) return;
  const unsigned item = (unsigned)(idx - tok * per_token);
  const int head = item / per_head, ch = item - head * per_head;
  const int slot = __ldg(p.slots + tok);
  const bool is_q = head < p.heads, is_v = head >= p.heads + p.kv_heads;
  if (slot < 0 && !is_q) return;  // a row that is not cached
  int pos = 0;
  if (p.rope_cs) {
    pos = __ldg(p.positions + tok);
    if (pos < 0 || pos >= p.max_pos) {
      // padding has no position; a cached row needs one
      if (slot >= 0) record_device_error(FVB_ERR_INVALID_ARG);
      return;
    }
  }
  if (slot >= p.n_slots) {
    record_device_error(FVB_ERR_INVALID_ARG);
    return;
  }
  const bf16* src;
  bf16* dst;
  if (is_q) {
    src = p.q + tok * p.q_rs + head * p.q_hs;
    dst = p.q_out + tok * p.qo_rs + head * p.qo_hs;
  } else {
    const int page = slot / p.page_size, at = slot - page * p.page_size;
    const int h = head - p.heads - (is_v ? p.kv_heads : 0);
    src = is_v ? p.v + tok * p.v_rs + h * p.v_hs : p.k + tok * p.k_rs + h * p.k_hs;
    dst = is_v ? p.v_cache + page * p.vc_ps + at * p.vc_rs + h * p.vc_hs
               : p.k_cache + page * p.kc_ps + at * p.kc_rs + h * p.kc_hs;
  }
  const bool turn = !is_v && p.rope_cs;
  const float* cs = turn ? p.rope_cs + ((long long)pos * (p.dim / 2) + ch * (EL / 2)) * 2 : nullptr;
  // the two halves of the pairs: dims i and i + dim/2, or 2i and 2i + 1
  const int first = turn && !p.interleaved ? ch * (EL / 2) : ch * EL;
  const int second = turn && !p.interleaved ? first + p.dim / 2 : first + EL / 2;
  if (VEC) {
    uint4 u0 = *reinterpret_cast<const uint4*>(src + first);
    uint4 u1 = *reinterpret_cast<const uint4*>(src + second);
    if (turn) {
      float x[8], y[8];
      unpack8(u0, x);
      unpack8(u1, y);
      if (p.interleaved) {
        float a[8], b[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = x[2 * i]; b[i] = x[2 * i + 1];
          a[4 + i] = y[2 * i]; b[4 + i] = y[2 * i + 1];
        }
        rotate8(a, b, cs);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] = a[i]; x[2 * i + 1] = b[i];
          y[2 * i] = a[4 + i]; y[2 * i + 1] = b[4 + i];
        }
      } else {
        rotate8(x, y, cs);
      }
      u0 = pack8(x);
      u1 = pack8(y);
    }
    *reinterpret_cast<uint4*>(dst + first) = u0;
    *reinterpret_cast<uint4*>(dst + second) = u1;
  } else {
    bf16 a = src[first], b = src[second];
    if (turn) {
      const float fa = __bfloat162float(a), fb = __bfloat162float(b);
      const float c = __ldg(cs), s = __ldg(cs + 1);
      a = __float2bfloat16(fa * c - fb * s);
      b = __float2bfloat16(fb * c + fa * s);
    }
    dst[first] = a;
    dst[second] = b;
  }
}

// ---------------------------------------------------------------------------
// one new token of each sequence over its pages
//
// An item is (sequence, kv head, block of up to 8*NT query heads of the
// group); its keys are cut into units of 64.  All items' units are laid end
// to end and every CTA takes an equal run of them, whatever the lengths are:
// the lengths are read on the device, so the launch is the same for all of
// them.  A CTA whose run holds a whole item writes its output; the others
// write (O, max, sum) to the workspace, and the last of an item's CTAs to
// arrive joins them in the order of the keys.
//
// Inside a CTA each warp takes 16 of a unit's 64 keys with its own ring of
// tiles, maximum and sum, so that no barrier stands in the loop:
//   S^T [16 keys x 8 heads] = K [16 x dim] Q^T     (mma m16n8k16, K as stored)
//   O^T [dim x 8 heads]    += V^T [dim x 16 keys] P^T
// With the keys on the M side the heads of a group fill the 8 columns, where
// queries on the M side would leave half or more of 16 rows empty.  A row of
// K or V is one bulk copy of dim * 2 bytes to a padded shared-memory row, so
// pages of any size and any stride are read alike.
// ---------------------------------------------------------------------------
struct AttendDev {
  const bf16* q;
  long long q_rs, q_hs;
  const bf16* k;
  long long k_ps, k_rs, k_hs;
  const bf16* v;
  long long v_ps, v_rs, v_hs;
  bf16* o;
  long long o_rs, o_hs;
  float* lse;
  long long lse_rs;
  const int* table;
  long long ld_table;
  const int* lens;
  int batch, heads, kv_heads, group;
  int head_blocks;  // blocks of 8*NT heads in a group
  int n_pages, page_size, max_len;
  float scale_log2;
  int* arrivals;    // [CTAs], zero between calls; an item that several CTAs share
                    // counts at its first one, which is no other's first
  float* part_o;    // [CTAs][2][8*NT][dim]
  float* part_ml;   // [CTAs][2][8*NT][2]
};

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int SUB = 16;            // keys of one warp's tile
constexpr int UNIT = WARPS * SUB;  // keys of one unit

template <int D, int NT>
struct Cfg {
  static constexpr int HB = 8 * NT;                 // heads of one item
  static constexpr int PITCH = D * 2 + 16;          // bytes of a tile row
  static constexpr int TILE = 2 * SUB * PITCH;      // K rows, then V rows
  static constexpr int STAGES = D == 256 ? 3 : (D == 128 ? 6 : 10);
  static constexpr int RING = WARPS * STAGES * TILE;
  static constexpr int OPITCH = D + 4;              // floats of a joined row
  static_assert(WARPS * HB * OPITCH * 4 <= RING, "the join reuses the ring");
  static constexpr int OFF_ML = RING;               // [WARPS][HB][2] f32
  static constexpr int OFF_BAR = OFF_ML + WARPS * HB * 2 * 4;
  static constexpr int SMEM = OFF_BAR + WARPS * STAGES * 8;
};

__device__ __forceinline__ void bulk_row(uint32_t dst, const void* src, uint32_t bytes,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// transpose of an 8x8 tile of 16-bit values held as a matrix fragment
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ int clamped_len(const AttendDev& p, int b) {
  const int n = __ldg(p.lens + b);
  return min(max(n, 0), p.max_len);
}

// Where the runs of units lie: CTA c of C has units [total*c/C, total*(c+1)/C).
struct Plan {
  long long total;
  int ctas;
  __device__ long long first(int c) const { return total * c / ctas; }
  __device__ int owner(long long unit) const {
    return static_cast<int>(((unit + 1) * ctas - 1) / total);
  }
};

// Joins the partials of one item's CTAs c0..c1, in order, and writes the
// output rows (called by the CTA that arrived last).
template <int D, int NT>
__device__ __forceinline__ void join(const AttendDev& p, uint8_t* smem, int c0, int c1, int b,
                                     int head0, int n_heads) {
  using C = Cfg<D, NT>;
  const int tid = threadIdx.x, np = c1 - c0 + 1;
  float* wgt = reinterpret_cast<float*>(smem);  // [np][HB]
  for (int h = tid; h < C::HB; h += THREADS) {
    float m = -INFINITY;
    for (int i = 0; i < np; ++i) {
      const long long s = 2 * (c0 + i) + (i == 0);
      m = fmaxf(m, __ldcg(p.part_ml + (s * C::HB + h) * 2));
    }
    const float mu = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int i = 0; i < np; ++i) {
      const long long s = 2 * (c0 + i) + (i == 0);
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + (s * C::HB + h) * 2));
      const float f = exp2_fast(ml.x - mu);
      wgt[i * C::HB + h] = f;
      l += ml.y * f;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    for (int i = 0; i < np; ++i) wgt[i * C::HB + h] *= inv;
    if (h < n_heads && p.lse)
      p.lse[b * p.lse_rs + head0 + h] = (mu + log2f(l)) * 0.6931471805599453f;
  }
  __syncthreads();
  for (int e = tid; e < n_heads * (D / 4); e += THREADS) {
    const int h = e / (D / 4), d = (e % (D / 4)) * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < np; ++i) {
      const long long s = 2 * (c0 + i) + (i == 0);
      const float4 t =
          __ldcg(reinterpret_cast<const float4*>(p.part_o + (s * C::HB + h) * D + d));
      const float f = wgt[i * C::HB + h];
      a.x += t.x * f; a.y += t.y * f; a.z += t.z * f; a.w += t.w * f;
    }
    *reinterpret_cast<uint2*>(p.o + b * p.o_rs + (head0 + h) * p.o_hs + d) =
        make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
  }
  __syncthreads();
}

template <int D, int NT>
__global__ void __launch_bounds__(THREADS, 1) attend_kernel(const AttendDev p) {
  using C = Cfg<D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  float* s_o = reinterpret_cast<float*>(smem);
  float* s_ml = reinterpret_cast<float*>(smem + C::OFF_ML);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  __shared__ long long s_scan[THREADS];
  __shared__ int s_at[4];
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint64_t* full = bars + warp * C::STAGES;
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * C::TILE;
  if (lane == 0)
    for (int s = 0; s < C::STAGES; ++s) mbar_init(&full[s], 1);
  fence_barrier_init();
  griddep_wait();
  griddep_launch_dependents();
  const int per_seq = p.kv_heads * p.head_blocks;  // items of one sequence

  // total units, and the empty sequences' rows
  long long mine = 0;
  for (int b = tid; b < p.batch; b += THREADS) {
    const int n = clamped_len(p, b);
    if (n != __ldg(p.lens + b)) record_device_error(FVB_ERR_INVALID_ARG);
    mine += (n + UNIT - 1) / UNIT;
  }
  s_scan[tid] = mine;
  __syncthreads();
  long long total = 0;
  for (int i = 0; i < THREADS; ++i) total += s_scan[i];
  __syncthreads();
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (clamped_len(p, b) > 0) continue;
    for (int e = tid; e < p.heads * (D / 4); e += THREADS)
      *reinterpret_cast<uint2*>(p.o + b * p.o_rs + (e / (D / 4)) * p.o_hs + (e % (D / 4)) * 4) =
          make_uint2(0u, 0u);
    if (p.lse)
      for (int h = tid; h < p.heads; h += THREADS) p.lse[b * p.lse_rs + h] = -INFINITY;
  }
  if (total == 0) return;
  Plan plan;
  plan.total = total * per_seq;
  plan.ctas = static_cast<int>(min((long long)gridDim.x, plan.total));
  if ((int)blockIdx.x >= plan.ctas) return;
  long long u = plan.first(blockIdx.x);
  const long long u_end = plan.first(blockIdx.x + 1);

  // the sequence that holds unit u: units of 128 sequences at a time
  int b = 0;
  long long seq_first = 0;  // first unit of sequence b
  {
    long long base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += THREADS) {
      const int bb = b0 + tid;
      const int n = bb < p.batch ? clamped_len(p, bb) : 0;
      s_scan[tid] = (long long)((n + UNIT - 1) / UNIT) * per_seq;
      if (tid == 0) s_at[0] = -1;
      __syncthreads();
      for (int o = 1; o < THREADS; o <<= 1) {
        const long long t = tid >= o ? s_scan[tid - o] : 0;
        __syncthreads();
        s_scan[tid] += t;
        __syncthreads();
      }
      const long long hi = base + s_scan[tid];
      const long long lo = base + (tid ? s_scan[tid - 1] : 0);
      if (u >= lo && u < hi) s_at[0] = tid;
      __syncthreads();
      const int at = s_at[0];
      const long long before = at > 0 ? s_scan[at - 1] : 0;
      const long long sum = s_scan[THREADS - 1];
      __syncthreads();
      if (at >= 0) {
        b = b0 + at;
        seq_first = base + before;
        break;
      }
      base += sum;
    }
  }

  int cnt = 0;  // tiles this warp has taken, over all items
  bool alive = true;
  while (u < u_end && alive) {
    int len = clamped_len(p, b);
    int n_units = (len + UNIT - 1) / UNIT;
    while (u >= seq_first + (long long)n_units * per_seq) {
      seq_first += (long long)n_units * per_seq;
      ++b;
      len = clamped_len(p, b);
      n_units = (len + UNIT - 1) / UNIT;
    }
    const int item = static_cast<int>((u - seq_first) / n_units);
    const long long item_first = seq_first + (long long)item * n_units;
    const int kvh = item / p.head_blocks, hblk = item % p.head_blocks;
    const int head0 = kvh * p.group + hblk * C::HB;
    const int n_heads = min(C::HB, p.group - hblk * C::HB);
    const int k_first = static_cast<int>(u - item_first);
    const int k_last = static_cast<int>(min(u_end - item_first, (long long)n_units));  // excl.
    // this warp's tiles: one per unit, the last one may lie past the keys
    int n_tiles = k_last - k_first;
    if ((k_last - 1) * UNIT + warp * SUB >= len) --n_tiles;

    const bf16* kb = p.k + kvh * p.k_hs;
    const bf16* vb = p.v + kvh * p.v_hs;
    const int* table = p.table + b * p.ld_table;
    auto issue = [&](int i) {
      const int st = (cnt + i) % C::STAGES;
      const int k0 = (k_first + i) * UNIT + warp * SUB;
      const int nv = min(SUB, len - k0);
      const int r = lane & 15;
      if (lane == 0) mbar_arrive_expect_tx(&full[st], (uint32_t)(nv * 2 * D * 2));
      __syncwarp();
      if (r < nv) {
        const unsigned key = k0 + r, pg = key / (unsigned)p.page_size;
        const int at = key - pg * p.page_size;
        int page = __ldg(table + pg);
        if (page < 0 || page >= p.n_pages) {
          record_device_error(FVB_ERR_INVALID_ARG);
          page = 0;
        }
        const uint32_t dst = ring + st * C::TILE + lane * C::PITCH;
        const bf16* src = lane < 16 ? kb + page * p.k_ps + at * p.k_rs
                                    : vb + page * p.v_ps + at * p.v_rs;
        bulk_row(dst, src, D * 2, &full[st]);
      }
    };
    // queries: B fragments (dims x heads), heads past the group are zero
    uint32_t qf[NT][D / 16][2];
    {
      const int dd = 2 * (lane & 3);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int h = t * 8 + (lane >> 2);
        const bf16* qp = p.q + b * p.q_rs + (head0 + h) * p.q_hs + dd;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          qf[t][j][0] = h < n_heads ? *reinterpret_cast<const uint32_t*>(qp + 16 * j) : 0u;
          qf[t][j][1] = h < n_heads ? *reinterpret_cast<const uint32_t*>(qp + 16 * j + 8) : 0u;
        }
      }
    }
    for (int i = 0; i < min(n_tiles, C::STAGES); ++i) issue(i);

    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][j][e] = 0.f;
    }
    for (int i = 0; i < n_tiles; ++i) {
      const int st = (cnt + i) % C::STAGES;
      if (!mbar_wait_spin(&full[st], ((cnt + i) / C::STAGES) & 1)) { alive = false; break; }
      const uint32_t sk = ring + st * C::TILE, sv = sk + SUB * C::PITCH;
      const int nv = min(SUB, len - ((k_first + i) * UNIT + warp * SUB));
      // two chains of products, so that one does not wait for the other
      float s[2][NT][4];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[c][t][e] = 0.f;
      const uint32_t ka = sk + (lane & 15) * C::PITCH + (lane >> 4) * 16;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t a0, a1, a2, a3;
        ldsm_x4(ka + j * 32, a0, a1, a2, a3);
#pragma unroll
        for (int t = 0; t < NT; ++t)
          mma_bf16_16816(s[j & 1][t], a0, a1, a2, a3, qf[t][j][0], qf[t][j][1]);
      }
      const int key = lane >> 2;
      uint32_t ph[NT][2], pl[NT][2];
      bool grew = false;
      float alpha[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = (s[0][t][e] + s[1][t][e]) * p.scale_log2;
          if (key + (e >> 1) * 8 >= nv) x[e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(x[e], x[e + 2]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(m[t][e], mx);
          const float mu = mn == -INFINITY ? 0.f : mn;
          alpha[t][e] = exp2_fast(m[t][e] - mu);
          grew |= mn != m[t][e];
          m[t][e] = mn;
          x[e] = exp2_fast(x[e] - mu);
          x[e + 2] = exp2_fast(x[e + 2] - mu);
          l[t][e] = l[t][e] * alpha[t][e] + x[e] + x[e + 2];
        }
        // p as the sum of two bf16: a single one would add its rounding
        // (2^-9 of each weight) to the output's own
        const uint32_t h01 = pack_bf16x2(x[0], x[1]), h23 = pack_bf16x2(x[2], x[3]);
        const float2 f01 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&h01));
        const float2 f23 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&h23));
        ph[t][0] = transpose8(h01);
        ph[t][1] = transpose8(h23);
        pl[t][0] = transpose8(pack_bf16x2(x[0] - f01.x, x[1] - f01.y));
        pl[t][1] = transpose8(pack_bf16x2(x[2] - f23.x, x[3] - f23.y));
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][j][e] *= alpha[t][e & 1];
      }
      // keys past the last one: their tile rows hold what was there before,
      // which times a weight of zero may still be NaN
      const int kk = 2 * (lane & 3);
      const uint32_t m0 = (kk < nv ? 0xffffu : 0u) | (kk + 1 < nv ? 0xffff0000u : 0u);
      const uint32_t m1 = (kk + 8 < nv ? 0xffffu : 0u) | (kk + 9 < nv ? 0xffff0000u : 0u);
      const uint32_t va = sv + ((lane & 7) + ((lane >> 4) & 1) * 8) * C::PITCH +
                          ((lane >> 3) & 1) * 16;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t a0, a1, a2, a3;
        ldsm_x4_t(va + j * 32, a0, a1, a2, a3);
        if (nv < SUB) { a0 &= m0; a1 &= m0; a2 &= m1; a3 &= m1; }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma_bf16_16816(o[t][j], a0, a1, a2, a3, ph[t][0], ph[t][1]);
          mma_bf16_16816(o[t][j], a0, a1, a2, a3, pl[t][0], pl[t][1]);
        }
      }
      __syncwarp();
      if (i + C::STAGES < n_tiles) issue(i + C::STAGES);
    }
    cnt += n_tiles;
    // every wait that ran out ends the CTA here, together
    if (__syncthreads_or(!alive)) return;

    // join the warps: factors from the common maximum, then the sum of O
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 4);
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 8);
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 16);
        if (lane < 4) {
          const int h = t * 8 + 2 * lane + e;
          s_ml[(warp * C::HB + h) * 2] = m[t][e];
          s_ml[(warp * C::HB + h) * 2 + 1] = l[t][e];
        }
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = t * 8 + 2 * (lane & 3) + e;
        float mx = -INFINITY;
        for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, s_ml[(w * C::HB + h) * 2]);
        const float f = exp2_fast(m[t][e] - (mx == -INFINITY ? 0.f : mx));
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          const int d = j * 16 + (lane >> 2);
          s_o[(warp * C::HB + h) * C::OPITCH + d] = o[t][j][e] * f;
          s_o[(warp * C::HB + h) * C::OPITCH + d + 8] = o[t][j][e + 2] * f;
        }
      }
    __syncthreads();
    const bool whole = k_first == 0 && k_last == n_units;
    const int c0 = plan.owner(item_first), c1 = plan.owner(item_first + n_units - 1);
    const long long slot = 2ll * blockIdx.x + ((int)blockIdx.x == c0 ? 1 : 0);
    for (int e = tid; e < C::HB * (D / 4); e += THREADS) {
      const int h = e / (D / 4), d = (e % (D / 4)) * 4;
      float mx = -INFINITY, sum = 0.f;
      for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, s_ml[(w * C::HB + h) * 2]);
      const float mu = mx == -INFINITY ? 0.f : mx;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < WARPS; ++w) {
        sum += s_ml[(w * C::HB + h) * 2 + 1] * exp2_fast(s_ml[(w * C::HB + h) * 2] - mu);
        const float4 t =
            *reinterpret_cast<const float4*>(s_o + (w * C::HB + h) * C::OPITCH + d);
        a.x += t.x; a.y += t.y; a.z += t.z; a.w += t.w;
      }
      if (whole) {
        if (h < n_heads) {
          const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
          *reinterpret_cast<uint2*>(p.o + b * p.o_rs + (head0 + h) * p.o_hs + d) =
              make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
          if (d == 0 && p.lse)
            p.lse[b * p.lse_rs + head0 + h] = (mu + log2f(sum)) * 0.6931471805599453f;
        }
      } else {
        *reinterpret_cast<float4*>(p.part_o + (slot * C::HB + h) * D + d) = a;
        if (d == 0)
          *reinterpret_cast<float2*>(p.part_ml + (slot * C::HB + h) * 2) = make_float2(mx, sum);
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        int* a = p.arrivals + c0;
        const int old = atomicAdd(a, 1);
        s_last = old == c1 - c0;
        if (s_last) *a = 0;  // as the next call finds it
        __threadfence();
      }
      __syncthreads();
      if (s_last) join<D, NT>(p, smem, c0, c1, b, head0, n_heads);
    }
    // generic accesses of the ring end before the next item's bulk copies
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    u = item_first + k_last;
  }
}

}  // namespace paged
}  // namespace fvb
