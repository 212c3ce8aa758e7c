// A key-value cache in pages, [pages, page_size, kv_heads, dim] bf16 with any
// strides: rows are appended with the rotary positions applied on the way
// (append_kernel), and one new token of each sequence attends over the pages
// of its table row (attend_kernel).
//
// The kernels start while the one before them in the stream may still write
// what they read, so everything is read by ordinary loads after griddep_wait:
// the read-only path (__ldg) is for data that nothing writes in the kernel's
// life, its start before that wait included.
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
  int heads_per_thread;  // VEC
  long long n_slots;
};

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
__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
  const float x = a, y = b;
  a = x * c - y * s;
  b = y * c + x * s;
}

// Where one head's row of a token comes from and goes to; false if nowhere.
struct Row {
  const bf16* src;
  bf16* dst;
};
__device__ __forceinline__ bool row_of(const AppendDev& p, long long tok, int head, int slot,
                                       Row* r) {
  if (head < p.heads) {
    r->src = p.q + tok * p.q_rs + head * p.q_hs;
    r->dst = p.q_out + tok * p.qo_rs + head * p.qo_hs;
    return true;
  }
  if (slot < 0) return false;  // a row that is not cached
  const int page = slot / p.page_size, at = slot - page * p.page_size;
  int h = head - p.heads;
  if (h < p.kv_heads) {
    r->src = p.k + tok * p.k_rs + h * p.k_hs;
    r->dst = p.k_cache + page * p.kc_ps + at * p.kc_rs + h * p.kc_hs;
  } else {
    h -= p.kv_heads;
    r->src = p.v + tok * p.v_rs + h * p.v_hs;
    r->dst = p.v_cache + page * p.vc_ps + at * p.vc_rs + h * p.vc_hs;
  }
  return true;
}

// A token's slot and position; false if its rows are left alone.
__device__ __forceinline__ bool token_of(const AppendDev& p, long long tok, int* slot, int* pos) {
  *slot = p.slots[tok];
  *pos = 0;
  bool ok = *slot < p.n_slots;
  if (p.rope_cs) {
    *pos = p.positions[tok];
    if (*pos < 0 || *pos >= p.max_pos) {
      if (*slot < 0) return false;  // padding has no position; a cached row needs one
      ok = false;
    }
  }
  if (!ok) record_device_error(FVB_ERR_INVALID_ARG);
  return ok;
}

// Bound by HBM: a thread moves 16 elements (8 rotary pairs, one chunk) of
// heads_per_thread heads of one token with 16-byte accesses, two heads in
// flight, and reads the chunk's cosines and sines once for them (a thread per
// head read them from L1 for every head: 13056 x 10 heads of 256 took 38 us, now
// 25.7; four heads in flight, whose registers leave fewer threads, 28.6).
__global__ void __launch_bounds__(256) append_vec_kernel(const AppendDev p) {
  griddep_wait();
  griddep_launch_dependents();
  const unsigned per_head = p.dim / 16, total = p.heads + 2 * p.kv_heads;
  const unsigned blocks = (total + p.heads_per_thread - 1) / p.heads_per_thread;
  const unsigned per_token = per_head * blocks;
  const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long tok = idx / per_token;
  if (tok >= p.tokens) return;
  const unsigned item = (unsigned)(idx - tok * per_token);
  const int blk = item / per_head, ch = item - blk * per_head;
  const int h0 = blk * p.heads_per_thread;
  const int h1 = min(h0 + p.heads_per_thread, (int)total);
  const int rotated = p.rope_cs ? p.heads + p.kv_heads : 0;
  int slot, pos;
  if (!token_of(p, tok, &slot, &pos)) return;
  float4 cs[4];
  if (h0 < rotated) {
    const float4* t = reinterpret_cast<const float4*>(p.rope_cs + ((long long)pos * (p.dim / 2) + ch * 8) * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) cs[i] = t[i];
  }
  constexpr int U = 2;
  for (int hb = h0; hb < h1; hb += U) {
    Row row[U];
    uint4 u[U][2];
    bool in[U];
    int first[U], second[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      // the two halves of the pairs: dims i and i + dim/2, or 2i and 2i + 1
      const bool half = hb + i < rotated && !p.interleaved;
      first[i] = ch * (half ? 8 : 16);
      second[i] = first[i] + (half ? p.dim / 2 : 8);
      in[i] = hb + i < h1 && row_of(p, tok, hb + i, slot, &row[i]);
      if (in[i]) {
        u[i][0] = *reinterpret_cast<const uint4*>(row[i].src + first[i]);
        u[i][1] = *reinterpret_cast<const uint4*>(row[i].src + second[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (!in[i]) continue;
      if (hb + i < rotated) {
        float x[8], y[8];
        unpack8(u[i][0], x);
        unpack8(u[i][1], y);
        if (p.interleaved) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            rotate(x[4 * j], x[4 * j + 1], cs[j].x, cs[j].y);
            rotate(x[4 * j + 2], x[4 * j + 3], cs[j].z, cs[j].w);
            rotate(y[4 * j], y[4 * j + 1], cs[2 + j].x, cs[2 + j].y);
            rotate(y[4 * j + 2], y[4 * j + 3], cs[2 + j].z, cs[2 + j].w);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            rotate(x[2 * j], y[2 * j], cs[j].x, cs[j].y);
            rotate(x[2 * j + 1], y[2 * j + 1], cs[j].z, cs[j].w);
          }
        }
        u[i][0] = pack8(x);
        u[i][1] = pack8(y);
      }
      *reinterpret_cast<uint4*>(row[i].dst + first[i]) = u[i][0];
      *reinterpret_cast<uint4*>(row[i].dst + second[i]) = u[i][1];
    }
  }
}

// One rotary pair of one head a thread, where alignment or the head size rule
// 16-byte accesses out: bound by its 2-byte accesses, 112 us on 13056 tokens of
// 10 heads of 256 whose rows are an odd number of values apart.
__global__ void __launch_bounds__(256) append_kernel(const AppendDev p) {
  griddep_wait();
  griddep_launch_dependents();
  const unsigned per_head = p.dim / 2;
  const unsigned per_token = per_head * (p.heads + 2 * p.kv_heads);
  const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long tok = idx / per_token;
  if (tok >= p.tokens) return;
  const unsigned item = (unsigned)(idx - tok * per_token);
  const int head = item / per_head, ch = item - head * per_head;
  int slot, pos;
  Row row;
  if (!token_of(p, tok, &slot, &pos) || !row_of(p, tok, head, slot, &row)) return;
  const bool turn = p.rope_cs && head < p.heads + p.kv_heads;
  const bool half = turn && !p.interleaved;
  const int first = half ? ch : 2 * ch, second = half ? ch + p.dim / 2 : 2 * ch + 1;
  bf16 a = row.src[first], b = row.src[second];
  if (turn) {
    const float2 cs = reinterpret_cast<const float2*>(p.rope_cs)[(long long)pos * per_head + ch];
    float x = __bfloat162float(a), y = __bfloat162float(b);
    rotate(x, y, cs.x, cs.y);
    a = __float2bfloat16(x);
    b = __float2bfloat16(y);
  }
  row.dst[first] = a;
  row.dst[second] = b;
}

// ---------------------------------------------------------------------------
// one new token of each sequence over its pages
//
// An item is (sequence, kv head, block of up to 8*NT query heads of the
// group); its keys are cut into units of 128.  All items' units are laid end
// to end and every CTA takes an equal run of them, whatever the lengths are:
// the lengths are read on the device, so the launch is the same for all of
// them.  A CTA whose run holds a whole item writes its output; the others
// write (O, max, sum) to the workspace.  Of every 8 neighbouring CTAs of an
// item the last to arrive joins the partials of the 8 in the order of the
// keys, and the last group to be done joins the groups' (one CTA that joined
// all 148 partials of a long sequence took 30 us for it).
//
// Inside a CTA each of 8 warps takes 16 of a unit's keys with its own ring of
// tiles (16 rows of K, then the same 16 of V), maximum and sum, so that no
// barrier stands in the loop:
//   S^T [16 keys x 8 heads] = K [16 x dim] Q^T     (mma m16n8k16, K as stored)
//   O^T [dim x 8 heads]    += V^T [dim x 16 keys] P^T
// With the keys on the M side the heads of a group fill the 8 columns, where
// queries on the M side would leave half or more of 16 rows empty.
//
// BOXES: where 16 keys always lie in one page (page_size % 16 == 0) a tile is
// dim / 64 tensor-map boxes of 16 rows x 128 bytes, swizzled.  Other pages are
// read with one bulk copy for each row of dim * 2 bytes, to padded rows; an SM
// starts one such copy in about 16 clocks, whatever its size, which holds rows
// of 128 bytes to 2.2 TB/s and rows of 256 to 4.5.
//
// NT = 2 (9 to 16 heads of a group) at 256 dims needs more registers than there
// are, and spills some 100 bytes: 16 x 20000 keys take 82 us (4.0 TB/s), with
// 8 heads 66 us (5.0 TB/s).
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
  int* arrivals;    // [CTAs][3], zero between calls: arrivals at the group that
                    // begins with this CTA inside an item, at the one that
                    // begins with the item's first CTA, and groups of the item
                    // that begins here
  float* part_o;    // [CTAs][2][8*NT][dim]
  float* part_ml;   // [CTAs][2][8*NT][2]
};

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int SUB = 16;            // keys of one warp's tile
constexpr int UNIT = WARPS * SUB;  // keys of one unit

template <int D, int NT, bool BOXES>
struct Cfg {
  static constexpr int HB = 8 * NT;                 // heads of one item
  static constexpr int PITCH = D * 2 + 16;          // bytes of a tile row (not BOXES)
  static constexpr int TILE = BOXES ? SUB * D * 2 : SUB * PITCH;  // 16 rows of K or of V
  static constexpr int SLOTS = D == 256 ? 3 : (D == 128 ? 6 : 12);
  static constexpr int RING = WARPS * SLOTS * TILE;
  static_assert(8 * D * 4 <= TILE && SLOTS > NT, "8 heads of O fit a slot");
  static constexpr int OFF_ML = RING;               // [WARPS][HB][2] f32
  static constexpr int OFF_TOT = OFF_ML + WARPS * HB * 2 * 4;   // [HB][2] f32
  static constexpr int OFF_SLOT = OFF_TOT + HB * 2 * 4;         // [WARPS] int
  static constexpr int OFF_BAR = OFF_SLOT + WARPS * 4;
  static constexpr int SMEM = OFF_BAR + WARPS * SLOTS * 8 + 1024;
};

__device__ __forceinline__ void bulk_row(uint32_t dst, const void* src, uint32_t bytes,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void box_row16(uint32_t dst, const CUtensorMap* map, int x, int row,
                                          int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(head), "r"(page),
      "r"(smem_u32(bar))
      : "memory");
}

// place of (head h of 8, dim d) in a warp's O: the pairs of heads that a
// matrix fragment holds fall on different banks
template <int D>
__device__ __forceinline__ int o_at(int h, int d) {
  return h * D + (d ^ ((h >> 1) * 8));
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
  const int n = p.lens[b];
  return min(max(n, 0), p.max_len);
}

// Where the runs of units lie: each CTA has `per` of them, the first `more`
// CTAs one more.
struct Plan {
  int per, more;
  __device__ Plan(int total, int ctas) : per(total / ctas), more(total % ctas) {}
  __device__ int first(int c) const { return c * per + min(c, more); }
  __device__ int owner(int unit) const {
    const int big = more * (per + 1);
    return unit < big ? unit / (per + 1) : more + (unit - big) / per;
  }
};

constexpr int JOIN = 8;  // partials of one group

// Partials of CTAs c, c + step, .. (n of them) of an item whose first CTA is
// c0, joined in order: into the output rows, or (!FINAL) into the first one's
// place.  A CTA's partial of the item that begins in it has slot 1, of the one
// that began before it slot 0.
template <int D, int NT, bool FINAL>
__device__ __forceinline__ void join(const AttendDev& p, int c0, int c, int n, int step, int b,
                                     int head0, int n_heads) {
  constexpr int HB = 8 * NT;
  auto slot = [&](int i) { return 2ll * (c + i * step) + (c + i * step == c0); };
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  for (int e = threadIdx.x; e < (FINAL ? n_heads : HB) * (D / 4); e += THREADS) {
    const int h = e / (D / 4), d = (e % (D / 4)) * 4;
    float mx = -INFINITY, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < n; i0 += JOIN) {
      // all loads of 8 partials at once
      float2 t[JOIN];
      float4 v[JOIN];
#pragma unroll
      for (int i = 0; i < JOIN; ++i) {
        const long long at = slot(i0 + i) * HB + h;
        const bool in = i0 + i < n;
        t[i] = in ? __ldcg(ml + at) : make_float2(-INFINITY, 0.f);
        v[i] = in ? __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D + d))
                  : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      const float before = mx;
#pragma unroll
      for (int i = 0; i < JOIN; ++i) mx = fmaxf(mx, t[i].x);
      const float mu = mx == -INFINITY ? 0.f : mx;
      const float r = exp2_fast(before - mu);
      l *= r; a.x *= r; a.y *= r; a.z *= r; a.w *= r;
#pragma unroll
      for (int i = 0; i < JOIN; ++i) {
        const float f = exp2_fast(t[i].x - mu);
        l = fmaf(t[i].y, f, l);
        a.x = fmaf(v[i].x, f, a.x); a.y = fmaf(v[i].y, f, a.y);
        a.z = fmaf(v[i].z, f, a.z); a.w = fmaf(v[i].w, f, a.w);
      }
    }
    const float mu = mx == -INFINITY ? 0.f : mx;
    if (FINAL) {
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      *reinterpret_cast<uint2*>(p.o + b * p.o_rs + (head0 + h) * p.o_hs + d) =
          make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
      if (d == 0 && p.lse) p.lse[b * p.lse_rs + head0 + h] = (mu + log2f(l)) * 0.6931471805599453f;
    } else {
      *reinterpret_cast<float4*>(p.part_o + (slot(0) * HB + h) * D + d) = a;
    }
  }
  if (FINAL) return;
  __syncthreads();  // the threads of a head have read its (max, sum)
  if (threadIdx.x < HB) {
    const int h = threadIdx.x;
    float2 t[JOIN];
    float mx = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < JOIN; ++i) {
      t[i] = i < n ? __ldcg(ml + slot(i) * HB + h) : make_float2(-INFINITY, 0.f);
      mx = fmaxf(mx, t[i].x);
    }
    const float mu = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int i = 0; i < JOIN; ++i) l = fmaf(t[i].y, exp2_fast(t[i].x - mu), l);
    *reinterpret_cast<float2*>(p.part_ml + (slot(0) * HB + h) * 2) = make_float2(mx, l);
  }
}

// A run of units of one item.
struct Run {
  int b, len, n_units;
  int first;             // the item's first unit
  int k_first, k_last;   // the run's units in it (the last one excluded)
  int kvh, head0, n_heads;
  int n_tiles;           // of this warp
};

template <int D, int NT, bool BOXES>
__global__ void __launch_bounds__(THREADS, 1)
    attend_kernel(const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const AttendDev p) {
  using C = Cfg<D, NT, BOXES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_ml = reinterpret_cast<float*>(smem + C::OFF_ML);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  __shared__ int s_sum[WARPS], s_first, s_b, s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint64_t* full = bars + warp * C::SLOTS;
  uint8_t* ring_ptr = smem + warp * C::SLOTS * C::TILE;
  const uint32_t ring = smem_u32(ring_ptr);
  if (lane == 0)
    for (int s = 0; s < C::SLOTS; ++s) mbar_init(&full[s], 1);
  if (BOXES && tid == 0) {
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  fence_barrier_init();
  griddep_wait();
  griddep_launch_dependents();
  const int per_seq = p.kv_heads * p.head_blocks;  // items of one sequence

  // units before each thread's sequences, by a scan over the CTA
  const int chunk = (p.batch + THREADS - 1) / THREADS;
  const int b_lo = min(tid * chunk, p.batch), b_hi = min(b_lo + chunk, p.batch);
  int mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int n = clamped_len(p, b);
    if (n != p.lens[b]) record_device_error(FVB_ERR_INVALID_ARG);
    mine += (n + UNIT - 1) / UNIT;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += t;
  }
  if (lane == 31) s_sum[warp] = upto;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w == warp) upto += total;
    total += s_sum[w];
  }
  // the rows of empty sequences, each by one CTA once it has nothing else to do
  auto zero_rows = [&]() {
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
      if (clamped_len(p, b) > 0) continue;
      for (int e = tid; e < p.heads * (D / 4); e += THREADS)
        *reinterpret_cast<uint2*>(p.o + b * p.o_rs + (e / (D / 4)) * p.o_hs + e % (D / 4) * 4) =
            make_uint2(0u, 0u);
      if (p.lse)
        for (int h = tid; h < p.heads; h += THREADS) p.lse[b * p.lse_rs + h] = -INFINITY;
    }
  };
  if (total == 0) {
    zero_rows();
    return;
  }
  const int ctas = min((int)gridDim.x, total * per_seq);
  if ((int)blockIdx.x >= ctas) {
    zero_rows();
    return;
  }
  const Plan plan(total * per_seq, ctas);
  const int u0 = plan.first(blockIdx.x), u_end = plan.first(blockIdx.x + 1);
  if (u0 >= (upto - mine) * per_seq && u0 < upto * per_seq) {
    int f = (upto - mine) * per_seq, b = b_lo;
    while (true) {
      const int n = (clamped_len(p, b) + UNIT - 1) / UNIT * per_seq;
      if (u0 < f + n) break;
      f += n;
      ++b;
    }
    s_b = b;
    s_first = f;
  }
  __syncthreads();
  int b_at = s_b, b_first = s_first;  // sequence of the next run, its first unit

  auto locate = [&](int u) {
    Run r;
    r.len = clamped_len(p, b_at);
    r.n_units = (r.len + UNIT - 1) / UNIT;
    while (u >= b_first + r.n_units * per_seq) {
      b_first += r.n_units * per_seq;
      r.len = clamped_len(p, ++b_at);
      r.n_units = (r.len + UNIT - 1) / UNIT;
    }
    r.b = b_at;
    const int item = (u - b_first) / r.n_units;
    r.first = b_first + item * r.n_units;
    r.kvh = item / p.head_blocks;
    const int h = (item - r.kvh * p.head_blocks) * C::HB;
    r.head0 = r.kvh * p.group + h;
    r.n_heads = min(C::HB, p.group - h);
    r.k_first = u - r.first;
    r.k_last = min(u_end - r.first, r.n_units);
    // one tile per unit; the last one may lie past the keys
    r.n_tiles = r.k_last - r.k_first;
    if ((r.k_last - 1) * UNIT + warp * SUB >= r.len) --r.n_tiles;
    return r;
  };

  Run run = locate(u0);
  int slot = 0, next = 0;  // of the ring: the tile to be read, to be requested
  uint32_t phase = 0;
  int requested = 0;
  // Pages ahead of use.  BOXES: lane i has the page of tile 32 * k + i, loaded
  // 16 tiles before.  Otherwise each lane has its own key's page of the next
  // tile.
  int pages = 0, pages_ahead = 0;
  auto load_pages = [&](int tile) {
    const int t = BOXES ? tile + lane : tile;
    const int k = (run.k_first + t) * UNIT + warp * SUB + (BOXES ? 0 : lane & (SUB - 1));
    return t < run.n_tiles && k < run.len
               ? p.table[run.b * p.ld_table + (unsigned)k / (unsigned)p.page_size] : 0;
  };
  auto start_pages = [&]() { pages_ahead = load_pages(0); };
  int page = 0, at = 0;  // of the tile that is requested
  // requests the run's next tile: K and V of the same keys in turn
  auto request = [&]() {
    if (requested >= 2 * run.n_tiles) return;
    const int tile = requested >> 1;
    const int k0 = (run.k_first + tile) * UNIT + warp * SUB;
    const int nv = min(SUB, run.len - k0);
    if (!(requested & 1)) {
      if (BOXES) {
        if ((tile & 31) == 0) pages = pages_ahead;
        if ((tile & 31) == 16) pages_ahead = load_pages(tile + 16);
        page = __shfl_sync(0xffffffffu, pages, tile & 31);
      } else {
        page = pages_ahead;
        pages_ahead = load_pages(tile + 1);
      }
      if (page < 0 || page >= p.n_pages) {
        record_device_error(FVB_ERR_INVALID_ARG);
        page = 0;
      }
      at = (unsigned)(k0 + (BOXES ? 0 : lane & (SUB - 1))) % (unsigned)p.page_size;
    }
    const uint32_t dst = ring + next * C::TILE;
    if (BOXES) {
      if (lane == 0) {
        const CUtensorMap* map = requested & 1 ? &map_v : &map_k;
        mbar_arrive_expect_tx(&full[next], C::TILE);
#pragma unroll
        for (int x = 0; x < D; x += 64)
          box_row16(dst + x / 64 * 2048, map, x, at, run.kvh, page, &full[next]);
      }
    } else {
      if (lane == 0) mbar_arrive_expect_tx(&full[next], (uint32_t)(nv * D * 2));
      __syncwarp();
      if (lane < nv) {
        const bf16* src = requested & 1 ? p.v + run.kvh * p.v_hs + page * p.v_ps + at * p.v_rs
                                        : p.k + run.kvh * p.k_hs + page * p.k_ps + at * p.k_rs;
        bulk_row(dst + lane * C::PITCH, src, D * 2, &full[next]);
      }
    }
    ++requested;
    if (++next == C::SLOTS) next = 0;
  };
  // Offsets in a tile of the matrices that this lane addresses: rows and dims
  // of K as they stand, rows of V for the transposed reads.  In a box the
  // 16-byte pieces of a row are swizzled by the row: four offsets, which
  // repeat from box to box.
  uint32_t k_off[4], v_off[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int kr = lane & 15, kp = 2 * j + (lane >> 4);
    const int vr = (lane & 7) + ((lane >> 4) & 1) * 8, vp = 2 * j + ((lane >> 3) & 1);
    k_off[j] = BOXES ? kr * 128 + (((kp ^ kr) & 7) << 4) : kr * C::PITCH + kp * 16;
    v_off[j] = BOXES ? vr * 128 + (((vp ^ vr) & 7) << 4) : vr * C::PITCH + vp * 16;
  }
  constexpr int BOX = BOXES ? 2048 : 128;  // bytes from 64 dims to the next 64
  // gives the slot that was read back to the ring
  auto advance = [&]() {
    __syncwarp();
    request();
    if (++slot == C::SLOTS) {
      slot = 0;
      phase ^= 1;
    }
  };
  // the next tile is here, for all lanes alike: false if the wait ran out
  auto arrived = [&]() {
    return __all_sync(0xffffffffu, mbar_wait_spin(&full[slot], phase)) != 0;
  };
  // queries: B fragments (dims x heads), heads past the group are zero
  uint32_t qf[NT][D / 16][2];
  auto load_q = [&]() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int h = t * 8 + (lane >> 2);
      const bf16* qp = p.q + run.b * p.q_rs + (run.head0 + h) * p.q_hs + 2 * (lane & 3);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        qf[t][j][0] = h < run.n_heads ? *reinterpret_cast<const uint32_t*>(qp + 16 * j) : 0u;
        qf[t][j][1] = h < run.n_heads ? *reinterpret_cast<const uint32_t*>(qp + 16 * j + 8) : 0u;
      }
    }
  };
  start_pages();
#pragma unroll 1
  for (int i = 0; i < C::SLOTS; ++i) request();
  load_q();

  bool alive = true;
  while (true) {
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
    for (int i = 0; i < run.n_tiles; ++i) {
      if (!(alive = arrived())) break;
      const int nv = min(SUB, run.len - ((run.k_first + i) * UNIT + warp * SUB));
      // four sums at a time, so that one product does not wait for another
      constexpr int CH = NT == 1 ? 4 : 2;
      float s[CH][NT][4];
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[c][t][e] = 0.f;
      const uint32_t kt = ring + slot * C::TILE;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t a0, a1, a2, a3;
        ldsm_x4(kt + k_off[j & 3] + (j >> 2) * BOX, a0, a1, a2, a3);
#pragma unroll
        for (int t = 0; t < NT; ++t)
          mma_bf16_16816(s[j % CH][t], a0, a1, a2, a3, qf[t][j][0], qf[t][j][1]);
      }
      advance();
      const int key = lane >> 2;
      uint32_t ph[NT][2], pl[NT][2];
      bool grew = false;
      float alpha[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = s[0][t][e] + s[1][t][e];
          if (CH == 4) x[e] += s[2 % CH][t][e] + s[3 % CH][t][e];
          x[e] *= p.scale_log2;
          if (key + (e >> 1) * 8 >= nv) x[e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(x[e], x[e + 2]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          // the reference is raised when a score passes it by 2^8: weights
          // and sums stay far inside f32, and O is seldom rescaled
          const float mn = mx > m[t][e] + 8.f ? mx : m[t][e];
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
      if (!(alive = arrived())) break;
      // keys past the last one: their tile rows hold what was there before,
      // which times a weight of zero may still be NaN
      const int kk = 2 * (lane & 3);
      const uint32_t m0 = (kk < nv ? 0xffffu : 0u) | (kk + 1 < nv ? 0xffff0000u : 0u);
      const uint32_t m1 = (kk + 8 < nv ? 0xffffu : 0u) | (kk + 9 < nv ? 0xffff0000u : 0u);
      const uint32_t vt = ring + slot * C::TILE;
      // four at a time, so that the two products of a sum are apart
#pragma unroll
      for (int j0 = 0; j0 < D / 16; j0 += 4) {
        uint32_t a[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          ldsm_x4_t(vt + v_off[j] + (j0 >> 2) * BOX, a[j][0], a[j][1], a[j][2], a[j][3]);
        if (nv < SUB) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            a[j][0] &= m0; a[j][1] &= m0; a[j][2] &= m1; a[j][3] &= m1;
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_bf16_16816(o[t][j0 + j], a[j][0], a[j][1], a[j][2], a[j][3], ph[t][0], ph[t][1]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_bf16_16816(o[t][j0 + j], a[j][0], a[j][1], a[j][2], a[j][3], pl[t][0], pl[t][1]);
        }
      }
      advance();
    }
    // every wait that ran out ends the CTA here, together, once the copies that
    // are still under way into its rings have ended (or had as long again)
    if (__syncthreads_or(!alive)) {
      if (!alive) {
        do {
          mbar_wait_limit(&full[slot], phase, FVB_WAIT_LIMIT_NS / 8);
          if (++slot == C::SLOTS) {
            slot = 0;
            phase ^= 1;
          }
        } while (slot != next);
      }
      return;
    }

    // the next run's first tiles arrive while this one is joined; the ring
    // keeps NT slots free, where each warp puts its O
    const Run done = run;
    const int u = done.first + done.k_last;
    const bool more = u < u_end;
    if (more) {
      run = locate(u);
      requested = 0;
      start_pages();
#pragma unroll 1
      for (int i = 0; i < C::SLOTS - NT; ++i) request();
      load_q();
    }
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
    // O of heads 8t.. goes to the slot t + 1 before the next to be read
    auto o_slot = [&](int w_slot, int t) { return (w_slot + C::SLOTS - 1 - t) % C::SLOTS; };
    // each warp's ring stands where it stands: its slot is told with (m, l)
    int* s_slot = reinterpret_cast<int*>(smem + C::OFF_SLOT);
    if (lane == 0) s_slot[warp] = slot;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float* ow = reinterpret_cast<float*>(ring_ptr + o_slot(slot, t) * C::TILE);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = 2 * (lane & 3) + e;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, s_ml[(w * C::HB + t * 8 + h) * 2]);
        const float f = exp2_fast(m[t][e] - (mx == -INFINITY ? 0.f : mx));
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          const int d = j * 16 + (lane >> 2);
          ow[o_at<D>(h, d)] = o[t][j][e] * f;
          ow[o_at<D>(h, d + 8)] = o[t][j][e + 2] * f;
        }
      }
    }
    // the maximum and sum of each head over the warps
    float2* s_tot = reinterpret_cast<float2*>(smem + C::OFF_TOT);
    if (tid < C::HB) {
      float2 t[WARPS];
      float mx = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        t[w] = reinterpret_cast<const float2*>(s_ml)[w * C::HB + tid];
        mx = fmaxf(mx, t[w].x);
      }
#pragma unroll
      for (int w = 0; w < WARPS; ++w)
        sum = fmaf(t[w].y, exp2_fast(t[w].x - (mx == -INFINITY ? 0.f : mx)), sum);
      s_tot[tid] = make_float2(mx, sum);
    }
    __syncthreads();
    const bool whole = done.k_first == 0 && done.k_last == done.n_units;
    const int c0 = plan.owner(done.first), c1 = plan.owner(done.first + done.n_units - 1);
    const long long part = 2ll * blockIdx.x + ((int)blockIdx.x == c0 ? 1 : 0);
    for (int e = tid; e < C::HB * (D / 4); e += THREADS) {
      const int h = e / (D / 4), d = (e % (D / 4)) * 4;
      const float mx = s_tot[h].x, sum = s_tot[h].y, mu = mx == -INFINITY ? 0.f : mx;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float* ow = reinterpret_cast<const float*>(
            smem + (w * C::SLOTS + o_slot(s_slot[w], h >> 3)) * C::TILE);
        const float4 t = *reinterpret_cast<const float4*>(ow + o_at<D>(h & 7, d));
        a.x += t.x; a.y += t.y; a.z += t.z; a.w += t.w;
      }
      if (whole) {
        if (h < done.n_heads) {
          const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
          *reinterpret_cast<uint2*>(p.o + done.b * p.o_rs + (done.head0 + h) * p.o_hs + d) =
              make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
          if (d == 0 && p.lse)
            p.lse[done.b * p.lse_rs + done.head0 + h] = (mu + log2f(sum)) * 0.6931471805599453f;
        }
      } else {
        *reinterpret_cast<float4*>(p.part_o + (part * C::HB + h) * D + d) = a;
        if (d == 0)
          *reinterpret_cast<float2*>(p.part_ml + (part * C::HB + h) * 2) = make_float2(mx, sum);
      }
    }
    if (!whole) {
      const int me = blockIdx.x, n = c1 - c0 + 1;
      const int g0 = c0 + (me - c0) / JOIN * JOIN, gn = min(JOIN, c1 - g0 + 1);
      const int groups = (n + JOIN - 1) / JOIN;
      // adds one arrival; true in the CTA that makes them `of`
      auto last_of = [&](int* a, int of) {
        __syncthreads();
        if (tid == 0) {
          // releases the CTA's partials, acquires the others'
          int old;
          asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;"
                       : "=r"(old) : "l"(a) : "memory");
          s_last = old == of - 1;
          if (s_last) *a = 0;  // as the next call finds it
        }
        __syncthreads();
        return s_last != 0;
      };
      if (last_of(p.arrivals + 3 * g0 + (g0 == c0), gn)) {
        if (groups == 1) {
          join<D, NT, true>(p, c0, g0, gn, 1, done.b, done.head0, done.n_heads);
        } else {
          join<D, NT, false>(p, c0, g0, gn, 1, done.b, done.head0, done.n_heads);
          if (last_of(p.arrivals + 3 * c0 + 2, groups))
            join<D, NT, true>(p, c0, c0, groups, JOIN, done.b, done.head0, done.n_heads);
        }
      }
    }
    if (!more) break;
    // generic accesses of the slots end before the bulk copies into them
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < NT; ++i) request();
  }
  zero_rows();
}

}  // namespace paged
}  // namespace fvb
