// C ABI of the operators that serve several requests at once (declared in
// include/fluxvla_b200.h): e4m3 norm and product, paged append and attention.
// Host side: argument checks, tensor maps, launch shapes.  No entry point
// allocates, synchronises or exits.
#include "host.cuh"

#include "gemm_fp8.cuh"
#include "norm_fp8.cuh"
#include "paged.cuh"

using namespace fvb_host;

// This translation unit's status word (common.cuh), read and reset through
// fvb_get_device_status once one of its kernels has been launched.
static std::atomic<bool> g_used{false};

int fvb_serving_device_status(int* status, int reset) {
  if (!g_used.load(std::memory_order_relaxed)) {
    *status = FVB_OK;
    return FVB_OK;
  }
  cudaError_t e = cudaMemcpyFromSymbol(status, g_fvb_device_status, sizeof(int));
  if (e == cudaSuccess && reset) {
    const int z = 0;
    e = cudaMemcpyToSymbol(g_fvb_device_status, &z, sizeof(int));
  }
  if (e != cudaSuccess) return fail(FVB_ERR_CUDA, "read status: %s", cudaGetErrorString(e));
  return FVB_OK;
}

namespace {

bool aligned(const void* p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// 2-D byte tensor map over [rows, k] (row stride ld bytes), box [box_rows,
// 128] with the 128-byte swizzle; out-of-range reads fill zeros.
int make_map_u8(CUtensorMap* m, const void* ptr, int64_t rows, int64_t k, int64_t ld,
                int box_rows) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return fail(FVB_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides,
                   box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(FVB_ERR_INVALID_ARG, "tensor map encode failed (%d)", (int)r);
  return FVB_OK;
}

template <typename TX, int DT, int KIND, bool VECS>
int launch_norm_rows(const fvb::n8::Dev& d, int rows, cudaStream_t st) {
  namespace N = fvb::n8;
  const int chunks = (d.dim + N::VEC - 1) / N::VEC;
  const int vpt = chunks <= N::MAX_THREADS ? 1 : (chunks <= 2 * N::MAX_THREADS ? 2 : 4);
  const int t = ((chunks + vpt - 1) / vpt + 31) / 32 * 32;
  auto kern = vpt == 1   ? N::norm_fp8_kernel<TX, DT, 1, KIND, VECS>
              : vpt == 2 ? N::norm_fp8_kernel<TX, DT, 2, KIND, VECS>
                         : N::norm_fp8_kernel<TX, DT, 4, KIND, VECS>;
  return launch_k("fvb_norm_fp8", kern, dim3(rows), dim3(t), VECS ? 0 : t * 32, st, d);
}

template <typename TX, int DT, bool VECS>
int launch_norm_fp8(const fvb::n8::Dev& d, int rows, cudaStream_t st) {
  namespace N = fvb::n8;
  if (d.mode == FVB_NORM_ADA_RMS) return launch_norm_rows<TX, DT, N::SHIFT, VECS>(d, rows, st);
  if (d.mode != FVB_NORM_NONE) return launch_norm_rows<TX, DT, N::SCALE, VECS>(d, rows, st);
  // no row statistics: runs of 4096 columns, each its own CTA.  (Two vectors a
  // thread: 848 x 16384 takes 10.5 us, with one 12.4, whose maxima and scales
  // serve half the columns, with four 12.4, whose registers leave fewer warps.)
  const int chunks = (d.dim + 2 * N::VEC - 1) / (2 * N::VEC);
  const int t = chunks < 256 ? (chunks + 31) / 32 * 32 : 256;
  return launch_k("fvb_norm_fp8", N::norm_fp8_kernel<TX, DT, 2, N::CODES, VECS>,
                  dim3(rows, (chunks + t - 1) / t), dim3(t), VECS ? 0 : t * 32, st, d);
}

template <typename TX, bool VECS>
int launch_norm_fp8(const fvb::n8::Dev& d, int delta, int rows, cudaStream_t st) {
  namespace N = fvb::n8;
  if (delta == N::DELTA_NONE) return launch_norm_fp8<TX, N::DELTA_NONE, VECS>(d, rows, st);
  if (delta == N::DELTA_F32) return launch_norm_fp8<TX, N::DELTA_F32, VECS>(d, rows, st);
  return launch_norm_fp8<TX, N::DELTA_BF16, VECS>(d, rows, st);
}

int launch_gemm_fp8(const void* kern, const CUtensorMap& ma, const CUtensorMap& mb,
                    const fvb::g8::Dev& d, int ctas, int cluster, int smem, cudaStream_t st) {
  if (int r = ensure_smem(kern, fvb::g8::ClusterCfg::MAX_SMEM, "fvb_gemm_fp8")) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(fvb::g8::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = cluster;
  attrs[0].val.clusterDim.y = 1;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  void* args[] = {const_cast<CUtensorMap*>(&ma), const_cast<CUtensorMap*>(&mb),
                  const_cast<fvb::g8::Dev*>(&d)};
  cudaError_t e = cudaLaunchKernelExC(&cfg, kern, args);
  if (e != cudaSuccess)
    return fail(FVB_ERR_CUDA, "fvb_gemm_fp8: launch failed: %s", cudaGetErrorString(e));
  return check_launch("fvb_gemm_fp8");
}

template <bool MULTI>
const void* cluster_kernel(int epi) {
  namespace G = fvb::g8;
  if (epi == FVB_EPI_BF16)
    return reinterpret_cast<const void*>(G::gemm_fp8_cluster<FVB_EPI_BF16, MULTI>);
  if (epi == FVB_EPI_GEGLU)
    return reinterpret_cast<const void*>(G::gemm_fp8_cluster<FVB_EPI_GEGLU, MULTI>);
  return reinterpret_cast<const void*>(G::gemm_fp8_cluster<FVB_EPI_F32_STORE, MULTI>);
}
template <bool VEC>
const void* pair_kernel(int epi) {
  namespace G = fvb::g8;
  if (epi == FVB_EPI_BF16) return reinterpret_cast<const void*>(G::gemm_fp8_pair<FVB_EPI_BF16, VEC>);
  if (epi == FVB_EPI_GEGLU)
    return reinterpret_cast<const void*>(G::gemm_fp8_pair<FVB_EPI_GEGLU, VEC>);
  return reinterpret_cast<const void*>(G::gemm_fp8_pair<FVB_EPI_F32_STORE, VEC>);
}

// Clusters of 1..8 CTAs of the cluster kernel (one CTA per SM) that the device
// runs at once: fewer than its SMs over the size, since a cluster stays in one
// GPC (148, 74, 45, 33, 26, 22, 15, 15 on a B200).
const int* cluster_slots() {
  static std::mutex mu;
  static int slots[128][9] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) dev = 0;
  std::lock_guard<std::mutex> lk(mu);
  if (slots[dev][1]) return slots[dev];
  const void* kern = cluster_kernel<false>(FVB_EPI_BF16);
  for (int c = 8; c >= 1; --c) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c * 256);
    cfg.blockDim = dim3(fvb::g8::THREADS);
    cfg.dynamicSmemBytes = fvb::g8::ClusterCfg::MAX_SMEM;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = c;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) n = 0;
    cudaGetLastError();
    slots[dev][c] = n > 0 ? n : (c == 1 ? sm_count() : 0);
  }
  return slots[dev];
}

constexpr int64_t ATTEND_COUNTER_BYTES = 4096;  // three ints per CTA

// Launch shape of an attention call: blocks of 8 or 16 heads, one CTA per SM.
struct AttendShape {
  int nt, head_blocks, ctas;
  int64_t off_o, off_ml, bytes;
};

int attend_prepare(const fvb_paged_attn_args* a, AttendShape* s) {
  if (!a) return fail(FVB_ERR_INVALID_ARG, "args is NULL");
  if (a->batch < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads)
    return fail(FVB_ERR_INVALID_ARG,
                "fvb_paged_attention: bad batch %d or heads %d / %d", a->batch, a->heads,
                a->kv_heads);
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return fail(FVB_ERR_UNSUPPORTED, "fvb_paged_attention: head_dim %d (64, 128 or 256)",
                a->head_dim);
  const int group = a->heads / a->kv_heads;
  s->nt = group <= 8 ? 1 : 2;
  s->head_blocks = (group + 8 * s->nt - 1) / (8 * s->nt);
  s->ctas = sm_count() < 340 ? sm_count() : 340;
  const int64_t rows = 2ll * s->ctas * 8 * s->nt;
  // the counters keep their place whatever the shape, so that calls of
  // several shapes may share a workspace one after the other
  s->off_o = ATTEND_COUNTER_BYTES;
  s->off_ml = s->off_o + rows * a->head_dim * 4;
  s->bytes = s->off_ml + rows * 8;
  return FVB_OK;
}

// Tensor map of a paged cache, box of 16 rows x 64 dims of one head and page.
// Strides of a dimension of size 1 mean nothing and may be anything.
bool make_cache_map(CUtensorMap* m, const void* ptr, int dim, int page_size, int kv_heads,
                    int n_pages, int64_t row, int64_t head, int64_t page) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return false;
  if (kv_heads == 1) head = dim;
  if (n_pages == 1) page = dim;
  if (row <= 0 || head <= 0 || page <= 0) return false;
  cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)page_size, (cuuint64_t)kv_heads,
                        (cuuint64_t)n_pages};
  cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)head * 2, (cuuint64_t)page * 2};
  cuuint32_t box[4] = {64, 16, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NT, bool BOXES>
int launch_attend(const CUtensorMap& mk, const CUtensorMap& mv, const fvb::paged::AttendDev& d,
                  int ctas, cudaStream_t st) {
  using C = fvb::paged::Cfg<D, NT, BOXES>;
  auto kern = fvb::paged::attend_kernel<D, NT, BOXES>;
  if (int r = ensure_smem(reinterpret_cast<const void*>(kern), C::SMEM, "fvb_paged_attention"))
    return r;
  return launch_k("fvb_paged_attention", kern, dim3(ctas), dim3(fvb::paged::THREADS),
                  (size_t)C::SMEM, st, mk, mv, d);
}

template <int D>
int launch_attend(int nt, bool boxes, const CUtensorMap& mk, const CUtensorMap& mv,
                  const fvb::paged::AttendDev& d, int ctas, cudaStream_t st) {
  if (boxes)
    return nt == 1 ? launch_attend<D, 1, true>(mk, mv, d, ctas, st)
                   : launch_attend<D, 2, true>(mk, mv, d, ctas, st);
  return nt == 1 ? launch_attend<D, 1, false>(mk, mv, d, ctas, st)
                 : launch_attend<D, 2, false>(mk, mv, d, ctas, st);
}

}  // namespace

extern "C" {

int fvb_norm_fp8(const fvb_norm_fp8_args* a, void* stream) {
  if (!a) return fail(FVB_ERR_INVALID_ARG, "args is NULL");
  if (a->rows < 0 || a->dim <= 0)
    return fail(FVB_ERR_INVALID_ARG, "fvb_norm_fp8: bad shape %d x %d", a->rows, a->dim);
  if (a->mode != FVB_NORM_GEMMA_RMS && a->mode != FVB_NORM_ADA_RMS && a->mode != FVB_NORM_RMS &&
      a->mode != FVB_NORM_NONE)
    return fail(FVB_ERR_INVALID_ARG, "fvb_norm_fp8: bad mode %d", a->mode);
  if (a->mode != FVB_NORM_NONE && a->dim > FVB_NORM_FP8_MAX_DIM)
    return fail(FVB_ERR_UNSUPPORTED, "fvb_norm_fp8: dim %d over %d", a->dim,
                FVB_NORM_FP8_MAX_DIM);
  // without one, within what 2^16 - 1 CTAs of 4096 columns cover
  if (a->dim > 65535 * 2048)
    return fail(FVB_ERR_UNSUPPORTED, "fvb_norm_fp8: dim %d over %d", a->dim, 65535 * 2048);
  if (!a->x || !a->q || !a->scales)
    return fail(FVB_ERR_INVALID_ARG, "fvb_norm_fp8: NULL operand");
  if (a->mode == FVB_NORM_GEMMA_RMS && !a->w)
    return fail(FVB_ERR_INVALID_ARG, "fvb_norm_fp8: weight required");
  if (a->mode == FVB_NORM_ADA_RMS && !a->mod)
    return fail(FVB_ERR_INVALID_ARG, "fvb_norm_fp8: modulation required");
  if ((a->delta == nullptr) != (a->res == nullptr))
    return fail(FVB_ERR_INVALID_ARG, "fvb_norm_fp8: delta and res come together");
  const int groups = (a->dim + 127) / 128;
  if (a->ld_x < a->dim || a->ld_q < a->dim || a->ld_scales < groups ||
      (a->delta && (a->ld_delta < a->dim || a->ld_res < a->dim)))
    return fail(FVB_ERR_INVALID_ARG, "fvb_norm_fp8: a row stride is shorter than its row");
  if (!(a->eps >= 0)) return fail(FVB_ERR_INVALID_ARG, "fvb_norm_fp8: bad eps");
  if (a->rows == 0) return FVB_OK;
  g_used.store(true, std::memory_order_relaxed);
  const int xb = a->x_f32 ? 4 : 2, db = a->delta_f32 ? 4 : 2;
  auto rows16 = [](const void* p, int64_t ld, int eb) { return aligned16(p) && ld * eb % 16 == 0; };
  fvb::n8::Dev d;
  d.mode = a->mode;
  d.x = a->x; d.ld_x = a->ld_x;
  d.delta = a->delta; d.ld_delta = a->ld_delta;
  d.res = a->res; d.ld_res = a->ld_res;
  d.w = (const bf16*)a->w; d.mod = a->mod;
  d.q = (uint8_t*)a->q; d.ld_q = a->ld_q;
  d.scales = a->scales; d.ld_scales = a->ld_scales;
  d.dim = a->dim; d.eps = a->eps; d.inv_dim = 1.0 / a->dim;
  // vector accesses where every row starts on 16 bytes (8 of the codes)
  const bool vec =
      rows16(a->x, a->ld_x, xb) && aligned(a->q, 8) && a->ld_q % 8 == 0 &&
      (!a->delta || (rows16(a->delta, a->ld_delta, db) && rows16(a->res, a->ld_res, xb))) &&
      (a->mode != FVB_NORM_GEMMA_RMS || aligned16(a->w)) &&
      (a->mode != FVB_NORM_ADA_RMS || (aligned16(a->mod) && a->dim % 4 == 0));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int delta = !a->delta ? fvb::n8::DELTA_NONE
                              : (a->delta_f32 ? fvb::n8::DELTA_F32 : fvb::n8::DELTA_BF16);
  if (a->x_f32)
    return vec ? launch_norm_fp8<float, true>(d, delta, a->rows, st)
               : launch_norm_fp8<float, false>(d, delta, a->rows, st);
  return vec ? launch_norm_fp8<bf16, true>(d, delta, a->rows, st)
             : launch_norm_fp8<bf16, false>(d, delta, a->rows, st);
}

int fvb_gemm_fp8(const fvb_gemm_fp8_args* a, void* stream) {
  if (!a) return fail(FVB_ERR_INVALID_ARG, "args is NULL");
  if (a->m < 0 || a->n <= 0 || a->k <= 0)
    return fail(FVB_ERR_INVALID_ARG, "fvb_gemm_fp8: bad shape %d x %d x %d", a->m, a->n, a->k);
  if (a->epilogue != FVB_EPI_BF16 && a->epilogue != FVB_EPI_F32_STORE &&
      a->epilogue != FVB_EPI_GEGLU)
    return fail(FVB_ERR_INVALID_ARG, "fvb_gemm_fp8: bad epilogue %d", a->epilogue);
  if (a->epilogue == FVB_EPI_GEGLU && a->n % 2)
    return fail(FVB_ERR_INVALID_ARG, "fvb_gemm_fp8: GEGLU needs an even feature count");
  // rows of the last tile are counted past the last token and feature
  constexpr int MOST = INT32_MAX - 256;
  if (a->m > MOST || a->n > MOST || a->k > MOST)
    return fail(FVB_ERR_UNSUPPORTED, "fvb_gemm_fp8: too large");
  if (!a->a || !a->a_scale || !a->b || !a->b_scale || !a->out)
    return fail(FVB_ERR_INVALID_ARG, "fvb_gemm_fp8: NULL operand");
  const int groups = (a->k + 127) / 128;
  const int nf = a->epilogue == FVB_EPI_GEGLU ? a->n / 2 : a->n;
  if (a->lda < a->k || a->ldb < a->k || a->ld_as < groups || a->ld_bs < groups || a->ldo < nf)
    return fail(FVB_ERR_INVALID_ARG, "fvb_gemm_fp8: a row stride is shorter than its row");
  if (!aligned16(a->a) || !aligned16(a->b) || a->lda % 16 || a->ldb % 16)
    return fail(FVB_ERR_INVALID_ARG,
                "fvb_gemm_fp8: operands must be 16B aligned with row strides in multiples of 16");
  if (a->m == 0) return FVB_OK;
  g_used.store(true, std::memory_order_relaxed);
  fvb::g8::Dev d;
  d.m = a->m; d.n = a->n; d.groups = groups;
  d.sa = a->a_scale; d.ld_sa = a->ld_as;
  d.sb = a->b_scale; d.ld_sb = a->ld_bs;
  d.out = a->out; d.ldo = a->ldo;
  const int eb = a->epilogue == FVB_EPI_F32_STORE ? 4 : 2;
  d.vec_out = aligned16(a->out) && a->ldo * eb % 16 == 0 && nf * eb % 16 == 0 && a->n % 8 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // The shape with the least time by a count of clocks, fitted to measured
  // products: a group costs the cluster kernel 600 clocks, a call 3000, a tile
  // 1500 more (3000 with an exchange), the pair kernel 970 and 3500 for a tile
  // of twice the height and width.  816 x 32768 x 2048 GEGLU at 1965 MHz: pair
  // 74 us, clusters 109 us; 816 x 2560 x 2048: the other way round, 40 pair tiles
  // leave SMs idle.  The count ranks shapes; where rows are no multiple of 128
  // bytes and a tile is 128 rows high it is far too low (768 x 1152 x 4304: 8.2 us
  // counted, 15 us taken).
  if (int rr = ensure_smem(cluster_kernel<false>(FVB_EPI_BF16), fvb::g8::ClusterCfg::MAX_SMEM,
                           "fvb_gemm_fp8"))
    return rr;
  const int* slots = cluster_slots();
  const int64_t f_tiles = (a->n + 127) / 128, t_tiles = (a->m + 127) / 128;
  const int64_t tiles = f_tiles * t_tiles;
  const int64_t f_pair = (a->n + 255) / 256, t_pair = (a->m + 255) / 256;
  auto waves = [](int64_t n, int64_t at_once) { return (n + at_once - 1) / at_once; };
  int64_t best = INT64_MAX;
  d.cl = 1;
  for (int c = 1; c <= 8 && c <= groups; ++c) {
    if (!slots[c]) continue;
    const int64_t t = c > 1 ? waves(tiles, slots[c]) * ((groups + c - 1) / c * 600 + 6000)
                            : waves(tiles, slots[1]) * (groups * 600 + 1500) + 3000;
    if (t < best) {
      best = t;
      d.cl = c;
    }
  }
  const bool pair = slots[2] && waves(f_pair * t_pair, slots[2]) * (groups * 970ll + 3500) < best;
  const int64_t most = INT32_MAX / 8 / groups;
  if (tiles > most) return fail(FVB_ERR_UNSUPPORTED, "fvb_gemm_fp8: too large");
  CUtensorMap mt, mf;
  int r = make_map_u8(&mf, a->b, a->n, a->k, a->ldb, 128);
  if (r) return r;
  if (pair) {
    d.t_tiles = (int)t_pair; d.f_tiles = (int)f_pair;
    r = make_map_u8(&mt, a->a, a->m, a->k, a->lda, 128);
    if (r) return r;
    const int pairs = (int)(f_pair * t_pair < slots[2] ? f_pair * t_pair : slots[2]);
    const void* two = d.vec_out ? pair_kernel<true>(a->epilogue) : pair_kernel<false>(a->epilogue);
    return launch_gemm_fp8(two, mt, mf, d, 2 * pairs, 2,
                           fvb::g8::PairCfg::SMEM, st);
  }
  // tiles of equal height
  d.f_tiles = (int)f_tiles; d.t_tiles = (int)t_tiles;
  d.rows = (int)((a->m + t_tiles - 1) / t_tiles + 7) / 8 * 8;
  d.stages = fvb::g8::ClusterCfg::stages(d.rows);
  r = make_map_u8(&mt, a->a, a->m, a->k, a->lda, d.rows);
  if (r) return r;
  const int ctas = d.cl > 1 ? (int)tiles * d.cl : (int)(tiles < slots[1] ? tiles : slots[1]);
  const bool multi = d.cl == 1 && tiles > ctas;
  const void* kern = multi ? cluster_kernel<true>(a->epilogue) : cluster_kernel<false>(a->epilogue);
  return launch_gemm_fp8(kern, mt, mf, d, ctas, d.cl,
                         fvb::g8::ClusterCfg::smem(d.rows), st);
}

int fvb_paged_append(const fvb_paged_append_args* a, void* stream) {
  if (!a) return fail(FVB_ERR_INVALID_ARG, "args is NULL");
  if (a->tokens < 0 || a->heads < 0 || a->kv_heads <= 0 || a->head_dim <= 0 || a->head_dim % 2)
    return fail(FVB_ERR_INVALID_ARG, "fvb_paged_append: bad shape");
  if (a->page_size <= 0 || a->n_pages < 0)
    return fail(FVB_ERR_INVALID_ARG, "fvb_paged_append: bad cache shape");
  // (a cache without pages has no address)
  if (!a->k || !a->v || !a->slots || (a->n_pages > 0 && (!a->k_cache || !a->v_cache)))
    return fail(FVB_ERR_INVALID_ARG, "fvb_paged_append: NULL operand");
  if (a->heads > 0 && (!a->q || !a->q_out))
    return fail(FVB_ERR_INVALID_ARG, "fvb_paged_append: queries need q and q_out");
  if (a->rope_cs && (!a->positions || a->max_pos <= 0 || !aligned(a->rope_cs, 8)))
    return fail(FVB_ERR_INVALID_ARG, "fvb_paged_append: rope_cs needs positions and max_pos");
  if (a->tokens == 0) return FVB_OK;
  g_used.store(true, std::memory_order_relaxed);
  fvb::paged::AppendDev d;
  d.q = (const bf16*)a->q; d.q_rs = a->q_row_stride; d.q_hs = a->q_head_stride;
  d.k = (const bf16*)a->k; d.k_rs = a->k_row_stride; d.k_hs = a->k_head_stride;
  d.v = (const bf16*)a->v; d.v_rs = a->v_row_stride; d.v_hs = a->v_head_stride;
  d.q_out = (bf16*)a->q_out; d.qo_rs = a->q_out_row_stride; d.qo_hs = a->q_out_head_stride;
  d.k_cache = (bf16*)a->k_cache; d.v_cache = (bf16*)a->v_cache;
  d.kc_ps = a->kc_page_stride; d.kc_rs = a->kc_row_stride; d.kc_hs = a->kc_head_stride;
  d.vc_ps = a->vc_page_stride; d.vc_rs = a->vc_row_stride; d.vc_hs = a->vc_head_stride;
  d.slots = a->slots; d.positions = a->positions; d.rope_cs = a->rope_cs;
  d.tokens = a->tokens; d.heads = a->heads; d.kv_heads = a->kv_heads; d.dim = a->head_dim;
  d.page_size = a->page_size; d.max_pos = a->max_pos; d.interleaved = a->rope_interleaved;
  d.n_slots = (long long)a->n_pages * a->page_size;
  bool vec = a->head_dim % 16 == 0 && (!a->rope_cs || aligned16(a->rope_cs));
  const void* ptrs[] = {a->q, a->k, a->v, a->q_out, a->k_cache, a->v_cache};
  for (const void* p : ptrs) vec = vec && aligned16(p);
  const int64_t strides[] = {d.q_rs, d.q_hs, d.k_rs, d.k_hs, d.v_rs, d.v_hs, d.qo_rs, d.qo_hs,
                             d.kc_ps, d.kc_rs, d.kc_hs, d.vc_ps, d.vc_rs, d.vc_hs};
  for (int i = a->heads > 0 ? 0 : 2; i < 14; ++i)
    if (a->heads > 0 || (i != 6 && i != 7)) vec = vec && strides[i] % 8 == 0;
  // all heads of a token in one thread where the tokens fill the GPU by
  // themselves, else a head each
  const int64_t heads = (int64_t)a->heads + 2ll * a->kv_heads;
  const int64_t chunks = a->head_dim / (vec ? 16 : 2);
  const bool many = chunks * a->tokens >= 256ll * 2 * sm_count();
  d.heads_per_thread = many && heads < INT32_MAX ? (int)heads : 1;
  const int64_t per_token = vec && many ? chunks : heads * chunks;
  const int64_t blocks = (per_token * a->tokens + 255) / 256;
  if (heads * chunks > INT32_MAX || blocks > INT32_MAX)
    return fail(FVB_ERR_UNSUPPORTED, "fvb_paged_append: too many rows");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return launch_k("fvb_paged_append",
                  vec ? fvb::paged::append_vec_kernel : fvb::paged::append_kernel,
                  dim3((unsigned)blocks), dim3(256), 0, st, d);
}

int64_t fvb_paged_attention_workspace_bytes(const fvb_paged_attn_args* a) {
  AttendShape s;
  if (attend_prepare(a, &s)) return -1;
  return s.bytes;
}

int fvb_paged_attention(const fvb_paged_attn_args* a, void* stream) {
  AttendShape s;
  int r = attend_prepare(a, &s);
  if (r) return r;
  // a cache without pages has no address, nor has a table without columns
  if (!a->q || !a->seq_lens || !a->out ||
      (a->n_pages > 0 &&
       (!a->k_cache || !a->v_cache || (a->max_pages > 0 && !a->page_table))))
    return fail(FVB_ERR_INVALID_ARG, "fvb_paged_attention: NULL operand");
  if (a->n_pages < 0 || a->page_size <= 0 || a->max_pages < 0 || a->ld_table < a->max_pages)
    return fail(FVB_ERR_INVALID_ARG, "fvb_paged_attention: bad cache shape");
  const int64_t max_len = (int64_t)a->max_pages * a->page_size;
  // the kernel counts keys in 32 bits, up to the end of the last unit and of the
  // pages that it looks up ahead (48 units)
  constexpr int AHEAD = 64 * fvb::paged::UNIT;
  if (max_len > INT32_MAX - AHEAD)
    return fail(FVB_ERR_UNSUPPORTED, "fvb_paged_attention: %lld keys a sequence",
                (long long)max_len);
  // units of 128 keys over all sequences and heads are counted in 32 bits, and
  // so are sequences, in strides of the block and of the grid, and a row's values
  if ((int64_t)a->heads * a->head_dim > INT32_MAX)
    return fail(FVB_ERR_UNSUPPORTED, "fvb_paged_attention: %d heads", a->heads);
  if (a->batch > INT32_MAX - 1024 ||
      (max_len / fvb::paged::UNIT + 1) * a->batch > INT32_MAX / (a->kv_heads * s.head_blocks))
    return fail(FVB_ERR_UNSUPPORTED, "fvb_paged_attention: %d sequences of up to %lld keys",
                a->batch, (long long)max_len);
  // the stride of a dimension of size 1 means nothing, and is taken as 0
  auto step = [](int64_t stride, int32_t size) { return size == 1 ? 0 : stride; };
  const int64_t s8[] = {step(a->kc_page_stride, a->n_pages), step(a->kc_row_stride, a->page_size),
                        step(a->kc_head_stride, a->kv_heads), step(a->vc_page_stride, a->n_pages),
                        step(a->vc_row_stride, a->page_size), step(a->vc_head_stride, a->kv_heads)};
  bool ok = aligned16(a->k_cache) && aligned16(a->v_cache);
  for (int64_t v : s8) ok = ok && v % 8 == 0;
  if (!ok)
    return fail(FVB_ERR_INVALID_ARG,
                "fvb_paged_attention: cache rows must be 16B aligned (strides in multiples of 8)");
  const int64_t q_rs = step(a->q_row_stride, a->batch), q_hs = step(a->q_head_stride, a->heads),
                o_rs = step(a->out_row_stride, a->batch), o_hs = step(a->out_head_stride, a->heads);
  if (!aligned(a->q, 4) || q_rs % 2 || q_hs % 2 || !aligned(a->out, 8) || o_rs % 4 || o_hs % 4)
    return fail(FVB_ERR_INVALID_ARG,
                "fvb_paged_attention: q needs 4-byte, out 8-byte aligned rows");
  if (!a->workspace || a->workspace_bytes < s.bytes || !aligned16(a->workspace))
    return fail(FVB_ERR_WORKSPACE, "fvb_paged_attention: workspace needs %lld bytes",
                (long long)s.bytes);
  if (a->batch == 0) return FVB_OK;
  g_used.store(true, std::memory_order_relaxed);
  fvb::paged::AttendDev d;
  d.q = (const bf16*)a->q; d.q_rs = q_rs; d.q_hs = q_hs;
  d.k = (const bf16*)a->k_cache; d.k_ps = s8[0]; d.k_rs = s8[1]; d.k_hs = s8[2];
  d.v = (const bf16*)a->v_cache; d.v_ps = s8[3]; d.v_rs = s8[4]; d.v_hs = s8[5];
  d.o = (bf16*)a->out; d.o_rs = o_rs; d.o_hs = o_hs;
  d.lse = a->lse; d.lse_rs = a->lse_row_stride;
  d.table = a->page_table; d.ld_table = a->ld_table; d.lens = a->seq_lens;
  d.batch = a->batch; d.heads = a->heads; d.kv_heads = a->kv_heads;
  d.group = a->heads / a->kv_heads; d.head_blocks = s.head_blocks;
  // without a page no key can be read, so every length is taken as 0 (and
  // neither the cache nor the table is touched)
  d.n_pages = a->n_pages; d.page_size = a->page_size;
  d.max_len = a->n_pages > 0 ? (int)max_len : 0;
  d.scale_log2 = a->scale * 1.4426950408889634f;
  d.arrivals = (int*)a->workspace;
  d.part_o = (float*)((char*)a->workspace + s.off_o);
  d.part_ml = (float*)((char*)a->workspace + s.off_ml);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  CUtensorMap mk, mv;
  memset(&mk, 0, sizeof(mk));
  memset(&mv, 0, sizeof(mv));
  const bool boxes =
      a->page_size % 16 == 0 && a->n_pages > 0 &&
      make_cache_map(&mk, a->k_cache, a->head_dim, a->page_size, a->kv_heads, a->n_pages, s8[1],
                     s8[2], s8[0]) &&
      make_cache_map(&mv, a->v_cache, a->head_dim, a->page_size, a->kv_heads, a->n_pages, s8[4],
                     s8[5], s8[3]);
  if (a->head_dim == 256) return launch_attend<256>(s.nt, boxes, mk, mv, d, s.ctas, st);
  if (a->head_dim == 128) return launch_attend<128>(s.nt, boxes, mk, mv, d, s.ctas, st);
  return launch_attend<64>(s.nt, boxes, mk, mv, d, s.ctas, st);
}

}  // extern "C"
