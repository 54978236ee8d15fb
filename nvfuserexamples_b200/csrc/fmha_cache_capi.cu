// fmha_cache_capi.cu — extern "C" entry points of the paged cache: argument validation, tensor maps, launches.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/fmha_sm100.h"
#include "fmha_cache_args.h"
#include "fmha_capi_common.h"
#include "fmha_kernel_args.h"

namespace fmha {

// [rows, heads, D] view of 16-bit values: 16-byte pieces of a row at 16-byte addresses.
static bool rows_ok(const fmha_tensor4& t, int heads) {
  return t.ptr != nullptr && (reinterpret_cast<uintptr_t>(t.ptr) & 15) == 0 && t.stride_s > 0 && t.stride_s % 8 == 0 &&
         (heads <= 1 || (t.stride_h > 0 && t.stride_h % 8 == 0));
}
// A [pages, H, rows, .] view, strides in units of `unit` bytes.
static bool pages_ok(const fmha_tensor4& t, const fmha_kv_cache& c, int unit, bool row_stride) {
  const int step = 16 / unit;
  if (t.ptr == nullptr || (reinterpret_cast<uintptr_t>(t.ptr) & 15) != 0) return false;
  if (row_stride && (t.stride_s <= 0 || t.stride_s % step != 0)) return false;
  if (c.H_kv > 1 && (t.stride_h <= 0 || t.stride_h % step != 0)) return false;
  return c.pages <= 1 || (t.stride_b > 0 && t.stride_b % step == 0);
}

static int validate_cache(const fmha_kv_cache& c, int B) {
  if (c.bits != 16 && c.bits != 4) return FMHA_ERR_UNSUPPORTED;
  if (c.D != 64 && c.D != 128) return FMHA_ERR_UNSUPPORTED;
  if (c.pages < 0 || c.page_rows <= 0 || c.page_rows % 16 != 0 || c.H_kv < 0 || c.table_width < 0) return FMHA_ERR_BAD_ARG;
  if (c.page_rows > kMaxPageRows || c.H_kv > 65535 || B > 65535) return FMHA_ERR_TOO_LARGE;
  // positions are 32-bit
  if (static_cast<int64_t>(c.table_width) * c.page_rows > (1ll << 31) - kMaxPageRows) return FMHA_ERR_TOO_LARGE;
  if (c.H_kv == 0) return FMHA_ERR_BAD_ARG;
  if (c.pages > 0 && (!pages_ok(c.k, c, c.bits == 4 ? 1 : 2, true) || !pages_ok(c.v, c, c.bits == 4 ? 1 : 2, true))) return FMHA_ERR_BAD_ARG;
  if (c.pages > 0 && c.bits == 4 && (!pages_ok(c.k_params, c, 2, false) || !pages_ok(c.v_params, c, 2, false))) return FMHA_ERR_BAD_ARG;
  if (c.table_width > 0 && B > 0 && (c.table == nullptr || c.table_stride < 0)) return FMHA_ERR_BAD_ARG;
  return FMHA_OK;
}

// Rows of a packed batch without offsets: the same number for every sequence.
static bool rows_each(int total, int B, const void* cu, int* each) {
  *each = B > 0 ? total / B : 0;
  return cu != nullptr || (B > 0 && total % B == 0);
}

// Tensor map of a cache's rows: {values, rows, heads, pages}, boxes of `cols` values x `rows` rows.  Axes of length 1 get a stride that the
// encoder accepts.
static int map_rows(CUtensorMap* out, const fmha_tensor4& t, const fmha_kv_cache& c, CUtensorMapDataType type, int unit, int values, int cols, int rows,
                    CUtensorMapSwizzle swizzle) {
  auto enc = get_encode_fn();
  if (enc == nullptr) return FMHA_ERR_LAUNCH;
  const int64_t ss = t.stride_s, sh = c.H_kv > 1 ? t.stride_h : ss * c.page_rows, sb = c.pages > 1 ? t.stride_b : sh * c.H_kv;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(values), static_cast<cuuint64_t>(c.page_rows), static_cast<cuuint64_t>(c.H_kv),
                              static_cast<cuuint64_t>(c.pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(ss) * unit, static_cast<cuuint64_t>(sh) * unit, static_cast<cuuint64_t>(sb) * unit};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(cols), static_cast<cuuint32_t>(rows), 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(out, type, 4, t.ptr, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FMHA_OK : cuda_fail(static_cast<cudaError_t>(r));
}
// ... and of its scales and bases: a page's rows of a head are one dense line of 32-bit (scale, base) pairs.
static int map_params(CUtensorMap* out, const fmha_tensor4& t, const fmha_kv_cache& c, int rows) {
  auto enc = get_encode_fn();
  if (enc == nullptr) return FMHA_ERR_LAUNCH;
  const int groups = c.D / kCacheGroup;
  const int64_t line = static_cast<int64_t>(c.page_rows) * groups * 2, sh = c.H_kv > 1 ? t.stride_h : line, sb = c.pages > 1 ? t.stride_b : sh * c.H_kv;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(c.page_rows) * groups, static_cast<cuuint64_t>(c.H_kv), static_cast<cuuint64_t>(c.pages)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(sb) * 2};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(rows * groups), 1, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, t.ptr, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FMHA_OK : cuda_fail(static_cast<cudaError_t>(r));
}

static int validate_paged(const fmha_paged_params* p) {
  if (p == nullptr || p->struct_bytes != static_cast<int>(sizeof(fmha_paged_params))) return FMHA_ERR_BAD_ARG;
  if (p->dtype != FMHA_DTYPE_F16 && p->dtype != FMHA_DTYPE_BF16) return FMHA_ERR_UNSUPPORTED;
  if (p->B < 0 || p->H <= 0 || p->total_rows < 0 || p->max_rows < 0) return FMHA_ERR_BAD_ARG;
  const int rc = validate_cache(p->cache, p->B);
  if (rc != FMHA_OK) return rc;
  if (p->H % p->cache.H_kv != 0) return FMHA_ERR_BAD_ARG;
  if (!(p->scale > 0.f) || !std::isfinite(p->scale)) return FMHA_ERR_BAD_ARG;
  // units are counted in 32 bits
  const int64_t tiles = (static_cast<int64_t>(p->max_rows) * (p->H / p->cache.H_kv) + 7) / 8;
  if (p->H > 65535 || tiles * p->cache.H_kv > (1 << 19) || tiles * p->cache.H_kv * p->B > 0x7fffffffll) return FMHA_ERR_TOO_LARGE;
  return FMHA_OK;
}
static PagedGrid grid_of(const fmha_paged_params* p) {
  return paged_grid(sm_count(), p->max_rows, p->H / p->cache.H_kv, static_cast<int64_t>(p->cache.H_kv) * p->B,
                    static_cast<int64_t>(p->cache.table_width) * p->cache.page_rows, p->cache.D, p->cache.bits);
}

}  // namespace fmha

using namespace fmha;

extern "C" {

int fmha_sm100_kv_append(const fmha_kv_append_params* p, void* stream) {
  if (p == nullptr || p->struct_bytes != static_cast<int>(sizeof(fmha_kv_append_params))) return FMHA_ERR_BAD_ARG;
  if (p->dtype != FMHA_DTYPE_F16 && p->dtype != FMHA_DTYPE_BF16) return FMHA_ERR_UNSUPPORTED;
  if (p->B < 0 || p->H < 0 || p->total_rows < 0 || p->n_freq < 0 || (p->flags & ~FMHA_KV_INTERLEAVED)) return FMHA_ERR_BAD_ARG;
  int rc = validate_cache(p->cache, p->B);
  if (rc != FMHA_OK) return rc;
  if (p->H > 65535) return FMHA_ERR_TOO_LARGE;
  if (2 * static_cast<int64_t>(p->n_freq) > p->cache.D || p->n_freq % (p->cache.bits == 4 ? 32 : 8) != 0) return FMHA_ERR_UNSUPPORTED;
  if (p->total_rows == 0) return FMHA_OK;
  KvAppendArgs a;
  std::memset(&a, 0, sizeof(a));
  if (p->B == 0 || p->seqlens == nullptr || !rows_each(p->total_rows, p->B, p->cu_rows, &a.rows_each)) return FMHA_ERR_BAD_ARG;
  if (!rows_ok(p->k, p->cache.H_kv) || !rows_ok(p->v, p->cache.H_kv)) return FMHA_ERR_BAD_ARG;
  if (p->H > 0 && (!rows_ok(p->q, p->H) || !rows_ok(p->q_out, p->H))) return FMHA_ERR_BAD_ARG;
  if (p->n_freq > 0 && p->inv_freq == nullptr) return FMHA_ERR_BAD_ARG;
  rc = check_device();
  if (rc != FMHA_OK) return rc;
  a.q = p->q; a.k = p->k; a.v = p->v; a.q_out = p->q_out;
  a.cache = p->cache;
  a.seqlens = p->seqlens;
  a.cu = p->cu_rows;
  a.B = p->B; a.H = p->H; a.total_rows = p->total_rows;
  a.inv_freq = p->inv_freq;
  a.n_freq = p->n_freq;
  const int e = launch_kv_append(a, p->dtype, (p->flags & FMHA_KV_INTERLEAVED) != 0, static_cast<cudaStream_t>(stream));
  return e != 0 ? cuda_fail(static_cast<cudaError_t>(e)) : FMHA_OK;
}

int fmha_sm100_kv_read(const fmha_kv_read_params* p, void* stream) {
  if (p == nullptr || p->struct_bytes != static_cast<int>(sizeof(fmha_kv_read_params))) return FMHA_ERR_BAD_ARG;
  if (p->dtype != FMHA_DTYPE_F16 && p->dtype != FMHA_DTYPE_BF16) return FMHA_ERR_UNSUPPORTED;
  if (p->B < 0 || p->total_rows < 0) return FMHA_ERR_BAD_ARG;
  int rc = validate_cache(p->cache, p->B);
  if (rc != FMHA_OK) return rc;
  if (p->total_rows == 0) return FMHA_OK;
  if (p->B == 0 || p->cu_rows == nullptr || !rows_ok(p->k, p->cache.H_kv) || !rows_ok(p->v, p->cache.H_kv)) return FMHA_ERR_BAD_ARG;
  rc = check_device();
  if (rc != FMHA_OK) return rc;
  const KvReadArgs a = {p->k, p->v, p->cache, p->cu_rows, p->B, p->total_rows};
  const int e = launch_kv_read(a, p->dtype, static_cast<cudaStream_t>(stream));
  return e != 0 ? cuda_fail(static_cast<cudaError_t>(e)) : FMHA_OK;
}

int fmha_sm100_paged_workspace_bytes(const fmha_paged_params* p, size_t* bytes) {
  if (bytes == nullptr) return FMHA_ERR_BAD_ARG;
  const int rc = validate_paged(p);
  if (rc != FMHA_OK) return rc;
  *bytes = paged_workspace(grid_of(p), p->cache.D);
  return FMHA_OK;
}

int fmha_sm100_paged_fwd(const fmha_paged_params* p, void* stream) {
  int rc = validate_paged(p);
  if (rc != FMHA_OK) return rc;
  if (p->total_rows == 0) return FMHA_OK;
  PagedArgs a;
  std::memset(&a, 0, sizeof(a));
  const fmha_kv_cache& c = p->cache;
  if (p->B == 0 || p->max_rows == 0 || p->seqlens == nullptr || !rows_each(p->total_rows, p->B, p->cu_rows, &a.rows_each)) return FMHA_ERR_BAD_ARG;
  if (p->cu_rows == nullptr && p->max_rows < a.rows_each) return FMHA_ERR_BAD_ARG;
  if (!rows_ok(p->q, p->H) || !rows_ok(p->o, p->H) || c.pages == 0) return FMHA_ERR_BAD_ARG;
  rc = check_device();
  if (rc != FMHA_OK) return rc;
  const PagedGrid grid = grid_of(p);
  const size_t need = paged_workspace(grid, c.D);
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need || (reinterpret_cast<uintptr_t>(p->workspace) & 255))) return FMHA_ERR_BAD_ARG;
  paged_places(a, p->workspace, grid, c.D);
  a.piece = c.page_rows % 64 == 0 ? 64 : c.page_rows % 32 == 0 ? 32 : 16;
  if (c.bits == 4) {
    const CUtensorMapSwizzle sw = c.D == 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;   // that of a row's length
    if ((rc = map_rows(&a.tm_k, c.k, c, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.D / 2, c.D / 2, a.piece, sw))) return rc;
    if ((rc = map_rows(&a.tm_v, c.v, c, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.D / 2, c.D / 2, a.piece, sw))) return rc;
    if ((rc = map_params(&a.tm_kp, c.k_params, c, a.piece))) return rc;
    if ((rc = map_params(&a.tm_vp, c.v_params, c, a.piece))) return rc;
  } else {
    const CUtensorMapDataType type = p->dtype == FMHA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if ((rc = map_rows(&a.tm_k, c.k, c, type, 2, c.D, 64, a.piece, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
    if ((rc = map_rows(&a.tm_v, c.v, c, type, 2, c.D, 64, a.piece, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
  }
  a.q_ptr = p->q.ptr; a.q_ss = p->q.stride_s; a.q_sh = p->H > 1 ? p->q.stride_h : 0;
  a.o_ptr = p->o.ptr; a.o_ss = p->o.stride_s; a.o_sh = p->H > 1 ? p->o.stride_h : 0;
  a.lse = p->lse;
  a.table = c.table; a.table_stride = c.table_stride; a.table_width = c.table_width;
  a.pages = c.pages; a.page_rows = c.page_rows;
  a.seqlens = p->seqlens;
  a.cu = p->cu_rows;
  a.B = p->B; a.H = p->H; a.H_kv = c.H_kv; a.group = p->H / c.H_kv;
  a.total_rows = p->total_rows;
  a.max_rows = p->max_rows;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  a.status = p->status;
  const int e = launch_paged(a, p->dtype, c.D, c.bits, static_cast<cudaStream_t>(stream));
  return e != 0 ? cuda_fail(static_cast<cudaError_t>(e)) : FMHA_OK;
}

}  // extern "C"
