// fmha_cache_args.h — parameter blocks and launchers of the paged-cache kernels, and the bits of arithmetic they share.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fmha_sm100.h"

namespace fmha {

constexpr int kCacheGroup = 32;            // values of a row that share a scale and a base in a 4-bit cache
constexpr float kCacheLimit = 20000.0f;    // what a 4-bit cache holds at most: scale <= 42 667 and base >= -62 667 then fit fp16
constexpr int kMaxPageRows = 1 << 16;

struct KvAppendArgs {
  fmha_tensor4 q, k, v, q_out;
  fmha_kv_cache cache;
  const int* seqlens;
  const int* cu;     // null: rows_each rows a sequence
  int B, H, total_rows, rows_each;
  const float* inv_freq;
  int n_freq;
  int parts;         // warps that share a row
};

struct KvReadArgs {
  fmha_tensor4 k, v;
  fmha_kv_cache cache;
  const int* cu;
  int B, total_rows;
};

struct PagedArgs {
  alignas(64) CUtensorMap tm_k;    // 16-bit rows, or codes
  alignas(64) CUtensorMap tm_v;
  alignas(64) CUtensorMap tm_kp;   // 4 bits: scales and bases
  alignas(64) CUtensorMap tm_vp;
  const void* q_ptr;
  int64_t q_ss, q_sh;
  void* o_ptr;
  int64_t o_ss, o_sh;
  float* lse;
  const int* table;
  int64_t table_stride;
  int table_width, pages, page_rows;
  int piece;         // rows of one copy: it divides a page and a key step
  const int* seqlens;
  const int* cu;     // null: rows_each rows a sequence
  int B, H, H_kv, group, total_rows, rows_each, max_rows;
  int tile_rows, row_tiles, whole, ctas;   // PagedGrid
  float scale_log2;
  float4* part_o;    // [ctas, 2, tile_rows / 8, D / 16, 32] unnormalised O of pieces of units, in the accumulators' order
  float4* part_ml;   // [ctas, 2, tile_rows / 8, 4] maximum (log2 domain) and sum of two rows each
  int2* part_info;   // [ctas] the unit that a CTA begins in the middle of, or -1; the place of its last part, if that is not its unit's end
  int* status;
};

int launch_kv_append(const KvAppendArgs& a, int dtype, bool interleaved, cudaStream_t stream);
int launch_kv_read(const KvReadArgs& a, int dtype, cudaStream_t stream);
struct PagedGrid {
  int tile_rows;       // (new row, head of the group) pairs of a tile: 8 or 16
  int64_t row_tiles;   // that max_rows new rows make
  bool whole;          // no unit is cut
  int ctas;
};
PagedGrid paged_grid(int64_t sms, int64_t max_rows, int64_t group, int64_t heads, int64_t max_keys, int D, int bits);   // heads: key heads of all sequences
size_t paged_workspace(const PagedGrid& g, int D);
void paged_places(PagedArgs& a, void* workspace, const PagedGrid& g, int D);   // lays the workspace out
int launch_paged(const PagedArgs& a, int dtype, int D, int bits, cudaStream_t stream);

#ifdef __CUDACC__
// The sequence that packed row `row` belongs to, by a whole warp: b (-1: none), its first row, how many it has, and its entry of `lens`.  Lanes look at a
// sequence each, and everything about it comes with the same round of loads.
struct RowSequence {
  int b, first, n, len;
};
__device__ __forceinline__ RowSequence sequence_of_row(const int* cu, const int* lens, int B, int row) {
  const int lane = threadIdx.x & 31;
  RowSequence s = {-1, 0, 0, 0};
#pragma unroll 4
  for (int i0 = 0; i0 < B; i0 += 32) {   // (no early end, so that the loads of a large batch are in flight together)
    const int i = i0 + lane;
    int lo = 0, hi = 0, len = 0;
    if (i < B) {
      lo = cu[i];
      hi = cu[i + 1];
      if (lens != nullptr) len = lens[i];
    }
    if (lo <= row && row < hi) s = {i, lo, hi - lo, len};
  }
  const uint32_t found = __ballot_sync(0xffffffffu, s.b >= 0);
  const int at = found != 0u ? __ffs(found) - 1 : 0;
  return {__shfl_sync(0xffffffffu, s.b, at), __shfl_sync(0xffffffffu, s.first, at), __shfl_sync(0xffffffffu, s.n, at),
          __shfl_sync(0xffffffffu, s.len, at)};
}
#endif

}  // namespace fmha
