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
PagedGrid paged_grid(int64_t sms, int64_t max_rows, int64_t group, int64_t heads, int64_t max_keys);   // heads: key heads of all sequences
size_t paged_workspace(const PagedGrid& g, int D);
void paged_places(PagedArgs& a, void* workspace, const PagedGrid& g, int D);   // lays the workspace out
int launch_paged(const PagedArgs& a, int dtype, int D, int bits, cudaStream_t stream);

#ifdef __CUDACC__
// The sequence that packed row `row` belongs to, by a whole warp: how many sequences end at or before it.  -1 in front of the first, B behind the last.
__device__ __forceinline__ int sequence_of_row(const int* cu, int B, int row) {
  const int lane = threadIdx.x & 31;
  if (row < cu[0]) return -1;
  int n = 0;
  for (int i = 0; i < B; i += 32) {
    const bool ended = i + lane < B && cu[i + lane + 1] <= row;
    n += __popc(__ballot_sync(0xffffffffu, ended));
  }
  return n;
}
#endif

}  // namespace fmha
