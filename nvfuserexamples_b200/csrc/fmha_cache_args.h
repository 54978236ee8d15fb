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
constexpr int kPagedKeyStep = 64;          // keys per step of the paged attention kernel
constexpr int kPagedRows = 16;             // query rows of one of its tiles
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
  int n_split;       // CTAs that may share a sequence's keys
  float scale_log2;
  float* part_o;     // [total_rows * H, n_split, D] unnormalised shares of O, when n_split > 1
  float2* part_ml;   // [total_rows * H, n_split] their maximum (log2 domain) and sum
  int* status;
};

int launch_kv_append(const KvAppendArgs& a, int dtype, bool interleaved, cudaStream_t stream);
int launch_kv_read(const KvReadArgs& a, int dtype, cudaStream_t stream);
int paged_splits(int64_t sms, int64_t tiles, int64_t max_keys, int D, int bits);   // n_split for these sizes
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
