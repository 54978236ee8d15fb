// fmha_paged_sm100.cu — attention of a few new rows per sequence over all its rows in a paged cache, held in 16 or 4 bits ("decode").
//
// Bound by bringing the cache in: a key row is used by the T x group query rows of its head, 4 flops per byte and row in 16 bits.  Four consumer warps
// take their own keys of a step, each with a running softmax of its own; a producer warp keeps several steps in flight through TMA, a copy per page (or
// per 64 rows of one).  The query rows of a tile are the group's heads of consecutive new rows, so K and V are read once for all of them.  A page
// number outside the cache is a coordinate outside the tensor map, which TMA fills with zeros.
//
// Products.  m16n8k16 MMAs from registers with the cache as the operand of 16 rows: S^T = K Q^T and O^T = V^T P^T, so that 8 query rows (a group of
// heads and one new row, as a rule) cost half of what a tile of 16 would, and the accumulators half of the registers; 9 to 16 rows take two such columns.  P^T
// comes out of the first product with keys along the rows and goes into the second with keys along the pairs: an 8 x 8 transposition per 8 keys.
//
// Work.  A unit is (8 or 16 query rows, key head, sequence), its weight its key steps, which only the device knows.  The units stand in one line, and each
// CTA takes an equal piece of it, cutting through units where that falls: all CTAs are busy to the end whatever the lengths are, and there is no bubble
// between units, for the producer goes on to the next one.  A CTA that has a unit from its first to its last step writes the result; a piece of one
// goes to the workspace (at most two of a CTA), and a second kernel joins the pieces of the units that were cut.
//
// 4 bits: b + s (1 + c/16).  Codes are operands of the MMA as they are: four bits at the bottom of a half are the subnormal c 2^-24, those above it c 2^-20, and
// tensor cores take subnormals.  A word of codes thus costs four ANDs and a shift for four pairs.  K: the sums over the 32 dimensions that share a
// scale (the query's even values are taken 16-fold) are multiplied by it in 32 bits; what does not depend on codes, the sum of (b + s) times the query's
// values, is one more MMA of the scales and bases as they lie in memory against those values' sums (in two parts of 11 bits).  So scores are as exact
// as 32 bits allow.  V: P is multiplied by the key's scale of each 32 dimensions, the product with the codes is scaled at the end, and the sum of P (b + s)
// is one more MMA of the transposed scales and bases.  P is rounded to 11 bits for both, and its product with a scale once more.  Both have to stay normal numbers of
// fp16 for that, however small V's values or the probabilities of most keys are.  So the row maximum is kept exactly here (16 bits: up to 2^8), P is taken up to
// 2^15-fold by way of the exponent, and each warp follows the largest scale it has seen, as it does the maximum: scales of 2 to 32 take so much of the factor of P,
// and below 2^-7 or from 32 on the scales are multiplied by a power of two (p_top, v_factor).  (Without that, o was off by 2 % for values of 1e-4, and by more than itself
// where the largest probability, 2^24 times the others, had a value of zero; it costs 3 %, a load and some ten instructions a step.)
//
// Measured (device time, 32/8 heads of 128; bytes of the cache once).  16 bits: 32 sequences of 8000 rows, one new row: 157 to 162 us, 6.7 to 6.5 TB/s, of 1000-8192 98 us, 6.2 TB/s; 16 of 200-4000, four new
// rows: 34.6 us, 4.0 TB/s.  4 bits: two of 90 001-131 072: 63.5 us, 4.5 TB/s; 32 of 1000-8192: 48.5 us, 3.9 TB/s.  Of a short run some 4.5 us pass before the
// first keys have landed and 3 at the join; in 4 bits the steady state is bound by issue and latency (1.6 to 1.8 instructions a cycle and SM; ALU 37-43 %, tensor
// pipe 24 %, DRAM 44-50 %).  More than 8 query rows of a key head in 4 bits (two columns; at D = 128 in 168 registers with 224 bytes of spill stores, 280 of loads): 32 of
// 500-4000, 64/4 heads 32.8 us, D = 64 21.9; 16 of 200-4000, four new rows, 32/8 heads 32.6.  Not meant for new rows by the hundred: every 16 query rows read the whole
// cache again (256 new rows of 4 sequences of 4000, 32/8 heads: 366 us, 476 in 4 bits, where the products would take 41).  Before: tiles of 16 query rows and a grid of splits 39 / 107 / 122 us (four new rows / batch / long), a line of work 46 / 86 / 117,
// the cache as the operand of 16 rows 48 / 55 / 71, shares in the accumulators' order 45 / 54 / 69, starts counted in the line 35 / 47 / 61.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "../../include/fmha_sm100.h"
#include "fmha_cache_args.h"
#include "fmha_device_utils.cuh"
#include "fmha_kernel_args.h"
#include "sm100_ptx.cuh"

namespace fmha {

namespace {

constexpr int kPgWarps = 4;   // consumer warps
constexpr int kPgThreads = 32 * (kPgWarps + 1);
constexpr int kPgMinKeys = 64;     // a CTA's piece of the line holds at least so many
constexpr int kPgWholeKeys = 512;  // units stay whole where no sequence can have more
constexpr int kPgUnitCost = 4;     // what a unit counts in the line beside its steps: its queries, its write-out
constexpr float kPgLn2 = 0.6931471805599453f;

enum PgWaitSite { kPgFull = 191, kPgEmpty = 192, kPgSmemBase = 193 };

// NQ: columns of 8 query rows.
template <int D, bool FOUR, int NQ>
struct PgSmem {
  static constexpr int kUnits = FOUR ? 2 : 1;                  // 16-key blocks of a warp's share of a step
  static constexpr int kKeys = kPgWarps * 16 * kUnits;         // keys of a step
  static constexpr int kRowBytes = FOUR ? D / 2 : D * 2;
  static constexpr int kParBytes = FOUR ? D / kCacheGroup * 4 : 0;
  static constexpr int kTile = kKeys * kRowBytes;              // K or V of a step
  static constexpr int kParTile = kKeys * kParBytes;           // its scales and bases
  static constexpr int kSub = kKeys * 128;                     // 16 bits: a 64-column sub-tile (128-byte swizzle)
  static constexpr int kStage = 2 * (kTile + kParTile);        // K, V, parameters of K, of V
  static constexpr int kCtas = FOUR && D == 64 && NQ == 1 ? 3 : 2;   // of an SM, at the most (paged_grid)
  static constexpr int kStages = FOUR ? (D == 128 ? 4 : NQ == 1 ? 5 : 7) : D == 128 ? 3 : 6;
  // O of the four warps on its way to be added up, a column of 8 rows at a time, in the accumulators' order (16 bytes of a lane), and statistics
  static constexpr int kBlocks = D / 16;
  static constexpr int kOffShare = kStages * kStage;
  static constexpr int kOffStats = kOffShare + kPgWarps * kBlocks * 512;
  static constexpr int kOffBar = kOffStats + kPgWarps * 8 * NQ * 8;
  static constexpr int kOffMisc = kOffBar + 2 * kStages * 8;
  static constexpr int kDynBytes = kOffMisc + 16;   // 1024-byte aligned base: checked by the kernel
  static_assert(kCtas * (kDynBytes + 1024) <= 233472, "so many CTAs share an SM");
  static_assert(kStage % 1024 == 0 || (FOUR && kStage % 512 == 0), "swizzled tiles begin at multiples of 1024 bytes (64-byte rows: 512)");
};

// D = A B + C
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t saddr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr) : "memory");
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix_x2(uint32_t& r0, uint32_t& r1, uint32_t saddr) {
  if constexpr (TRANS) asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(saddr) : "memory");
  else asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(saddr) : "memory");
}
// Lane (g, t) holds elements (g, 2t) and (g, 2t + 1) of an 8 x 8 matrix: afterwards (2t, g) and (2t + 1, g).
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
__device__ __forceinline__ uint32_t lds32(uint32_t saddr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(saddr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t saddr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(saddr));
  return v;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The eight codes of a word, or four codes of either of two keys, as pairs of subnormal halves: codes 0 and 4 (times 2^-24), 1 and 5 (2^-20), 2 and 6
// (2^-24), 3 and 7 (2^-20).
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t (&v)[4]) {
  v[0] = w & 0x000F000Fu;
  v[1] = w & 0x00F000F0u;
  v[2] = (w >> 8) & 0x000F000Fu;
  v[3] = (w >> 8) & 0x00F000F0u;
}

// 4 bits, by the exponent field of V's largest scale (which is 2^(field - 15) to twice that; an infinity counts as the largest number): P is taken
// 2^p_top-fold and the scales 2^v_factor-fold, so that P times a scale stays below 2^16.  Scales from 2^-7 to 32 are left as they are; next to larger ones
// a scale is rounded to 2^-30 of the largest, which only shows where a key with nearly all of the probability has values a millionth of another's.
__device__ __forceinline__ int p_top(int field) { return 15 - min(max(field - 15, 0), 4); }
__device__ __forceinline__ int v_factor(int field) { return field >= 20 ? 19 - min(field, 30) : field >= 8 ? 0 : 15 - field; }
// 2^k as a half, -14 <= k <= 15, twice
__device__ __forceinline__ uint32_t half2_pow2(int k) { return (static_cast<uint32_t>(15 + k) << 10) * 0x00010001u; }

// A sequence: its new rows and its keys.
struct PgSeq {
  int row0, n_new, len;   // first new row, how many take part, rows in the cache
  int n_all;              // new rows there are: the i-th sees len - n_all + i + 1 keys
};
__device__ __forceinline__ PgSeq sequence(const PagedArgs& a, int b) {
  PgSeq s;
  s.row0 = b * a.rows_each;
  s.n_all = a.rows_each;
  if (a.cu != nullptr) {
    s.row0 = a.cu[b];
    s.n_all = a.cu[b + 1] - s.row0;
  }
  s.n_new = s.row0 < 0 ? 0 : min(min(s.n_all, a.max_rows), a.total_rows - s.row0);
  s.len = a.seqlens[b];
  return s;
}
// Keys that the new rows up to `row` see; a sequence ends at its line of the page table.
__device__ __forceinline__ int keys_of(const PagedArgs& a, const PgSeq& s, int row) {
  const int64_t most = static_cast<int64_t>(a.table_width) * a.page_rows;
  return static_cast<int>(max(min(static_cast<int64_t>(s.len) - s.n_all + row + 1, most), static_cast<int64_t>(0)));
}
// A group of units: the key heads of a tile of query rows.  A unit's place in the line is its steps and kPgUnitCost more in front of them (without which
// CTAs with many short units were the last by far, for a switch from unit to unit takes as long as two to four steps: B=16, 200 to 4000 keys 45.6 us, with
// 2 more 36.2, 3 34.9, 4 34.9, 6 35.0; B=32, 1000 to 8192 keys in 4 bits 52.4, 48.2, 47.7, 46.8, 48.9).
struct PgGroup {
  int n_rows, k_limit, steps, weight;   // rows that exist; keys that the last of them sees; what a unit of it counts in the line
};
__device__ __forceinline__ PgGroup group_of(const PagedArgs& a, int b, int tile, int keys) {
  PgGroup u = {0, 0, 0, 0};
  const PgSeq s = sequence(a, b);
  const int r0 = tile * a.tile_rows;
  u.n_rows = min(a.tile_rows, s.n_new * a.group - r0);
  if (u.n_rows <= 0) return u;
  u.k_limit = keys_of(a, s, (r0 + u.n_rows - 1) / a.group);
  u.steps = (u.k_limit + keys - 1) / keys;
  u.weight = a.whole ? 1 : u.steps + kPgUnitCost;   // rows that see no key are written as well
  return u;
}

// A CTA's way along the line, the same in each of its warps: its piece of a unit, then the next.
struct PgWay {
  int tiles, groups;   // row tiles of a sequence, groups in all
  int g, b, tile, hk;  // the unit
  PgGroup u;
  int j0, j1;          // its steps
  int left, n;         // of the CTA's piece of the line, this part included; how many parts came before
  bool first, last;    // the part holds the unit's first step, its last one
};
template <int KEYS>
__device__ __forceinline__ void way_part(const PagedArgs& a, PgWay& w, int off) {
  const int take = min(w.u.weight - off, w.left);
  w.first = off == 0;
  w.last = off + take == w.u.weight;
  w.j0 = a.whole ? 0 : max(off - kPgUnitCost, 0);
  w.j1 = a.whole ? w.u.steps : max(off + take - kPgUnitCost, 0);
  w.left -= take;
}
// False: nothing for this CTA.  Lanes look at 32 groups together; up to 32 of them the lengths are read once.  With more, a lane sums a block of consecutive
// groups, its loads in flight together, and only the block that holds the CTA's first unit is looked through (all of them, 32 at a time, twice: 1000 sequences of
// up to 64 keys, 8/2 heads of 64, 41.0 us, 256 of 100-512, 32/8 heads of 128, 74.4 us, instead of 26.9 and 71.2).
template <int KEYS>
__device__ __forceinline__ bool way_begin(const PagedArgs& a, PgWay& w) {
  const int lane = threadIdx.x & 31;
  w.tiles = a.row_tiles;
  w.groups = a.B * w.tiles;
  auto look = [&](int g) {
    PgGroup u = {0, 0, 0, 0};
    if (g < w.groups) u = w.tiles == 1 ? group_of(a, g, 0, KEYS) : group_of(a, g / w.tiles, g % w.tiles, KEYS);
    return u;
  };
  PgGroup u;
  const int block = (w.groups + 31) / 32;
  long long total, blocks = 0, before = 0;   // of all groups; of those up to this lane's block; of the groups passed
  if (block == 1) {
    u = look(lane);
    total = __reduce_add_sync(0xffffffffu, u.weight);
  } else {
#pragma unroll 8
    for (int i = 0; i < block; ++i) blocks += look(lane * block + i).weight;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
      const long long y = __shfl_up_sync(0xffffffffu, blocks, m);
      if (lane >= m) blocks += y;
    }
    total = __shfl_sync(0xffffffffu, blocks, 31);
  }
  total *= a.H_kv;
  const int least = a.whole ? 1 : max(1, kPgMinKeys / KEYS) + kPgUnitCost, ctas = gridDim.x;
  // a piece of the line (in 32 bits, where a division takes a third of the time, if the line is that short)
  const long long chunk = max(static_cast<long long>(least), total < (1ll << 30) ? (static_cast<int>(total) + ctas - 1) / ctas : (total + ctas - 1) / ctas);
  const long long w0 = chunk * blockIdx.x;
  if (w0 >= total) return false;
  w.left = static_cast<int>(min(chunk, total - w0));
  int g0 = 0;
  if (block > 1) {
    const int at = __ffs(__ballot_sync(0xffffffffu, blocks * a.H_kv > w0)) - 1;   // (there is one: w0 < total)
    if (at > 0) before = __shfl_sync(0xffffffffu, blocks, at - 1);
    g0 = at * block;
    u = look(g0 + lane);
  }
  for (;; u = look(g0 + lane)) {
    int sum = u.weight;   // inclusive
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, sum, m);
      if (lane >= m) sum += y;
    }
    const uint32_t beyond = __ballot_sync(0xffffffffu, (before + sum) * a.H_kv > w0);
    if (beyond != 0u) {
      const int at = __ffs(beyond) - 1;
      w.g = g0 + at;
      before += __shfl_sync(0xffffffffu, sum - u.weight, at);
      w.u.n_rows = __shfl_sync(0xffffffffu, u.n_rows, at);
      w.u.k_limit = __shfl_sync(0xffffffffu, u.k_limit, at);
      w.u.steps = __shfl_sync(0xffffffffu, u.steps, at);
      w.u.weight = __shfl_sync(0xffffffffu, u.weight, at);
      break;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
    g0 += 32;
  }
  w.b = w.tiles == 1 ? w.g : w.g / w.tiles;
  w.tile = w.g - w.b * w.tiles;
  const long long within = w0 - before * a.H_kv;   // (a group's key heads together may have 2^31 steps and more: 2^31 rows of 64 heads)
  w.hk = static_cast<int>(within < (1ll << 31) ? static_cast<unsigned>(within) / static_cast<unsigned>(w.u.weight) : within / w.u.weight);
  w.n = 0;
  way_part<KEYS>(a, w, static_cast<int>(within - static_cast<long long>(w.hk) * w.u.weight));
  return true;
}
template <int KEYS>
__device__ __forceinline__ bool way_next(const PagedArgs& a, PgWay& w) {
  if (w.left == 0) return false;
  ++w.n;
  if (++w.hk == a.H_kv) {
    w.hk = 0;
    do {   // (a sequence's tiles without rows are its last ones)
      if (w.u.weight == 0 || ++w.tile == w.tiles) {
        w.tile = 0;
        if (++w.b >= a.B) return false;   // (the line's length says that there is one: if offsets are changed meanwhile, none is looked for behind them)
      }
      w.u = group_of(a, w.b, w.tile, KEYS);
    } while (w.u.weight == 0);
    w.g = w.b * w.tiles + w.tile;
  }
  way_part<KEYS>(a, w, 0);
  return true;
}

// Block c of O^T of the 8 rows from r0 on (of which n exist): a lane's dimensions of rows 2t and 2t + 1, divided by their sums, to O.
template <bool BF16, bool FOUR>
__device__ __forceinline__ void store_block(const PagedArgs& a, const PgSeq& seq, int r0, int n, int hk, int c, const float4& x, const float (&l)[2]) {
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (2 * t + e >= n) continue;
    const int r = r0 + 2 * t + e;
    const float inv = l[e] > 0.f ? 1.0f / l[e] : 0.f;   // no key: zeros (a NaN among the scores stays one: its accumulator is)
    unsigned short* dst = static_cast<unsigned short*>(a.o_ptr) + static_cast<int64_t>(seq.row0 + r / a.group) * a.o_ss + (hk * a.group + r % a.group) * a.o_sh;
    const uint32_t v = pack2<BF16>((e ? x.y : x.x) * inv, (e ? x.w : x.z) * inv);
    if constexpr (FOUR) {
      *reinterpret_cast<uint32_t*>(dst + 32 * (c / 2) + 4 * g + 2 * (c & 1)) = v;
    } else {
      dst[16 * c + g] = static_cast<unsigned short>(v);
      dst[16 * c + 8 + g] = static_cast<unsigned short>(v >> 16);
    }
  }
}
__device__ __forceinline__ void store_lse(const PagedArgs& a, const PgSeq& seq, int r0, int n, int hk, const float (&m)[2], const float (&l)[2]) {
  const int t = threadIdx.x & 3;
  if (a.lse == nullptr) return;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (2 * t + e >= n) continue;
    const int r = r0 + 2 * t + e;
    a.lse[static_cast<int64_t>(hk * a.group + r % a.group) * a.total_rows + seq.row0 + r / a.group] =
        l[e] == 0.f ? -INFINITY : (m[e] + fast_log2(l[e])) * kPgLn2;
  }
}

}  // namespace

template <int D, bool BF16, bool FOUR, int NQ>
__global__ void __launch_bounds__(kPgThreads, PgSmem<D, FOUR, NQ>::kCtas) fmha_paged_kernel(const __grid_constant__ PagedArgs a) {
  using L = PgSmem<D, FOUR, NQ>;
  constexpr int ST = L::kStages, UN = L::kUnits, KEYS = L::kKeys, ROWS = 8 * NQ;
  constexpr bool MMA_BF16 = BF16 && !FOUR;
  constexpr float kLazy = FOUR ? 0.f : 8.f;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {
    griddep_wait();
    if (threadIdx.x == 0 && a.status != nullptr) atomicCAS(a.status, 0, kPgSmemBase);
    return;
  }
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);   // [ST] a step has landed
  uint64_t* empty = full + ST;                                       // [ST] ... and the four consumer warps are done with it
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc);
  const WaitCtx wctx{abort_flag, a.status};
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < ST; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, kPgWarps);
    }
    mbar_fence_init();
  }
  if (threadIdx.x == 32) {
    tma_prefetch_desc(&a.tm_k);
    tma_prefetch_desc(&a.tm_v);
    if constexpr (FOUR) {
      tma_prefetch_desc(&a.tm_kp);
      tma_prefetch_desc(&a.tm_vp);
    }
  }
  griddep_wait();   // up to here nothing of global memory has been touched
  PgWay w;
  const bool any = way_begin<KEYS>(a, w);
  // What the second kernel needs to know: the unit that this CTA begins in the middle of, and which of its two places its last part is in.
  if (threadIdx.x == 0 && a.part_info != nullptr) a.part_info[blockIdx.x] = make_int2(any && !w.first ? w.g * a.H_kv + w.hk : -1, -1);
  __syncthreads();

  if (!any) {
    // nothing of the line
  } else if (warp == kPgWarps) {
    // ============================ TMA producer ======================================
    // Lane i brings piece i of the step: the page number of the next step is read while this one's buffers are waited for.
    const int pieces = KEYS / a.piece;   // up to 8
    int i = 0;
    do {
      const int* line = a.table + w.b * a.table_stride;
      const int k_limit = w.u.k_limit, hk = w.hk;
      auto page_of = [&](int j) {
        const int key = j * KEYS + lane * a.piece;
        return lane < pieces && key < k_limit ? line[key / a.page_rows] : -1;   // rows behind the last key: zeros
      };
      int page = w.j0 < w.j1 ? page_of(w.j0) : -1;
      for (int j = w.j0; j < w.j1; ++j, ++i) {
        const int s = i % ST;
        const int now = page;
        if (j + 1 < w.j1) page = page_of(j + 1);
        if (lane == 0) {
          if (i >= ST) mbar_wait(empty + s, (i / ST - 1) & 1, wctx, kPgEmpty);
          mbar_arrive_expect_tx(full + s, L::kStage);
        }
        __syncwarp();
        if (lane < pieces) {
          uint8_t* k = smem + s * L::kStage;
          uint8_t* v = k + L::kTile;
          const int at = lane * a.piece, row = (j * KEYS + at) % a.page_rows;
          const int pg = now < 0 ? a.pages : now;   // (a negative one is outside as well)
          if constexpr (FOUR) {
            tma_load_4d(k + at * L::kRowBytes, &a.tm_k, full + s, 0, row, hk, pg);
            tma_load_4d(v + at * L::kRowBytes, &a.tm_v, full + s, 0, row, hk, pg);
            uint8_t* par = v + L::kTile + at * L::kParBytes;
            tma_load_3d(par, &a.tm_kp, full + s, row * (D / kCacheGroup), hk, pg);
            tma_load_3d(par + L::kParTile, &a.tm_vp, full + s, row * (D / kCacheGroup), hk, pg);
          } else {
#pragma unroll
            for (int c = 0; c < D / 64; ++c) tma_load_4d(k + c * L::kSub + at * 128, &a.tm_k, full + s, c * 64, row, hk, pg);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) tma_load_4d(v + c * L::kSub + at * 128, &a.tm_v, full + s, c * 64, row, hk, pg);
          }
        }
        __syncwarp();
      }
    } while (way_next<KEYS>(a, w));
  } else {
    // ============================ consumers =========================================
    const int g = lane >> 2, t = lane & 3;   // this thread's MMA rows are g and g + 8, its columns (query rows) 2t and 2t + 1
    const int tid = threadIdx.x;
    float4* share = reinterpret_cast<float4*>(smem + L::kOffShare);   // [4][kBlocks][32]
    float2* stats = reinterpret_cast<float2*>(smem + L::kOffStats);   // [4][ROWS] (maximum, sum)
    const int mi = lane >> 3, r8 = lane & 7;   // ldmatrix: lane (mi, r8) addresses row r8 of 8x8 block mi
    const int kw = warp * 16 * UN;             // this warp's keys in a step
    // 4 bits: where this lane's row of a ldmatrix lies for groups 0 and 1, and for 2 and 3; blocks: (keys 0-7, group c), (keys 8-15, group c),
    // (keys 0-7, group c + 1), (keys 8-15, group c + 1); the swizzle goes by the row within 8
    [[maybe_unused]] const uint32_t ld_key = (kw + (mi & 1) * 8 + r8) * L::kRowBytes;
    [[maybe_unused]] const uint32_t ld_at[2] = {ld_key + (D == 128 ? ((mi >> 1) ^ (r8 >> 1)) << 4 : ((mi >> 1) ^ (r8 >> 2)) << 4),
                                                ld_key + (((2 + (mi >> 1)) ^ (r8 >> 1)) << 4)};
    [[maybe_unused]] const float inv_sl2 = fminf(1.0f / a.scale_log2, 1e30f);   // (a subnormal scale: finite, as -infinity may be added to 8 times it)
    int i = 0;   // steps so far
    do {
      const PgSeq seq = sequence(a, w.b);
      const int r0 = w.tile * ROWS, n_rows = w.u.n_rows, k_limit = w.u.k_limit;
      const int lim_min = keys_of(a, seq, r0 / a.group);   // all rows see the keys before it
      // ---- Q^T: column n of k-step ks is query row n; the keys that rows 2t and 2t + 1 see ----
      uint32_t qf[NQ][D / 16][2];
      int limit[NQ][2];
      float sl2[NQ][2];
      [[maybe_unused]] uint32_t af[NQ][2];   // the row's sums over the groups of 32 dimensions, twice: high and low part
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        const int r = r0 + nq * 8 + g;
        const bool exists = nq * 8 + g < n_rows;
        const int row = r / a.group, h = w.hk * a.group + r % a.group;
        const unsigned short* q = static_cast<const unsigned short*>(a.q_ptr) + static_cast<int64_t>(seq.row0 + row) * a.q_ss + h * a.q_sh;
        float mul = a.scale_log2;
        if constexpr (FOUR) {
          // thread t has dimensions 32 c + 8 t to + 7 of group c, one word of codes: two k-steps
          uint4 x[D / 32];
          float top = 0.f;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            x[c] = make_uint4(0u, 0u, 0u, 0u);
            if (exists) x[c] = __ldg(reinterpret_cast<const uint4*>(q + c * 32 + t * 8));
            const uint32_t ws[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmax3(top, fabsf(unpack_lo<BF16>(ws[e])), fabsf(unpack_hi<BF16>(ws[e])));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // Rows with values of 1024 and more are scaled down by a power of two, so that the sums of 32, and 16-fold values, fit fp16; the scores are scaled back.
          const int e2 = top >= 1024.f && top < INFINITY ? ilogbf(top) - 9 : 0;
          const float down = __int_as_float((127 - e2) << 23);
          mul *= __int_as_float((127 + e2) << 23);
          af[nq][0] = af[nq][1] = 0u;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            const uint32_t ws[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
            uint32_t hs[4];
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              hs[e] = pack2<false>(unpack_lo<BF16>(ws[e]) * down, unpack_hi<BF16>(ws[e]) * down);
              sum += unpack_lo<false>(hs[e]) + unpack_hi<false>(hs[e]);
            }
            // pairs (0, 4) and (2, 6) 16-fold, see code_pairs
            qf[nq][2 * c][0] = hmul2(prmt(hs[0], hs[2], 0x5410u), 0x4C004C00u);
            qf[nq][2 * c][1] = prmt(hs[0], hs[2], 0x7632u);
            qf[nq][2 * c + 1][0] = hmul2(prmt(hs[1], hs[3], 0x5410u), 0x4C004C00u);
            qf[nq][2 * c + 1][1] = prmt(hs[1], hs[3], 0x7632u);
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (c == t) {
              const float hi = unpack_lo<false>(pack2<false>(sum, 0.f));
              af[nq][0] = pack2<false>(hi, hi);
              af[nq][1] = pack2<false>(sum - hi, sum - hi);
            }
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              qf[nq][ks][e] = exists ? __ldg(reinterpret_cast<const unsigned int*>(q + ks * 16 + e * 8 + 2 * t)) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {   // of the columns this thread has in the accumulators
          sl2[nq][e] = FOUR ? __shfl_sync(0xffffffffu, mul, (2 * t + e) * 4) : mul;
          const int rr = nq * 8 + 2 * t + e;
          limit[nq][e] = rr < n_rows ? keys_of(a, seq, (r0 + rr) / a.group) : 0;
        }
      }

      // running maximum of the unscaled scores; what exponents are shifted by (minus the scaled maximum; 0 before the first key); running sum
      float m[NQ][2];
      float2 shift[NQ], l[NQ];
      float o[NQ][D / 16][4];   // 16 bits: dimensions 16 mt + g and + 8; 4 bits: block 2 c + e has 32 c + 4 g + 2 e and + 1
      [[maybe_unused]] float ob[NQ][4];   // 4 bits: rows are scales and bases
      // 4 bits: the first number above all with the exponent of V's largest scale so far; v_factor of that
      [[maybe_unused]] uint32_t v_limit = 1u << 10;
      [[maybe_unused]] int v_up = v_factor(0);
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        m[nq][0] = m[nq][1] = -INFINITY;
        shift[nq] = l[nq] = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) o[nq][c][0] = o[nq][c][1] = o[nq][c][2] = o[nq][c][3] = 0.f;
        ob[nq][0] = ob[nq][1] = ob[nq][2] = ob[nq][3] = 0.f;
      }

      for (int j = w.j0; j < w.j1; ++j, ++i) {
        const int s = i % ST;
        const int key0 = j * KEYS + kw;   // this warp's first key
        mbar_wait(full + s, (i / ST) & 1, wctx, kPgFull);
        if (key0 < k_limit) {
          const uint32_t sk = smem_u32(smem + s * L::kStage), sv = sk + L::kTile;
          const bool whole = key0 + 16 * UN <= k_limit;
          // 4 bits: V's largest scale, of which the sums of products follow the exponent as they do the maximum; a lane looks at one key's
          [[maybe_unused]] uint32_t v_scale = 0u;
          if constexpr (FOUR) {
            const uint32_t at = sv + L::kTile + L::kParTile + (kw + lane) * L::kParBytes;
            if constexpr (D == 128) {
              const uint4 x = lds128(at);
              v_scale = max(max(x.x & 0x7fffu, x.y & 0x7fffu), max(x.z & 0x7fffu, x.w & 0x7fffu));
            } else {
              const uint2 x = lds64(at);
              v_scale = max(x.x & 0x7fffu, x.y & 0x7fffu);
            }
            if (key0 + lane >= k_limit) v_scale = 0u;
          }
          // ---- S^T ----------------------------------------------------------------------
          float sc[UN][NQ][4];   // keys 16 un + g (rows 2t, 2t + 1), + 8
#pragma unroll
          for (int un = 0; un < UN; ++un) {
            const float zero[4] = {0.f, 0.f, 0.f, 0.f};
            const int kb = kw + un * 16;
            if constexpr (FOUR) {
              const uint32_t par = sv + L::kTile;
              // scales of keys g and g + 8 in 32 bits; (scale, base) of group t of either as the operand of the sums
              float ks[2][D / 32];
              uint32_t pw[4];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t at = par + (kb + g + 8 * e) * L::kParBytes;
                if constexpr (D == 128) {
                  const uint4 x = lds128(at);
                  ks[e][0] = unpack_lo<false>(x.x); ks[e][1] = unpack_lo<false>(x.y); ks[e][2] = unpack_lo<false>(x.z); ks[e][3] = unpack_lo<false>(x.w);
                } else {
                  const uint2 x = lds64(at);
                  ks[e][0] = unpack_lo<false>(x.x); ks[e][1] = unpack_lo<false>(x.y);
                }
                pw[e] = pw[2 + e] = lds32(at + (t % (D / 32)) * 4);
              }
              float2 acc[NQ][2];
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq) acc[nq][0] = acc[nq][1] = make_float2(0.f, 0.f);
#pragma unroll
              for (int c = 0; c < D / 32; c += 2) {
                uint32_t wd[4];   // word t of key g of each block
                ldmatrix_x4<false>(wd, sk + ld_at[c / 2] + un * 16 * L::kRowBytes);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  uint32_t v0[4], v1[4];
                  code_pairs(wd[2 * e], v0);
                  code_pairs(wd[2 * e + 1], v1);
                  const uint32_t a0[4] = {v0[0], v1[0], v0[1], v1[1]}, a1[4] = {v0[2], v1[2], v0[3], v1[3]};
#pragma unroll
                  for (int nq = 0; nq < NQ; ++nq) {
                    float mm[4], m2[4];
                    mma_16816<false>(mm, a0, qf[nq][2 * (c + e)][0], qf[nq][2 * (c + e)][1], zero);
                    mma_16816<false>(m2, a1, qf[nq][2 * (c + e) + 1][0], qf[nq][2 * (c + e) + 1][1], mm);
                    acc[nq][0] = __ffma2_rn(make_float2(ks[0][c + e], ks[0][c + e]), make_float2(m2[0], m2[1]), acc[nq][0]);
                    acc[nq][1] = __ffma2_rn(make_float2(ks[1][c + e], ks[1][c + e]), make_float2(m2[2], m2[3]), acc[nq][1]);
                  }
                }
              }
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq) {
                float base[4];
                mma_16816<false>(base, pw, af[nq][0], af[nq][1], zero);
#pragma unroll
                for (int e = 0; e < 2; ++e) {   // c 2^-20 times 2^16 is c / 16
                  const float2 x = __ffma2_rn(acc[nq][e], make_float2(65536.f, 65536.f), make_float2(base[2 * e], base[2 * e + 1]));
                  sc[un][nq][2 * e] = x.x;
                  sc[un][nq][2 * e + 1] = x.y;
                }
              }
            } else {
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq) sc[un][nq][0] = sc[un][nq][1] = sc[un][nq][2] = sc[un][nq][3] = 0.f;
#pragma unroll
              for (int ks = 0; ks < D / 16; ++ks) {
                uint32_t kf[4];   // blocks: (keys 0-7, dims lo), (keys 8-15, dims lo), (0-7, hi), (8-15, hi)
                ldmatrix_x4<false>(kf, sk + (ks / 4) * L::kSub + sw128_offset(kb + (mi & 1) * 8 + r8, (ks % 4) * 2 + (mi >> 1)));
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) mma_16816<MMA_BF16>(sc[un][nq], kf, qf[nq][ks][0], qf[nq][ks][1], sc[un][nq]);
              }
            }
          }
          // ---- running maximum, exponentials -------------------------------------------------------
          if (key0 + 16 * UN > lim_min) {
#pragma unroll
            for (int un = 0; un < UN; ++un)
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (key0 + un * 16 + (e >> 1) * 8 + g >= limit[nq][e & 1]) sc[un][nq][e] = -INFINITY;
          }
          float mx[NQ][2];
          bool more = FOUR && v_scale >= v_limit;
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = fmaxf(sc[0][nq][e], sc[0][nq][2 + e]);
#pragma unroll
              for (int un = 1; un < UN; ++un) x = fmax3(x, sc[un][nq][e], sc[un][nq][2 + e]);
              mx[nq][e] = x;
              more |= x > (FOUR ? m[nq][e] : fmaf(kLazy, inv_sl2, m[nq][e]));
            }
          if (__any_sync(0xffffffffu, more)) {   // the maximum of a row has moved, or that of the scales
            [[maybe_unused]] float top = 0.f, top_by = 0.f, v_by = 1.f;
            if constexpr (FOUR) {
              const int old = static_cast<int>(v_limit >> 10) - 1, field = max(old, static_cast<int>(__reduce_max_sync(0xffffffffu, v_scale) >> 10));
              top = static_cast<float>(p_top(field));
              top_by = static_cast<float>(p_top(old) - p_top(field));
              v_by = __int_as_float((127 + v_factor(field) - v_up) << 23);
              v_limit = static_cast<uint32_t>(field + 1) << 10;
              v_up = v_factor(field);
            }
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
              float alpha[2], new_shift[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float x = mx[nq][e];
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                const bool moved = x > (FOUR ? m[nq][e] : fmaf(kLazy, inv_sl2, m[nq][e]));
                const float old = e ? shift[nq].y : shift[nq].x;
                // (4 bits: rounded so that no exponent, a multiply-add rounded once, passes `top`, however large the scores are)
                if constexpr (FOUR) new_shift[e] = moved ? __fsub_rd(top, __fmul_ru(x, sl2[nq][e])) : __fsub_rd(old, top_by);
                else new_shift[e] = moved ? -x * sl2[nq][e] : old;
                alpha[e] = !moved && (!FOUR || top_by == 0.f) ? 1.0f : m[nq][e] == -INFINITY ? 0.f : fast_exp2(new_shift[e] - old);
                if (moved) m[nq][e] = x;
              }
              shift[nq] = make_float2(new_shift[0], new_shift[1]);
              l[nq].x *= alpha[0];
              l[nq].y *= alpha[1];
              if constexpr (FOUR) {
                ob[nq][0] *= alpha[0];
                ob[nq][1] *= alpha[1];
                alpha[0] *= v_by;
                alpha[1] *= v_by;
              }
#pragma unroll
              for (int c = 0; c < D / 16; ++c) {
                o[nq][c][0] *= alpha[0];
                o[nq][c][1] *= alpha[1];
                o[nq][c][2] *= alpha[0];
                o[nq][c][3] *= alpha[1];
              }
            }
          }
          uint32_t p[UN][NQ][2];   // P^T as the second operand: keys 2t, 2t + 1 (and 8 further on) of row g
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int un = 0; un < UN; ++un)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 x = __ffma2_rn(make_float2(sc[un][nq][2 * e], sc[un][nq][2 * e + 1]), make_float2(sl2[nq][0], sl2[nq][1]), shift[nq]);
                const float2 y = make_float2(fast_exp2(x.x), fast_exp2(x.y));
                l[nq] = __fadd2_rn(l[nq], y);
                p[un][nq][e] = transpose_8x8(pack2<MMA_BF16>(y.x, y.y));
              }
          // ---- O^T --------------------------------------------------------------------------------
          // What lies behind the last key is not a number that a zero probability could be trusted with: keys 16 un + 8 e + 2t and the next
          auto keep = [&](int un, int e) {
            const int rest = k_limit - key0 - un * 16 - e * 8 - 2 * t;
            return rest >= 2 ? 0xffffffffu : rest == 1 ? 0x0000ffffu : 0u;
          };
#pragma unroll
          for (int un = 0; un < UN; ++un) {
            const int kb = kw + un * 16;
            if constexpr (FOUR) {
              const uint32_t par = sv + L::kTile + L::kParTile;
              uint32_t ss[2][D / 32], pt[4] = {};   // scales of keys 2t, 2t + 1 (8 e further on); transposed scales and bases: row g = value g of a key's
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t at = par + (kb + 8 * e + 2 * t) * L::kParBytes;
                if constexpr (D == 128) {
                  const uint4 x = lds128(at), y = lds128(at + 16);
                  ss[e][0] = prmt(x.x, y.x, 0x5410u); ss[e][1] = prmt(x.y, y.y, 0x5410u); ss[e][2] = prmt(x.z, y.z, 0x5410u); ss[e][3] = prmt(x.w, y.w, 0x5410u);
                } else {
                  const uint4 x = lds128(at);   // both keys
                  ss[e][0] = prmt(x.x, x.z, 0x5410u); ss[e][1] = prmt(x.y, x.w, 0x5410u);
                  const uint32_t lo = g & 2 ? x.y : x.x, hi = g & 2 ? x.w : x.z;
                  pt[2 * e] = g < 4 ? prmt(lo, hi, g & 1 ? 0x7632u : 0x5410u) : 0u;
                }
              }
              if constexpr (D == 128) ldmatrix_x2<true>(pt[0], pt[2], par + (kb + (lane & 15)) * 16);
              if (!whole) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint32_t kp = keep(un, e);
                  pt[2 * e] &= kp;
#pragma unroll
                  for (int c = 0; c < D / 32; ++c) ss[e][c] &= kp;
                }
              }
              if (v_up != 0) {
                const uint32_t by = half2_pow2(v_up);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                  for (int c = 0; c < D / 32; ++c) ss[e][c] = hmul2(ss[e][c], by);
              }
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq) mma_16816<false>(ob[nq], pt, p[un][nq][0], p[un][nq][1], ob[nq]);
#pragma unroll
              for (int c = 0; c < D / 32; c += 2) {
                uint32_t wd[4];   // as for K, transposed: four codes (4g and on of the group) of keys 2t and 2t + 1
                ldmatrix_x4<true>(wd, sv + ld_at[c / 2] + un * 16 * L::kRowBytes);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  uint32_t v0[4], v1[4];
                  code_pairs(wd[2 * e], v0);
                  code_pairs(wd[2 * e + 1], v1);
                  const uint32_t a0[4] = {v0[0], v0[1], v1[0], v1[1]}, a1[4] = {v0[2], v0[3], v1[2], v1[3]};
#pragma unroll
                  for (int nq = 0; nq < NQ; ++nq) {
                    const uint32_t b0 = hmul2(p[un][nq][0], ss[0][c + e]), b1 = hmul2(p[un][nq][1], ss[1][c + e]);
                    mma_16816<false>(o[nq][2 * (c + e)], a0, b0, b1, o[nq][2 * (c + e)]);
                    mma_16816<false>(o[nq][2 * (c + e) + 1], a1, b0, b1, o[nq][2 * (c + e) + 1]);
                  }
                }
              }
            } else {
#pragma unroll
              for (int mt = 0; mt < D / 16; ++mt) {
                uint32_t vf[4];   // transposed blocks: (keys 0-7, dims lo), (keys 0-7, dims hi), (8-15, lo), (8-15, hi)
                ldmatrix_x4<true>(vf, sv + (mt / 4) * L::kSub + sw128_offset(kb + (mi >> 1) * 8 + r8, (mt % 4) * 2 + (mi & 1)));
                if (!whole) {
                  const uint32_t k0 = keep(un, 0), k1 = keep(un, 1);
                  vf[0] &= k0;
                  vf[1] &= k0;
                  vf[2] &= k1;
                  vf[3] &= k1;
                }
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) mma_16816<MMA_BF16>(o[nq][mt], vf, p[un][nq][0], p[un][nq][1], o[nq][mt]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + s);
      }

      // ============================ add up the four warps ===============================
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = e ? l[nq].y : l[nq].x;
#pragma unroll
          for (int k = 4; k < 32; k *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, k);
          // (the maximum in the log2 domain, as the exponents were shifted by it)
          if (g == 0) stats[warp * ROWS + nq * 8 + 2 * t + e] = make_float2(m[nq][e] == -INFINITY ? -INFINITY : -(e ? shift[nq].y : shift[nq].x), sum);
        }
      const bool done = w.first && w.last;
      const int place = 2 * blockIdx.x + (w.n == 0 ? 0 : 1);
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        if (nq * 8 >= n_rows) break;
#pragma unroll
        for (int c = 0; c < L::kBlocks; ++c) {
          float4 x = make_float4(o[nq][c][0], o[nq][c][1], o[nq][c][2], o[nq][c][3]);
          if constexpr (FOUR) {
            // the sum of P (b + s) of the group is in lanes 2 (c/2) and 2 (c/2) + 1 of the rows of scales and bases
            const int at = 8 * (c / 2) + t;
            const float b0 = __shfl_sync(0xffffffffu, ob[nq][0], at) + __shfl_sync(0xffffffffu, ob[nq][0], at + 4);
            const float b1 = __shfl_sync(0xffffffffu, ob[nq][1], at) + __shfl_sync(0xffffffffu, ob[nq][1], at + 4);
            const float f20 = __int_as_float((127 + 20 - v_up) << 23), f16 = __int_as_float((127 + 16 - v_up) << 23);
            x = make_float4(fmaf(x.x, f20, b0), fmaf(x.y, f20, b1), fmaf(x.z, f16, b0), fmaf(x.w, f16, b1));
          }
          share[(warp * L::kBlocks + c) * 32 + lane] = x;
        }
        named_bar_sync(1, 32 * kPgWarps);
        // a warp takes a quarter of the blocks: the rows' factors first
        float f[kPgWarps][2], m_all[2], l_all[2] = {0.f, 0.f};
        {
          float4 st[kPgWarps];   // (maximum, sum) of rows 2t and 2t + 1
#pragma unroll
          for (int k = 0; k < kPgWarps; ++k) st[k] = *reinterpret_cast<const float4*>(stats + k * ROWS + nq * 8 + 2 * t);
          m_all[0] = fmaxf(fmaxf(st[0].x, st[1].x), fmaxf(st[2].x, st[3].x));
          m_all[1] = fmaxf(fmaxf(st[0].z, st[1].z), fmaxf(st[2].z, st[3].z));
#pragma unroll
          for (int k = 0; k < kPgWarps; ++k) {   // (a warp without keys counts nothing)
            f[k][0] = st[k].x == -INFINITY ? 0.f : fast_exp2(st[k].x - m_all[0]);
            f[k][1] = st[k].z == -INFINITY ? 0.f : fast_exp2(st[k].z - m_all[1]);
            l_all[0] = fmaf(f[k][0], st[k].y, l_all[0]);
            l_all[1] = fmaf(f[k][1], st[k].w, l_all[1]);
          }
        }
        if (*abort_flag == 0) {
#pragma unroll
          for (int c = warp; c < L::kBlocks; c += kPgWarps) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kPgWarps; ++k) {
              const float4 y = share[(k * L::kBlocks + c) * 32 + lane];
              x.x = fmaf(f[k][0], y.x, x.x);
              x.y = fmaf(f[k][1], y.y, x.y);
              x.z = fmaf(f[k][0], y.z, x.z);
              x.w = fmaf(f[k][1], y.w, x.w);
            }
            if (done) store_block<BF16, FOUR>(a, seq, r0 + nq * 8, n_rows - nq * 8, w.hk, c, x, l_all);
            else a.part_o[(static_cast<int64_t>(place * NQ + nq) * L::kBlocks + c) * 32 + lane] = x;
          }
          if (warp == 0 && g == 0) {
            if (done) store_lse(a, seq, r0 + nq * 8, n_rows - nq * 8, w.hk, m_all, l_all);
            else a.part_ml[(place * NQ + nq) * 4 + t] = make_float4(m_all[0], l_all[0], m_all[1], l_all[1]);
          }
        }
        named_bar_sync(1, 32 * kPgWarps);   // the shares (and at the end the statistics) may be overwritten
      }
      if (tid == 0 && !w.last) a.part_info[blockIdx.x].y = place;   // the CTA's last part, whose unit goes on in the next CTA
    } while (way_next<KEYS>(a, w));
  }
  // Rows that no unit stands for: outside the sequences, or past max_rows of theirs.
  {
    auto zero = [&](int64_t from, int64_t to) {
      from = max(from, static_cast<int64_t>(0));
      to = min(to, static_cast<int64_t>(a.total_rows));
      const int per_row = a.H * (D / 8);
      for (int64_t i = threadIdx.x; i < (to - from) * per_row; i += kPgThreads) {
        const int64_t row = from + i / per_row;
        const int h = static_cast<int>(i % per_row) / (D / 8), ch = static_cast<int>(i % (D / 8));
        *reinterpret_cast<uint4*>(static_cast<unsigned short*>(a.o_ptr) + row * a.o_ss + h * a.o_sh + ch * 8) = make_uint4(0u, 0u, 0u, 0u);
        if (ch == 0 && a.lse != nullptr) a.lse[static_cast<int64_t>(h) * a.total_rows + row] = -INFINITY;
      }
    };
    if (a.cu != nullptr) {
      for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
        const int64_t from = a.cu[b], to = a.cu[b + 1];
        if (to - from > a.max_rows) zero(from + a.max_rows, to);
        if (b == 0) zero(0, from);
        if (b == a.B - 1) zero(max(from, to), a.total_rows);
      }
    }
  }
  __syncthreads();
  if (*abort_flag) {
    for (int k = 0; k < 20; ++k) __nanosleep(1000000);   // copies in flight end before the CTA does
    __syncthreads();
  }
}

// Joins the pieces of a unit that was cut: block c - 1 takes the unit that CTA c begins in the middle of, if CTA c - 1 began elsewhere; the
// pieces are the last part of CTA c - 1 and the first ones of CTA c and all after it that begin in the same unit.  A warp takes a block of O^T (16
// dimensions).  All there is to it is a chain of loads, so those that can be are made together: which pieces there are, then the first eight of them and
// their statistics (its launch is hidden under the kernel before it).
template <int D, bool BF16, bool FOUR>
__global__ void __launch_bounds__(2 * D) paged_join_kernel(const __grid_constant__ PagedArgs a) {
  griddep_wait();
  constexpr int kBlocks = D / 16, kAhead = 8;
  const int lane = threadIdx.x & 31, block = threadIdx.x >> 5, t = lane & 3, g = lane >> 2;
  const int c = blockIdx.x + 1, nqs = a.tile_rows / 8, nq = blockIdx.y;
  const int2 here = a.part_info[c], before = a.part_info[c - 1];
  int follow = -2;
  if (c + 1 + lane < a.ctas) follow = a.part_info[c + 1 + lane].x;
  const int unit = here.x;
  if (unit < 0 || before.x == unit) return;
  int n = 2;   // pieces
  for (int k0 = c + 1;;) {
    const uint32_t same = __ballot_sync(0xffffffffu, follow == unit);
    n += same == 0xffffffffu ? 32 : __ffs(~same) - 1;
    if (same != 0xffffffffu) break;
    k0 += 32;
    follow = k0 + lane < a.ctas ? a.part_info[k0 + lane].x : -2;
  }
  auto place = [&](int k) { return (k == 0 ? before.y : 2 * (c + k - 1)) * nqs + nq; };
  float4 x[kAhead];
  auto load = [&](int k0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + k < n) x[k] = a.part_o[(static_cast<int64_t>(place(k0 + k)) * kBlocks + block) * 32 + lane];
    }
  };
  load(0);
  // maxima and sums of rows 2t and 2t + 1: lane (g, t) looks at pieces g, g + 8, ...; up to 32 of them are read once
  float4 st[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    st[k] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    if (8 * k + g < n) st[k] = a.part_ml[place(8 * k + g) * 4 + t];
  }
  const int hk = unit % a.H_kv, tile = unit / a.H_kv % a.row_tiles, b = unit / a.H_kv / a.row_tiles;
  const PgSeq seq = sequence(a, b);
  float m_all[2] = {fmaxf(fmaxf(st[0].x, st[1].x), fmaxf(st[2].x, st[3].x)), fmaxf(fmaxf(st[0].z, st[1].z), fmaxf(st[2].z, st[3].z))};
  for (int k = 32 + g; k < n; k += 8) {
    const float4 y = a.part_ml[place(k) * 4 + t];
    m_all[0] = fmaxf(m_all[0], y.x);
    m_all[1] = fmaxf(m_all[1], y.z);
  }
#pragma unroll
  for (int k = 4; k < 32; k *= 2) {
    m_all[0] = fmaxf(m_all[0], __shfl_xor_sync(0xffffffffu, m_all[0], k));
    m_all[1] = fmaxf(m_all[1], __shfl_xor_sync(0xffffffffu, m_all[1], k));
  }
  float l_all[2] = {0.f, 0.f};
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = 0; k0 < n; k0 += kAhead) {
    // factors of the eight pieces, of this lane's one: a piece without keys that a row sees counts nothing
    float4 s = st[0];
    if (k0 > 0) s = k0 + g < n ? a.part_ml[place(k0 + g) * 4 + t] : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    const float f0 = s.x == -INFINITY ? 0.f : fast_exp2(s.x - m_all[0]), f1 = s.z == -INFINITY ? 0.f : fast_exp2(s.z - m_all[1]);
    l_all[0] = fmaf(f0, s.y, l_all[0]);
    l_all[1] = fmaf(f1, s.w, l_all[1]);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const float k_f0 = __shfl_sync(0xffffffffu, f0, 4 * k + t), k_f1 = __shfl_sync(0xffffffffu, f1, 4 * k + t);
      acc.x = fmaf(k_f0, x[k].x, acc.x);
      acc.y = fmaf(k_f1, x[k].y, acc.y);
      acc.z = fmaf(k_f0, x[k].z, acc.z);
      acc.w = fmaf(k_f1, x[k].w, acc.w);
    }
    if (k0 + kAhead < n) load(k0 + kAhead);
  }
#pragma unroll
  for (int k = 4; k < 32; k *= 2) {
    l_all[0] += __shfl_xor_sync(0xffffffffu, l_all[0], k);
    l_all[1] += __shfl_xor_sync(0xffffffffu, l_all[1], k);
  }
  const int r0 = tile * a.tile_rows + nq * 8, n_rows = min(8, seq.n_new * a.group - r0);
  store_block<BF16, FOUR>(a, seq, r0, n_rows, hk, block, acc, l_all);
  if (block == 0 && g == 0) store_lse(a, seq, r0, n_rows, hk, m_all, l_all);
}

// The rules, each with both sides measured (us, 32/8 heads of 128, one new row if not said; 16 bits if not said):
// - 8 query rows as one column where a unit has no more, else tiles of 16.  Four rows of a group: 54.3 against 55.4 with tiles of 16 (32 sequences of
//   500-4000), in 4 bits 30.3 against 44.2.  Twelve rows: 60.2 with a tile of 16, 87.3 with two of 8, which read the cache twice.
// - Units whole (no workspace, no second kernel) up to 512 keys.  One sequence of 250 keys: 6.9, cut 9.1; of 512: 9.3, cut 9.4, in 4 bits 8.5 and 10.0;
//   64 of 100-512: 23.7 and 25.8; but one of 700: 11.2 and 8.9, of 1000: 14.2 and 9.8.
// - Pieces of at least 64 keys.  At least 128 and 256: one sequence of 700 keys 9.8 and 11.4 against 8.9, of 2000: 10.0 and 11.2 against 9.8; of 30 000
//   every CTA has more than that.
// - Two CTAs per SM, but no more than the most keys that there can be would occupy.  Three, of fewer stages, against two: D = 128, 4 bits, 32 sequences of
//   1000-8192 48.7 and 46.7, two of 90 001-131 072 64.2 and 60.8; D = 64, 16/4 heads, 16 bits: 64 of 500-4000 32.3 and 32.2, one of 60 000 24.6 and 21.9; 4 bits,
//   tiles of 16: 22.1 and 21.4.  What a CTA costs at its start and at the join outweighs the warps that it adds, but for D = 64 in 4 bits with one
//   column, where a step is mostly instructions: three from 2/3 of a unit per SM on.  64 sequences of 500-4000, 16/4 heads (256 units): 23.3 and 27.1; 64 of
//   100-3000, 12/12: 42.6 and 55.6; 128 of 300-2000, 32/8: 42.4 and 49.1; 16 of 500-4000, 32/8 (128 units): 15.1 and 16.1; 100 of 100-3000, 8/1: 18.2 and
//   18.7; the other way 8 of 500-4000, 32/8 (64 units): 12.5 and 11.6; one of 60 000, 16/4: 19.1 and 18.0; units that stay whole, 512 of up to 200 keys: 11.6 and 10.8.
PagedGrid paged_grid(int64_t sms, int64_t max_rows, int64_t group, int64_t heads, int64_t max_keys, int D, int bits) {
  PagedGrid g;
  g.tile_rows = max_rows * group <= 8 ? 8 : 16;
  g.row_tiles = (max_rows * group + g.tile_rows - 1) / g.tile_rows;
  g.whole = max_keys <= kPgWholeKeys;
  const int64_t units = g.row_tiles * heads, most = units * std::max<int64_t>(1, (max_keys + kPgMinKeys - 1) / kPgMinKeys);
  const bool three = D == 64 && bits == 4 && g.tile_rows == 8 && !g.whole && 3 * units >= 2 * sms;
  g.ctas = static_cast<int>(std::max<int64_t>(1, std::min((three ? 3 : 2) * sms, most)));
  return g;
}
size_t paged_workspace(const PagedGrid& g, int D) {
  return g.whole ? 0 : static_cast<size_t>(g.ctas) * (2 * g.tile_rows * (D * sizeof(float) + sizeof(float2)) + sizeof(int2));
}
void paged_places(PagedArgs& a, void* workspace, const PagedGrid& g, int D) {
  a.whole = g.whole;
  a.ctas = g.ctas;
  a.tile_rows = g.tile_rows;
  a.row_tiles = static_cast<int>(g.row_tiles);
  if (g.whole) return;
  const size_t rows = static_cast<size_t>(g.ctas) * 2 * g.tile_rows;
  a.part_o = static_cast<float4*>(workspace);
  a.part_ml = a.part_o + rows * D / 4;
  a.part_info = reinterpret_cast<int2*>(a.part_ml + rows / 2);
}

template <int D, bool BF16, bool FOUR, int NQ>
static int launch_paged_impl(const PagedArgs& a, cudaStream_t stream) {
  using L = PgSmem<D, FOUR, NQ>;
  auto kfn = fmha_paged_kernel<D, BF16, FOUR, NQ>;
  static std::atomic<bool> configured[64] = {};   // per device; set after the attribute call succeeded
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  cudaError_t e = launch_overlapped(kfn, dim3(a.ctas), dim3(kPgThreads), L::kDynBytes, stream, a);
  if (e == cudaSuccess && !a.whole && a.ctas > 1) e = launch_overlapped(paged_join_kernel<D, BF16, FOUR>, dim3(a.ctas - 1, NQ), dim3(2 * D), 0, stream, a);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

int launch_paged(const PagedArgs& a, int dtype, int D, int bits, cudaStream_t stream) {
  const bool bf = dtype == FMHA_DTYPE_BF16, four = bits == 4;
#define FMHA_PAGED_CASE(DD, BF, F4) \
  if (D == DD && bf == BF && four == F4) return a.tile_rows == 8 ? launch_paged_impl<DD, BF, F4, 1>(a, stream) : launch_paged_impl<DD, BF, F4, 2>(a, stream);
  FMHA_PAGED_CASE(64, false, false)
  FMHA_PAGED_CASE(64, true, false)
  FMHA_PAGED_CASE(128, false, false)
  FMHA_PAGED_CASE(128, true, false)
  FMHA_PAGED_CASE(64, false, true)
  FMHA_PAGED_CASE(64, true, true)
  FMHA_PAGED_CASE(128, false, true)
  FMHA_PAGED_CASE(128, true, true)
#undef FMHA_PAGED_CASE
  return static_cast<int>(cudaErrorInvalidValue);
}

}  // namespace fmha
