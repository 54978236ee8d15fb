// fmha_paged_sm100.cu — attention of a few new rows per sequence over all its rows in a paged cache, held in 16 or 4 bits ("decode").
//
// Bound by bringing the cache in: a key row is used by the T x group query rows of its head, 4 flops per byte and row in 16 bits.  As in
// fmha_fwd_rows_sm100.cu, m16n8k16 MMAs from registers fit the row count, each of four consumer warps takes 16 of every 64 keys with a running
// softmax of its own, and a producer warp keeps several steps in flight through TMA, a copy per page (or per 64 rows of one).  The query rows of a
// tile are the group's heads of consecutive new rows, so K and V are read once for all of them.  A page number outside the cache is a coordinate
// outside the tensor map, which TMA fills with zeros.
//
// The keys of a sequence are dealt out over CTAs (splits_of) by its own length, which only the device knows; each leaves its unnormalised O, maximum and
// sum in the workspace, and a second kernel joins them.  Where a sequence has one share, its CTA writes the result itself.
//
// 4 bits: a thread takes eight codes from a word as four pairs of halves: a code in the low bits of the half 1024 is 1024 + c, one in bits 4 to 7 of the half
// 64 is 64 + c; minus 1024 or 64 that is c, exactly, and b + s + (s / 16) c is one fused multiply-add.  The dimensions of K are permuted in the
// MMA's contraction, and those of V over its columns, so that a word's codes are one thread's operands; keys keep their order, in which P comes out of
// the first MMA.
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

constexpr int kPgWarps = 4;   // consumer warps, 16 keys of a step each
constexpr int kPgThreads = 32 * (kPgWarps + 1);
constexpr int kPgMinSteps = 4;   // key steps of a share
constexpr float kPgLn2 = 0.6931471805599453f;

enum PgWaitSite { kPgFull = 191, kPgEmpty = 192 };

template <int D, bool FOUR>
struct PgSmem {
  static constexpr int kRowBytes = FOUR ? D / 2 : D * 2;
  static constexpr int kParBytes = FOUR ? D / kCacheGroup * 4 : 0;
  static constexpr int kTile = kPagedKeyStep * kRowBytes;      // K or V of a step
  static constexpr int kParTile = kPagedKeyStep * kParBytes;   // its scales and bases
  static constexpr int kSub = kPagedKeyStep * 128;             // 16 bits: a 64-column sub-tile (128-byte swizzle)
  static constexpr int kStage = 2 * (kTile + kParTile);        // K, V, parameters of K, of V
  static constexpr int kStages = FOUR ? (D == 128 ? 8 : 12) : D == 128 ? 3 : 6;
  static constexpr int kOffBar = kStages * kStage;
  static constexpr int kOffMisc = kOffBar + 2 * kStages * 8;
  static constexpr int kDynBytes = kOffMisc + 16 + 1024;
  // after the key loop, over the stages: O of the four warps, [16][D + 8] fp32 each, and their row statistics
  static constexpr int kRowFloats = D + 8;
  static constexpr int kShare = kPagedRows * kRowFloats * 4;
  static constexpr int kOffStats = kPgWarps * kShare;
  static_assert(kOffStats + kPgWarps * kPagedRows * 8 <= kOffBar, "the shares fit over the stages");
  static_assert(kStage % 1024 == 0 || FOUR, "swizzled tiles begin at multiples of 1024 bytes");
  static_assert(kStage % 512 == 0, "and those of 64-byte rows at multiples of 512");
};

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
__device__ __forceinline__ uint32_t lds32(uint32_t saddr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(saddr));
  return v;
}
__device__ __forceinline__ uint32_t hadd2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// (w & mask) | magic, one instruction
__device__ __forceinline__ uint32_t mask_or(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(mask), "r"(magic));
  return d;
}
// The values of a word's eight codes as four pairs: pair j holds codes j (low half) and j + 4.  step = s / 16 and first = b + s of either half.
__device__ __forceinline__ void values4(uint32_t w, uint32_t step, uint32_t first, uint32_t (&v)[4]) {
  const uint32_t w8 = w >> 8;
  v[0] = hfma2(hadd2(mask_or(w, 0x000F000Fu, 0x64006400u), 0xE400E400u), step, first);
  v[1] = hfma2(hadd2(mask_or(w, 0x00F000F0u, 0x54005400u), 0xD400D400u), step, first);
  v[2] = hfma2(hadd2(mask_or(w8, 0x000F000Fu, 0x64006400u), 0xE400E400u), step, first);
  v[3] = hfma2(hadd2(mask_or(w8, 0x00F000F0u, 0x54005400u), 0xD400D400u), step, first);
}
// Two finite 16-bit values of the query type as halves that stay finite.
template <bool BF16>
__device__ __forceinline__ uint32_t to_half2(uint32_t w) {
  if constexpr (!BF16) return w;
  auto clamp = [](float x) { return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.f), 65504.f) : x; };
  return pack2<false>(clamp(unpack_lo<true>(w)), clamp(unpack_hi<true>(w)));
}

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
// Over how many CTAs the keys of a tile are dealt out: by their number alone, so that both kernels find the same.
__device__ __forceinline__ int splits_of(int keys, int n_split) {
  const int steps = (keys + kPagedKeyStep - 1) / kPagedKeyStep;
  return max(1, min(n_split, steps / kPgMinSteps));
}

}  // namespace

template <int D, bool BF16, bool FOUR>
__global__ void __launch_bounds__(kPgThreads, 2) fmha_paged_kernel(const __grid_constant__ PagedArgs a) {
  griddep_wait();
  using L = PgSmem<D, FOUR>;
  constexpr int ST = L::kStages;
  constexpr bool MMA_BF16 = BF16 && !FOUR;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);   // [ST] a step has landed
  uint64_t* empty = full + ST;                                       // [ST] ... and the four consumer warps are done with it
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc);
  const WaitCtx wctx{abort_flag, a.status};

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int split = blockIdx.x, hk = blockIdx.y % a.H_kv, tile = blockIdx.y / a.H_kv, b = blockIdx.z;
  const PgSeq seq = sequence(a, b);

  // Rows that no tile of the grid stands for: outside the sequences, or past max_rows of theirs.
  if (split == 0 && tile == 0) {
    auto zero = [&](int64_t from, int64_t to, int h0, int h1) {
      from = max(from, static_cast<int64_t>(0));
      to = min(to, static_cast<int64_t>(a.total_rows));
      const int per_row = (h1 - h0) * (D / 8);
      for (int64_t i = threadIdx.x; i < (to - from) * per_row; i += kPgThreads) {
        const int64_t row = from + i / per_row;
        const int h = h0 + static_cast<int>(i % per_row) / (D / 8), ch = static_cast<int>(i % (D / 8));
        *reinterpret_cast<uint4*>(static_cast<unsigned short*>(a.o_ptr) + row * a.o_ss + h * a.o_sh + ch * 8) = make_uint4(0u, 0u, 0u, 0u);
        if (ch == 0 && a.lse != nullptr) a.lse[static_cast<int64_t>(h) * a.total_rows + row] = -INFINITY;
      }
    };
    const int h0 = hk * a.group, h1 = h0 + a.group;
    if (seq.n_all > a.max_rows) zero(static_cast<int64_t>(seq.row0) + a.max_rows, static_cast<int64_t>(seq.row0) + seq.n_all, h0, h1);
    if (b == 0) zero(0, seq.row0, h0, h1);
    if (b == a.B - 1) zero(static_cast<int64_t>(seq.row0) + max(seq.n_all, 0), a.total_rows, h0, h1);
  }
  const int r0 = tile * kPagedRows;                                  // row r of the head's (new row, head of the group) pairs
  const int n_rows = min(kPagedRows, seq.n_new * a.group - r0);
  if (n_rows <= 0) return;
  const int k_limit = keys_of(a, seq, (r0 + n_rows - 1) / a.group);  // of the tile's last row
  const int n_split = splits_of(k_limit, a.n_split);
  if (split >= n_split) return;
  const int n_steps = (k_limit + kPagedKeyStep - 1) / kPagedKeyStep;
  const int j0 = static_cast<int>(static_cast<int64_t>(n_steps) * split / n_split), j1 = static_cast<int>(static_cast<int64_t>(n_steps) * (split + 1) / n_split);

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < ST; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, kPgWarps);
    }
    mbar_fence_init();
  }
  __syncthreads();

  const int g = lane >> 2, t = lane & 3;   // this thread's MMA rows are g and g + 8
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  if (warp == kPgWarps) {
    // ============================ TMA producer ======================================
    // Lane i brings piece i of the step: the page number of the next step is read while this one's buffers are waited for.
    const int pieces = kPagedKeyStep / a.piece;   // 1, 2 or 4
    const int* line = a.table + b * a.table_stride;
    auto page_of = [&](int j) {
      const int key = j * kPagedKeyStep + lane * a.piece;
      return lane < pieces && key < k_limit ? line[key / a.page_rows] : -1;   // rows behind the last key: zeros
    };
    int page = j0 < j1 ? page_of(j0) : -1;
    for (int j = j0; j < j1; ++j) {
      const int i = j - j0, s = i % ST;
      const int now = page;
      if (j + 1 < j1) page = page_of(j + 1);
      if (lane == 0) {
        if (i >= ST) mbar_wait(empty + s, (i / ST - 1) & 1, wctx, kPgEmpty);
        mbar_arrive_expect_tx(full + s, L::kStage);
      }
      __syncwarp();
      if (lane < pieces) {
        uint8_t* k = smem + s * L::kStage;
        uint8_t* v = k + L::kTile;
        const int at = lane * a.piece, row = (j * kPagedKeyStep + at) % a.page_rows;
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
  } else {
    // ============================ consumers =========================================
    // Q fragments of the 16 rows (rows that do not exist are zeros), and the keys that rows g and g + 8 see
    uint32_t qf[D / 16][4];
    int limit[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = r0 + g + hf * 8;
      const bool exists = g + hf * 8 < n_rows;
      const int row = r / a.group, h = hk * a.group + r % a.group;
      limit[hf] = exists ? keys_of(a, seq, row) : 0;
      const unsigned short* q = static_cast<const unsigned short*>(a.q_ptr) + static_cast<int64_t>(seq.row0 + row) * a.q_ss + h * a.q_sh;
      if constexpr (FOUR) {
        // thread t has the dimensions [t D/4, +D/4) of the contraction, eight (a word of codes) to two k-steps; pair j is (j, j + 4)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint4 w = make_uint4(0u, 0u, 0u, 0u);
          if (exists) w = __ldg(reinterpret_cast<const uint4*>(q + t * (D / 4) + i * 8));
          const uint32_t x = to_half2<BF16>(w.x), y = to_half2<BF16>(w.y), z = to_half2<BF16>(w.z), u = to_half2<BF16>(w.w);
          qf[2 * i][hf] = prmt(x, z, 0x5410u);
          qf[2 * i][2 + hf] = prmt(x, z, 0x7632u);
          qf[2 * i + 1][hf] = prmt(y, u, 0x5410u);
          qf[2 * i + 1][2 + hf] = prmt(y, u, 0x7632u);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            qf[ks][e * 2 + hf] = exists ? __ldg(reinterpret_cast<const unsigned int*>(q + ks * 16 + e * 8 + 2 * t)) : 0u;
      }
    }
    const float sl2 = a.scale_log2;
    // 16 bits, ldmatrix: lane (mi, r) addresses row r of 8x8 block mi
    const int mi = lane >> 3, r = lane & 7;
    const int k_row = warp * 16 + (mi >> 1) * 8 + r, k_ch = mi & 1;
    const int v_row = warp * 16 + (mi & 1) * 8 + r, v_ch = mi >> 1;

    for (int j = j0; j < j1; ++j) {
      const int i = j - j0, s = i % ST;
      const int key0 = j * kPagedKeyStep + warp * 16;   // this warp's 16 keys
      mbar_wait(full + s, (i / ST) & 1, wctx, kPgFull);
      if (key0 < k_limit) {
        const uint32_t sk = smem_u32(smem + s * L::kStage), sv = sk + L::kTile;
        const bool whole = key0 + 16 <= k_limit;
        float sc[2][4] = {};
        if constexpr (FOUR) {
          const uint32_t par = sv + L::kTile;
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const int key = warp * 16 + nt * 8 + g;
            // thread t's D / 4 dimensions lie in one group of 32
            const uint32_t sb = lds32(par + key * L::kParBytes + (D == 128 ? t : t >> 1) * 4);
            const uint32_t ss = prmt(sb, sb, 0x1010u), bb = prmt(sb, sb, 0x3232u);
            const uint32_t step = hmul2(ss, 0x2C002C00u), first = hadd2(bb, ss);   // s / 16, b + s
            uint32_t w[D / 32];
            if constexpr (D == 128) {
              const uint4 x = lds128(sk + key * 64 + ((t ^ ((key >> 1) & 3)) << 4));   // 64-byte swizzle
              w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            } else {
              w[0] = lds32(sk + key * 32 + t * 8);
              w[1] = lds32(sk + key * 32 + t * 8 + 4);
            }
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
              uint32_t v[4];
              values4(w[q], step, first, v);
              mma_16816<false>(sc[nt], qf[2 * q], v[0], v[1]);
              mma_16816<false>(sc[nt], qf[2 * q + 1], v[2], v[3]);
            }
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t kf[4];
            ldmatrix_x4<false>(kf, sk + (ks / 4) * L::kSub + sw128_offset(k_row, (ks % 4) * 2 + k_ch));
            mma_16816<MMA_BF16>(sc[0], qf[ks], kf[0], kf[1]);
            mma_16816<MMA_BF16>(sc[1], qf[ks], kf[2], kf[3]);
          }
        }
        // scaled scores in the log2 domain
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = sc[nt][e] * sl2;
            if (key0 + nt * 8 + 2 * t + (e & 1) >= limit[e >> 1]) x = -INFINITY;
            sc[nt][e] = x;
          }
        uint32_t p[4];
        float alpha[2];
        bool moved = false;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          float mx = fmaxf(fmaxf(sc[0][2 * hf], sc[0][2 * hf + 1]), fmaxf(sc[1][2 * hf], sc[1][2 * hf + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          float m_new = fmaxf(m[hf], mx);
          if (m[hf] != -INFINITY && m_new - m[hf] <= 8.0f) m_new = m[hf];   // lazy: exponentials stay below 2^8
          alpha[hf] = m_new == m[hf] ? 1.0f : fast_exp2(m[hf] - m_new);
          moved |= m_new != m[hf];
          m[hf] = m_new;
          const float neg_m = m_new == -INFINITY ? 0.f : -m_new;   // no key seen so far
          float e[2][2];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) e[nt][c] = fast_exp2(sc[nt][2 * hf + c] + neg_m);
          l[hf] = l[hf] * alpha[hf] + ((e[0][0] + e[0][1]) + (e[1][0] + e[1][1]));
          p[hf] = pack2<MMA_BF16>(e[0][0], e[0][1]);
          p[2 + hf] = pack2<MMA_BF16>(e[1][0], e[1][1]);
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int nt = 0; nt < D / 8; ++nt) {
            o[nt][0] *= alpha[0];
            o[nt][1] *= alpha[0];
            o[nt][2] *= alpha[1];
            o[nt][3] *= alpha[1];
          }
        }
        // What lies behind the last key is not a number that a zero probability could be trusted with: keys 2t, 2t + 1 and 8 + 2t, 9 + 2t
        auto keep = [&](int nt) {
          const int left = k_limit - key0 - nt * 8 - 2 * t;
          return left >= 2 ? 0xffffffffu : left == 1 ? 0x0000ffffu : 0u;
        };
        if constexpr (FOUR) {
          // Thread (g, t) has the codes of keys 2t, 2t + 1, 8 + 2t, 9 + 2t in word g (D = 128: and g + 8) of their rows.  In a load the threads of odd t
          // (D = 64: of upper t) take the keys of a pair in the other order, which spreads the rows over the banks; `sel` undoes it.
          const uint32_t par = sv + L::kTile + L::kParTile;
          const int odd = D == 128 ? t & 1 : t >> 1;
          const uint32_t sel_lo = odd ? 0x1054u : 0x5410u, sel_hi = odd ? 0x3276u : 0x7632u;
          auto word = [&](int key, int h) {
            const int wd = g + 8 * h;
            return lds32(sv + key * L::kRowBytes + (D == 128 ? (((wd >> 2) ^ ((key >> 1) & 3)) << 4) + (wd & 3) * 4 : wd * 4));
          };
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            uint32_t vb[2][8];   // B fragments: [key pair][value of the word], (key, key + 1)
#pragma unroll
            for (int kp = 0; kp < 2; ++kp) {
              const int key = warp * 16 + kp * 8 + 2 * t;
              const uint32_t x = word(key + odd, h), y = word(key + (odd ^ 1), h);
              const int grp = 2 * h + (g >> 2);   // of dimensions 64 h + 8 g ...
              const uint32_t px = lds32(par + (key + odd) * L::kParBytes + grp * 4), py = lds32(par + (key + (odd ^ 1)) * L::kParBytes + grp * 4);
              uint32_t ss = prmt(px, py, sel_lo), bb = prmt(px, py, sel_hi);
              if (!whole) {
                const uint32_t kpm = keep(kp);
                ss &= kpm;
                bb &= kpm;
              }
              const uint32_t step = hmul2(ss, 0x2C002C00u), first = hadd2(bb, ss);
              const uint32_t lo = prmt(x, y, sel_lo), hi = prmt(x, y, sel_hi);   // codes 0..3 of either key, codes 4..7
              const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
              vb[kp][0] = hfma2(hadd2(mask_or(lo, 0x000F000Fu, 0x64006400u), 0xE400E400u), step, first);
              vb[kp][1] = hfma2(hadd2(mask_or(lo, 0x00F000F0u, 0x54005400u), 0xD400D400u), step, first);
              vb[kp][2] = hfma2(hadd2(mask_or(lo8, 0x000F000Fu, 0x64006400u), 0xE400E400u), step, first);
              vb[kp][3] = hfma2(hadd2(mask_or(lo8, 0x00F000F0u, 0x54005400u), 0xD400D400u), step, first);
              vb[kp][4] = hfma2(hadd2(mask_or(hi, 0x000F000Fu, 0x64006400u), 0xE400E400u), step, first);
              vb[kp][5] = hfma2(hadd2(mask_or(hi, 0x00F000F0u, 0x54005400u), 0xD400D400u), step, first);
              vb[kp][6] = hfma2(hadd2(mask_or(hi8, 0x000F000Fu, 0x64006400u), 0xE400E400u), step, first);
              vb[kp][7] = hfma2(hadd2(mask_or(hi8, 0x00F000F0u, 0x54005400u), 0xD400D400u), step, first);
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) mma_16816<false>(o[8 * h + c], p, vb[0][c], vb[1][c]);
          }
        } else {
#pragma unroll
          for (int np = 0; np < D / 16; ++np) {
            uint32_t vf[4];
            ldmatrix_x4<true>(vf, sv + (np / 4) * L::kSub + sw128_offset(v_row, (np % 4) * 2 + v_ch));
            if (!whole) {
              const uint32_t m0 = keep(0), m1 = keep(1);
              vf[0] &= m0;
              vf[1] &= m1;
              vf[2] &= m0;
              vf[3] &= m1;
            }
            mma_16816<MMA_BF16>(o[2 * np], p, vf[0], vf[1]);
            mma_16816<MMA_BF16>(o[2 * np + 1], p, vf[2], vf[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + s);
    }
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
    }
  }
  __syncthreads();   // every stage has been read: the shares may overwrite them

  // ============================ combine the four warps ================================
  float2* stats = reinterpret_cast<float2*>(smem + L::kOffStats);   // [4][16] (maximum, sum)
  if (warp < kPgWarps) {
    float* share = reinterpret_cast<float*>(smem + warp * L::kShare);
    if constexpr (FOUR) {
      // n-tile 8 h + c: columns 2t, 2t + 1 are dimensions 64 h + 16 t + c and + 8
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int c = 0; c < 8; c += 4) {
            float* dst = share + g * L::kRowFloats + 64 * h + 16 * t + 8 * e + c;
            *reinterpret_cast<float4*>(dst) = make_float4(o[8 * h + c][e], o[8 * h + c + 1][e], o[8 * h + c + 2][e], o[8 * h + c + 3][e]);
            *reinterpret_cast<float4*>(dst + 8 * L::kRowFloats) =
                make_float4(o[8 * h + c][2 + e], o[8 * h + c + 1][2 + e], o[8 * h + c + 2][2 + e], o[8 * h + c + 3][2 + e]);
          }
    } else {
#pragma unroll
      for (int nt = 0; nt < D / 8; ++nt) {
        *reinterpret_cast<float2*>(share + g * L::kRowFloats + nt * 8 + 2 * t) = make_float2(o[nt][0], o[nt][1]);
        *reinterpret_cast<float2*>(share + (g + 8) * L::kRowFloats + nt * 8 + 2 * t) = make_float2(o[nt][2], o[nt][3]);
      }
    }
    if (t == 0) {
      stats[warp * kPagedRows + g] = make_float2(m[0], l[0]);
      stats[warp * kPagedRows + g + 8] = make_float2(m[1], l[1]);
    }
  }
  __syncthreads();
  const int items = *abort_flag ? 0 : n_rows * (D / 8);   // (row, 8 columns)
  for (int i = threadIdx.x; i < items; i += kPgThreads) {
    const int row = i / (D / 8), ch = i % (D / 8);
    float m_all = -INFINITY, l_all = 0.f, acc[8] = {};
#pragma unroll
    for (int k = 0; k < kPgWarps; ++k) m_all = fmaxf(m_all, stats[k * kPagedRows + row].x);
#pragma unroll
    for (int k = 0; k < kPgWarps; ++k) {
      const float2 st = stats[k * kPagedRows + row];
      const float w = st.x == -INFINITY ? 0.f : fast_exp2(st.x - m_all);   // a warp without keys
      l_all = fmaf(w, st.y, l_all);
      const float4* src = reinterpret_cast<const float4*>(smem + k * L::kShare + (row * L::kRowFloats + ch * 8) * 4);
      const float4 x = src[0], y = src[1];
      acc[0] = fmaf(w, x.x, acc[0]); acc[1] = fmaf(w, x.y, acc[1]); acc[2] = fmaf(w, x.z, acc[2]); acc[3] = fmaf(w, x.w, acc[3]);
      acc[4] = fmaf(w, y.x, acc[4]); acc[5] = fmaf(w, y.y, acc[5]); acc[6] = fmaf(w, y.z, acc[6]); acc[7] = fmaf(w, y.w, acc[7]);
    }
    const int64_t at = seq.row0 + (r0 + row) / a.group;
    const int h = hk * a.group + (r0 + row) % a.group;
    if (n_split == 1) {
      const float inv = l_all > 0.f ? 1.0f / l_all : 0.f;   // no key: zeros (a NaN among the scores stays one: its accumulator is)
      *reinterpret_cast<uint4*>(static_cast<unsigned short*>(a.o_ptr) + at * a.o_ss + h * a.o_sh + ch * 8) =
          make_uint4(pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv), pack2<BF16>(acc[4] * inv, acc[5] * inv),
                     pack2<BF16>(acc[6] * inv, acc[7] * inv));
      if (ch == 0 && a.lse != nullptr)
        a.lse[static_cast<int64_t>(h) * a.total_rows + at] = l_all == 0.f ? -INFINITY : (m_all + fast_log2(l_all)) * kPgLn2;
    } else {
      const int64_t share = (at * a.H + h) * a.n_split + split;
      float4* dst = reinterpret_cast<float4*>(a.part_o + share * D + ch * 8);
      dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (ch == 0) a.part_ml[share] = make_float2(m_all, l_all);
    }
  }
  if (*abort_flag) {
    for (int k = 0; k < 20; ++k) __nanosleep(1000000);   // copies in flight end before the CTA does
    __syncthreads();
  }
}

// Joins the shares of rows whose keys were dealt out: a warp per (new row, head).
template <int D, bool BF16>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ PagedArgs a) {
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t rh = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (rh >= static_cast<int64_t>(a.total_rows) * a.H) return;
  const int row = static_cast<int>(rh / a.H), h = static_cast<int>(rh % a.H);
  const int b = a.cu != nullptr ? sequence_of_row(a.cu, a.B, row) : row / a.rows_each;
  if (b < 0 || b >= a.B) return;
  const PgSeq seq = sequence(a, b);
  const int i = row - seq.row0;
  if (i >= seq.n_new) return;
  // the tile of this row, and how many shares it had
  const int r0 = (i * a.group + h % a.group) / kPagedRows * kPagedRows, n_rows = min(kPagedRows, seq.n_new * a.group - r0);
  const int n = splits_of(keys_of(a, seq, (r0 + n_rows - 1) / a.group), a.n_split);
  if (n == 1) return;
  const float2* ml = a.part_ml + rh * a.n_split;
  const float* po = a.part_o + rh * a.n_split * D;
  float m_all = -INFINITY;
  for (int s = lane; s < n; s += 32) m_all = fmaxf(m_all, ml[s].x);
#pragma unroll
  for (int k = 16; k > 0; k /= 2) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, k));
  float l_all = 0.f;
  constexpr int V = D / 32;   // values of a lane
  float acc[V] = {};
  for (int s0 = 0; s0 < n; s0 += 32) {
    float w = 0.f;
    if (s0 + lane < n) {
      const float2 x = ml[s0 + lane];
      w = x.x == -INFINITY ? 0.f : fast_exp2(x.x - m_all);   // a share without keys that this row sees
      l_all = fmaf(w, x.y, l_all);
    }
    const int some = min(32, n - s0);
#pragma unroll 4
    for (int s = 0; s < some; ++s) {
      const float ws = __shfl_sync(0xffffffffu, w, s);
      const float* src = po + static_cast<int64_t>(s0 + s) * D + lane * V;
      if constexpr (V == 4) {
        const float4 x = *reinterpret_cast<const float4*>(src);
        acc[0] = fmaf(ws, x.x, acc[0]); acc[1] = fmaf(ws, x.y, acc[1]); acc[2] = fmaf(ws, x.z, acc[2]); acc[3] = fmaf(ws, x.w, acc[3]);
      } else {
        const float2 x = *reinterpret_cast<const float2*>(src);
        acc[0] = fmaf(ws, x.x, acc[0]); acc[1] = fmaf(ws, x.y, acc[1]);
      }
    }
  }
#pragma unroll
  for (int k = 16; k > 0; k /= 2) l_all += __shfl_xor_sync(0xffffffffu, l_all, k);
  const float inv = l_all > 0.f ? 1.0f / l_all : 0.f;
  unsigned short* dst = static_cast<unsigned short*>(a.o_ptr) + static_cast<int64_t>(row) * a.o_ss + h * a.o_sh + lane * V;
  if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv));
  else *reinterpret_cast<uint32_t*>(dst) = pack2<BF16>(acc[0] * inv, acc[1] * inv);
  if (lane == 0 && a.lse != nullptr)
    a.lse[static_cast<int64_t>(h) * a.total_rows + row] = l_all == 0.f ? -INFINITY : (m_all + fast_log2(l_all)) * kPgLn2;
}

// CTAs that may share a tile's keys: enough of them for two on every SM and a few to spare, since sequences differ in length.
int paged_splits(int64_t sms, int64_t tiles, int64_t max_keys, int D, int bits) {
  (void)D;
  (void)bits;
  if (sms <= 0 || tiles <= 0) return 1;
  const int64_t most = std::max<int64_t>(1, (max_keys + kPagedKeyStep - 1) / kPagedKeyStep / kPgMinSteps);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({most, 4 * sms / tiles, 128})));
}

template <int D, bool BF16, bool FOUR>
static int launch_paged_impl(const PagedArgs& a, cudaStream_t stream) {
  using L = PgSmem<D, FOUR>;
  auto kfn = fmha_paged_kernel<D, BF16, FOUR>;
  static std::atomic<bool> configured[64] = {};   // per device; set after the attribute call succeeded
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int64_t row_tiles = (static_cast<int64_t>(a.max_rows) * a.group + kPagedRows - 1) / kPagedRows;
  cudaError_t e = launch_overlapped(kfn, dim3(a.n_split, static_cast<unsigned>(a.H_kv * row_tiles), a.B), dim3(kPgThreads), L::kDynBytes, stream, a);
  if (e == cudaSuccess && a.n_split > 1) {
    const int64_t rows = static_cast<int64_t>(a.total_rows) * a.H;
    e = launch_overlapped(paged_join_kernel<D, BF16>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, stream, a);
  }
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

int launch_paged(const PagedArgs& a, int dtype, int D, int bits, cudaStream_t stream) {
  const bool bf = dtype == FMHA_DTYPE_BF16, four = bits == 4;
#define FMHA_PAGED_CASE(DD, BF, F4) \
  if (D == DD && bf == BF && four == F4) return launch_paged_impl<DD, BF, F4>(a, stream);
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
