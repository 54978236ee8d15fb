// fmha_kv_cache_sm100.cu — rows into a paged cache (rotated by their positions, in 16 or 4 bits) and out of it.
//
// Bound by memory: a row's heads are read once and written once.  A warp takes a row, or a part of its heads where there are too few rows to
// fill the chip; a lane takes the same 16 values of every head (8 of a rotated pair's first and 8 of its second halves), so the sixteen angles' cosines and
// sines it needs stay in registers over all heads: each lane computes one or two of the row's angles and gets the others by shuffles.  The angle is
// position * inv_freq in 64 bits, where the product is
// exact for positions below 2^29; in 32 bits an angle of 2^20 would be off by up to 0.03.  Rotated values are formed in 32 bits and rounded once, to the
// type of k; a 4-bit cache codes those.
//
// Measured (device time): appending 9 389 rows of 32/8 heads of 128, 16 bits, 42 us, 5.5 TB/s of what is read and written; one row of 64 sequences 3.0 us, little
// more than an empty launch, 3.4 in 4 bits; 5 321 rows of 16/4 heads of 64 in 4 bits 9.8 us, 2.9 TB/s: 7.05 million warp instructions, which take 6.2 us at one a
// cycle of each scheduler (4.4 by bytes), the rest latency: 1.4 of 4.8 warps of a scheduler can issue, 59 % of the cycles do (24 warps an SM at 80 registers); reading back 9 600 rows of 8 heads of
// 128 14.2 us, 5.6 TB/s, and 8 100 of 4 heads of 64 from 4 bits 5.0 us, 2.2 TB/s (few loads a warp: its row's place, then its heads).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../../include/fmha_sm100.h"
#include "fmha_cache_args.h"
#include "fmha_device_utils.cuh"
#include "fmha_kernel_args.h"
#include "sm100_ptx.cuh"

namespace fmha {

namespace {
constexpr int kKvWarps = 8;   // warps of a block

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = unpack_lo<BF16>(ws[i]);
    x[2 * i + 1] = unpack_hi<BF16>(ws[i]);
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]), pack2<BF16>(x[6], x[7]));
}

// Eight values of a row, of whose 32 the lanes lane ^ 1, ^ 2 and ^ 3 have the others: their codes, and scale and base of the 32.  All products,
// differences and quotients are rounded one by one, so that the codes are the definition's and not the compiler's.  The eight quotients by one scale
// take its rounded reciprocal once: a quotient within one unit, its exact remainder, and the correction are correctly rounded then (Markstein's theorem; the
// scale has 11 bits, so its last bits are not all ones).  A number in [0, 15] is rounded by adding 1.5 * 2^23, whose last bits then hold it.
// (With a division and two conversions a value, append and read together took 17.3 us instead of 14.3 at 5 321 rows, 16/4 heads of 64.)
__device__ __forceinline__ uint32_t code8(const float (&x)[8], __half2& scale_base) {
  float lo = INFINITY, hi = -INFINITY, bad = 0.f, f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bad = fmaf(x[i], 0.f, bad);   // NaN where an infinity or NaN was among them
    f[i] = fminf(fmaxf(x[i], -kCacheLimit), kCacheLimit);
    lo = fminf(lo, f[i]);
    hi = fmaxf(hi, f[i]);
  }
#pragma unroll
  for (int m = 1; m <= 2; m *= 2) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    bad += __shfl_xor_sync(0xffffffffu, bad, m);
  }
  const __half s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 16.0f / 15.0f));
  const float sf = __half2float(s);
  const __half b = __float2half_rn(__fsub_rn(lo, sf));
  const float bf = __half2float(b);
  scale_base = bad == 0.f ? __halves2half2(s, b) : __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff));
  uint32_t codes = 0u;
  if (sf > 0.f && bad == 0.f) {
    const float r = __frcp_rn(sf);
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      const float x0 = __fsub_rn(f[i], bf), q = __fmul_rn(x0, r), quotient = __fmaf_rn(__fmaf_rn(-q, sf, x0), r, q);
      const float c = __fmaf_rn(quotient, 16.0f, -16.0f);   // 16 (quotient - 1): 16 is a power of two
      codes = codes << 4 | (__float_as_uint(__fadd_rn(fminf(fmaxf(c, 0.f), 15.f), 12582912.0f)) & 15u);
    }
  }
  return codes;
}
}  // namespace

// Units of 16 values: unit u < n_freq / 8 of a head holds the values [8u, +8) and [n_freq + 8u, +8), the others likewise the two halves of what
// is not rotated.  A warp's step covers 32 units: four heads of 128 values or eight of 64, each lane always the same unit.
template <int D, bool BF16, bool FOUR, bool INTER>
__global__ void __launch_bounds__(32 * kKvWarps, FOUR ? 3 : 4) kv_append_kernel(const __grid_constant__ KvAppendArgs a) {
  griddep_wait();
  constexpr int kUnits = D / 16, kHeads = 32 / kUnits;
  const int lane = threadIdx.x & 31;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * kKvWarps + (threadIdx.x >> 5);
  const int row = static_cast<int>(task / a.parts), part = static_cast<int>(task % a.parts);
  if (row >= a.total_rows) return;
  const int Hk = a.cache.H_kv, heads = a.H + 2 * Hk;   // of q, then k, then v
  const int steps = (heads + kHeads - 1) / kHeads;
  const int s0 = steps * part / a.parts, s1 = steps * (part + 1) / a.parts;
  const int unit = lane % kUnits, sub = lane / kUnits;
  const int n_freq = a.n_freq;
  const bool turned = unit < n_freq / 8;
  const int half = turned ? n_freq : (D - 2 * n_freq) / 2;                       // distance of the unit's two pieces
  const int at = turned ? 8 * unit : 2 * n_freq + 8 * (unit - n_freq / 8);

  auto source = [&](int step) -> const uint4* {   // null: no such head
    const int h = step * kHeads + sub;
    if (step >= s1 || h >= heads) return nullptr;
    const fmha_tensor4& t = h < a.H ? a.q : h < a.H + Hk ? a.k : a.v;
    const int hh = h < a.H ? h : h < a.H + Hk ? h - a.H : h - a.H - Hk;
    return reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(t.ptr) + static_cast<int64_t>(row) * t.stride_s + hh * t.stride_h + at);
  };
  uint4 xa = {}, xb = {};   // the next step's values: the first are on their way while the row's place is looked up
  auto load = [&](int step) {
    const uint4* p = source(step);
    if (p != nullptr) {
      xa = __ldg(p);
      xb = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned short*>(p) + half));
    }
  };
  load(s0);

  // ---- the row's sequence, position and place -----------------------------------------
  RowSequence seq;
  if (a.cu != nullptr) {
    seq = sequence_of_row(a.cu, a.seqlens, a.B, row);
  } else {
    const int b = row / a.rows_each;
    seq = {b, b * a.rows_each, a.rows_each, a.seqlens[b]};
  }
  const int pos = seq.b >= 0 ? seq.len - seq.n + (row - seq.first) : -1;
  const int slot = pos >= 0 ? pos / a.cache.page_rows : 0;
  int page = -1;
  if (pos >= 0 && slot < a.cache.table_width) page = a.cache.table[seq.b * a.cache.table_stride + slot];
  const int in_page = pos - slot * a.cache.page_rows;

  // ---- cosine and sine of the lane's eight angles ---------------------------------------
  float cs[8], sn[8];
  if (n_freq > 0) {
    float c0[2] = {1.f, 1.f}, s0a[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int j = i * 32 + lane;
      if (j < n_freq) {
        double s, c;
        sincospi(static_cast<double>(pos) * static_cast<double>(a.inv_freq[j]) * 0.31830988618379067154, &s, &c);   // the angle over pi
        c0[i] = static_cast<float>(c);
        s0a[i] = static_cast<float>(s);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // pairs of a unit: (8u + i, n_freq + 8u + i); interleaved, (8u + 2i, 8u + 2i + 1) of either piece
      const int j = INTER ? (i < 4 ? 4 * unit + i : n_freq / 2 + 4 * unit + i - 4) : 8 * unit + i;
      cs[i] = __shfl_sync(0xffffffffu, c0[0], j & 31);
      sn[i] = __shfl_sync(0xffffffffu, s0a[0], j & 31);
      if (D == 128) {
        const float c1 = __shfl_sync(0xffffffffu, c0[1], j & 31), s1v = __shfl_sync(0xffffffffu, s0a[1], j & 31);
        if (j >= 32) {
          cs[i] = c1;
          sn[i] = s1v;
        }
      }
    }
  }

  for (int step = s0; step < s1; ++step) {
    const uint4 wa = xa, wb = xb;
    load(step + 1);
    const int h = step * kHeads + sub;
    const bool is_q = h < a.H, is_v = h >= a.H + Hk, exists = h < heads;
    uint4 ya = wa, yb = wb;
    float va[8], vb[8];
    if (FOUR || (turned && !is_v)) {
      unpack8<BF16>(wa, va);
      unpack8<BF16>(wb, vb);
    }
    if (turned && !is_v) {
      float ra[8], rb[8];
      auto turn = [](float x, float y, float c, float s, float& u, float& v) {
        u = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
        v = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
      };
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (INTER) {
          if (i < 4) turn(va[2 * i], va[2 * i + 1], cs[i], sn[i], ra[2 * i], ra[2 * i + 1]);
          else turn(vb[2 * i - 8], vb[2 * i - 7], cs[i], sn[i], rb[2 * i - 8], rb[2 * i - 7]);
        } else {
          turn(va[i], vb[i], cs[i], sn[i], ra[i], rb[i]);
        }
      }
      ya = pack8<BF16>(ra);
      yb = pack8<BF16>(rb);
      if constexpr (FOUR) {   // the cache codes what a 16-bit cache would hold
        unpack8<BF16>(ya, va);
        unpack8<BF16>(yb, vb);
      }
    }
    if (FOUR && (step + 1) * kHeads > a.H) {   // not where all heads are of q
      __half2 pa, pb;
      const uint32_t ca = code8(va, pa), cb = code8(vb, pb);   // whole warp: the lanes of 32 values are in it together
      if (exists && !is_q && page >= 0 && page < a.cache.pages) {
        const fmha_tensor4& t = is_v ? a.cache.v : a.cache.k;
        const fmha_tensor4& tp = is_v ? a.cache.v_params : a.cache.k_params;
        const int hh = h - a.H - (is_v ? Hk : 0);
        uint8_t* dst = static_cast<uint8_t*>(t.ptr) + page * t.stride_b + hh * t.stride_h + in_page * t.stride_s;
        *reinterpret_cast<uint32_t*>(dst + at / 2) = ca;
        *reinterpret_cast<uint32_t*>(dst + (at + half) / 2) = cb;
        if (unit % 4 == 0) {
          __half2* par = reinterpret_cast<__half2*>(static_cast<__half*>(tp.ptr) + page * tp.stride_b + hh * tp.stride_h) + in_page * (D / kCacheGroup);
          par[at / kCacheGroup] = pa;
          par[(at + half) / kCacheGroup] = pb;
        }
      }
    }
    if constexpr (!FOUR) {
      if (exists && !is_q && page >= 0 && page < a.cache.pages) {
        const fmha_tensor4& t = is_v ? a.cache.v : a.cache.k;
        const int hh = h - a.H - (is_v ? Hk : 0);
        unsigned short* dst = static_cast<unsigned short*>(t.ptr) + page * t.stride_b + hh * t.stride_h + in_page * t.stride_s + at;
        *reinterpret_cast<uint4*>(dst) = ya;
        *reinterpret_cast<uint4*>(dst + half) = yb;
      }
    }
    if (exists && is_q) {
      unsigned short* dst = static_cast<unsigned short*>(a.q_out.ptr) + static_cast<int64_t>(row) * a.q_out.stride_s + h * a.q_out.stride_h + at;
      if (pos < 0) ya = yb = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(dst) = ya;
      *reinterpret_cast<uint4*>(dst + half) = yb;
    }
  }
}

// A warp per row of the result; a lane takes 16 values of a head at a time.
template <int D, bool BF16, bool FOUR>
__global__ void __launch_bounds__(32 * kKvWarps) kv_read_kernel(const __grid_constant__ KvReadArgs a) {
  griddep_wait();
  constexpr int kUnits = D / 16, kHeads = 32 / kUnits;
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kKvWarps + (threadIdx.x >> 5);
  if (row >= a.total_rows) return;
  const int unit = lane % kUnits, sub = lane / kUnits, Hk = a.cache.H_kv;
  const RowSequence seq = sequence_of_row(a.cu, nullptr, a.B, static_cast<int>(row));
  int page = -1, in_page = 0;
  if (seq.b >= 0) {
    const int pos = static_cast<int>(row) - seq.first, slot = pos / a.cache.page_rows;
    in_page = pos - slot * a.cache.page_rows;
    if (slot < a.cache.table_width) page = a.cache.table[seq.b * a.cache.table_stride + slot];
    if (page >= a.cache.pages) page = -1;
  }
  constexpr int kAhead = 4;
  for (int h0 = 0; h0 < 2 * Hk; h0 += kAhead * kHeads) {
    uint4 x[kAhead][2];
    uint2 codes[kAhead];
    __half2 par[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + i * kHeads + sub, hh = h < Hk ? h : h - Hk;
      x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
      codes[i] = make_uint2(0u, 0u);
      par[i] = __half2half2(__ushort_as_half(0));
      if (h < 2 * Hk && page >= 0) {
        const fmha_tensor4& t = h < Hk ? a.cache.k : a.cache.v;
        if constexpr (FOUR) {
          const fmha_tensor4& tp = h < Hk ? a.cache.k_params : a.cache.v_params;
          codes[i] = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(t.ptr) + page * t.stride_b + hh * t.stride_h + in_page * t.stride_s) + unit);
          par[i] = __ldg(reinterpret_cast<const __half2*>(static_cast<const __half*>(tp.ptr) + page * tp.stride_b + hh * tp.stride_h) +
                         in_page * (D / kCacheGroup) + unit / 2);
        } else {
          const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(t.ptr) + page * t.stride_b + hh * t.stride_h + in_page * t.stride_s);
          x[i][0] = __ldg(p + unit);   // the two halves of a head: whole sectors an instruction
          x[i][1] = __ldg(p + kUnits + unit);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + i * kHeads + sub, hh = h < Hk ? h : h - Hk;
      if (h >= 2 * Hk) continue;
      const fmha_tensor4& t = h < Hk ? a.k : a.v;
      uint4* dst = reinterpret_cast<uint4*>(static_cast<unsigned short*>(t.ptr) + row * t.stride_s + hh * t.stride_h);
      if constexpr (FOUR) {
        const float s = __low2float(par[i]), base = __high2float(par[i]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t c = k == 0 ? codes[i].x : codes[i].y;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = fmaf(s, 1.0f + static_cast<float>((c >> (4 * e)) & 15u) * 0.0625f, base);
          dst[2 * unit + k] = pack8<BF16>(v);
        }
      } else {
        dst[unit] = x[i][0];
        dst[kUnits + unit] = x[i][1];
      }
    }
  }
}

template <int D, bool BF16, bool FOUR, bool INTER>
static int append_impl(const KvAppendArgs& a, cudaStream_t stream) {
  KvAppendArgs args = a;
  const int steps = (a.H + 2 * a.cache.H_kv + 512 / D - 1) / (512 / D);
  const int64_t fill = static_cast<int64_t>(sm_count()) * 16;   // warps that keep the memory busy (rows of 32/8 heads, 4 / 8 / 16 / 32 per SM: 64 rows 3.2 3.0 3.0 3.0 us, 512 rows 8.2 5.7 4.8 5.3)
  args.parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(steps, fill / std::max(a.total_rows, 1))));
  const int64_t warps = static_cast<int64_t>(a.total_rows) * args.parts;
  const cudaError_t e = launch_overlapped(kv_append_kernel<D, BF16, FOUR, INTER>, dim3(static_cast<unsigned>((warps + kKvWarps - 1) / kKvWarps)),
                                          dim3(32 * kKvWarps), 0, stream, args);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

int launch_kv_append(const KvAppendArgs& a, int dtype, bool interleaved, cudaStream_t stream) {
  const bool bf = dtype == FMHA_DTYPE_BF16, four = a.cache.bits == 4;
#define FMHA_APPEND_CASE(DD, BF, F4, IN) \
  if (a.cache.D == DD && bf == BF && four == F4 && interleaved == IN) return append_impl<DD, BF, F4, IN>(a, stream);
#define FMHA_APPEND_CASES(DD, BF) \
  FMHA_APPEND_CASE(DD, BF, false, false) FMHA_APPEND_CASE(DD, BF, false, true) FMHA_APPEND_CASE(DD, BF, true, false) FMHA_APPEND_CASE(DD, BF, true, true)
  FMHA_APPEND_CASES(64, false)
  FMHA_APPEND_CASES(64, true)
  FMHA_APPEND_CASES(128, false)
  FMHA_APPEND_CASES(128, true)
#undef FMHA_APPEND_CASES
#undef FMHA_APPEND_CASE
  return static_cast<int>(cudaErrorInvalidValue);
}

template <int D, bool BF16, bool FOUR>
static int read_impl(const KvReadArgs& a, cudaStream_t stream) {
  const cudaError_t e = launch_overlapped(kv_read_kernel<D, BF16, FOUR>, dim3((a.total_rows + kKvWarps - 1) / kKvWarps), dim3(32 * kKvWarps), 0, stream, a);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

int launch_kv_read(const KvReadArgs& a, int dtype, cudaStream_t stream) {
  const bool bf = dtype == FMHA_DTYPE_BF16;
  if (a.cache.bits == 16) return a.cache.D == 64 ? read_impl<64, false, false>(a, stream) : read_impl<128, false, false>(a, stream);   // moved as they are
  if (a.cache.D == 64) return bf ? read_impl<64, true, true>(a, stream) : read_impl<64, false, true>(a, stream);
  return bf ? read_impl<128, true, true>(a, stream) : read_impl<128, false, true>(a, stream);
}

}  // namespace fmha
