// Device parts shared by the product kernels: how a block finds its tile, the matrix steps, the epilogue.
//
// All products run with the weights as the matrix unit's first operand, so an accumulator lane holds one row of x and
// four consecutive columns of the result: its scale is one number and its four results leave in one store.
#pragma once
#include "blocks.hpp"
#include "common.hpp"

namespace aeisu {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// An operand step is 128 bytes of a row: 128 E4M3 codes or 64 sixteen-bit values.  A fragment is what one lane holds of
// it, two pieces of 16 bytes: lane l has row l & 15 and the pieces l >> 4 and 4 + (l >> 4).  Which columns of the step
// these are does not matter as long as both operands agree.
struct Frag {
  i4 lo, hi;
};
constexpr int kStepBytes = 128;

// Steps of E4M3 codes as exact products: codes widen to FP16 without loss, and the FP16 unit keeps FP32 sums.
__device__ __forceinline__ f4 step_e4m3_exact(const Frag& w, const Frag& x) {
  f4 r = {0.f, 0.f, 0.f, 0.f};
  r = mfma_f16(e4m3x8_to_h8(w.lo[0], w.lo[1]), e4m3x8_to_h8(x.lo[0], x.lo[1]), r);
  r = mfma_f16(e4m3x8_to_h8(w.lo[2], w.lo[3]), e4m3x8_to_h8(x.lo[2], x.lo[3]), r);
  r = mfma_f16(e4m3x8_to_h8(w.hi[0], w.hi[1]), e4m3x8_to_h8(x.hi[0], x.hi[1]), r);
  return mfma_f16(e4m3x8_to_h8(w.hi[2], w.hi[3]), e4m3x8_to_h8(x.hi[2], x.hi[3]), r);
}
template <int TYPE>
__device__ __forceinline__ f4 step_16bit(const Frag& w, const Frag& x, f4 acc) {
  if constexpr (TYPE == AEISU_TYPE_F16) {
    acc = mfma_f16(__builtin_bit_cast(h8, w.lo), __builtin_bit_cast(h8, x.lo), acc);
    return mfma_f16(__builtin_bit_cast(h8, w.hi), __builtin_bit_cast(h8, x.hi), acc);
  } else {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, w.lo), __builtin_bit_cast(b8, x.lo), acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, w.hi), __builtin_bit_cast(b8, x.hi), acc, 0, 0, 0);
  }
}

// Rows [lo, hi) of x that one block works on, all of expert `expert` (-1: rows of no expert, whose results are 0).
struct RowTile {
  int64_t lo, hi;
  int expert;
};

// The t-th tile of at most BM rows.  Every wave finds it by itself: 64 segments at a time, one a lane.  The segments
// are the rows before the first offset, each expert's and those after the last offset; a running maximum of the
// offsets, kept within the rows, bounds them, so they cover every row once whatever the offsets hold.
template <int BM>
__device__ __forceinline__ bool find_tile(const int32_t* offsets, int experts, int64_t rows, int64_t t, RowTile& out) {
  if (!offsets) {
    out.lo = t * BM;
    out.hi = out.lo + BM < rows ? out.lo + BM : rows;
    out.expert = 0;
    return out.lo < rows;
  }
  const int lane = lane_id(), m = (int)rows;
  int before = 0;                                    // the previous segments' end
  int64_t first = 0;                                 // and their tiles
  for (int s0 = 0; s0 < experts + 2; s0 += 64) {
    const int s = s0 + lane;                         // segment s ends at offsets[s]; the last one at `rows`
    int end = s <= experts ? offsets[s] : m;
    end = end < 0 ? 0 : end > m ? m : end;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(end, d);
      if (lane >= d) end = end > o ? end : o;
    }
    end = end > before ? end : before;
    int begin = __shfl_up(end, 1);
    if (lane == 0) begin = before;
    const int tiles = (end - begin + BM - 1) / BM;
    int sum = tiles;                                 // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    const uint64_t past = __ballot(first + sum > t);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int64_t at = __shfl(begin, l) + (t - first - (__shfl(sum, l) - __shfl(tiles, l))) * BM;
      const int64_t e = __shfl(end, l);
      const int seg = s0 + l;
      out.lo = at;
      out.hi = at + BM < e ? at + BM : e;
      out.expert = seg >= 1 && seg <= experts ? seg - 1 : -1;
      return true;
    }
    first += __shfl(sum, 63);
    before = __shfl(end, 63);
  }
  return false;
}

// Most tiles of BM rows that the segments can make: each full tile has BM rows and each segment at most one other.
inline int64_t most_tiles(int64_t rows, int experts, bool grouped, int bm) {
  if (!grouped) return (rows + bm - 1) / bm;
  const int64_t t = rows / bm + experts + 2;
  return t < rows ? t : rows;
}

// Four results of row m from column n on: bias, activation, one rounding to the result's type.
__device__ __forceinline__ void finish4(const aeisu_product& p, int64_t m, int64_t n, f4 v, const float* bias, bool wide) {
  const int64_t left = p.n - n;
  if (left <= 0) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bias) v[i] += bias[n + (i < left ? i : 0)];
    const float neg = p.slope > 0.f ? v[i] * p.slope : 0.f;
    v[i] = v[i] < 0.f ? neg : v[i];
  }
  const int64_t at = m * p.out_stride + n;
  if (p.out_type == AEISU_TYPE_F32) {
    float* o = static_cast<float*>(p.out) + at;
    if (wide && left >= 4) *reinterpret_cast<f4*>(o) = v;
    else
      for (int i = 0; i < 4 && i < left; ++i) o[i] = v[i];
    return;
  }
  unsigned short b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    b[i] = p.out_type == AEISU_TYPE_F16 ? __builtin_bit_cast(unsigned short, (_Float16)v[i])
                                        : __builtin_bit_cast(unsigned short, (__bf16)v[i]);
  unsigned short* o = static_cast<unsigned short*>(p.out) + at;
  if (wide && left >= 4) *reinterpret_cast<uint2*>(o) = uint2{b[0] | (unsigned)b[1] << 16, b[2] | (unsigned)b[3] << 16};
  else
    for (int i = 0; i < 4 && i < left; ++i) o[i] = b[i];
}

}  // namespace aeisu
