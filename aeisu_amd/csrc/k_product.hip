// Matrix products of block-scaled E4M3, FP16 or BF16 operands, for one weight or for weights grouped by expert:
//
//   out[m][n] = act( sum_j sx[j][m] sw[n / 128][j] sum_{k in block j} x[m][k] w[n][k]  + bias[n] )
//
// (16-bit operands: one sum, no scales).  The sum over a block's 128 codes is made by the matrix unit from zero, and one
// FMA per result adds it, scaled, to the FP32 sum.
#include "product.hpp"

namespace aeisu {
namespace {

// 64 x 64 tiles of the result, one for each block of four waves (2 x 2, each 32 x 32); operands staged through registers,
// so rows may start at any address and end anywhere.
template <int TYPE>
__global__ __launch_bounds__(256) void product_kernel(aeisu_product p, const int32_t* offsets, int experts, int64_t ntiles) {
  constexpr int BM = 64, BN = 64;
  constexpr bool kE4M3 = TYPE == AEISU_TYPE_E4M3;
  constexpr int ES = kE4M3 ? 1 : 2, PER = 16 / ES, STEP = kStepBytes / ES;
  __shared__ i4 lds[2][BM * 8];                      // x, w: 16-row pieces of 128 fragments' halves, in lane order
  RowTile tile;
  if (!find_tile<BM>(offsets, experts, p.rows, blockIdx.x / ntiles, tile)) return;
  const int64_t n0 = (int64_t)(blockIdx.x % ntiles) * BN;
  const int lane = lane_id(), wave = threadIdx.x >> 6, wm = (wave & 1) * 2, wn = (wave >> 1) * 2;
  const int e = tile.expert < 0 ? 0 : tile.expert;
  const char* xb = static_cast<const char*>(p.x);
  const char* wb = static_cast<const char*>(p.w) + e * p.w_expert_stride * ES;
  const int64_t kb = (p.k + kBlock - 1) / kBlock;
  const float* sw = kE4M3 ? p.w_scales + (e * ((p.n + kBlock - 1) / kBlock) + n0 / kBlock) * kb : nullptr;
  f4 acc[2][2] = {};
  const int64_t steps = tile.expert < 0 ? 0 : (p.k + STEP - 1) / STEP;
  int64_t xm[2];                                     // rows whose scales this lane applies
  for (int i = 0; i < 2; ++i) {
    const int64_t m = tile.lo + (wm + i) * 16 + (lane & 15);
    xm[i] = m < tile.hi ? m : tile.hi - 1;
  }
  for (int64_t s = 0; s < steps; ++s) {
    i4 st[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = threadIdx.x + 256 * (i & 1);     // 512 pieces of 16 bytes an operand
      const int row = (c >> 7) * 16 + (c & 15), piece = ((c >> 6) & 1) * 4 + ((c & 63) >> 4);
      const int64_t left = kE4M3 ? PER : p.k - (s * STEP + piece * PER);
      int64_t r;
      const char* src;
      if (i < 2) {
        r = tile.lo + row < tile.hi ? tile.lo + row : tile.hi - 1;
        src = xb + r * p.x_stride * ES;
      } else {
        r = n0 + row < p.n ? n0 + row : p.n - 1;
        src = wb + r * p.w_stride * ES;
      }
      src += s * kStepBytes + piece * 16;
      st[i] = i4{0, 0, 0, 0};
      if (left >= PER) __builtin_memcpy(&st[i], src, 16);
      else if (left > 0) {
        unsigned short h[8] = {};
        for (int j = 0; j < 8; ++j)
          if (j < left) h[j] = reinterpret_cast<const unsigned short*>(src)[j];
        __builtin_memcpy(&st[i], h, 16);
      }
    }
    __syncthreads();                                 // the previous step's fragments have been read
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[i >> 1][threadIdx.x + 256 * (i & 1)] = st[i];
    __syncthreads();
    Frag x[2], w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[i] = Frag{lds[0][(wm + i) * 128 + lane], lds[0][(wm + i) * 128 + 64 + lane]};
      w[i] = Frag{lds[1][(wn + i) * 128 + lane], lds[1][(wn + i) * 128 + 64 + lane]};
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float sc = 0.f;
      if constexpr (kE4M3) sc = p.x_scales[s * p.x_scales_stride + xm[i]] * sw[s];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (kE4M3) {
          const f4 part = step_e4m3_exact(w[j], x[i]);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(part[r], sc, acc[i][j][r]);
        } else {
          acc[i][j] = step_16bit<TYPE>(w[j], x[i], acc[i][j]);
        }
      }
    }
  }
  const size_t vec = p.out_type == AEISU_TYPE_F32 ? 16 : 8;
  const bool wide = (reinterpret_cast<uintptr_t>(p.out) % vec) == 0 && p.out_stride % 4 == 0;
  const float* bias = p.bias && tile.expert >= 0 ? p.bias + (int64_t)e * p.n : nullptr;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = tile.lo + (wm + i) * 16 + (lane & 15);
    if (m >= tile.hi) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j) finish4(p, m, n0 + (wn + j) * 16 + 4 * (lane >> 4), acc[i][j], bias, wide);
  }
}

}  // namespace

hipError_t launch_product(const aeisu_product& p, const int32_t* offsets, int experts, hipStream_t stream) {
  const int64_t ntiles = (p.n + 63) / 64;
  const int64_t blocks = most_tiles(p.rows, experts, offsets != nullptr, 64) * ntiles;
  if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
  auto go = [&](auto kernel) { kernel<<<(unsigned)blocks, 256, 0, stream>>>(p, offsets, experts, ntiles); };
  if (p.type == AEISU_TYPE_E4M3) go(product_kernel<AEISU_TYPE_E4M3>);
  else if (p.type == AEISU_TYPE_F16) go(product_kernel<AEISU_TYPE_F16>);
  else go(product_kernel<AEISU_TYPE_BF16>);
  return hipGetLastError();
}

}  // namespace aeisu
