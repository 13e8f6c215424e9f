// Matrix products of block-scaled E4M3, FP16 or BF16 operands, for one weight or for weights grouped by expert:
//
//   out[m][n] = act( sum_j sx[j][m] sw[n / 128][j] sum_{k in block j} x[m][k] w[n][k]  + bias[n] )
//
// (16-bit operands: one sum, no scales).  The sum over a block's 128 codes is made by the matrix unit from zero, and one
// FMA per result adds it, scaled, to the FP32 sum.
#include <algorithm>
#include <atomic>
#include <cmath>

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
  if (!find_tile<BM>(offsets, experts, p.rows, (int)(blockIdx.x / ntiles), tile)) return;
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

hipError_t launch_product_any(const aeisu_product& p, const int32_t* offsets, int experts, hipStream_t stream) {
  const int64_t ntiles = (p.n + 63) / 64;
  const int64_t blocks = most_tiles(p.rows, experts, offsets != nullptr, 64) * ntiles;
  if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
  auto go = [&](auto kernel) { kernel<<<(unsigned)blocks, 256, 0, stream>>>(p, offsets, experts, ntiles); };
  if (p.type == AEISU_TYPE_E4M3) go(product_kernel<AEISU_TYPE_E4M3>);
  else if (p.type == AEISU_TYPE_F16) go(product_kernel<AEISU_TYPE_F16>);
  else go(product_kernel<AEISU_TYPE_BF16>);
  return hipGetLastError();
}

namespace {

// CUs of the current device
int compute_units() {
  static std::atomic<int> known[64];
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64) return 256;
  int n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n < 8) n = 256;
    known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Which kernel: the one with the least expected time, in microseconds from what each measured (E4M3 to BF16, a step is
// 128 bytes of k):
//   * 256 x 256: 1.55 a step and 6 for the stores of each round of a tile on every CU (8192 x 10240 x 5120: 346);
//   * 128 x 128: 0.62 a step for a tile on every CU, two of which fit (485 there; 512 x 4096 x 4096: 27, where
//     256 x 256 leaves 7/8 of the CUs idle and takes 42);
//   * 16 a x 16 b with k split over a block's waves: (1 + 1.1 a + 0.75 b + 0.45 a b) / 32 a step (a 4, b 4, 256 x 4096 x 4096:
//     19 against 27 for 128 x 128; a 1, b 1, 1 x 4096 x 4096: 6.6 against 26);
//   * 64 x 64 through registers for rows that do not allow the first two: 1.1 a step, four blocks on a CU
//     (777 x 515 x 1003 over seven experts, FP16: 29 against 21 for a 2, b 2).
// FP32 results of E4M3 operands are exact products at half the rate, and 256 x 256 does not have the registers for them.
// Tiles of grouped rows are estimated: where every expert's last tile is half full.
struct Choice {
  enum { kAny, k128, k256, kRows } kernel;
  int mt, nt;
};
Choice choose(const aeisu_product& p, bool grouped, int experts, int cus) {
  const bool e4m3 = p.type == AEISU_TYPE_E4M3, exact = e4m3 && p.out_type == AEISU_TYPE_F32;
  const int64_t es = e4m3 ? 1 : 2;
  const double steps = double((p.k * es + kStepBytes - 1) / kStepBytes);
  const double groups = grouped ? double(p.rows < experts ? p.rows : experts) : 0;
  auto share = [&](int bm, int bn) {                 // blocks for each CU
    const double m = grouped ? std::max(double(p.rows) / bm + 0.5 * groups, 0.9 * groups) : double((p.rows + bm - 1) / bm);
    return std::max(m, 1.0) * double((p.n + bn - 1) / bn) / cus;
  };
  Choice best{Choice::kAny, 0, 0};
  double least = 5 + steps * 1.1 * std::ceil(share(64, 64)) / (share(64, 64) > 1 ? 2 : 1);
  auto offer = [&](double t, Choice c) {
    if (t < least) least = t, best = c;
  };
  for (int mt = 1; mt <= 4; mt *= 2)
    for (int nt = 1; nt <= mt + 1 && nt <= 4; nt *= 2)
      offer(3 + steps / 32 * (1 + 1.1 * mt + 0.75 * nt + 0.45 * mt * nt) * std::max(1.0, share(16 * mt, 16 * nt)),
            Choice{Choice::kRows, mt, nt});
  // 16-byte pieces of rows, and 32-bit offsets within a tile
  const bool pieces = e4m3 || (p.k % 8 == 0 && p.x_stride % 8 == 0 && p.w_stride % 8 == 0 && p.w_expert_stride % 8 == 0 &&
                               (reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w)) % 16 == 0);
  if (pieces && std::max(p.x_stride, p.w_stride) * es <= (int64_t(1) << 32) / 256 - kStepBytes) {
    offer(5 + steps * (exact ? 0.97 : 0.62) * std::ceil(share(128, 128)), Choice{Choice::k128, 0, 128});
    if (!exact) offer(8 + (steps * 1.55 + 6) * std::ceil(share(256, 256)), Choice{Choice::k256, 0, 0});
  }
  return best;
}

}  // namespace

hipError_t launch_product(const aeisu_product& p, const int32_t* offsets, int experts, hipStream_t stream) {
  const int cus = compute_units();
  const Choice c = choose(p, offsets != nullptr, experts, cus);
  switch (c.kernel) {
    case Choice::k256: return launch_product_256(p, offsets, experts, cus, stream);
    case Choice::k128: return launch_product_128(p, offsets, experts, c.nt, stream);
    case Choice::kRows: return launch_product_rows(p, offsets, experts, c.mt, c.nt, stream);
    default: return launch_product_any(p, offsets, experts, stream);
  }
}

}  // namespace aeisu
