// Products of few rows: blocks of 16 MT rows x 16 NT columns, the columns of the operands split over a block's eight
// waves.  Each wave reads its fragments from memory into registers and keeps sums of its own, which meet in LDS in the
// order of the waves.
#include "product.hpp"

namespace aeisu {
namespace {

constexpr int kWaves = 8;

template <int TYPE, bool EXACT, bool ODD, int MT, int NT>
__global__ __launch_bounds__(64 * kWaves) void product_rows_kernel(aeisu_product p, const int32_t* offsets, int experts, int nblocks) {
  constexpr bool kE4M3 = TYPE == AEISU_TYPE_E4M3;
  constexpr int ES = kE4M3 ? 1 : 2, STEP = kStepBytes / ES, U = 2;
  __shared__ f4 sums[kWaves][MT * NT][64];
  RowTile tile;
  if (!find_tile<16 * MT>(offsets, experts, p.rows, (int)(blockIdx.x / nblocks), tile)) return;
  const int64_t n0 = (int64_t)(blockIdx.x % nblocks) * 16 * NT;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const int e = tile.expert < 0 ? 0 : tile.expert;
  const int kb = (int)((p.k + kBlock - 1) / kBlock);
  const int steps = tile.expert < 0 ? 0 : (int)((p.k + STEP - 1) / STEP);
  const char *x[MT], *w[NT];
  const float* sx[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    int64_t m = tile.lo + i * 16 + (lane & 15);
    m = m < tile.hi ? m : tile.hi - 1;
    x[i] = static_cast<const char*>(p.x) + m * p.x_stride * ES + g * 16;
    sx[i] = kE4M3 ? p.x_scales + m : nullptr;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    int64_t n = n0 + j * 16 + (lane & 15);
    n = n < p.n ? n : p.n - 1;
    w[j] = static_cast<const char*>(p.w) + (e * p.w_expert_stride + n * p.w_stride) * ES + g * 16;
  }
  const float* sw = kE4M3 ? p.w_scales + ((int64_t)e * ((p.n + kBlock - 1) / kBlock) + n0 / kBlock) * kb : nullptr;
  f4 acc[MT][NT] = {};
  for (int s0 = wave; s0 < steps; s0 += U * kWaves) {
    Piece<ES, ODD> xf[U][MT][2], wf[U][NT][2];
    float sc[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * kWaves < steps ? s0 + u * kWaves : steps - 1;
      const int64_t at = (int64_t)s * kStepBytes, left = p.k - (int64_t)s * STEP - g * 8;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        wf[u][j][0] = load_piece<ES, ODD>(w[j] + at, left, s > 0 || g > 0);
        wf[u][j][1] = load_piece<ES, ODD>(w[j] + at + 64, left - 32, true);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xf[u][i][0] = load_piece<ES, ODD>(x[i] + at, left, s > 0 || g > 0);
        xf[u][i][1] = load_piece<ES, ODD>(x[i] + at + 64, left - 32, true);
        if constexpr (kE4M3) sc[u][i] = sx[i][s * p.x_scales_stride] * sw[s];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * kWaves >= steps) break;
      Frag wq[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) wq[j] = Frag{wf[u][j][0].whole(), wf[u][j][1].whole()};
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const Frag xq{xf[u][i][0].whole(), xf[u][i][1].whole()};
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if constexpr (kE4M3) {
            const f4 part = EXACT ? step_e4m3_exact(wq[j], xq) : step_e4m3(wq[j], xq);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(part[r], sc[u][i], acc[i][j][r]);
          } else {
            acc[i][j] = step_16bit<TYPE>(wq[j], xq, acc[i][j]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) sums[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  const size_t vec = p.out_type == AEISU_TYPE_F32 ? 16 : 8;
  const bool wide = (reinterpret_cast<uintptr_t>(p.out) % vec) == 0 && p.out_stride % 4 == 0;
  const float* bias = p.bias && tile.expert >= 0 ? p.bias + (int64_t)e * p.n : nullptr;
  const int used = steps < kWaves ? steps : kWaves;
  for (int t = wave; t < MT * NT; t += kWaves) {
    const int64_t m = tile.lo + (t / NT) * 16 + (lane & 15);
    if (m >= tile.hi) continue;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    for (int q = 0; q < used; ++q) v += sums[q][t][lane];
    finish4(p, m, n0 + (t % NT) * 16 + 4 * g, v, bias, wide);
  }
}

template <int TYPE, bool EXACT, bool ODD, int MT, int NT>
hipError_t launch(const aeisu_product& p, const int32_t* offsets, int experts, hipStream_t stream) {
  const int64_t nblocks = (p.n + 16 * NT - 1) / (16 * NT);
  const int64_t blocks = most_tiles(p.rows, experts, offsets != nullptr, 16 * MT) * nblocks;
  if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
  product_rows_kernel<TYPE, EXACT, ODD, MT, NT><<<(unsigned)blocks, 64 * kWaves, 0, stream>>>(p, offsets, experts, (int)nblocks);
  return hipGetLastError();
}

template <int MT, int NT>
hipError_t launch_type(const aeisu_product& p, const int32_t* offsets, int experts, hipStream_t stream) {
  const bool odd = odd_rows(p);
  if (p.type == AEISU_TYPE_F16)
    return odd ? launch<AEISU_TYPE_F16, false, true, MT, NT>(p, offsets, experts, stream)
               : launch<AEISU_TYPE_F16, false, false, MT, NT>(p, offsets, experts, stream);
  if (p.type == AEISU_TYPE_BF16)
    return odd ? launch<AEISU_TYPE_BF16, false, true, MT, NT>(p, offsets, experts, stream)
               : launch<AEISU_TYPE_BF16, false, false, MT, NT>(p, offsets, experts, stream);
  if (p.out_type == AEISU_TYPE_F32) return launch<AEISU_TYPE_E4M3, true, false, MT, NT>(p, offsets, experts, stream);
  return launch<AEISU_TYPE_E4M3, false, false, MT, NT>(p, offsets, experts, stream);
}

}  // namespace

hipError_t launch_product_rows(const aeisu_product& p, const int32_t* offsets, int experts, int mt, int nt, hipStream_t stream) {
  if (mt == 1) return nt == 1 ? launch_type<1, 1>(p, offsets, experts, stream) : launch_type<1, 2>(p, offsets, experts, stream);
  if (mt == 2) return nt == 1 ? launch_type<2, 1>(p, offsets, experts, stream) : launch_type<2, 2>(p, offsets, experts, stream);
  if (nt == 1) return launch_type<4, 1>(p, offsets, experts, stream);
  return nt == 2 ? launch_type<4, 2>(p, offsets, experts, stream) : launch_type<4, 4>(p, offsets, experts, stream);
}

}  // namespace aeisu
