// Products of few rows: blocks of 16 MT rows x 16 NT columns, the columns of the operands split over a block's eight
// waves.  Each wave reads its fragments from memory into registers and keeps sums of its own, which meet in LDS in the
// order of the waves.
#include "product.hpp"

namespace aeisu {
namespace {

constexpr int kWaves = 8;

// 16 bytes of a row of which `left` elements are its own; zeros for the others.  Rows may start anywhere.
template <int ES>
__device__ __forceinline__ i4 piece(const char* p, int64_t left) {
  i4 v = {0, 0, 0, 0};
  if (ES == 1 || left >= 8) {
    __builtin_memcpy(&v, p, 16);
  } else if (left > 0) {
    unsigned short h[8] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) h[j] = reinterpret_cast<const unsigned short*>(p)[j];
    __builtin_memcpy(&v, h, 16);
  }
  return v;
}

template <int TYPE, bool EXACT, int MT, int NT>
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
    Frag xf[U][MT], wf[U][NT];
    float sc[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * kWaves < steps ? s0 + u * kWaves : steps - 1;
      const int64_t at = (int64_t)s * kStepBytes, left = p.k - (int64_t)s * STEP - g * 8;
#pragma unroll
      for (int j = 0; j < NT; ++j) wf[u][j] = Frag{piece<ES>(w[j] + at, left), piece<ES>(w[j] + at + 64, left - 32)};
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xf[u][i] = Frag{piece<ES>(x[i] + at, left), piece<ES>(x[i] + at + 64, left - 32)};
        if constexpr (kE4M3) sc[u][i] = sx[i][s * p.x_scales_stride] * sw[s];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * kWaves >= steps) break;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if constexpr (kE4M3) {
            const f4 part = EXACT ? step_e4m3_exact(wf[u][j], xf[u][i]) : step_e4m3(wf[u][j], xf[u][i]);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(part[r], sc[u][i], acc[i][j][r]);
          } else {
            acc[i][j] = step_16bit<TYPE>(wf[u][j], xf[u][i], acc[i][j]);
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

template <int TYPE, bool EXACT, int MT, int NT>
hipError_t launch(const aeisu_product& p, const int32_t* offsets, int experts, hipStream_t stream) {
  const int64_t nblocks = (p.n + 16 * NT - 1) / (16 * NT);
  const int64_t blocks = most_tiles(p.rows, experts, offsets != nullptr, 16 * MT) * nblocks;
  if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
  product_rows_kernel<TYPE, EXACT, MT, NT><<<(unsigned)blocks, 64 * kWaves, 0, stream>>>(p, offsets, experts, (int)nblocks);
  return hipGetLastError();
}

template <int MT, int NT>
hipError_t launch_type(const aeisu_product& p, const int32_t* offsets, int experts, hipStream_t stream) {
  if (p.type == AEISU_TYPE_F16) return launch<AEISU_TYPE_F16, false, MT, NT>(p, offsets, experts, stream);
  if (p.type == AEISU_TYPE_BF16) return launch<AEISU_TYPE_BF16, false, MT, NT>(p, offsets, experts, stream);
  if (p.out_type == AEISU_TYPE_F32) return launch<AEISU_TYPE_E4M3, true, MT, NT>(p, offsets, experts, stream);
  return launch<AEISU_TYPE_E4M3, false, MT, NT>(p, offsets, experts, stream);
}

}  // namespace

hipError_t launch_product_rows(const aeisu_product& p, const int32_t* offsets, int experts, int mt, int nt, hipStream_t stream) {
  if (mt == 1) return nt == 1 ? launch_type<1, 1>(p, offsets, experts, stream) : launch_type<1, 2>(p, offsets, experts, stream);
  if (mt == 2) return nt == 1 ? launch_type<2, 1>(p, offsets, experts, stream) : launch_type<2, 2>(p, offsets, experts, stream);
  if (nt == 1) return launch_type<4, 1>(p, offsets, experts, stream);
  return nt == 2 ? launch_type<4, 2>(p, offsets, experts, stream) : launch_type<4, 4>(p, offsets, experts, stream);
}

}  // namespace aeisu
