// Quantisation to E4M3 blocks: rows in blocks of 1 x 128 (activations), weights in tiles of 128 x 128.
//
//   scale = max(m / 448, 2^-126), m = largest finite |y| of the block;   code = E4M3(fl32(y / scale))
//
// One pass over the data: sixteen lanes hold a row's block (eight values each), reduce m among themselves and write
// eight codes each.  A workgroup takes sixteen rows at one block column, so that the block-major scales leave as
// 64 consecutive bytes.
#include "blocks.hpp"
#include "common.hpp"

namespace aeisu {
namespace {

typedef unsigned short us8 __attribute__((ext_vector_type(8)));

template <int TYPE>
using elem_t = typename std::conditional<TYPE == AEISU_TYPE_F32, float, unsigned short>::type;

template <int TYPE>
__device__ __forceinline__ float widen(elem_t<TYPE> v) {
  if constexpr (TYPE == AEISU_TYPE_F32) return v;
  else if constexpr (TYPE == AEISU_TYPE_F16) return (float)__builtin_bit_cast(_Float16, v);
  else return __builtin_bit_cast(float, (unsigned)v << 16);
}

// Eight values of a row from column c on, zeros past `left` of them.  Rows need only the alignment of an element:
// the load of eight is one instruction wherever it starts.
template <int TYPE>
__device__ __forceinline__ void load8(const elem_t<TYPE>* p, int64_t left, float v[8]) {
  if (left >= 8) {
    elem_t<TYPE> e[8];
    __builtin_memcpy(e, p, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = widen<TYPE>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? widen<TYPE>(p[i]) : 0.f;
  }
}

// Largest finite magnitude of eight values
__device__ __forceinline__ float finite_max(const float v[8]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = __builtin_fabsf(v[i]);
    m = a < __builtin_inff() ? __builtin_fmaxf(m, a) : m;     // false for NaN too
  }
  return m;
}

__device__ __forceinline__ float block_scale(float m) { return __builtin_fmaxf(m / kE4M3Max, 0x1p-126f); }

// Codes of eight values.  |y / scale| <= 448 (1 + 2^-23) for a finite y, which rounds to at most 448, and the
// conversion gives the NaN code for NaN and infinity: no clamp.
__device__ __forceinline__ uint2 encode8(const float v[8], float scale) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = v[i] / scale;
  uint2 r;
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  r.x = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
  r.y = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], lo, true);
  return r;
}

template <int TYPE, bool GATED>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeRows q) {
  const int lane = threadIdx.x & 15;
  const int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (r >= q.rows) return;                           // whole groups of sixteen lanes
  int64_t src = r;
  if (q.index) src = q.index[r];
  const bool have = src >= 0 && src < q.x_rows;
  const elem_t<TYPE>* x = static_cast<const elem_t<TYPE>*>(q.x) + (have ? src : 0) * q.x_stride;
  const int64_t nb = (q.cols + kBlock - 1) / kBlock;
  for (int64_t j = blockIdx.y; j < nb; j += gridDim.y) {
    const int64_t c = j * kBlock + lane * 8;
    const int64_t left = have ? q.cols - c : 0;
    float v[8];
    load8<TYPE>(x + c, left, v);
    if constexpr (GATED) {
      float b[8];
      load8<TYPE>(x + q.cols + c, left, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] / (1.f + expf(-v[i])) * b[i];
    }
    float m = finite_max(v);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) m = __builtin_fmaxf(m, __shfl_xor(m, d, 16));
    const float s = block_scale(m);
    *reinterpret_cast<uint2*>(q.codes + r * q.codes_stride + c) = encode8(v, s);
    if (lane == 0) q.scales[j * q.scales_stride + r] = s;
  }
}

// One workgroup per tile: sixteen rows a pass, the 64 values of each thread stay in registers.
template <int TYPE>
__global__ __launch_bounds__(256) void quantize_weight_kernel(QuantizeWeight q) {
  __shared__ float part[4];
  const int lane = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int64_t nb = (q.n + kBlock - 1) / kBlock, kb = (q.k + kBlock - 1) / kBlock, kp = kb * kBlock;
  const int64_t jk = blockIdx.x % kb, jn = blockIdx.x / kb, e = blockIdx.y;
  const elem_t<TYPE>* w = static_cast<const elem_t<TYPE>*>(q.w) + e * q.expert_stride;
  const int64_t c = jk * kBlock + lane * 8;
  float v[8][8], m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = jn * kBlock + i * 16 + row;
    load8<TYPE>(w + (r < q.n ? r : 0) * q.row_stride + c, r < q.n ? q.k - c : 0, v[i]);
    m = __builtin_fmaxf(m, finite_max(v[i]));
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = __builtin_fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  const float s = block_scale(__builtin_fmaxf(__builtin_fmaxf(part[0], part[1]), __builtin_fmaxf(part[2], part[3])));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = jn * kBlock + i * 16 + row;
    if (r < q.n) *reinterpret_cast<uint2*>(q.codes + (e * q.n + r) * kp + c) = encode8(v[i], s);
  }
  if (threadIdx.x == 0) q.scales[(e * nb + jn) * kb + jk] = s;
}

}  // namespace

hipError_t launch_quantize_rows(const QuantizeRows& q, int type, bool gated, hipStream_t stream) {
  const int64_t nb = blocks_of(q.cols);
  const dim3 grid((unsigned)((q.rows + 15) / 16), (unsigned)(nb < 65535 ? nb : 65535));
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(q); };
  if (type == AEISU_TYPE_F16) gated ? go(quantize_rows_kernel<AEISU_TYPE_F16, true>) : go(quantize_rows_kernel<AEISU_TYPE_F16, false>);
  else if (type == AEISU_TYPE_BF16)
    gated ? go(quantize_rows_kernel<AEISU_TYPE_BF16, true>) : go(quantize_rows_kernel<AEISU_TYPE_BF16, false>);
  else gated ? go(quantize_rows_kernel<AEISU_TYPE_F32, true>) : go(quantize_rows_kernel<AEISU_TYPE_F32, false>);
  return hipGetLastError();
}

hipError_t launch_quantize_weight(const QuantizeWeight& q, int type, int64_t experts, hipStream_t stream) {
  const int64_t tiles = blocks_of(q.n) * blocks_of(q.k);
  if (tiles > 0x7fffffff) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)tiles, (unsigned)experts);
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(q); };
  if (type == AEISU_TYPE_F16) go(quantize_weight_kernel<AEISU_TYPE_F16>);
  else if (type == AEISU_TYPE_BF16) go(quantize_weight_kernel<AEISU_TYPE_BF16>);
  else go(quantize_weight_kernel<AEISU_TYPE_F32>);
  return hipGetLastError();
}

}  // namespace aeisu
