// Quantisation to E4M3 blocks: rows in blocks of 1 x 128 (activations), weights in tiles of 128 x 128.
//
//   scale = max(m / 448, 2^-126), m = largest finite |y| of the block;   code = E4M3(fl32(y / scale))
//
// One pass over the data: sixteen lanes hold a row's block (eight values each), reduce m among themselves and write
// eight codes each.  A workgroup takes sixteen rows (or groups of them) at one block column, so that the block-major
// scales leave as 64 consecutive bytes.
// Bound by memory: 16,384 x 4096 BF16 40.5 us (5.0 TB/s; a large copy reaches 5.3), 136,640 x 128 FP16 10.9 us (4.8), gated
// 4096 x 2816 BF16 12.5 us (4.7); gathered rows that are picked twice come from the caches: 16,384 of 8192 34 us, 5.9 TB/s
// of loads and stores.  What gathered and gated rows gain over 39 and 14 us came from fewer instructions a value: one
// correction a quotient for two, largest magnitudes of 16-bit values found two at a time on their bits, 32-bit columns,
// the exponential from its instruction.
#include "blocks.hpp"
#include "common.hpp"

namespace aeisu {
namespace {

template <int TYPE>
using elem_t = typename std::conditional<TYPE == AEISU_TYPE_F32, float, unsigned short>::type;

template <int TYPE>
__device__ __forceinline__ float widen(elem_t<TYPE> v) {
  if constexpr (TYPE == AEISU_TYPE_F32) return v;
  else if constexpr (TYPE == AEISU_TYPE_F16) return (float)__builtin_bit_cast(_Float16, v);
  else return __builtin_bit_cast(float, (unsigned)v << 16);
}

template <int TYPE>
struct Eight {
  elem_t<TYPE> e[8];
};

// Eight values of a row, zeros past `left` of them.  Rows need only the alignment of an element: the load of eight is
// one instruction (FP32: two) wherever it starts.
template <int TYPE>
__device__ __forceinline__ Eight<TYPE> load8(const elem_t<TYPE>* p, int left) {
  Eight<TYPE> r;
  if (left >= 8) {
    __builtin_memcpy(r.e, p, sizeof(r.e));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.e[i] = i < left ? p[i] : elem_t<TYPE>(0);
  }
  return r;
}
template <int TYPE>
__device__ __forceinline__ void widen8(const Eight<TYPE>& r, float v[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = widen<TYPE>(r.e[i]);
}

// Largest finite magnitude of eight values.  `bad` becomes NaN where one is not finite (v * 0); only then are they
// looked at one by one.
__device__ __forceinline__ float finite_max(const float v[8]) {
  float m = 0.f, bad = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m = __builtin_fmaxf(m, __builtin_fabsf(v[i]));
    bad = __builtin_fmaf(v[i], 0.f, bad);
  }
  if (bad != bad) {
    m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = __builtin_fabsf(v[i]);
      m = a < __builtin_inff() ? __builtin_fmaxf(m, a) : m;   // false for NaN too
    }
  }
  return m;
}
// Largest of sixteen adjacent lanes: rotations within a lane row
template <int BY>
__device__ __forceinline__ unsigned rotated(unsigned m) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)m, (int)m, 0x120 + BY, 0xf, 0xf, false);
}
__device__ __forceinline__ unsigned max16(unsigned m) {
  auto larger = [](unsigned a, unsigned b) { return a > b ? a : b; };
  m = larger(m, rotated<8>(m));
  m = larger(m, rotated<4>(m));
  m = larger(m, rotated<2>(m));
  return larger(m, rotated<1>(m));
}
// of magnitudes, whose order is that of their bits
__device__ __forceinline__ float max16(float m) { return __builtin_bit_cast(float, max16(__builtin_bit_cast(unsigned, m))); }

// Largest finite magnitude of sixteen lanes' values.  16-bit values are compared two at a time as they are, magnitudes in
// the order of their bits; where the largest is no finite value, those that are not are left out.
template <int TYPE>
__device__ __forceinline__ float block_max(const Eight<TYPE>& r, const float v[8]) {
  if constexpr (TYPE == AEISU_TYPE_F32) return max16(finite_max(v));
  else {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    us2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      m = __builtin_elementwise_max(m, us2{r.e[i], r.e[i + 1]} & us2{0x7fff, 0x7fff});
    const unsigned top = max16((unsigned)(m[0] > m[1] ? m[0] : m[1]));
    if (__builtin_expect(top >= (TYPE == AEISU_TYPE_F16 ? 0x7c00u : 0x7f80u), 0)) return max16(finite_max(v));
    return widen<TYPE>((unsigned short)top);
  }
}

// Quotients y / by, correctly rounded, without a division for each: with r + s = 1 / by to 48 bits, fma(y, r, y s) lies within a
// unit in the last place, and from there one correction q + r (y - q by) gives the nearest (Markstein's theorem, r being
// the nearest to 1 / by and y - q by exact).  That remainder is exact while |y| 2^-47 is no denormal number.
struct Divisor {
  float by, r, s;
  __device__ __forceinline__ float quotient(float y) const {
    const float q = __builtin_fmaf(y, r, y * s);
    return __builtin_fmaf(__builtin_fmaf(-q, by, y), r, q);
  }
};
__device__ __forceinline__ Divisor divisor(float by) {
  const float r = 1.f / by;
  return {by, r, __builtin_fmaf(-by, r, 1.f) * r};
}

// Scale and codes of eight values of a block whose largest finite magnitude is m: scale = max(m / 448, 2^-126).
// |y / scale| <= 448 (1 + 2^-23) for a finite y, which rounds to at most 448, and the conversion gives the NaN code for NaN
// and infinity (whose quotients are NaN): no clamp.
// Below m = 2^-80 true divisions: there the remainders would no longer be exact wherever the quotient reaches 2^-10, and
// under that every code is 0.
struct Scaled {
  uint2 codes;
  float scale;
};
__device__ __forceinline__ Scaled encode8(const float v[8], float m) {
  float q[8], scale;
  if (__builtin_expect(m >= 0x1p-80f, 1)) {
    scale = Divisor{kE4M3Max, 1.f / 448.f, (float)(1.0 / 448.0 - (double)(1.f / 448.f))}.quotient(m);
    const Divisor d = divisor(scale);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = d.quotient(v[i]);
  } else {
    scale = __builtin_fmaxf(m / kE4M3Max, 0x1p-126f);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = v[i] / scale;
  }
  Scaled r;
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  r.codes.x = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
  r.codes.y = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], lo, true);
  r.scale = scale;
  return r;
}

// SiLU(a) b.  With t = exp(-|a|) the logistic function is 1 / (1 + t) or t / (1 + t): nothing overflows, and 1 + t in [1, 2]
// suits the reciprocal instruction (one unit in the last place).  t = e e and e = 2^(h + l), h + l = -|a| / (2 ln 2) to 48
// bits, as 2^h (1 + l ln 2): a factor e before b and one after it keep large b with a down to -170 from an underflow of t
// (the exponential instruction gives no denormal numbers).
__device__ __forceinline__ float gate(float a, float b) {
  constexpr float half = 0.72134752f, rest = (float)(0.72134752044448170 - (double)half);
  const float x = __builtin_fmaxf(-__builtin_fabsf(a), -200.f), h = x * half;
  const float l = __builtin_fmaf(x, rest, __builtin_fmaf(x, half, -h)), p = __builtin_amdgcn_exp2f(h);
  const float e = __builtin_fmaf(p * l, 0.69314718f, p), f = a < 0.f ? e : 1.f;
  return a * f * __builtin_amdgcn_rcpf(__builtin_fmaf(e, e, 1.f)) * b * f;
}

// CU block columns for each thread, all loads before the first use.
template <int TYPE, bool GATED, int CU>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeRows q) {
  const int lane = threadIdx.x & 15;
  const int cols = (int)q.cols, nb = (cols + kBlock - 1) / kBlock;
  const int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (r >= q.rows) return;                           // whole groups of sixteen lanes
  const int64_t src = q.index ? q.index[r] : r;
  const bool have = src >= 0 && src < q.x_rows;
  const elem_t<TYPE>* x = static_cast<const elem_t<TYPE>*>(q.x) + (have ? src : 0) * q.x_stride;
  uint8_t* codes = q.codes + r * q.codes_stride;
  for (int j0 = blockIdx.y * CU; j0 < nb; j0 += gridDim.y * CU) {
    Eight<TYPE> a[CU], b[GATED ? CU : 1];
#pragma unroll
    for (int j = 0; j < CU; ++j) {
      const int c = (j0 + j) * kBlock + lane * 8, left = have ? cols - c : 0;
      a[j] = load8<TYPE>(x + c, left);
      if constexpr (GATED) b[j] = load8<TYPE>(x + cols + c, left);
    }
#pragma unroll
    for (int j = 0; j < CU; ++j) {
      if (j0 + j >= nb) break;
      float v[8], m;
      widen8<TYPE>(a[j], v);
      if constexpr (GATED) {
        float u[8];
        widen8<TYPE>(b[j], u);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = gate(v[k], u[k]);
        m = max16(finite_max(v));
      } else {
        m = block_max<TYPE>(a[j], v);
      }
      const Scaled s = encode8(v, m);
      *reinterpret_cast<uint2*>(codes + (j0 + j) * kBlock + lane * 8) = s.codes;
      if (lane == 0) q.scales[(j0 + j) * q.scales_stride + r] = s.scale;
    }
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
    widen8<TYPE>(load8<TYPE>(w + (r < q.n ? r : 0) * q.row_stride + c, r < q.n ? (int)(q.k - c) : 0), v[i]);
    m = __builtin_fmaxf(m, finite_max(v[i]));
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = __builtin_fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  m = __builtin_fmaxf(__builtin_fmaxf(part[0], part[1]), __builtin_fmaxf(part[2], part[3]));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = jn * kBlock + i * 16 + row;
    const Scaled s = encode8(v[i], m);
    if (r < q.n) *reinterpret_cast<uint2*>(q.codes + (e * q.n + r) * kp + c) = s.codes;
    if (i == 0 && threadIdx.x == 0) q.scales[(e * nb + jn) * kb + jk] = s.scale;
  }
}

}  // namespace

namespace {

template <int TYPE, bool GATED, int CU>
hipError_t launch_rows(const QuantizeRows& q, hipStream_t stream) {
  const int64_t nb = (blocks_of(q.cols) + CU - 1) / CU;
  const dim3 grid((unsigned)((q.rows + 15) / 16), (unsigned)(nb < 65535 ? nb : 65535));
  quantize_rows_kernel<TYPE, GATED, CU><<<grid, 256, 0, stream>>>(q);
  return hipGetLastError();
}
template <int TYPE, bool GATED>
hipError_t launch_rows(const QuantizeRows& q, hipStream_t stream) {
  // Two block columns a thread share the row's index and address where there are enough of them: 16,384 rows of 4096
  // gathered 33 us against 38 with one, 35 with four; rows as they are 40 (5.1 TB/s) against 42 and 43.  Gated rows (12.2
  // us against 15.4 with two, 4096 x 2816) and rows of one block (136,640 of 128: 10.8 against 11.7) lose by it: they run
  // in fewer, longer workgroups whose loads and arithmetic overlap less.
  if constexpr (!GATED) {
    if (blocks_of(q.cols) >= 2 && (q.rows + 15) / 16 * blocks_of(q.cols) >= 4096) return launch_rows<TYPE, GATED, 2>(q, stream);
  }
  return launch_rows<TYPE, GATED, 1>(q, stream);
}

}  // namespace

hipError_t launch_quantize_rows(const QuantizeRows& all, int type, bool gated, hipStream_t stream) {
  constexpr int64_t kRows = int64_t(1) << 27;        // rows a launch: 2^31 threads in x
  const int64_t size = type == AEISU_TYPE_F32 ? 4 : 2;
  for (int64_t r = 0; r < all.rows; r += kRows) {
    QuantizeRows q = all;
    q.rows = all.rows - r < kRows ? all.rows - r : kRows;
    q.codes += r * all.codes_stride;
    q.scales += r;
    if (all.index) q.index += r;
    else q.x = static_cast<const char*>(all.x) + r * all.x_stride * size, q.x_rows -= r;
    hipError_t e;
    if (type == AEISU_TYPE_F16) e = gated ? launch_rows<AEISU_TYPE_F16, true>(q, stream) : launch_rows<AEISU_TYPE_F16, false>(q, stream);
    else if (type == AEISU_TYPE_BF16) e = gated ? launch_rows<AEISU_TYPE_BF16, true>(q, stream) : launch_rows<AEISU_TYPE_BF16, false>(q, stream);
    else e = gated ? launch_rows<AEISU_TYPE_F32, true>(q, stream) : launch_rows<AEISU_TYPE_F32, false>(q, stream);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
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
