// Row operators in front of a column-sparse layer: the residual addition with
// the root-mean-square norm, and the rounding of rows to e4m3 with one scale
// per row, each written out over the next layer's alive columns only.
//
//   s[m, k] = x[m, k] + r[m, k]                                  (fp32; stored rounded once)
//   y[m, j] = s[m, c_j] * rsqrt(mean_k s[m, k]^2 + eps) * g[c_j]   c = alive list, or all columns
//   e4m3:  scale[m] = max(max_j |y[m, j]| / 448, 2^-126),  q[m, j] = e4m3(y[m, j] / scale[m])
// The plain rounding (gw_quantize_rows) takes y[m, j] = x[m, c_j].
//
// The norm uses the unrounded fp32 sum, so y and s are each rounded once. The
// largest magnitude is taken on the bit patterns of |y| as unsigned integers:
// that order agrees with the order of the values, and puts NaN above infinity
// above every finite value, so a row with a NaN gets a NaN scale and a row
// with an infinity an infinite one (its values then read back as NaN).
#include <algorithm>

#include "gw_common.cuh"
#include "gw_internal.h"

namespace gw {

namespace {

constexpr float kE4m3Max = 448.0f;                 // largest finite e4m3 value
constexpr float kScaleMin = 1.17549435082e-38f;    // 2^-126: a row of zeros divides by it

// Two values rounded to e4m3 (nearest even, saturating, NaN kept): lo in bits 0-7.
__device__ __forceinline__ uint32_t e4m3_pack2(float lo, float hi) {
  uint16_t v;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(v) : "f"(hi), "f"(lo));
  return v;
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
  const float s = __uint_as_float(amax_bits) / kE4m3Max;
  return s < kScaleMin ? kScaleMin : s;            // NaN compares false and stays
}

template <bool Q8, int DT> struct RowOut { using raw = typename Elem<DT>::raw; };
template <int DT> struct RowOut<true, DT> { using raw = uint8_t; };

// Sum of v and maximum of m over the CTA (any number of whole warps).
__device__ __forceinline__ void block_reduce(float& v, uint32_t& m, float* red_v, uint32_t* red_m) {
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  __syncthreads();                                 // the buffers' previous values have been read
  if (lane == 0) {
    red_v[warp] = v;
    red_m[warp] = m;
  }
  __syncthreads();
  v = lane < warps ? red_v[lane] : 0.0f;
  m = lane < warps ? red_m[lane] : 0u;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  m = __reduce_max_sync(0xFFFFFFFFu, m);
}

// Any width, any alignment, any list (longer than the row, unordered,
// repeated): one CTA per row that reads the row again for each pass, the sum
// written last, so that it may take the place of x or of r.
template <int DT, bool Q8, bool NORM>
__global__ void __launch_bounds__(1024) rows_any_kernel(const RowParams p) {
  using raw = typename Elem<DT>::raw;
  using out = typename RowOut<Q8, DT>::raw;
  __shared__ float red_v[32];
  __shared__ uint32_t red_m[32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  bool bad = false;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const raw* x = static_cast<const raw*>(p.x) + row * p.ldx;
    const raw* r = p.r ? static_cast<const raw*>(p.r) + row * p.ldr : nullptr;
    raw* s = p.s ? static_cast<raw*>(p.s) + row * p.lds : nullptr;
    const raw* g = static_cast<const raw*>(p.g);
    out* y = static_cast<out*>(p.y) + row * p.ldy;
    auto sum_at = [&](int64_t k) {
      const float v = Elem<DT>::to_f(x[k]);
      return r ? v + Elem<DT>::to_f(r[k]) : v;
    };
    float rstd = 1.0f;
    if constexpr (NORM) {
      float ss = 0.0f;
      uint32_t unused = 0;
      for (int64_t k = threadIdx.x; k < p.cols; k += blockDim.x) {
        const float v = sum_at(k);
        ss = fmaf(v, v, ss);
      }
      block_reduce(ss, unused, red_v, red_m);
      rstd = rsqrtf(ss / static_cast<float>(p.cols) + p.eps);
    }
    auto out_at = [&](int64_t j) {
      const int64_t c = p.idx ? __ldg(p.idx + j) : j;
      if (c < 0 || c >= p.cols) { bad = true; return 0.0f; }
      const float v = sum_at(c);
      if constexpr (NORM) return g ? v * rstd * Elem<DT>::to_f(g[c]) : v * rstd;
      return v;
    };
    float scale = 1.0f;
    if constexpr (Q8) {
      uint32_t amax = 0;
      float unused = 0.0f;
      for (int64_t j = threadIdx.x; j < p.n; j += blockDim.x) amax = max(amax, abs_bits(out_at(j)));
      block_reduce(unused, amax, red_v, red_m);
      scale = row_scale(amax);
      if (threadIdx.x == 0) p.scale[row] = scale;
    }
    for (int64_t j = threadIdx.x; j < p.pad; j += blockDim.x) {
      const float v = j < p.n ? out_at(j) : 0.0f;
      if constexpr (Q8) y[j] = static_cast<out>(e4m3_pack2(v / scale, 0.0f));
      else y[j] = Elem<DT>::from_f(v);
    }
    if (s) {
      __syncthreads();                             // every read of x and r of this row is done
      for (int64_t k = threadIdx.x; k < p.cols; k += blockDim.x) s[k] = Elem<DT>::from_f(sum_at(k));
    }
  }
  if (bad) raise_error(p.err, GW_DERR_BAD_INDEX);
}

template <int DT, bool Q8, bool NORM>
cudaError_t launch_rows_any(const RowParams& p, int sm_count, cudaStream_t stream) {
  const int64_t width = std::max<int64_t>(p.cols, p.pad);
  const int threads = width <= 1024 ? 128 : width <= 8192 ? 256 : 1024;
  const int64_t grid = std::min<int64_t>(p.rows, static_cast<int64_t>(sm_count) * (2048 / threads));
  return launch_pdl(rows_any_kernel<DT, Q8, NORM>, dim3(static_cast<unsigned>(grid)), dim3(threads),
                    stream, p);
}

template <bool Q8, bool NORM>
cudaError_t launch_rows_dt(const RowParams& p, int dtype, int sm_count, cudaStream_t stream) {
  switch (dtype) {
    case GW_DTYPE_F16: return launch_rows_any<GW_DTYPE_F16, Q8, NORM>(p, sm_count, stream);
    case GW_DTYPE_BF16: return launch_rows_any<GW_DTYPE_BF16, Q8, NORM>(p, sm_count, stream);
    default: return launch_rows_any<GW_DTYPE_F32, Q8, NORM>(p, sm_count, stream);
  }
}

}  // namespace

cudaError_t launch_rows(const RowParams& p, int dtype, bool q8, bool norm, int sm_count,
                        cudaStream_t stream) {
  if (p.rows == 0) return cudaSuccess;
  if (q8) return norm ? launch_rows_dt<true, true>(p, dtype, sm_count, stream)
                      : launch_rows_dt<true, false>(p, dtype, sm_count, stream);
  return launch_rows_dt<false, true>(p, dtype, sm_count, stream);
}

}  // namespace gw
