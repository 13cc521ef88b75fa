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
// largest magnitude is taken on the bit patterns as unsigned integers: that
// order agrees with the order of the values, and puts NaN above infinity above
// every finite value, so a row with a NaN gets a NaN scale and a row with an
// infinity an infinite one (its values then read back as NaN).
//
// e4m3 values are taken from u[m, j] = s[m, c_j] g[c_j], from which the norm's
// factor cancels: y / scale = 448 u / max|u|, computed as (0.875 u) / (max|u| / 512).
// With 16-bit inputs 0.875 u is mostly exact in fp32 (u has up to 21 bits), so a
// quotient that lies exactly between two e4m3 values, which 16-bit data meets
// often, comes out exact and rounds to even; dividing by a rounded scale would
// send it either way.
//
// What bounds these kernels is HBM: a row is read and written once. rows_kernel
// keeps a row in registers (E elements per thread, a warp or a CTA per row),
// and passes it through shared memory only to pick alive columns from it;
// rows_any_kernel takes what that one does not.
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

// The scale of a row whose largest |u| is umax and whose norm factor is rstd,
// and the divisor d for which y / scale = 0.875 u / d. NaN compares false and stays.
struct RowScale {
  float scale, d;
};
__device__ __forceinline__ RowScale row_scale(uint32_t umax_bits, float rstd) {
  const float umax = __uint_as_float(umax_bits);
  RowScale q;
  q.scale = umax * rstd / kE4m3Max;
  q.d = umax * (1.0f / 512.0f);
  if (q.scale < kScaleMin) {
    q.scale = kScaleMin;
    q.d = 0.875f * kScaleMin / rstd;
  }
  return q;
}
__device__ __forceinline__ float to_scale(float u, float d) { return 0.875f * u / d; }

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
      return NORM && g ? v * Elem<DT>::to_f(g[c]) : v;
    };
    RowScale q8 = {1.0f, 1.0f};
    if constexpr (Q8) {
      uint32_t amax = 0;
      float unused = 0.0f;
      for (int64_t j = threadIdx.x; j < p.n; j += blockDim.x) amax = max(amax, abs_bits(out_at(j)));
      block_reduce(unused, amax, red_v, red_m);
      q8 = row_scale(amax, rstd);
      if (threadIdx.x == 0) p.scale[row] = q8.scale;
    }
    for (int64_t j = threadIdx.x; j < p.pad; j += blockDim.x) {
      const float v = j < p.n ? out_at(j) : 0.0f;
      if constexpr (Q8) y[j] = static_cast<out>(e4m3_pack2(to_scale(v, q8.d), 0.0f));
      else y[j] = Elem<DT>::from_f(v * rstd);
    }
    if (s) {
      __syncthreads();                             // every read of x and r of this row is done
      for (int64_t k = threadIdx.x; k < p.cols; k += blockDim.x) s[k] = Elem<DT>::from_f(sum_at(k));
    }
  }
  if (bad) raise_error(p.err, GW_DERR_BAD_INDEX);
}

// ---------------------------------------------------------------------------
// Rows of up to 32768 columns, read and written once.
// ---------------------------------------------------------------------------
// A group of G threads (a warp, or the whole CTA) holds a row: E elements per
// thread, in 16-byte vectors (VEC: element k = (i G + t) V + j of vector i) or
// one by one (k = i G + t). GATHER passes u = s g through shared memory and
// picks the alive columns there; the list is kept there too, as 16-bit
// positions, loaded once for all the rows of a CTA. For the e4m3 scale each
// thread knows which of its columns the list names (one bit each), so the sum
// of squares and the largest |u| take one reduction.
constexpr int kRowsMaxCols = 32768;
constexpr uint32_t kNoColumn = 0xFFFFu;            // zero output (bad index or padding)

template <int DT>
__device__ __forceinline__ uint4 ld_row_v4(const void* base, int64_t vec) {
  // Read once: kept out of L1 (the residual may be written in place, so not the read-only path).
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(static_cast<const uint4*>(base) + vec) : "memory");
  return v;
}

// One 16-byte vector as floats.
template <int DT>
__device__ __forceinline__ void unpack16(const uint4 q, float* f) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == GW_DTYPE_F32) {
      f[i] = __uint_as_float(w[i]);
    } else {
      f[2 * i] = Elem<DT>::to_f(static_cast<uint16_t>(w[i] & 0xFFFFu));
      f[2 * i + 1] = Elem<DT>::to_f(static_cast<uint16_t>(w[i] >> 16));
    }
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack16(const float* f) {
  if constexpr (DT == GW_DTYPE_F32)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    return make_uint4(Elem<DT>::pack2(f[0], f[1]), Elem<DT>::pack2(f[2], f[3]),
                      Elem<DT>::pack2(f[4], f[5]), Elem<DT>::pack2(f[6], f[7]));
}

// Where element k of a row lies in its shared-memory copy. A thread stores a
// 16-bit vector's eight floats as two 16-byte halves; the halves go to two
// planes, so that neighbouring threads' stores are adjacent.
template <int DT, bool VEC>
__device__ __forceinline__ int row_pos(int k, int cols) {
  if constexpr (VEC && DT != GW_DTYPE_F32)
    return ((k >> 2) & 1) * (cols >> 1) + (k >> 3) * 4 + (k & 3);
  else
    return k;
}

template <int DT, bool Q8, bool GATHER, bool VEC, int E, bool WARP, int MAXT>
__global__ void __launch_bounds__(MAXT) rows_kernel(const RowParams p, int y_vec) {
  using raw = typename Elem<DT>::raw;
  using out = typename RowOut<Q8, DT>::raw;
  constexpr int V = VEC ? static_cast<int>(16 / sizeof(raw)) : 1;
  constexpr int I = E / V;                                        // vectors (or elements) per thread
  constexpr int kPack = Q8 ? 4 : sizeof(raw) == 2 ? 2 : 1;        // outputs per 4-byte store
  extern __shared__ __align__(16) uint8_t smem[];
  const int G = WARP ? 32 : static_cast<int>(blockDim.x);
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int group = WARP ? (threadIdx.x >> 5) : 0;
  const int groups = WARP ? (blockDim.x >> 5) : 1;
  const int cols = static_cast<int>(p.cols);
  const int n = static_cast<int>(p.n);
  const int pad = static_cast<int>(p.pad);
  float* red_v = reinterpret_cast<float*>(smem);                  // [2][32]
  uint32_t* red_m = reinterpret_cast<uint32_t*>(smem) + 64;       // [2][32]
  float* srow = reinterpret_cast<float*>(smem + 512) + group * ((cols + 3) & ~3);
  uint16_t* spos = reinterpret_cast<uint16_t*>(smem + 512 + groups * ((cols + 3) & ~3) * 4);
  const int npos = (pad + 3) & ~3;

  // The inputs may come from the previous kernel of the stream.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  uint32_t named = 0xFFFFFFFFu;                                   // this thread's columns in the list
  if constexpr (GATHER) {
    bool bad = false;
    uint32_t* bits = reinterpret_cast<uint32_t*>(spos + npos);    // Q8: one bit per column
    if constexpr (Q8) {
      for (int i = threadIdx.x; i < (cols + 31) / 32; i += blockDim.x) bits[i] = 0;
      __syncthreads();
    }
    for (int j = threadIdx.x; j < npos; j += blockDim.x) {
      uint32_t pos = kNoColumn;
      if (j < n) {
        const int64_t c = __ldg(p.idx + j);
        if (c < 0 || c >= cols) {
          bad = true;
        } else {
          pos = row_pos<DT, VEC>(static_cast<int>(c), cols);
          if constexpr (Q8) atomicOr(&bits[c >> 5], 1u << (c & 31));
        }
      }
      spos[j] = static_cast<uint16_t>(pos);
    }
    if (bad && blockIdx.x == 0) raise_error(p.err, GW_DERR_BAD_INDEX);
    __syncthreads();
    if constexpr (Q8) {
      named = 0;
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int k = (i * G + t) * V;
        if (k < cols) named |= ((bits[k >> 5] >> (k & 31)) & ((1u << V) - 1u)) << (i * V);
      }
    }
  }

  const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
  int buf = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * groups + group; row < p.rows; row += step) {
    const raw* x = static_cast<const raw*>(p.x) + row * p.ldx;
    const raw* r = static_cast<const raw*>(p.r) + row * p.ldr;
    raw* sum = static_cast<raw*>(p.s) + row * p.lds;
    const raw* g = static_cast<const raw*>(p.g);
    float u[E];
    if constexpr (VEC) {
      uint4 xv[I], rv[I];
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int k = (i * G + t) * V;
        xv[i] = k < cols ? ld_row_v4<DT>(x, i * G + t) : make_uint4(0, 0, 0, 0);
      }
      if (p.r) {
#pragma unroll
        for (int i = 0; i < I; ++i) {
          const int k = (i * G + t) * V;
          rv[i] = k < cols ? ld_row_v4<DT>(r, i * G + t) : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < I; ++i) unpack16<DT>(xv[i], u + i * V);
      if (p.r) {
#pragma unroll
        for (int i = 0; i < I; ++i) {
          float f[V];
          unpack16<DT>(rv[i], f);
#pragma unroll
          for (int j = 0; j < V; ++j) u[i * V + j] += f[j];
        }
      }
      if (p.s) {
#pragma unroll
        for (int i = 0; i < I; ++i)
          if ((i * G + t) * V < cols) reinterpret_cast<uint4*>(sum)[i * G + t] = pack16<DT>(u + i * V);
      }
    } else {
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int k = i * G + t;
        u[i] = k < cols ? Elem<DT>::to_f(x[k]) : 0.0f;
      }
      if (p.r) {
#pragma unroll
        for (int i = 0; i < I; ++i)
          if (i * G + t < cols) u[i] += Elem<DT>::to_f(r[i * G + t]);
      }
      if (p.s) {
#pragma unroll
        for (int i = 0; i < I; ++i)
          if (i * G + t < cols) sum[i * G + t] = Elem<DT>::from_f(u[i]);
      }
    }
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) ss = fmaf(u[e], u[e], ss);
    if (g) {
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int k = (i * G + t) * V;
        if (k < cols) {
          if constexpr (VEC) {
            float f[V];
            unpack16<DT>(__ldg(reinterpret_cast<const uint4*>(g) + i * G + t), f);
#pragma unroll
            for (int j = 0; j < V; ++j) u[i * V + j] *= f[j];
          } else {
            u[i] *= Elem<DT>::to_f(__ldg(g + k));
          }
        }
      }
    }
    uint32_t umax = 0;
    if constexpr (Q8) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!GATHER || ((named >> e) & 1u)) umax = max(umax, abs_bits(u[e]));
    }
    if constexpr (GATHER) {
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int k = (i * G + t) * V;
        if (k < cols) {
          if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < V; j += 4)
              *reinterpret_cast<float4*>(srow + row_pos<DT, VEC>(k + j, cols)) =
                  make_float4(u[i * V + j], u[i * V + j + 1], u[i * V + j + 2], u[i * V + j + 3]);
          } else {
            srow[k] = u[i];
          }
        }
      }
    }
    // Sum of squares and largest |u| of the row; publishes srow too.
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    if constexpr (Q8) umax = __reduce_max_sync(0xFFFFFFFFu, umax);
    if constexpr (WARP) {
      __syncwarp();
    } else {
      const int lane = t & 31;
      if (lane == 0) {
        red_v[buf * 32 + (t >> 5)] = ss;
        red_m[buf * 32 + (t >> 5)] = umax;
      }
      __syncthreads();
      const bool in = lane < (G >> 5);
      ss = in ? red_v[buf * 32 + lane] : 0.0f;
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
      if constexpr (Q8) umax = __reduce_max_sync(0xFFFFFFFFu, in ? red_m[buf * 32 + lane] : 0u);
      buf ^= 1;
    }
    const float rstd = p.norm ? rsqrtf(ss / static_cast<float>(cols) + p.eps) : 1.0f;
    RowScale q8 = {1.0f, 1.0f};
    if constexpr (Q8) {
      q8 = row_scale(umax, rstd);
      if (t == 0) p.scale[row] = q8.scale;
    }
    out* y = static_cast<out*>(p.y) + row * p.ldy;
    auto value = [&](float v) { return Q8 ? to_scale(v, q8.d) : v * rstd; };
    auto store1 = [&](int j, float v) {
      if constexpr (Q8) y[j] = static_cast<out>(e4m3_pack2(v, 0.0f));
      else y[j] = Elem<DT>::from_f(v);
    };
    if constexpr (GATHER) {
      // Neighbouring threads take neighbouring groups of outputs: 4-byte
      // stores, and shared-memory reads within a narrow window of the row.
      for (int j = t * kPack; j < pad; j += G * kPack) {
        float v[kPack];
        uint16_t pos[kPack];
        if constexpr (kPack == 4) *reinterpret_cast<uint2*>(pos) = *reinterpret_cast<const uint2*>(spos + j);
        else if constexpr (kPack == 2) *reinterpret_cast<uint32_t*>(pos) = *reinterpret_cast<const uint32_t*>(spos + j);
        else pos[0] = spos[j];
#pragma unroll
        for (int q = 0; q < kPack; ++q) v[q] = pos[q] == kNoColumn ? 0.0f : value(srow[pos[q]]);
        if (y_vec && j + kPack <= pad) {
          uint32_t w;
          if constexpr (Q8) w = e4m3_pack2(v[0], v[1]) | (e4m3_pack2(v[2], v[3]) << 16);
          else if constexpr (kPack == 2) w = Elem<DT>::pack2(v[0], v[1]);
          else w = __float_as_uint(v[0]);
          *reinterpret_cast<uint32_t*>(y + j) = w;
        } else {
#pragma unroll
          for (int q = 0; q < kPack; ++q)
            if (j + q < pad) store1(j + q, v[q]);
        }
      }
      // The next row overwrites srow.
      if constexpr (WARP) __syncwarp();
      else __syncthreads();
    } else {
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int k = (i * G + t) * V;
        if (k < cols) {
#pragma unroll
          for (int j = 0; j < V; ++j) u[i * V + j] = value(u[i * V + j]);
          if constexpr (!VEC) {
            store1(k, u[i]);
          } else if constexpr (!Q8) {
            *reinterpret_cast<uint4*>(y + k) = pack16<DT>(u + i * V);
          } else {
            const float* f = u + i * V;
            const uint32_t lo = e4m3_pack2(f[0], f[1]) | (e4m3_pack2(f[2], f[3]) << 16);
            if constexpr (V == 8) {
              const uint32_t hi = e4m3_pack2(f[4], f[5]) | (e4m3_pack2(f[6], f[7]) << 16);
              *reinterpret_cast<uint2*>(y + k) = make_uint2(lo, hi);
            } else {
              *reinterpret_cast<uint32_t*>(y + k) = lo;
            }
          }
        }
      }
      for (int j = n + t; j < pad; j += G) y[j] = 0;
    }
  }
}

template <int DT, bool Q8, bool GATHER, bool VEC, int E, bool WARP, int MAXT>
cudaError_t launch_rows_variant(const RowParams& p, int y_vec, int sm_count, cudaStream_t stream) {
  auto kern = rows_kernel<DT, Q8, GATHER, VEC, E, WARP, MAXT>;
  const int cols4 = static_cast<int>((p.cols + 3) & ~int64_t{3});
  const int warps = WARP ? 4 : static_cast<int>((p.cols + 32 * E - 1) / (32 * E));
  const int groups = WARP ? 4 : 1;
  const int npos = static_cast<int>((p.pad + 3) & ~int64_t{3});
  int smem = 512;
  if (GATHER) smem += groups * cols4 * 4 + npos * 2 + (Q8 ? (cols4 + 31) / 32 * 4 : 0);
  if (smem > 232448) return cudaErrorInvalidValue;
  cudaError_t e = cudaSuccess;
  if (smem > 48 * 1024) {
    e = ensure_smem_attr(reinterpret_cast<const void*>(kern), 232448);
    if (e != cudaSuccess) return e;
  }
  // As many CTAs as the SMs can hold by threads and shared memory; each takes
  // rows in steps of the grid, so the list is loaded once per CTA.
  const int64_t per_sm = std::max(1, std::min(2048 / (warps * 32), 232448 / (smem + 1024)));
  const int64_t grid = std::min<int64_t>((p.rows + groups - 1) / groups, per_sm * sm_count);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(warps * 32));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, y_vec);
}

template <int DT, bool Q8, bool GATHER, bool VEC>
cudaError_t launch_rows_fast(const RowParams& p, int y_vec, int sm_count, cudaStream_t stream) {
  if (p.cols <= 256) return launch_rows_variant<DT, Q8, GATHER, VEC, 8, true, 128>(p, y_vec, sm_count, stream);
  if (p.cols <= 1024) return launch_rows_variant<DT, Q8, GATHER, VEC, 32, true, 128>(p, y_vec, sm_count, stream);
  if (p.cols <= 8192) return launch_rows_variant<DT, Q8, GATHER, VEC, 16, false, 512>(p, y_vec, sm_count, stream);
  return launch_rows_variant<DT, Q8, GATHER, VEC, 32, false, 1024>(p, y_vec, sm_count, stream);
}

// The rows_kernel for these operands, or cudaErrorNotSupported where only
// rows_any_kernel takes them: longer rows, lists longer than the row.
template <int DT, bool Q8>
cudaError_t launch_rows_held(const RowParams& p, int sm_count, cudaStream_t stream) {
  if (p.cols < 1 || p.cols > kRowsMaxCols || p.n > p.cols || p.pad > p.cols + 128) return cudaErrorNotSupported;
  constexpr int eb = DT == GW_DTYPE_F32 ? 4 : 2;
  constexpr int V = 16 / eb;
  const int ob = Q8 ? 1 : eb;                      // bytes of an output
  auto aligned = [&](const void* q, int64_t ld, int bytes, int elem) {
    return !q || ((reinterpret_cast<uintptr_t>(q) % bytes) == 0 && (p.rows <= 1 || (ld * elem) % bytes == 0));
  };
  const bool gather = p.idx != nullptr || p.n == 0;
  bool vec = p.cols % V == 0 && aligned(p.x, p.ldx, 16, eb) && aligned(p.r, p.ldr, 16, eb) &&
             aligned(p.s, p.lds, 16, eb) && aligned(p.g, 0, 16, eb);
  if (!gather) vec = vec && aligned(p.y, p.ldy, V * ob, ob);
  const int y_vec = aligned(p.y, p.ldy, 4, ob) ? 1 : 0;
  if (gather)
    return vec ? launch_rows_fast<DT, Q8, true, true>(p, y_vec, sm_count, stream)
               : launch_rows_fast<DT, Q8, true, false>(p, y_vec, sm_count, stream);
  return vec ? launch_rows_fast<DT, Q8, false, true>(p, y_vec, sm_count, stream)
             : launch_rows_fast<DT, Q8, false, false>(p, y_vec, sm_count, stream);
}

template <int DT, bool Q8, bool NORM>
cudaError_t launch_rows_dt1(const RowParams& p, int sm_count, cudaStream_t stream) {
  const cudaError_t e = launch_rows_held<DT, Q8>(p, sm_count, stream);
  if (e != cudaErrorNotSupported) return e;
  const int64_t width = std::max<int64_t>(p.cols, p.pad);
  const int threads = width <= 1024 ? 128 : width <= 8192 ? 256 : 1024;
  const int64_t grid = std::min<int64_t>(p.rows, static_cast<int64_t>(sm_count) * (2048 / threads));
  return launch_pdl(rows_any_kernel<DT, Q8, NORM>, dim3(static_cast<unsigned>(grid)), dim3(threads),
                    stream, p);
}

template <bool Q8, bool NORM>
cudaError_t launch_rows_dt(const RowParams& p, int dtype, int sm_count, cudaStream_t stream) {
  switch (dtype) {
    case GW_DTYPE_F16: return launch_rows_dt1<GW_DTYPE_F16, Q8, NORM>(p, sm_count, stream);
    case GW_DTYPE_BF16: return launch_rows_dt1<GW_DTYPE_BF16, Q8, NORM>(p, sm_count, stream);
    default: return launch_rows_dt1<GW_DTYPE_F32, Q8, NORM>(p, sm_count, stream);
  }
}

}  // namespace

cudaError_t launch_rows(RowParams p, int dtype, bool q8, bool norm, int sm_count,
                        cudaStream_t stream) {
  if (p.rows == 0) return cudaSuccess;
  p.norm = norm ? 1 : 0;
  if (q8) return norm ? launch_rows_dt<true, true>(p, dtype, sm_count, stream)
                      : launch_rows_dt<true, false>(p, dtype, sm_count, stream);
  return launch_rows_dt<false, true>(p, dtype, sm_count, stream);
}

}  // namespace gw
