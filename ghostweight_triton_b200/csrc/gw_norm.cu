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
// factor cancels: y / scale = 448 u / max|u|, rounded to fp32 once (to_scale). With
// 16-bit inputs u is mostly exact in fp32, and quotients that lie exactly between
// two e4m3 values are common; they come out exact and round to even, where
// dividing by a rounded scale would send them either way.
//
// What bounds these kernels is HBM: a row is read and written once. rows_kernel
// keeps a row in registers (E elements per thread, a warp or a CTA per row),
// and passes it through shared memory only to pick alive columns from it;
// rows_any_kernel takes what that one does not. Share of the measured copy
// bandwidth (6453 GB/s) over the bytes of one read and one write: 4096 x 4096
// fp16 with residual, half alive, 19.6 us, 93%; all columns 20.2 us, 103%; 8192 x
// 8192 bf16 with residual to e4m3, 30% alive, 73.8 us, 89%; 1537 x 11008 bf16
// rounded 11.1 us, 71%.
// Rows of odd length run at a third to a half of it (4096 x 4097 bf16 with residual:
// 52 us half alive, 41 us full): their 2-byte accesses make instructions the limit.
// What rows_any_kernel takes (of these, the ones of more than 16384 columns) is read
// again for each pass, at a quarter: 1024 x 20001 bf16 with residual 96 us half
// alive, 108 us full, 120 us half alive to e4m3.
//
// No kernel here lets the next one of the stream start before it has finished
// (griddepcontrol.launch_dependents): the products request W' before they wait for
// the previous kernel, and W' may be what gw_quantize_rows has just written.
#include <algorithm>
#include <type_traits>

#include "gw_common.cuh"
#include "gw_internal.h"

namespace gw {

namespace {

constexpr float kE4m3Max = 448.0f;                 // largest finite e4m3 value
constexpr float kScaleMin = 0x1p-126f;             // a row of zeros divides by it

// Two values rounded to e4m3 (nearest even, saturating, NaN kept): lo in bits 0-7.
__device__ __forceinline__ uint32_t e4m3_pack2(float lo, float hi) {
  uint16_t v;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(v) : "f"(hi), "f"(lo));
  return v;
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The scale of a row whose largest |u| is umax and whose norm factor is rstd,
// and what turns u into y / scale = 448 u / umax = (0.875 u) / d, d = umax / 512:
// d and its reciprocal r (the hardware's approximation after one Newton step),
// of umax and u multiplied by m2, a power of two that keeps both in range. Where
// the scale is at its floor (2^-126), y / scale is u rstd 2^126 instead.
struct RowScale {
  float scale, d, r, m2;
  bool floor, odd;                                 // odd: at the floor, or m2 is not one
};
__device__ __forceinline__ RowScale row_scale(uint32_t umax_bits, float rstd) {
  const float umax = __uint_as_float(umax_bits);
  RowScale q;
  q.scale = umax * rstd * (1.0f / kE4m3Max);       // NaN compares false and stays
  q.m2 = umax < 0x1p-64f ? 0x1p64f : umax > 0x1p64f ? 0x1p-64f : 1.0f;
  q.d = umax * q.m2 * (1.0f / 512.0f);
  asm("rcp.approx.f32 %0, %1;" : "=f"(q.r) : "f"(q.d));
  q.r = fmaf(q.r, fmaf(-q.d, q.r, 1.0f), q.r);
  q.floor = q.scale < kScaleMin;
  if (q.floor) {
    q.scale = kScaleMin;
    q.r = rstd;
  }
  q.odd = q.floor || q.m2 != 1.0f;
  return q;
}
// The quotient rounded to nearest, by the remainder of a first estimate (Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor",
// 1990): v0 = h r with h = 0.875 u, v = v0 + (h - v0 d) r, where the remainder is
// exact in one fused operation. EXACT: 0.875 u needs no more than fp32's bits (16-bit
// values as they are); else its low part joins the remainder.
template <bool EXACT>
__device__ __forceinline__ float2 to_scale2(float2 u, const RowScale& q) {
  if (q.odd) {
    if (q.floor) return mul2(mul2(u, both(q.r)), both(0x1p126f));
    u = mul2(u, both(q.m2));
  }
  const float2 nh = mul2(u, both(-0.875f));                        // -h
  const float2 v0 = mul2(nh, both(-q.r));
  float2 t = fma2(v0, both(q.d), nh);                              // -(h - v0 d)
  if constexpr (!EXACT) t = fma2(fma2(u, both(0.875f), nh), both(-1.0f), t);
  return fma2(t, both(-q.r), v0);
}
template <bool EXACT>
__device__ __forceinline__ float to_scale(float u, const RowScale& q) {
  return to_scale2<EXACT>(make_float2(u, 0.0f), q).x;
}
// max(a, |b|), NaN if either is (its bits then lie above infinity's).
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
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
      return NORM && g ? v * Elem<DT>::to_f(g[c]) : v;
    };
    RowScale q8{};
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
      if constexpr (Q8) y[j] = static_cast<out>(e4m3_pack2(j < p.n ? to_scale<false>(v, q8) : 0.0f, 0.0f));
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
// Rows read and written once.
// ---------------------------------------------------------------------------
// A group of G threads (a warp for up to 1024 columns, else the CTA) works on a
// row. One thread copies whole rows of x and r into a ring of stages in shared
// memory (bulk copies counted on an mbarrier), up to kMaxStages rows ahead, so
// that loads are in flight while a row is reduced and written. Loading a row
// when its turn came left HBM idle during the reduction and the output: 34 us
// instead of 27 for 4096 x 4096 fp16 with residual, half of the columns alive.
//   kVec   rows of 16-byte vectors: thread t takes vectors i G + t of the stage;
//   kAny   rows of any alignment: the 16-byte granules that hold the row are
//          copied, thread t takes elements i G + t. Granules that reach past the
//          matrix (its first and last row) are not copied; those rows are read
//          from memory.
//   kLong  rows of vectors too long for the registers: both passes read the stage.
// In kVec and kAny each thread holds its E elements of u = s g in registers.
// GATHER passes them through shared memory as fp32 and picks the alive columns
// there, through a table of 16-bit places that a CTA makes from the list once for
// all its rows (kept in registers instead, the places and the weight behind them
// took every thread's share of the list to set up: 24 us instead of 11 for
// 8192 x 768 fp16, where a warp has three rows). For the e4m3 scale a thread
// knows which of its columns the list names (one bit each), so the sum of squares
// and the largest |u| take one reduction.
constexpr int kRowsHeldCols = 16384;               // 1024 threads x 16
constexpr int kRowsMaxCols = 65535;                // 16-bit positions
constexpr int kMaxStages = 4;
constexpr uint32_t kNoColumn = 0xFFFFu;            // zero output (bad index or padding)
// The two 16-bit values of a word as floats.
template <int DT>
__device__ __forceinline__ float lo_f(uint32_t w) {
  if constexpr (DT == GW_DTYPE_F16) return __low2float(*reinterpret_cast<const __half2*>(&w));
  return __uint_as_float(w << 16);
}
template <int DT>
__device__ __forceinline__ float hi_f(uint32_t w) {
  if constexpr (DT == GW_DTYPE_F16) return __high2float(*reinterpret_cast<const __half2*>(&w));
  return __uint_as_float(w & 0xFFFF0000u);
}
// Values of type DT kept in registers: two 16-bit ones in each.
template <int DT, int N>
struct Held {
  static constexpr int kWords = DT == GW_DTYPE_F32 ? N : (N + 1) / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  // After clear(); i known at compile time, each once.
  __device__ __forceinline__ void set(int i, typename Elem<DT>::raw v) {
    if constexpr (DT == GW_DTYPE_F32) w[i] = v;
    else w[i / 2] |= static_cast<uint32_t>(v) << (16 * (i & 1));
  }
  __device__ __forceinline__ void set16(int v, const uint4 q) {    // 16 bytes from value 16 / size * v on
    w[4 * v] = q.x;
    w[4 * v + 1] = q.y;
    w[4 * v + 2] = q.z;
    w[4 * v + 3] = q.w;
  }
  __device__ __forceinline__ float2 get2(int i) const {             // values i (even) and i + 1
    if constexpr (DT == GW_DTYPE_F32) return make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1]));
    else return make_float2(lo_f<DT>(w[i / 2]), hi_f<DT>(w[i / 2]));
  }
};
enum RowMode { kVec = 0, kAny = 1, kLong = 2 };

// `bytes` (a multiple of 16, both addresses 16-byte aligned) of this GPU's memory
// into shared memory, counted as transaction bytes on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
      :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
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
      f[2 * i] = lo_f<DT>(w[i]);
      f[2 * i + 1] = hi_f<DT>(w[i]);
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

// Shared memory of a CTA: [2][32] partial sums and maxima (512 bytes), mbarriers
// (groups x kMaxStages), the abort flag, then the ring, the fp32 rows, the list's
// places and (Q8) one byte per column.
struct RowShared {
  int stages = 0;            // rows in flight per group
  int operand_bytes = 0;     // room for one operand of one row
  int stage_bytes = 0;       // x and r of one row
  int ring = 0;              // offsets
  int srow = 0;
  int spos = 0;
  int flags = 0;
  int bytes = 0;
};
constexpr int kRowHead = 512 + 4 * kMaxStages * 8 + 64;

// NORM: residual, norm and weight; else (Q8) the rows as they are.
template <int DT, bool Q8, bool NORM, bool GATHER, int MODE, int E, bool WARP, int MAXT>
__global__ void __launch_bounds__(MAXT) rows_kernel(const RowParams p, const RowShared sh, int y_vec) {
  using raw = typename Elem<DT>::raw;
  using out = typename RowOut<Q8, DT>::raw;
  constexpr bool VEC = MODE != kAny;
  constexpr int V = VEC ? static_cast<int>(16 / sizeof(raw)) : 1;
  constexpr int I = E / V;                                        // vectors (or elements) per thread
  constexpr int kPack = Q8 ? 4 : sizeof(raw) == 2 ? 2 : 1;        // outputs per 4-byte store
  constexpr bool STAGED = GATHER && MODE != kLong;                // u passes through shared memory
  static_assert(NORM || Q8, "plain rows are only rounded");
  // Plain rows of 16-bit vectors: the largest magnitude of two values at a time,
  // on their bits (see the file comment), without turning them into floats.
  constexpr bool kBits16 = !NORM && !GATHER && VEC && sizeof(raw) == 2;
  extern __shared__ __align__(128) uint8_t smem[];
  const int G = WARP ? 32 : static_cast<int>(blockDim.x);
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int group = WARP ? (threadIdx.x >> 5) : 0;
  const int groups = WARP ? (blockDim.x >> 5) : 1;
  const int cols = static_cast<int>(p.cols);
  const int n = static_cast<int>(p.n);
  const int pad = static_cast<int>(p.pad);
  float* red_v = reinterpret_cast<float*>(smem);                  // [2][32]
  uint32_t* red_m = reinterpret_cast<uint32_t*>(smem) + 64;       // [2][32]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + 512 + 4 * kMaxStages * 8);
  uint8_t* ring = smem + sh.ring + group * sh.stages * sh.stage_bytes;
  float* srow = reinterpret_cast<float*>(smem + sh.srow) + group * ((cols + 3) & ~3);
  uint16_t* spos = reinterpret_cast<uint16_t*>(smem + sh.spos);   // srow bytes, or kLong: columns
  uint8_t* flags = smem + sh.flags;                               // Q8 and GATHER: 1 per listed column
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * groups + group;
  const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
  const uint32_t row_bytes = static_cast<uint32_t>(cols * sizeof(raw));
  const uint32_t bar0 = smem_u32(smem + 512) + static_cast<uint32_t>(group * kMaxStages * 8);
  const uint32_t ring_s = smem_u32(ring);

  if (t == 0) {
    for (int s = 0; s < sh.stages; ++s) mbar_init(bar0 + 8u * s, 1);
    if (group == 0) *abort_flag = 0;
    mbar_init_fence();
  }
  __syncthreads();
  // The inputs may come from the previous kernel of the stream.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // kAny: the granules that hold a row, and whether they lie within its matrix.
  auto granules = [&](const void* base, int64_t ld, int64_t row, uintptr_t& lo, uint32_t& bytes) {
    const uintptr_t first = reinterpret_cast<uintptr_t>(base);
    const uintptr_t a = first + static_cast<uintptr_t>(row * ld) * sizeof(raw);
    const uintptr_t last = first + static_cast<uintptr_t>((p.rows - 1) * ld) * sizeof(raw) + row_bytes;
    lo = a & ~static_cast<uintptr_t>(15);
    const uintptr_t hi = (a + row_bytes + 15) & ~static_cast<uintptr_t>(15);
    bytes = static_cast<uint32_t>(hi - lo);
    return lo >= first && hi <= last;
  };
  auto fetch = [&](int64_t row, int s) {           // one thread: x (and r) of the row into stage s
    const uint32_t dst = ring_s + static_cast<uint32_t>(s * sh.stage_bytes);
    const uint32_t bar = bar0 + 8u * s;
    if constexpr (VEC) {
      mbar_arrive_expect_tx(bar, NORM && p.r ? 2 * row_bytes : row_bytes);
      bulk_load(dst, static_cast<const raw*>(p.x) + row * p.ldx, row_bytes, bar);
      if (NORM && p.r) bulk_load(dst + sh.operand_bytes, static_cast<const raw*>(p.r) + row * p.ldr, row_bytes, bar);
    } else {
      uintptr_t xl, rl = 0;
      uint32_t xb, rb = 0;
      if (!granules(p.x, p.ldx, row, xl, xb)) xb = 0;
      if (!NORM || !p.r || !granules(p.r, p.ldr, row, rl, rb)) rb = 0;
      mbar_arrive_expect_tx(bar, xb + rb);
      if (xb) bulk_load(dst, reinterpret_cast<const void*>(xl), xb, bar);
      if (rb) bulk_load(dst + sh.operand_bytes, reinterpret_cast<const void*>(rl), rb, bar);
    }
  };
  if (t == 0)
    for (int s = 0; s < sh.stages && row0 + s * step < p.rows; ++s) fetch(row0 + s * step, s);

  uint32_t named = 0xFFFFFFFFu;                                   // this thread's columns in the list
  bool checked = false;                                           // some output has no column
  const raw* g = NORM ? static_cast<const raw*>(p.g) : nullptr;
  if constexpr (GATHER) {
    if constexpr (Q8) {
      for (int i = threadIdx.x; i < (cols + 3) / 4; i += blockDim.x) reinterpret_cast<uint32_t*>(flags)[i] = 0;
      __syncthreads();
    }
    bool bad = false;
    // Eight entries per thread at a time, all loaded before the first is used.
    const int entries = (pad + 3) & ~3;
    for (int j0 = threadIdx.x; j0 < entries; j0 += 8 * blockDim.x) {
      int64_t c64[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = j0 + i * static_cast<int>(blockDim.x);
        c64[i] = j < n ? __ldg(p.idx + j) : -1;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = j0 + i * static_cast<int>(blockDim.x);
        if (j >= entries) break;
        const uint32_t c = static_cast<uint32_t>(c64[i]);
        uint32_t place = kNoColumn;
        if (static_cast<uint64_t>(c64[i]) < static_cast<uint64_t>(cols)) {
          if constexpr (Q8) flags[c] = 1;
          place = MODE == kLong ? c : 4u * row_pos<DT, VEC>(static_cast<int>(c), cols);
        } else if (j < n) {
          bad = true;
        }
        spos[j] = static_cast<uint16_t>(place);
      }
    }
    if (bad && blockIdx.x == 0) raise_error(p.err, GW_DERR_BAD_INDEX);
    checked = __syncthreads_or(bad ? 1 : 0) != 0;
    if constexpr (Q8 && STAGED) {
      named = 0;
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int k = (i * G + t) * V;
        if (k < cols) {
#pragma unroll
          for (int j = 0; j < V; ++j) named |= static_cast<uint32_t>(flags[k + j]) << (i * V + j);
        }
      }
    }
  }
  Held<DT, MODE == kLong || !NORM ? 1 : E> gain;                  // this thread's share of the weight
  gain.clear();
  if constexpr (NORM && MODE != kLong) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int k = (i * G + t) * V;
      if (g && k < cols) {
        if constexpr (VEC) gain.set16(i, __ldg(reinterpret_cast<const uint4*>(g) + i * G + t));
        else gain.set(i, __ldg(g + k));
      }
    }
  }

  const float inv_cols = 1.0f / static_cast<float>(cols);
  int buf = 0, stage = 0;
  uint32_t phase = 0;
  // The row's place in each output, moved along with the row.
  raw* sum = NORM && p.s ? static_cast<raw*>(p.s) + row0 * p.lds : nullptr;
  out* y = static_cast<out*>(p.y) + row0 * p.ldy;
  const int64_t sum_step = NORM && p.s ? step * p.lds : 0;
  const int64_t y_step = step * p.ldy;
  for (int64_t row = row0; row < p.rows; row += step, sum += sum_step, y += y_step) {
    const uint8_t* xs = ring + stage * sh.stage_bytes;
    const uint8_t* rs = xs + sh.operand_bytes;
    // A wait that runs out raises the device error word and the abort flag; the
    // rest of this CTA's rows are then worked off quickly, with undefined outputs.
    mbar_wait(bar0 + 8u * stage, phase, abort_flag, p.err);
    __align__(16) float u[MODE == kLong ? V : E];
    float2 ss2 = make_float2(0.0f, 0.0f);
    float uabs = 0.0f;
    // Vector v of the row (the thread's i-th): the sum, rounded to `sum` and
    // squared into ss2 when `first`, times the weight.
    auto vector = [&](int v, int i, float* f, bool first) {
      unpack16<DT>(reinterpret_cast<const uint4*>(xs)[v], f);
      if constexpr (NORM) {
        float2* f2 = reinterpret_cast<float2*>(f);
        float q[V];
        if (p.r) {
          unpack16<DT>(reinterpret_cast<const uint4*>(rs)[v], q);
#pragma unroll
          for (int j = 0; j < V / 2; ++j) f2[j] = add2(f2[j], make_float2(q[2 * j], q[2 * j + 1]));
        }
        if (first) {
          if (sum) reinterpret_cast<uint4*>(sum)[v] = pack16<DT>(f);
#pragma unroll
          for (int j = 0; j < V / 2; ++j) ss2 = fma2(f2[j], f2[j], ss2);
        }
        if (g) {
          if constexpr (MODE == kLong) unpack16<DT>(__ldg(reinterpret_cast<const uint4*>(g) + v), q);
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            if constexpr (MODE == kLong) f2[j] = mul2(f2[j], make_float2(q[2 * j], q[2 * j + 1]));
            else f2[j] = mul2(f2[j], gain.get2(i * V + 2 * j));
          }
        }
      }
    };
    // kBits16: the largest bits of |x| so far, two 16-bit values.
    uint32_t largest = 0;
    auto vector_bits = [&](int v) {
      const uint4 q = reinterpret_cast<const uint4*>(xs)[v];
      largest = __vmaxu2(largest, __vmaxu2(__vmaxu2(q.x & 0x7FFF7FFFu, q.y & 0x7FFF7FFFu),
                                           __vmaxu2(q.z & 0x7FFF7FFFu, q.w & 0x7FFF7FFFu)));
    };
    if constexpr (MODE == kVec) {
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int v = i * G + t;
        float* f = u + i * V;
        if (v * V < cols) {
          vector(v, i, f, true);
          if constexpr (kBits16) vector_bits(v);
          if constexpr (STAGED) {
#pragma unroll
            for (int j = 0; j < V; j += 4)
              *reinterpret_cast<float4*>(srow + row_pos<DT, VEC>(v * V + j, cols)) =
                  make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) f[j] = 0.0f;
        }
      }
      if constexpr (Q8 && !kBits16) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!GATHER || ((named >> e) & 1u)) uabs = max_abs(uabs, u[e]);
      }
    } else if constexpr (MODE == kLong) {
#pragma unroll 4
      for (int v = t; v * V < cols; v += G) {
        if constexpr (kBits16) {
          vector_bits(v);
          continue;
        }
        vector(v, 0, u, true);
        if constexpr (Q8) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (!GATHER || flags[v * V + j]) uabs = max_abs(uabs, u[j]);
        }
      }
    } else {
      const raw* x = static_cast<const raw*>(p.x) + row * p.ldx;
      const raw* r = NORM && p.r ? static_cast<const raw*>(p.r) + row * p.ldr : nullptr;
      uintptr_t lo;
      uint32_t bytes;
      const bool in_x = granules(p.x, p.ldx, row, lo, bytes);
      const bool in_r = !r || granules(p.r, p.ldr, row, lo, bytes);
      if (in_x && in_r) {
        const raw* xr = reinterpret_cast<const raw*>(xs + (reinterpret_cast<uintptr_t>(x) & 15u));
        const raw* rr = reinterpret_cast<const raw*>(rs + (reinterpret_cast<uintptr_t>(r) & 15u));
#pragma unroll
        for (int i = 0; i < I; ++i) u[i] = i * G + t < cols ? Elem<DT>::to_f(xr[i * G + t]) : 0.0f;
        if (r) {
#pragma unroll
          for (int i = 0; i < I; ++i)
            if (i * G + t < cols) u[i] += Elem<DT>::to_f(rr[i * G + t]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < I; ++i) {
          const int k = i * G + t;
          u[i] = 0.0f;
          if (k < cols) {
            u[i] = Elem<DT>::to_f(x[k]);
            if (r) u[i] += Elem<DT>::to_f(r[k]);
          }
        }
      }
      if (sum) {
#pragma unroll
        for (int i = 0; i < I; ++i)
          if (i * G + t < cols) sum[i * G + t] = Elem<DT>::from_f(u[i]);
      }
      float2* u2 = reinterpret_cast<float2*>(u);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        if constexpr (NORM) {
          ss2 = fma2(u2[i], u2[i], ss2);
          if (g) u2[i] = mul2(u2[i], gain.get2(2 * i));
        }
      }
#pragma unroll
      for (int i = 0; i < I; ++i) {
        if constexpr (STAGED) {
          if (i * G + t < cols) srow[i * G + t] = u[i];
        }
        if constexpr (Q8) {
          if (!GATHER || ((named >> i) & 1u)) uabs = max_abs(uabs, u[i]);
        }
      }
    }
    float ss = ss2.x + ss2.y;
    uint32_t umax = __float_as_uint(uabs);
    if constexpr (kBits16)
      umax = __float_as_uint(Elem<DT>::to_f(static_cast<raw>(max(largest & 0xFFFFu, largest >> 16))));
    // Sum of squares and largest |u| of the row; publishes srow too.
    if constexpr (NORM) {
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    }
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
    }
    auto refill = [&] {                              // every thread is done with the stage
      const int64_t next = row + sh.stages * step;
      if (t == 0 && next < p.rows && !*abort_flag) fetch(next, stage);
      if (++stage == sh.stages) {
        stage = 0;
        phase ^= 1u;
      }
    };
    if constexpr (MODE != kLong) refill();
    if constexpr (!WARP) {
      const int lane = t & 31;
      const bool in = lane < (G >> 5);
      if constexpr (NORM) {
        ss = in ? red_v[buf * 32 + lane] : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
      }
      if constexpr (Q8) umax = __reduce_max_sync(0xFFFFFFFFu, in ? red_m[buf * 32 + lane] : 0u);
      buf ^= 1;
    }
    const float rstd = NORM ? rsqrtf(ss * inv_cols + p.eps) : 1.0f;
    RowScale q8{};
    if constexpr (Q8) {
      q8 = row_scale(umax, rstd);
      if (t == 0) p.scale[row] = q8.scale;
    }
    constexpr bool kExact = !NORM && sizeof(raw) == 2;
    auto value = [&](float v) { return Q8 ? to_scale<kExact>(v, q8) : v * rstd; };
    auto value2 = [&](float2 v) { return Q8 ? to_scale2<kExact>(v, q8) : mul2(v, both(rstd)); };
    auto store1 = [&](int j, float v) {
      if constexpr (Q8) y[j] = static_cast<out>(e4m3_pack2(v, 0.0f));
      else y[j] = Elem<DT>::from_f(v);
    };
    auto store_pack = [&](int j, const float* v) {   // outputs j .. j + kPack - 1, up to pad
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
    };
    auto store_vector = [&](int k, float* f) {       // outputs k .. k + V - 1 (aligned)
      if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < V; j += 2)
          *reinterpret_cast<float2*>(f + j) = value2(*reinterpret_cast<const float2*>(f + j));
      }
      if constexpr (!VEC) {
        store1(k, value(f[0]));
      } else if constexpr (!Q8) {
        *reinterpret_cast<uint4*>(y + k) = pack16<DT>(f);
      } else {
        const uint32_t lo = e4m3_pack2(f[0], f[1]) | (e4m3_pack2(f[2], f[3]) << 16);
        if constexpr (V == 8) {
          const uint32_t hi = e4m3_pack2(f[4], f[5]) | (e4m3_pack2(f[6], f[7]) << 16);
          *reinterpret_cast<uint2*>(y + k) = make_uint2(lo, hi);
        } else {
          *reinterpret_cast<uint32_t*>(y + k) = lo;
        }
      }
    };
    if constexpr (STAGED) {
      // Neighbouring threads take neighbouring groups of outputs: 4-byte
      // stores, and shared-memory reads within a narrow window of the row.
      const uint8_t* sr = reinterpret_cast<const uint8_t*>(srow);
      auto read = [&](int j, uint32_t* c) {          // the places of outputs j .. j + kPack - 1
        if constexpr (kPack == 4) {
          const uint2 q = *reinterpret_cast<const uint2*>(spos + j);
          c[0] = q.x & 0xFFFFu; c[1] = q.x >> 16; c[2] = q.y & 0xFFFFu; c[3] = q.y >> 16;
        } else if constexpr (kPack == 2) {
          const uint32_t q = *reinterpret_cast<const uint32_t*>(spos + j);
          c[0] = q & 0xFFFFu; c[1] = q >> 16;
        } else {
          c[0] = spos[j];
        }
      };
      int j = t * kPack;
      if (y_vec && !checked) {
        // Every output of these groups has a column: no checks.
        const int whole = n / kPack * kPack;
        uint32_t* yw = reinterpret_cast<uint32_t*>(y + j);
#pragma unroll 4
        for (; j < whole; j += G * kPack, yw += G) {
          uint32_t c[kPack];
          __align__(16) float v[kPack];
          read(j, c);
#pragma unroll
          for (int e = 0; e < kPack; ++e) v[e] = *reinterpret_cast<const float*>(sr + c[e]);
          if constexpr (kPack == 1) {
            *yw = __float_as_uint(value(v[0]));
          } else {
            const float2 a = value2(make_float2(v[0], v[1]));
            if constexpr (!Q8) {
              *yw = Elem<DT>::pack2(a.x, a.y);
            } else {
              const float2 b = value2(make_float2(v[2], v[3]));
              *yw = e4m3_pack2(a.x, a.y) | (e4m3_pack2(b.x, b.y) << 16);
            }
          }
        }
      }
      for (; j < pad; j += G * kPack) {
        uint32_t c[kPack];
        __align__(16) float v[kPack];
        read(j, c);
#pragma unroll
        for (int e = 0; e < kPack; ++e)
          v[e] = c[e] == kNoColumn ? 0.0f : value(*reinterpret_cast<const float*>(sr + c[e]));
        store_pack(j, v);
      }
      // The next row overwrites srow.
      if constexpr (WARP) __syncwarp();
      else __syncthreads();
    } else if constexpr (MODE == kLong && GATHER) {
      const raw* x = reinterpret_cast<const raw*>(xs);
      const raw* r = reinterpret_cast<const raw*>(rs);
      for (int j = t * kPack; j < pad; j += G * kPack) {
        float v[kPack];
#pragma unroll
        for (int e = 0; e < kPack; ++e) {
          const uint32_t c = spos[j + e];
          v[e] = 0.0f;
          if (c != kNoColumn) {
            float f = Elem<DT>::to_f(x[c]);
            if (NORM && p.r) f += Elem<DT>::to_f(r[c]);
            if (g) f *= Elem<DT>::to_f(__ldg(g + c));
            v[e] = value(f);
          }
        }
        store_pack(j, v);
      }
      __syncthreads();
      refill();
    } else {
      if constexpr (MODE == kLong) {
#pragma unroll 2
        for (int v = t; v * V < cols; v += G) {
          __align__(16) float f[V];
          vector(v, 0, f, false);
          store_vector(v * V, f);
        }
      } else {
#pragma unroll
        for (int i = 0; i < I; ++i)
          if ((i * G + t) * V < cols) store_vector((i * G + t) * V, u + i * V);
      }
      for (int j = n + t; j < pad; j += G) y[j] = 0;
      if constexpr (MODE == kLong) {
        __syncthreads();
        refill();
      }
    }
  }
  // After a wait that ran out, copies may still be on their way into this CTA's
  // shared memory: wait (bounded) for either phase of every stage once more.
  if (t == 0 && *abort_flag)
    for (int s = 0; s < sh.stages; ++s) {
      mbar_wait(bar0 + 8u * s, 0u, nullptr, p.err, 100000000ull);
      mbar_wait(bar0 + 8u * s, 1u, nullptr, p.err, 100000000ull);
    }
}

template <int DT, bool Q8, bool NORM, bool GATHER, int MODE, int E, bool WARP, int MAXT>
cudaError_t launch_rows_variant(const RowParams& p, int y_vec, int sm_count, cudaStream_t stream) {
  auto kern = rows_kernel<DT, Q8, NORM, GATHER, MODE, E, WARP, MAXT>;
  constexpr int kSmemLimit = 232448;
  const int cols = static_cast<int>(p.cols);
  const int cols4 = (cols + 3) & ~3;
  const int groups = WARP ? 4 : 1;
  const int warps = WARP ? groups : MODE == kLong ? (cols <= kRowsHeldCols ? 16 : 32)
                                                  : std::min(32, (cols + 32 * E - 1) / (32 * E));
  const int threads = warps * 32;
  const int npos = GATHER ? static_cast<int>((p.pad + 3) & ~int64_t{3}) : 0;
  const bool staged = GATHER && MODE != kLong;
  RowShared sh;
  const int fixed = kRowHead + (staged ? groups * cols4 * 4 : 0) + npos * 2 +
                    (GATHER && Q8 ? cols4 : 0);
  sh.operand_bytes = (cols * (DT == GW_DTYPE_F32 ? 4 : 2) + 15) / 16 * 16 + (MODE == kAny ? 16 : 0);
  sh.stage_bytes = sh.operand_bytes * (p.r ? 2 : 1);
  // As many CTAs as make 1024 threads per SM, each with up to four rows in
  // flight; fewer CTAs where two rows each would not fit.
  int per_sm = std::max(1, (MODE == kLong ? 2048 : 1024) / threads);
  for (;; per_sm = (per_sm + 1) / 2) {
    sh.stages = ((kSmemLimit + 1024) / per_sm - 1024 - fixed) / (groups * sh.stage_bytes);
    if (sh.stages >= (MODE == kLong && per_sm == 2 ? 1 : 2) || per_sm == 1) break;
  }
  if (sh.stages < 1) return cudaErrorNotSupported;
  sh.stages = std::min(sh.stages, kMaxStages);
  sh.ring = kRowHead;
  sh.srow = sh.ring + groups * sh.stages * sh.stage_bytes;
  sh.spos = sh.srow + (staged ? groups * cols4 * 4 : 0);
  sh.flags = sh.spos + npos * 2;
  sh.bytes = fixed + groups * sh.stages * sh.stage_bytes;
  cudaError_t e = cudaSuccess;
  if (sh.bytes > 48 * 1024) {
    e = ensure_smem_attr(reinterpret_cast<const void*>(kern), kSmemLimit);
    if (e != cudaSuccess) return e;
  }
  // Each CTA takes rows in steps of the grid, so the list is loaded once per CTA.
  const int64_t grid = std::min<int64_t>((p.rows + groups - 1) / groups, static_cast<int64_t>(per_sm) * sm_count);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(sh.bytes);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, sh, y_vec);
}

template <int DT, bool Q8, bool NORM, bool GATHER>
cudaError_t launch_rows_held(const RowParams& p, bool vec, int y_vec, int sm_count, cudaStream_t stream) {
  if (vec) {
    if (p.cols <= 256) return launch_rows_variant<DT, Q8, NORM, GATHER, kVec, 8, true, 128>(p, y_vec, sm_count, stream);
    if (p.cols <= 1024) return launch_rows_variant<DT, Q8, NORM, GATHER, kVec, 32, true, 128>(p, y_vec, sm_count, stream);
    cudaError_t e = cudaErrorNotSupported;
    if (p.cols <= kRowsHeldCols && (GATHER || p.cols <= 4096))
      e = launch_rows_variant<DT, Q8, NORM, GATHER, kVec, 16, false, 1024>(p, y_vec, sm_count, stream);
    if (e != cudaErrorNotSupported) return e;
    return launch_rows_variant<DT, Q8, NORM, GATHER, kLong, 16, false, 1024>(p, y_vec, sm_count, stream);
  }
  if (p.cols <= 256) return launch_rows_variant<DT, Q8, NORM, GATHER, kAny, 8, true, 128>(p, y_vec, sm_count, stream);
  if (p.cols <= 4096) return launch_rows_variant<DT, Q8, NORM, GATHER, kAny, 16, false, 256>(p, y_vec, sm_count, stream);
  if (p.cols <= kRowsHeldCols)
    return launch_rows_variant<DT, Q8, NORM, GATHER, kAny, 16, false, 1024>(p, y_vec, sm_count, stream);
  return cudaErrorNotSupported;
}

// The rows_kernel for these operands, or cudaErrorNotSupported where only
// rows_any_kernel takes them: rows too long for a stage (or too long and not
// aligned), lists longer than the row.
template <int DT, bool Q8, bool NORM>
cudaError_t launch_rows_once(const RowParams& p, int sm_count, cudaStream_t stream) {
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
  return gather ? launch_rows_held<DT, Q8, NORM, true>(p, vec, y_vec, sm_count, stream)
                : launch_rows_held<DT, Q8, NORM, false>(p, vec, y_vec, sm_count, stream);
}

template <int DT, bool Q8, bool NORM>
cudaError_t launch_rows_dt1(const RowParams& p, int sm_count, cudaStream_t stream) {
  const cudaError_t e = launch_rows_once<DT, Q8, NORM>(p, sm_count, stream);
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

cudaError_t launch_rows(const RowParams& p, int dtype, bool q8, bool norm, int sm_count,
                        cudaStream_t stream) {
  if (p.rows == 0) return cudaSuccess;
  if (q8) return norm ? launch_rows_dt<true, true>(p, dtype, sm_count, stream)
                      : launch_rows_dt<true, false>(p, dtype, sm_count, stream);
  return launch_rows_dt<false, true>(p, dtype, sm_count, stream);
}

}  // namespace gw
