// K3-fp32: exact single-precision gather-GEMM on the FP32 pipes (no TF32).
//
// The reference runs fp32 inputs through tl.dot with allow_tf32=False
// (ghostweight_triton/kernels/matmul.py:127-130) so results hold a 1e-4
// tolerance; tcgen05 has no exact-fp32 kind, so fp32 uses FFMA:
//   y[m, n] = act( sum_j x[m, idx[j]] * w[n, j] + bias[n] ) + residual[m, n]
// Every output is one chain of fused multiply-adds over j in ascending order,
// whatever the tile, so its bits do not depend on the tile chosen.
//
// What bounds it is the FP32 pipe for tall outputs (74 TFLOP/s at 148 x 128
// lanes and 1.96 GHz) and the latency of the k loop for small ones. Tiles of
// BM x BN outputs, BK columns per stage; both operands arrive by cp.async, the
// alive columns of x as single elements through the list (loaded a stage
// ahead), W' as 16-byte vectors, S - 1 stages ahead of the arithmetic. Shared
// rows hold BK + 4 floats: a thread reads four columns of a row as one vector,
// and eight neighbouring rows cover all 32 banks.
// Tiles of 64 x 64 outputs where they make four CTAs per SM, 32 x 64 below (their
// finer grain evens out the SMs' shares), 16 x 32 for at most 16 rows.
#include <algorithm>

#include "gw_common.cuh"
#include "gw_internal.h"

namespace gw {

namespace {

__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src, bool valid) {
  const uint32_t bytes = valid ? 4u : 0u;          // 0: the destination becomes zero
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" :: "r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const float* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory");
}

struct SimtParams {
  const float* x;
  int64_t M;
  int64_t K;
  int64_t ldx;
  const float* w;
  int64_t N;
  int64_t ldw;
  const int64_t* idx;
  int64_t n_alive;
  const float* bias;
  int epi;
  float* y;
  int64_t ldy;
  unsigned int* err;
  const int32_t* n_dev;      // the alive count on the device (n_alive is then an upper bound)
  const float* res;          // residual (or null), leading dimension ldr
  int64_t ldr;
  int w_vec;                 // W' rows may be read as 16-byte vectors
};

constexpr int64_t kGridRows = 32768;               // row tiles in grid.y

template <int BM, int BN, int BK, int TM, int TN, int S>
struct SimtCfg {
  static constexpr int kThreads = (BM / TM) * (BN / TN);
  static constexpr int kRow = BK + 4;                              // floats per shared row
  static constexpr int kStageFloats = (BM + BN) * kRow;
  static constexpr int kSmemBytes = S * kStageFloats * 4;
  static constexpr int kARows = kThreads / BK;                     // rows of x per pass of the threads
  static constexpr int kAPer = BM / kARows;                        // elements of x per thread and stage
  static constexpr int kBVecs = BN * (BK / 4);                     // vectors of W' per stage
  static constexpr int kBPer = (kBVecs + kThreads - 1) / kThreads;
  static_assert(kThreads % BK == 0 && BM % kARows == 0, "whole passes over the tile of x");
};

template <int BM, int BN, int BK, int TM, int TN, int S>
__global__ void __launch_bounds__((BM / TM) * (BN / TN))
gemm_f32_kernel(const SimtParams p) {
  using C = SimtCfg<BM, BN, BK, TM, TN, S>;
  extern __shared__ __align__(16) float smem_f[];
  const uint32_t smem_s = smem_u32(smem_f);
  int64_t n_alive = p.n_alive;
  if (p.n_dev) n_alive = min(n_alive, static_cast<int64_t>(max(*p.n_dev, 0)));
  const int tid = threadIdx.x;
  // Row tiles in two grid dimensions: one ends at 65535. (All tiles in grid.x costs
  // a division per CTA: 28.3 us instead of 25.9 for 1024 x 768 x 384.)
  const int64_t m0 = (static_cast<int64_t>(blockIdx.z) * kGridRows + blockIdx.y) * BM;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * BN;
  if (m0 >= p.M) return;                           // the last of grid.z, a whole CTA
  // A warp is 4 x 8 threads, eight neighbouring lanes 2 x 4 of them: a vector load
  // takes four rows of W' (two of x) for each eight lanes. 3 to 5% faster than
  // eight lanes along a row.
  const int lane = tid & 31;
  constexpr int kWarpsN = BN / (8 * TN);
  const int row_t = (tid >> 5) / kWarpsN * (4 * TM) + (((lane >> 4) << 1) | (lane & 1));   // rows row_t + 4 i
  const int col_t = (tid >> 5) % kWarpsN * (8 * TN) + ((lane >> 1) & 7);                  // columns col_t + 8 j
  const int lk = tid % BK;                           // this thread's column of x tiles
  const int lr = tid / BK;
  const int nk = static_cast<int>((n_alive + BK - 1) / BK);
  bool bad = false;

  auto column = [&](int kt) {                        // the alive column this thread loads in step kt
    const int64_t j = static_cast<int64_t>(kt) * BK + lk;
    if (j >= n_alive) return int64_t{-1};
    const int64_t c = __ldg(p.idx + j);
    if (c >= 0 && c < p.K) return c;
    bad = true;
    return int64_t{-1};
  };
  // This thread's rows of x and vectors of W', and where they go in a stage.
  const float* x_row[C::kAPer];
#pragma unroll
  for (int i = 0; i < C::kAPer; ++i) {
    const int64_t m = m0 + lr + i * C::kARows;
    x_row[i] = m < p.M ? p.x + m * p.ldx : nullptr;
  }
  const uint32_t a_dst = static_cast<uint32_t>((lr * C::kRow + lk) * 4);
  const float* w_vec[C::kBPer];
#pragma unroll
  for (int i = 0; i < C::kBPer; ++i) {
    const int v = tid + i * C::kThreads;
    const int64_t n = n0 + v / (BK / 4);
    w_vec[i] = v < C::kBVecs && n < p.N ? p.w + n * p.ldw + (v % (BK / 4)) * 4 : nullptr;
  }
  const uint32_t b_dst = static_cast<uint32_t>((BM * C::kRow + tid / (BK / 4) * C::kRow + (tid % (BK / 4)) * 4) * 4);
  static_assert(C::kThreads % (BK / 4) == 0, "a thread's vectors of W' share one column");
  const int n_cols = static_cast<int>(n_alive);
  auto load = [&](int kt, int stage, int64_t col) {  // both tiles of k step kt
    const uint32_t st = smem_s + static_cast<uint32_t>(stage * C::kStageFloats * 4);
#pragma unroll
    for (int i = 0; i < C::kAPer; ++i) {
      const bool ok = col >= 0 && x_row[i] != nullptr;
      cp_async4(st + a_dst + i * C::kARows * C::kRow * 4, ok ? x_row[i] + col : p.x, ok);
    }
    if (p.w_vec) {
      const int left = n_cols - (kt * BK + (tid % (BK / 4)) * 4);
      const uint32_t want = left >= 4 ? 16u : left > 0 ? static_cast<uint32_t>(left) * 4u : 0u;
#pragma unroll
      for (int i = 0; i < C::kBPer; ++i) {
        if (C::kBVecs % C::kThreads == 0 || tid + i * C::kThreads < C::kBVecs) {
          const uint32_t bytes = w_vec[i] ? want : 0u;
          cp_async16(st + b_dst + i * (C::kThreads / (BK / 4)) * C::kRow * 4, bytes ? w_vec[i] + kt * BK : p.w, bytes);
        }
      }
    } else {
      for (int e = tid; e < BN * BK; e += C::kThreads) {
        const int r = e / BK;
        const int64_t k = static_cast<int64_t>(kt) * BK + e % BK;
        const bool ok = n0 + r < p.N && k < n_alive;
        cp_async4(st + static_cast<uint32_t>((BM * C::kRow + r * C::kRow + e % BK) * 4),
                  ok ? p.w + (n0 + r) * p.ldw + k : p.w, ok);
      }
    }
  };

  float acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = 0.0f;

  // One commit per stage, empty at the end, so that the count of groups in
  // flight says which stage has landed. The list is read four stages ahead of
  // the loads that need it: an entry on its way from L2 held up every stage of
  // a small tile otherwise.
  constexpr int kAhead = 4;
  int64_t cols[S - 1 + kAhead];
#pragma unroll
  for (int s = 0; s < S - 1 + kAhead; ++s) cols[s] = s < nk ? column(s) : -1;
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
    if (s < nk) load(s, s, cols[s]);
    cp_async_commit();
  }
  int64_t next[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) next[i] = cols[S - 1 + i];
  int stage = 0, free_stage = S - 1;                 // of step kt, and of step kt + S - 1
  for (int kt = 0; kt < nk; ++kt) {
    cp_async_wait<S - 2>();
    __syncthreads();                                 // stage kt landed; stage kt - 1 is free
    if (kt + S - 1 < nk) load(kt + S - 1, free_stage, next[0]);
    free_stage = stage;
    cp_async_commit();
#pragma unroll
    for (int i = 0; i + 1 < kAhead; ++i) next[i] = next[i + 1];
    next[kAhead - 1] = kt + S - 1 + kAhead < nk ? column(kt + S - 1 + kAhead) : -1;
    const float* a_t = smem_f + stage * C::kStageFloats;
    if (++stage == S) stage = 0;
    const float* b_t = a_t + BM * C::kRow;
#pragma unroll
    for (int k = 0; k < BK; k += 4) {
      float4 b[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
        b[j] = *reinterpret_cast<const float4*>(b_t + (col_t + 8 * j) * C::kRow + k);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const float4 a = *reinterpret_cast<const float4*>(a_t + (row_t + 4 * i) * C::kRow + k);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          float v = fmaf(a.x, b[j].x, acc[i][j]);
          v = fmaf(a.y, b[j].y, v);
          v = fmaf(a.z, b[j].z, v);
          acc[i][j] = fmaf(a.w, b[j].w, v);
        }
      }
    }
  }
  cp_async_wait<0>();
  if (bad) raise_error(p.err, GW_DERR_BAD_INDEX);

  auto store = [&](const float (*r)[TN]) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t m = m0 + row_t + 4 * i;
      if (m >= p.M) continue;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int64_t n = n0 + col_t + 8 * j;
        if (n >= p.N) continue;
        float v = acc[i][j];
        if (p.bias) v += __ldg(p.bias + n);
        v = apply_epilogue(v, p.epi);
        if (r) v += r[i][j];
        p.y[m * p.ldy + n] = v;
      }
    }
  };
  if (p.res) {
    // All of the residual before the first store: y may be the residual, so a
    // load behind a store would wait for it.
    float r[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t m = m0 + row_t + 4 * i;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int64_t n = n0 + col_t + 8 * j;
        r[i][j] = m < p.M && n < p.N ? p.res[m * p.ldr + n] : 0.0f;
      }
    }
    store(r);
  } else {
    store(nullptr);
  }
}

template <int BM, int BN, int BK, int TM, int TN, int S>
cudaError_t launch_simt(const SimtParams& p, cudaStream_t stream) {
  using C = SimtCfg<BM, BN, BK, TM, TN, S>;
  const int64_t gx = (p.N + BN - 1) / BN;
  const int64_t gy = (p.M + BM - 1) / BM;
  const int64_t gz = (gy + kGridRows - 1) / kGridRows;
  if (gx > 0x7FFFFFFFll || gz > 65535) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(std::min(gy, kGridRows)),
                  static_cast<unsigned>(gz));
  auto kern = gemm_f32_kernel<BM, BN, BK, TM, TN, S>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), C::kSmemBytes);
  if (e != cudaSuccess) return e;
  kern<<<grid, C::kThreads, C::kSmemBytes, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gemm_f32(const float* x, int64_t M, int64_t K, int64_t ldx, const float* w,
                            int64_t N, int64_t ldw, const int64_t* idx, int64_t n_alive,
                            const float* bias, int epilogue, float* y, int64_t ldy,
                            unsigned int* err, cudaStream_t stream, const int32_t* n_dev,
                            const Residual& res) {
  if (M == 0 || N == 0) return cudaSuccess;
  SimtParams p{};
  p.x = x;
  p.M = M;
  p.K = K;
  p.ldx = ldx;
  p.w = w;
  p.N = N;
  p.ldw = ldw;
  p.idx = idx;
  p.n_alive = n_alive;
  p.bias = bias;
  p.epi = epilogue;
  p.y = y;
  p.ldy = ldy;
  p.err = err;
  p.n_dev = n_dev;
  p.res = static_cast<const float*>(res.p);
  p.ldr = res.ld;
  p.w_vec = ((reinterpret_cast<uintptr_t>(w) & 15u) == 0 && (N <= 1 || ldw % 4 == 0)) ? 1 : 0;
  // Measured (us) for M x N x K' = 1024 x 768 x 384, 100 x 4096 x 2048 and 4096 x
  // 4096 x 2048: 64 x 64 tiles 32, 116 and 1745; 32 x 64 tiles 26, 81 and 1904
  // (with 32 columns a stage 27, 98 and 2234); 128 x 128 tiles 92, 408 and 2000
  // (one CTA per SM holds their registers). 16 x 4096 x 2048: 16 x 32 tiles with 64
  // columns a stage 42, with 32 columns 62; 32 x 32 tiles 71.
  auto ctas = [&](int64_t bm, int64_t bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  constexpr int64_t kSms = 148;
  if (M <= 16) return launch_simt<16, 32, 64, 2, 2, 4>(p, stream);
  if (ctas(64, 64) < 4 * kSms) return launch_simt<32, 64, 64, 4, 4, 2>(p, stream);
  return launch_simt<64, 64, 32, 8, 4, 3>(p, stream);
}

}  // namespace gw
