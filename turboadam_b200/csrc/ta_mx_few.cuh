// ta_mx_few.cuh -- products with few rows of A (single tokens): bound by the bytes of B, which is
// read once.
//
// A tile of the product engine has 256 rows; with one token its matrix instructions would work
// on zeros, and its copies, one stage at a time and CTA pair, reach some 3.4 TB/s (35 us
// at 4096 > 14336, bf16, for 8 tokens). Here every lane has several 16-byte loads of B under
// way, which is what HBM asks for: 20.5 us for one token (5.7 TB/s), 22 us for two, 35.5 us for
// four, where a lane's arithmetic takes over (4096 > 4096: 8.4, 9.4 and 12.3 us, the tiles 23);
// beyond, the tiles are faster. Two forms, by which dimension of B is contiguous:
//   k_few_rows: the sum's (an output by input weight): a warp takes four rows of B;
//   k_few_cols: the result's: a lane takes eight columns, the sum is split over the warps of a
//               block and over blocks, and k_few_finish adds the blocks' parts in order (4096 >
//               14336: 25 us for one token, 26.5 for two, 43.5 for four).
#pragma once

#include "ta_mx_elementwise.cuh"

namespace ta {
namespace mx {

constexpr int kFewMax = 4;   // rows of A
constexpr int kFewRows = 4;  // rows of B a warp takes
// Steps of a warp's copies in shared memory. Four blocks an SM with three steps each measured 23 us
// for two tokens and 37 for four; loads into registers, one step ahead, 32 and 46 (their registers
// leave two blocks), two steps ahead 27 and 36; three blocks with four steps 30 and 37. One token
// takes 21.5 us from here and took 23 from registers (4096 > 4096: 8.4 and 7.7).
constexpr int kFewStages = 3;
constexpr size_t kFewRing = (size_t)8 * kFewStages * kFewRows * 32 * 16;  // bytes

struct FewArgs {
  const uint16_t* a;  // [tokens][K], rows lda apart
  const uint16_t* b;  // lines ldb apart
  int64_t lda, ldb;
  int32_t tokens, N, K;
  int32_t warps_n;    // k_few_rows: warps along N; the other of the block's 8 share the sum
  int32_t splits;     // k_few_cols: blocks along K
  float* part;        // k_few_cols: [splits][tokens][N]
  uint16_t* out;
  const uint16_t* aux;
  const void* bias;
  int16_t* deriv;
  int64_t ldo, ld_aux, ld_deriv;
  int32_t bias_dt, act;
};

template <int DT>
__device__ __forceinline__ void few_store(const FewArgs& g, int t, int n, float v) {
  if (g.bias) v += load_as_float(g.bias, n, g.bias_dt);
  float d = 1.f;
  if (g.act == ACT_RELU) activate<true>(ACT_RELU, v, &v, &d);
  else if (g.act == ACT_GELU) activate<true>(ACT_GELU, v, &v, &d);
  else if (g.act == ACT_GELU_TANH) activate<true>(ACT_GELU_TANH, v, &v, &d);
  else if (g.act == ACT_SILU) activate<true>(ACT_SILU, v, &v, &d);
  if (g.deriv) g.deriv[t * g.ld_deriv + n] = (int16_t)encode_deriv<DT>(d);
  if (g.aux) v += load_as_float(g.aux, t * g.ld_aux + n, DT);
  store_from_float(g.out, t * g.ldo + n, DT, v);
}

__device__ __forceinline__ uint4 load_once(const uint16_t* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(p));
  return v;
}
__device__ __forceinline__ void copy16_async(uint4* dst, const uint16_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
template <int DT>
__device__ __forceinline__ void unpack8(uint4 u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack16(w[i], DT);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Rows of both operands start on 16 bytes and K is a multiple of 8.
template <int DT, int T>
__global__ void __launch_bounds__(256, 4) k_few_rows(const __grid_constant__ FewArgs g) {
  chain_next();
  chain_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wn = warp % g.warps_n, wk = warp / g.warps_n, warps_k = 8 / g.warps_n;
  const int row0 = (blockIdx.x * g.warps_n + wn) * kFewRows;
  extern __shared__ __align__(16) uint4 few_ring[];
  float acc[kFewRows][T] = {};
  const uint16_t* b[kFewRows];
#pragma unroll
  for (int r = 0; r < kFewRows; ++r) b[r] = g.b + (int64_t)min(row0 + r, g.N - 1) * g.ldb;
  if (row0 < g.N) {
    // a lane copies its own pieces of B's rows kFewStages - 1 steps ahead, and reads them back itself
    uint4* ring = few_ring + warp * (kFewStages * kFewRows * 32) + lane;
    const uint32_t step = warps_k * 256, K = g.K, k0 = wk * 256 + lane * 8;
    const int steps = (int)((K + step - 1 - min(K + step - 1, wk * 256u)) / step);
    auto copy = [&](int s) {
      const uint32_t k = k0 + (uint32_t)s * step;
      if (s < steps && k < K) {
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
          copy16_async(ring + (s % kFewStages * kFewRows + r) * 32, b[r] + k);
      }
      copy_commit();
    };
#pragma unroll
    for (int s = 0; s < kFewStages - 1; ++s) copy(s);
    for (int s = 0; s < steps; ++s) {
      const uint32_t k = k0 + (uint32_t)s * step;
      __syncwarp();  // (the stage that is filled again was read in the last step)
      copy(s + kFewStages - 1);
      float y[T][8];
#pragma unroll
      for (int t = 0; t < T; ++t)
        unpack8<DT>(t < g.tokens && k < K ? *reinterpret_cast<const uint4*>(g.a + t * g.lda + k)
                                          : make_uint4(0, 0, 0, 0),
                    y[t]);
      copy_wait<kFewStages - 1>();
      if (k < K) {
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
          float x[8];
          unpack8<DT>(ring[(s % kFewStages * kFewRows + r) * 32], x);
#pragma unroll
          for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[r][t] = fmaf(x[i], y[t][i], acc[r][t]);
        }
      }
    }
    copy_wait<0>();
  }
  __syncthreads();  // (the sums lie where the copies did)
  float(*sums)[kFewRows * T] = reinterpret_cast<float(*)[kFewRows * T]>(few_ring);
#pragma unroll
  for (int r = 0; r < kFewRows; ++r)
#pragma unroll
    for (int t = 0; t < T; ++t) {
#pragma unroll
      for (int o = 16; o; o >>= 1) acc[r][t] += __shfl_xor_sync(0xffffffffu, acc[r][t], o);
      if (lane == 0) sums[warp][r * T + t] = acc[r][t];
    }
  __syncthreads();
  const int per = kFewRows * T;
  for (int e = threadIdx.x; e < g.warps_n * per; e += 256) {
    const int w = e / per, r = e % per / T, t = e % T;
    const int n = (blockIdx.x * g.warps_n + w) * kFewRows + r;
    if (n >= g.N || t >= g.tokens) continue;
    float v = 0.f;
    for (int k = 0; k < warps_k; ++k) v += sums[k * g.warps_n + w][r * T + t];
    few_store<DT>(g, t, n, v);
  }
}

// Rows of B start on 16 bytes and N is a multiple of 8.
template <int DT, int T>
__global__ void __launch_bounds__(256) k_few_cols(const __grid_constant__ FewArgs g) {
  chain_next();
  chain_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.x * 256 + lane * 8;
  const int k0 = (int)((int64_t)g.K * blockIdx.y / gridDim.y);
  const int k1 = (int)((int64_t)g.K * (blockIdx.y + 1) / gridDim.y);
  // a stretch of A in shared memory, a step's tokens side by side
  constexpr int kStretch = 1024 / T;
  __shared__ __align__(16) float xs[kStretch][T];
  float acc[T][8] = {};
  for (int64_t kc = k0; kc < k1; kc += kStretch) {
    const int len = (int)min((int64_t)kStretch, k1 - kc);
    __syncthreads();
    for (int e = threadIdx.x; e < len * T; e += 256) {
      const int t = e / len, k = e % len;
      xs[k][t] = t < g.tokens ? load_as_float(g.a, t * g.lda + kc + k, DT) : 0.f;
    }
    __syncthreads();
    if (c < g.N) {
#pragma unroll 4
      for (int k = warp; k < len; k += 8) {
        float x[8];
        unpack8<DT>(load_once(g.b + (kc + k) * g.ldb + c), x);
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const float y = xs[k][t];
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[t][i] = fmaf(x[i], y, acc[t][i]);
        }
      }
    }
  }
  __shared__ float sums[8][256];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    if (t >= g.tokens) break;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[warp][lane * 8 + i] = acc[t][i];
    __syncthreads();
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += sums[w][threadIdx.x];
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n < g.N) g.part[((int64_t)blockIdx.y * g.tokens + t) * g.N + n] = v;
  }
}

template <int DT>
__global__ void __launch_bounds__(256) k_few_finish(const __grid_constant__ FewArgs g) {
  chain_next();
  chain_wait();
  const int n = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
  if (n >= g.N) return;
  float v = 0.f;
  for (int s = 0; s < g.splits; ++s) v += g.part[((int64_t)s * g.tokens + t) * g.N + n];
  few_store<DT>(g, t, n, v);
}

}  // namespace mx
}  // namespace ta
