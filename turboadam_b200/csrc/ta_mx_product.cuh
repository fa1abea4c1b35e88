// ta_mx_product.cuh -- the tile engine of the matrix operators: one persistent,
// warp-specialised kernel for D[m][n] = epilogue(sum_k A[m][k] B[n][k]) over a
// list of products, on tcgen05 with TMA-fed 128-byte swizzled operand tiles.
//
// Why this shape. A 16-bit tensor-core product on sm_100a is fed from shared
// memory: an M x N x 16 instruction reads (M + N) * 32 bytes for M * N * 16
// multiply-adds, so the tile has to be large before the tensor pipe, and not
// shared memory, is what bounds it. CG == 2 runs a pair of SMs on one 256 x 256
// tile (each SM stages half of A and half of B: 8 bytes per 1024 multiply-adds);
// CG == 1 runs one SM on a 128 x 128 tile, for lists too small to give every
// pair of SMs a large tile. In both a CTA stages 32 KB per 64 k's, six stages
// deep, and keeps two accumulators in tensor memory, so that the epilogue of
// one tile runs under the products of the next.
//
// Roles of the 320 threads: warp 0 issues the TMA loads, warp 1 the matrix
// instructions (of the pair's first CTA, with CG == 2), warps 2..9 the
// epilogue: two warps for each 32-row quadrant of tensor memory, which take the
// tile's 32-column chunks in turn.
//
// Long sums with few tiles (the Gram matrix of a wide matrix; few tokens) are
// split over k: each split leaves its fp32 tile in the workspace, and the last
// one to arrive adds them in the order of the splits, so that the result does
// not depend on which came last.
#pragma once

#include "ta_mx_device.cuh"

namespace ta {
namespace mx {

constexpr int kRows = 128;    // rows of a CTA's operand tiles
constexpr int kDepth = 64;    // k's per stage: one 128-byte swizzled row
constexpr int kStages = 6;
constexpr int kTileBytes = kRows * kDepth * 2;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kMaxProblems = 8;  // per launch (they travel as kernel parameters)
constexpr size_t kProductSmem = (size_t)kStages * 2 * kTileBytes + 1024 + 256;

// What is done with a finished tile.
enum Epilogue {
  EPI_GRAM = 0,   // fp16, symmetric: alpha * acc, mirrored
  EPI_POLY = 1,   // fp16, symmetric: c0 I + c1 A + c2 acc (A read back), mirrored
  EPI_APPLY = 2,  // fp16: alpha * acc
  EPI_FINAL = 3,  // the orthogonalised update: stored, or applied to the parameter
  EPI_LINEAR = 4, // bias, activation (and its derivative), residual
  EPI_PLAIN = 5   // rounded to the output's type
};

// Per-matrix scale of a Newton-Schulz list: the stored fp16 input times `unit` is the
// normalised matrix (unit is NaN where the input holds a NaN or an infinity).
struct Scale {
  float pow2;  // stored = input * pow2
  float unit;
};

// One matrix of a Newton-Schulz list (device table).
struct Item {
  const void* g;     // input or gradient, [rows][cols]
  void* mom;         // momentum, updated in place (null: the input itself)
  void* out;         // parameter (updated in place) or result
  __half* x0;        // scaled input, [rows][ld]
  __half* x0_lo;     // its remainder (null: rounded once)
  double* partial;   // [chunks] sums of squares
  Scale* scale;
  int64_t n;         // rows * cols
  int32_t cols, ld;
  int32_t chunk0;    // first work chunk of this matrix
  int32_t chunks;
  int64_t chunk_elems;
  float keep, gain;  // parameter <- keep * parameter - gain * update
  int16_t g_dt, mom_dt, out_dt, update;
};

struct alignas(64) Problem {
  CUtensorMap ta, tb;
  int32_t M, N;
  int32_t kblocks;          // blocks of 64 k's in one part of the sum
  int32_t parts;            // the sum runs over this many operand pairs
  int32_t tiles_m, tiles_n, tiles;  // per matrix (tiles: of the upper triangle, if sym)
  int32_t first;            // first work unit of this problem in the launch
  int32_t batch, splits;
  int32_t za, zb;           // z coordinate of (matrix z, part p): z * za + p * (za > 1)
  int16_t a_mn, b_mn, sym, dt;  // dt: output type (EPI_LINEAR, EPI_PLAIN)
  int32_t ldo, ld_aux;
  void* out;
  int64_t out_zs;           // elements between matrices
  const void* aux;          // EPI_POLY: A; EPI_LINEAR: residual
  int64_t aux_zs;
  const Scale* scale;       // [batch]
  const Item* items;        // [batch] (EPI_FINAL)
  const void* bias;         // EPI_LINEAR
  int16_t* deriv;           // EPI_LINEAR: the activation's derivative, 2^-14 steps
  int32_t ld_deriv;
  int16_t bias_dt, act;
  float* split_ws;          // [unit / splits][splits][rows x columns of a CTA tile]
  uint32_t* split_count;    // zero before and after every launch
};

struct ProductArgs {
  Problem p[kMaxProblems];
  int32_t count;
  int32_t units;            // work units: tiles x matrices x splits, over all problems
  int32_t bf16;             // operand type (all problems of a launch)
  int32_t unit_pow;         // scale.unit enters alpha to this power (0, 1 or 2)
  float alpha, c0, c1, c2;
  uint32_t* status;
};

template <int CG>
struct TileCfg {
  static constexpr int kCols = CG == 2 ? 256 : 128;  // accumulator columns of a CTA
  static constexpr int kTileRows = kRows * CG;
  static constexpr int kTmemCols = 2 * kCols;
};

struct Unit {
  int p, z, m0, n0, split;
  bool mirror;  // an off-diagonal tile of a symmetric result
};

// Work unit u of the launch. Tiles of a general product run down groups of 8 tile rows, so that
// the CTAs in flight share operand tiles in L2; splits of one tile are neighbours.
template <int CG>
__device__ __forceinline__ Unit locate(const ProductArgs& g, int u, int p_hint) {
  Unit w;
  int p = p_hint;
  while (p + 1 < g.count && u >= g.p[p + 1].first) ++p;
  const Problem& P = g.p[p];
  w.p = p;
  int t = u - P.first;
  w.split = t % P.splits;
  t /= P.splits;
  w.z = t / P.tiles;
  t -= w.z * P.tiles;
  int i, j;
  if (P.sym) {  // t-th tile of the upper triangle, column by column
    j = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while (j * (j + 1) / 2 > t) --j;
    while ((j + 1) * (j + 2) / 2 <= t) ++j;
    i = t - j * (j + 1) / 2;
  } else {
    const int group = 8 * P.tiles_n;
    const int g0 = t / group * 8;
    const int rows = min(8, P.tiles_m - g0);
    const int r = t - t / group * group;
    i = g0 + r % rows;
    j = r / rows;
  }
  w.m0 = i * TileCfg<CG>::kTileRows;
  w.n0 = j * TileCfg<CG>::kCols;
  w.mirror = P.sym && i != j;
  return w;
}

__device__ __forceinline__ void split_range(const Problem& P, int split, int* k0, int* k1) {
  const int total = P.kblocks * P.parts;
  *k0 = (int)((int64_t)total * split / P.splits);
  *k1 = (int)((int64_t)total * (split + 1) / P.splits);
}

// ---- activations ---------------------------------------------------------------
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };

// y = act(z), d = act'(z). A NaN z gives NaN for both.
template <bool DERIV>
__device__ __forceinline__ void activate(int act, float z, float* y, float* d) {
  if (act == ACT_RELU) {
    *y = z < 0.f ? 0.f : z;  // keeps NaN
    if (DERIV) *d = z > 0.f ? 1.f : (z != z ? z : 0.f);
  } else if (act == ACT_GELU) {  // z Phi(z); derivative Phi(z) + z phi(z)
    const float cdf = 0.5f * erfcf(-0.70710678f * z);
    *y = z == -INFINITY ? 0.f : z * cdf;
    if (DERIV) *d = fabsf(z) == INFINITY ? cdf : cdf + z * (0.39894228f * expf(-0.5f * z * z));
  } else if (act == ACT_GELU_TANH) {  // z sigmoid(2 u), u = sqrt(2/pi) (z + 0.044715 z^3)
    const float u2 = 1.59576912f * z * (1.f + 0.044715f * z * z);
    const float s = 1.f / (1.f + expf(-u2));
    *y = z == -INFINITY ? 0.f : z * s;
    if (DERIV) {
      const float du2 = 1.59576912f * (1.f + 0.134145f * z * z);
      const float t = s * (1.f - s);
      *d = t == 0.f ? s : s + z * t * du2;
    }
  } else if (act == ACT_SILU) {  // z sigmoid(z)
    const float s = 1.f / (1.f + expf(-z));
    *y = z == -INFINITY ? 0.f : z * s;
    if (DERIV) {
      const float t = s * (1.f - s);
      *d = t == 0.f ? s : s + z * t;
    }
  } else {
    *y = z;
    if (DERIV) *d = z != z ? z : 1.f;
  }
}

// An activation's derivative lies in (-0.13, 1.13): a 16-bit fixed-point number in steps of 2^-14
// holds it to 2^-15 absolute, finer than an fp16 near 1, so a gradient computed from it loses
// nothing next to its own rounding to 16 bits. The lowest code stands for NaN.
constexpr int16_t kDerivNan = -32768;
__device__ __forceinline__ int16_t encode_deriv(float d) {
  return d != d ? kDerivNan : (int16_t)__float2int_rn(d * 16384.f);
}
__device__ __forceinline__ float decode_deriv(int16_t q) {
  return q == kDerivNan ? __int_as_float(0x7fc00000) : (float)q * (1.f / 16384.f);
}

// ---- row chunks of 32 columns --------------------------------------------------
// 16-bit elements [0, n) of a row chunk. vec: the chunk starts on 16 bytes and n == 32.
__device__ __forceinline__ void load_row(const void* p, int64_t at, int n, bool vec, int dt,
                                         float (&x)[32]) {
  if (vec && dt != DT_F32) {
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 u = q[i];
      float2 f;
      f = unpack16(u.x, dt); x[8 * i + 0] = f.x; x[8 * i + 1] = f.y;
      f = unpack16(u.y, dt); x[8 * i + 2] = f.x; x[8 * i + 3] = f.y;
      f = unpack16(u.z, dt); x[8 * i + 4] = f.x; x[8 * i + 5] = f.y;
      f = unpack16(u.w, dt); x[8 * i + 6] = f.x; x[8 * i + 7] = f.y;
    }
  } else if (vec) {
    const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 u = q[i];
      x[4 * i] = u.x; x[4 * i + 1] = u.y; x[4 * i + 2] = u.z; x[4 * i + 3] = u.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = i < n ? load_as_float(p, at + i, dt) : 0.f;
  }
}
__device__ __forceinline__ void store_row(void* p, int64_t at, int n, bool vec, int dt,
                                          const float (&x)[32]) {
  if (vec && dt != DT_F32) {
    uint4* q = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q[i] = make_uint4(pack16(x[8 * i], x[8 * i + 1], dt), pack16(x[8 * i + 2], x[8 * i + 3], dt),
                        pack16(x[8 * i + 4], x[8 * i + 5], dt),
                        pack16(x[8 * i + 6], x[8 * i + 7], dt));
  } else if (vec) {
    float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      q[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) store_from_float(p, at + i, dt, x[i]);
  }
}
// A 32-column chunk of rows `ld` elements apart keeps its 16-byte alignment in every row.
__device__ __forceinline__ bool row_vec(const void* p, int64_t ld, int n, int dt) {
  const int per = dt == DT_F32 ? 4 : 8;
  return n == 32 && ((uintptr_t)p & 15) == 0 && ld % per == 0;
}

// One thread's 32 finished sums: row `row`, columns [col, col + n).
template <int EPI>
__device__ __forceinline__ void finish(const ProductArgs& g, const Problem& P, const Unit& w,
                                       float alpha, int row, int col, int n, float (&v)[32]) {
  if constexpr (EPI == EPI_GRAM || EPI == EPI_POLY || EPI == EPI_APPLY) {
    // fp16 workspace matrices: rows start on 16 bytes
    __half* out = reinterpret_cast<__half*>(P.out) + (int64_t)w.z * P.out_zs;
    if constexpr (EPI == EPI_POLY) {
      float a[32];
      const __half* A = reinterpret_cast<const __half*>(P.aux) + (int64_t)w.z * P.aux_zs;
      load_row(A, (int64_t)row * P.ld_aux + col, n, n == 32, DT_F16, a);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        v[i] = fmaf(g.c2, v[i], fmaf(g.c1, a[i], row == col + i ? g.c0 : 0.f));
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= alpha;
    }
    store_row(out, (int64_t)row * P.ldo + col, n, n == 32, DT_F16, v);
    if (EPI != EPI_APPLY && w.mirror) {  // a warp's 32 rows are 64 consecutive bytes
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < n) out[(int64_t)(col + i) * P.ldo + row] = __float2half_rn(v[i]);
    }
  } else if constexpr (EPI == EPI_FINAL) {
    const Item& it = P.items[w.z];
    const int dt = it.out_dt;
    const int64_t at = (int64_t)row * P.N + col;
    const bool vec = row_vec(it.out, P.N, n, dt);
    if (it.update) {
      float p[32];
      load_row(it.out, at, n, vec, dt, p);
      const float keep = it.keep, gain = it.gain * alpha;
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = fmaf(-gain, v[i], keep * p[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= alpha;
    }
    store_row(it.out, at, n, vec, dt, v);
  } else if constexpr (EPI == EPI_LINEAR) {
    if (P.bias) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < n) v[i] += load_as_float(P.bias, col + i, P.bias_dt);
    }
    if (P.deriv) {
      const int64_t at = (int64_t)row * P.ld_deriv + col;
      float d[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float y;
        activate<true>(P.act, v[i], &y, &d[i]);
        v[i] = y;
      }
      if (n == 32) {  // the derivative's rows start on 16 bytes
        uint4* q = reinterpret_cast<uint4*>(P.deriv + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t u[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            u[k] = (uint32_t)(uint16_t)encode_deriv(d[8 * i + 2 * k]) |
                   ((uint32_t)(uint16_t)encode_deriv(d[8 * i + 2 * k + 1]) << 16);
          q[i] = make_uint4(u[0], u[1], u[2], u[3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < n) P.deriv[at + i] = encode_deriv(d[i]);
      }
    } else if (P.act != ACT_NONE) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float y;
        activate<false>(P.act, v[i], &y, nullptr);
        v[i] = y;
      }
    }
    if (P.aux) {
      float r[32];
      load_row(P.aux, (int64_t)row * P.ld_aux + col, n, row_vec(P.aux, P.ld_aux, n, P.dt), P.dt,
               r);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += r[i];
    }
    store_row(P.out, (int64_t)row * P.ldo + col, n, row_vec(P.out, P.ldo, n, P.dt), P.dt, v);
  } else {
    store_row(P.out, (int64_t)row * P.ldo + col, n, row_vec(P.out, P.ldo, n, P.dt), P.dt, v);
  }
}

template <int CG, int EPI>
__global__ void __launch_bounds__(kThreads, 1) k_product(const __grid_constant__ ProductArgs g) {
  using Cfg = TileCfg<CG>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* tile_a = smem;
  uint8_t* tile_b = smem + kStages * kTileBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + 2 * kStages * kTileBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile uint32_t* last_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const int worker = blockIdx.x / CG, workers = gridDim.x / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      bar_init(&full[s], 1);
      bar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      bar_init(&acc_full[b], 1);
      bar_init(&acc_empty[b], CG * kEpiWarps);
    }
    bar_init_fence();
  }
  if (warp == 1) tmem_alloc<CG>(tmem_slot, Cfg::kTmemCols);
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *(volatile uint32_t*)tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      int hint = 0;
      for (int u = worker; u < g.units && ok; u += workers) {
        const Unit w = locate<CG>(g, u, hint);
        hint = w.p;
        const Problem& P = g.p[w.p];
        int k0, k1;
        split_range(P, w.split, &k0, &k1);
        const int am = w.m0 + (int)rank * kRows, bn = w.n0 + (int)rank * kRows;
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const int s = it % kStages;
          if (!bar_wait(&empty[s], ((it / kStages) & 1) ^ 1, g.status)) {
            ok = false;
            break;
          }
          // with a pair, both CTAs' bytes are counted on the first CTA's barrier
          uint32_t bar = smem_addr(&full[s]);
          if (CG == 2) bar = map_to_rank(bar, 0);
          if (rank == 0) bar_expect_tx(&full[s], CG * 2 * kTileBytes);
          const int part = kb >= P.kblocks;
          const int k = (kb - part * P.kblocks) * kDepth;
          const int za = w.z * P.za + (P.za > 1 ? part : 0);
          const int zb = w.z * P.zb + (P.zb > 1 ? part : 0);
          const uint32_t a = smem_addr(tile_a + s * kTileBytes);
          const uint32_t b = smem_addr(tile_b + s * kTileBytes);
          if (P.a_mn) {
            tma_load<CG>(&P.ta, a, bar, am, k, za);
            tma_load<CG>(&P.ta, a + kTileBytes / 2, bar, am + 64, k, za);
          } else {
            tma_load<CG>(&P.ta, a, bar, k, am, za);
          }
          if (P.b_mn) {
            tma_load<CG>(&P.tb, b, bar, bn, k, zb);
            tma_load<CG>(&P.tb, b + kTileBytes / 2, bar, bn + 64, k, zb);
          } else {
            tma_load<CG>(&P.tb, b, bar, k, bn, zb);
          }
        }
      }
      // Leave no copy in flight: every stage that was filled has been read (its "empty" phase
      // completes), which the waits of a complete run establish here, each of them bounded.
      for (int s = 0; s < kStages && ok; ++s, ++it)
        if (it >= (uint32_t)kStages)
          ok = bar_wait(&empty[it % kStages], ((it / kStages) & 1) ^ 1, g.status);
      if (!ok)  // a wait ran out: let the copies that were issued land before the CTA ends
        for (const uint64_t t0 = now_ns(); now_ns() - t0 < 1000000ull;) {}
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      uint32_t it = 0, tile = 0;
      bool ok = true;
      int hint = 0;
      for (int u = worker; u < g.units && ok; u += workers) {
        const Unit w = locate<CG>(g, u, hint);
        hint = w.p;
        const Problem& P = g.p[w.p];
        int k0, k1;
        split_range(P, w.split, &k0, &k1);
        if (k0 == k1) continue;  // an empty sum: the epilogue takes zeros
        const int buf = tile & 1;
        const bool a_mn = P.a_mn, b_mn = P.b_mn;
        const uint32_t idesc = mma_idesc(g.bf16, a_mn, b_mn, Cfg::kTileRows, Cfg::kCols);
        const uint32_t step_a = mma_k_step(a_mn), step_b = mma_k_step(b_mn);
        const uint32_t d = tmem + buf * Cfg::kCols;
        if (!bar_wait(&acc_empty[buf], ((tile >> 1) & 1) ^ 1, g.status)) break;
        tc_fence_after();
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const int s = it % kStages;
          if (!bar_wait(&full[s], (it / kStages) & 1, g.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint64_t a = mma_smem_desc(smem_addr(tile_a + s * kTileBytes), a_mn);
          uint64_t b = mma_smem_desc(smem_addr(tile_b + s * kTileBytes), b_mn);
#pragma unroll
          for (int i = 0; i < kDepth / 16; ++i, a += step_a, b += step_b)
            tc_mma<CG>(d, a, b, idesc, kb > k0 || i > 0);
          tc_commit<CG>(&empty[s]);
        }
        if (ok) tc_commit<CG>(&acc_full[buf]);
        ++tile;
      }
    }
  } else {
    const int quad = warp & 3;             // the tensor-memory lanes this warp can read
    const int half = (warp - 2) >> 2;      // which of the quadrant's two warps
    const int r_local = quad * 32 + lane;
    uint32_t tile = 0;
    int hint = 0;
    bool ok = true;  // false once a wait has run out: units pass without results, so that the
                     // block barriers of the split sums still see every warp
    for (int u = worker; u < g.units; u += workers) {
      const Unit w = locate<CG>(g, u, hint);
      hint = w.p;
      const Problem& P = g.p[w.p];
      int k0, k1;
      split_range(P, w.split, &k0, &k1);
      const int buf = tile & 1;
      if (k1 > k0 && ok) {
        ok = __all_sync(0xffffffffu, bar_wait(&acc_full[buf], (tile >> 1) & 1, g.status));
        tc_fence_after();
      }
      const bool sums = k1 > k0 && ok;
      const int row = w.m0 + (int)rank * kRows + r_local;
      const uint32_t src = tmem + buf * Cfg::kCols + ((uint32_t)(quad * 32) << 16);
      float alpha = g.alpha;
      if (g.unit_pow) {
        const float unit = P.scale[w.z].unit;
        alpha *= g.unit_pow == 2 ? unit * unit : unit;
      }
      if (P.splits == 1) {
        for (int c = half; c < Cfg::kCols / 32; c += 2) {
          const int col = w.n0 + c * 32, n = min(32, P.N - col);
          if (n <= 0 || !ok) break;
          float v[32];
          if (sums) {
            tmem_ld32(src + c * 32, v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;
          }
          if (row < P.M) finish<EPI>(g, P, w, alpha, row, col, n, v);
        }
        if (sums) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive_cluster(map_to_rank(smem_addr(&acc_empty[buf]), 0));
        }
      } else {
        // this CTA's tile of the split: [split][column / 4][row] float4
        const int64_t tile_id = (int64_t)((u - P.first) / P.splits) * CG + rank;
        float4* mine = reinterpret_cast<float4*>(P.split_ws) +
                       (tile_id * P.splits + w.split) * (Cfg::kCols / 4 * kRows);
        for (int c = half; c < Cfg::kCols / 32; c += 2) {
          if (w.n0 + c * 32 >= P.N || !sums) break;  // a split has at least one k block
          float v[32];
          tmem_ld32(src + c * 32, v);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            __stcg(&mine[(c * 8 + i) * kRows + r_local],
                   make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
        }
        if (sums) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive_cluster(map_to_rank(smem_addr(&acc_empty[buf]), 0));
        }
        __threadfence();
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
        if (threadIdx.x == 64) {
          const bool all = ok && atomicAdd(&P.split_count[tile_id], 1u) == (uint32_t)P.splits - 1;
          *last_flag = all;
          if (all) P.split_count[tile_id] = 0;  // for the next launch
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
        const bool last = *last_flag && ok;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
        if (last) {
          __threadfence();
          const float4* parts = reinterpret_cast<const float4*>(P.split_ws) +
                                tile_id * P.splits * (Cfg::kCols / 4 * kRows);
          for (int c = half; c < Cfg::kCols / 32; c += 2) {
            const int col = w.n0 + c * 32, n = min(32, P.N - col);
            if (n <= 0) break;
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;
            for (int s = 0; s < P.splits; ++s) {
              const float4* q = parts + (int64_t)s * (Cfg::kCols / 4 * kRows);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 f = __ldcg(&q[(c * 8 + i) * kRows + r_local]);
                v[4 * i] += f.x;
                v[4 * i + 1] += f.y;
                v[4 * i + 2] += f.z;
                v[4 * i + 3] += f.w;
              }
            }
            if (row < P.M) finish<EPI>(g, P, w, alpha, row, col, n, v);
          }
        }
      }
      if (sums) ++tile;
    }
  }
  __syncwarp();
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_free<CG>(tmem, Cfg::kTmemCols);
}

}  // namespace mx
}  // namespace ta
