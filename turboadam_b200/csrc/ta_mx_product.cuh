// ta_mx_product.cuh -- the tile engine of the matrix operators: one persistent,
// warp-specialised kernel for D[m][n] = epilogue(sum_k A[m][k] B[n][k]) over a
// list of products, on tcgen05 with TMA-fed 128-byte swizzled operand tiles.
//
// Why this shape. A 16-bit tensor-core product on sm_100a takes both operands from shared
// memory, whose 128 bytes per cycle serve the matrix instructions' reads and the TMA writes
// alike. A pair of SMs (cta_group::2) computes a tile of 256 rows by C columns; each SM holds 128
// rows of A and C / 2 rows of B. Per 64 k's that is 16 KB + 64 C bytes written and as many read,
// or 256 + C cycles of shared memory, against 2 C cycles of the tensor pipe: C = 256 only just
// balances (measured 1200 TFLOP/s at 14336 x 4096 x 4096, loads and reads in each other's way),
// C = 512 leaves a quarter of the bandwidth free. So a wide tile is two instructions of C / 2
// columns that share A (the second takes it from the collector), over all 512 columns of tensor
// memory; a narrow one, for small results or short sums, is one instruction and leaves room for a
// second accumulator, so that its epilogue runs under the next tile's products.
//
// Roles of the 320 threads: warp 0 issues the TMA loads, warp 1 the matrix
// instructions (of the pair's first CTA), warps 2..9 the epilogue: two warps for
// each 32-row quadrant of tensor memory, which take the tile's 128-byte column
// groups in turn and pass them through shared memory, so that every global
// access of the epilogue covers whole lines.
//
// Long sums with few tiles (the Gram matrix of a wide matrix; few tokens) are
// split over k: each split leaves its fp32 tile in the workspace, and the last
// one to arrive adds them in the order of the splits, so that the result does
// not depend on which came last.
#pragma once

#include <type_traits>

#include "ta_mx_device.cuh"

namespace ta {
namespace mx {

constexpr int kRows = 128;      // rows of a CTA's operand tile of A
constexpr int kTileRows = 256;  // rows of a pair's tile
constexpr int kDepth = 64;      // k's per stage: one 128-byte swizzled row
constexpr int kTileABytes = kRows * kDepth * 2;
constexpr int kMaxStages = 8;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kTmemCols = 512;
constexpr int kMaxProblems = 8;  // per launch (they travel as kernel parameters)
constexpr int kGroupBytes = 128;                          // an epilogue group: 32 rows of a line
constexpr int kStageOutBytes = 32 * kGroupBytes;          // per epilogue warp
constexpr int kBiasBytes = 32 * 4;                        // per epilogue warp
constexpr size_t kOperandSpace = 192 * 1024;
constexpr size_t kProductSmem =
    1024 + kOperandSpace + kEpiWarps * (kStageOutBytes + kBiasBytes) + 256;

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
  int32_t tiles_m, tiles_n, tiles;  // per matrix (tiles: on and above the diagonal, if sym)
  int32_t first;            // first work unit of this problem in the launch
  int32_t batch, splits;
  int32_t za, zb;           // z coordinate of (matrix z, part p): z * za + p * (za > 1)
  int16_t a_mn, b_mn, sym, pad0;
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
  int32_t cols;             // tile width C: `halves` instructions of `half` columns
  int32_t half, halves;
  int32_t stages, buffers;
  int32_t unit_pow;         // scale.unit enters alpha to this power (0, 1 or 2)
  float alpha, c0, c1, c2;
  uint32_t* status;
};

struct Unit {
  int p, z, m0, n0, split;
};

// First tile column of tile row i of a symmetric result: the one that holds the diagonal block's
// first column. Columns left of the diagonal block are skipped by the epilogue, those right of it
// are mirrored, in groups of 32 or 64 columns (both widths divide 256 and every tile width).
__host__ __device__ __forceinline__ int sym_first(int i, int cols) { return i * kTileRows / cols; }

// Work unit u of the launch. Tiles of a general product run down groups of 8 tile rows, so that
// the CTAs in flight share operand tiles in L2; splits of one tile are neighbours.
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
  if (P.sym) {
    i = 0;
    for (;;) {
      const int n = P.tiles_n - sym_first(i, g.cols);
      if (t < n) break;
      t -= n;
      ++i;
    }
    j = sym_first(i, g.cols) + t;
  } else {
    const int group = 8 * P.tiles_n;
    const int g0 = t / group * 8;
    const int rows = min(8, P.tiles_m - g0);
    const int r = t - t / group * group;
    i = g0 + r % rows;
    j = r / rows;
  }
  w.m0 = i * kTileRows;
  w.n0 = j * g.cols;
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

// ---- epilogue groups ------------------------------------------------------------
// A warp's group is 32 rows by 128 bytes of one output (64 columns of a 16-bit type, 32 of
// fp32). In registers a thread holds 32 columns of one row; in global memory a row is a line. The
// group's shared-memory copy has its 16-byte pieces XORed with the row, which keeps both the
// row-wise accesses (a thread's own row) and the line-wise ones (8 threads a row) free of bank
// conflicts.
struct Group {
  uint32_t s;  // shared address of this warp's 4 KB
  int lane;
  int rows;    // valid rows (0 .. 32)
  __device__ __forceinline__ uint32_t piece(int row, int k) const {
    return s + row * kGroupBytes + ((k ^ (row & 7)) << 4);
  }
};

// Lines start on 16 bytes, and the group's columns are all there.
__device__ __forceinline__ bool whole_lines(const void* p, int64_t ld, int n, int size) {
  return n * size == kGroupBytes && (((uintptr_t)p | (uint64_t)(ld * size)) & 15) == 0;
}

// base points at the group's first element; n valid columns of SIZE bytes, lines ld elements
// apart. Loads the group. Eight threads take a line, so a warp's access covers four whole lines.
template <int SIZE>
__device__ __forceinline__ void group_load(const Group& g, const void* base, int64_t ld, int n) {
  using T = typename std::conditional<SIZE == 4, uint32_t, uint16_t>::type;
  const uint8_t* p = reinterpret_cast<const uint8_t*>(base);
  if (whole_lines(base, ld, n, SIZE)) {
    const int k = g.lane & 7, r0 = g.lane >> 3;
    const uint8_t* q = p + r0 * ld * SIZE + k * 16;
    const int64_t step = ld * (4 * SIZE);
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = r0 + 4 * i < g.rows ? *reinterpret_cast<const uint4*>(q + i * step)
                                 : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) sts16(g.piece(r0 + 4 * i, k), v[i]);
  } else {
    for (int r = 0; r < g.rows; ++r)
      for (int c = g.lane; c < n; c += 32)
        sts_elem<SIZE>(g.piece(r, c * SIZE >> 4) + (c * SIZE & 15),
                       reinterpret_cast<const T*>(base)[r * ld + c]);
  }
  __syncwarp();
}
template <int SIZE>
__device__ __forceinline__ void group_store(const Group& g, void* base, int64_t ld, int n) {
  using T = typename std::conditional<SIZE == 4, uint32_t, uint16_t>::type;
  __syncwarp();
  if (whole_lines(base, ld, n, SIZE)) {
    const int k = g.lane & 7, r0 = g.lane >> 3;
    uint8_t* q = reinterpret_cast<uint8_t*>(base) + r0 * ld * SIZE + k * 16;
    const int64_t step = ld * (4 * SIZE);
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = lds16(g.piece(r0 + 4 * i, k));
    if (g.rows == 32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(q + i * step) = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r0 + 4 * i < g.rows) *reinterpret_cast<uint4*>(q + i * step) = v[i];
    }
  } else {
    for (int r = 0; r < g.rows; ++r)
      for (int c = g.lane; c < n; c += 32)
        reinterpret_cast<T*>(base)[r * ld + c] =
            (T)lds_elem<SIZE>(g.piece(r, c * SIZE >> 4) + (c * SIZE & 15));
  }
  __syncwarp();
}
// This thread's row of the group, columns [32 h, 32 h + 32) (fp32: h = 0).
template <int DT>
__device__ __forceinline__ void row_get(const Group& g, int h, float (&x)[32]) {
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint4 u = lds16(g.piece(g.lane, k));
      x[4 * k] = __uint_as_float(u.x);
      x[4 * k + 1] = __uint_as_float(u.y);
      x[4 * k + 2] = __uint_as_float(u.z);
      x[4 * k + 3] = __uint_as_float(u.w);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint4 u = lds16(g.piece(g.lane, 4 * h + k));
      float2 f;
      f = unpack16(u.x, DT); x[8 * k + 0] = f.x; x[8 * k + 1] = f.y;
      f = unpack16(u.y, DT); x[8 * k + 2] = f.x; x[8 * k + 3] = f.y;
      f = unpack16(u.z, DT); x[8 * k + 4] = f.x; x[8 * k + 5] = f.y;
      f = unpack16(u.w, DT); x[8 * k + 6] = f.x; x[8 * k + 7] = f.y;
    }
  }
}
template <int DT>
__device__ __forceinline__ void row_put(const Group& g, int h, const float (&x)[32]) {
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      sts16(g.piece(g.lane, k),
            make_uint4(__float_as_uint(x[4 * k]), __float_as_uint(x[4 * k + 1]),
                       __float_as_uint(x[4 * k + 2]), __float_as_uint(x[4 * k + 3])));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      sts16(g.piece(g.lane, 4 * h + k),
            make_uint4(pack16(x[8 * k], x[8 * k + 1], DT), pack16(x[8 * k + 2], x[8 * k + 3], DT),
                       pack16(x[8 * k + 4], x[8 * k + 5], DT),
                       pack16(x[8 * k + 6], x[8 * k + 7], DT)));
  }
}

// Where a group's finished sums come from: tensor memory, the split workspace, or nothing (an
// empty sum).
struct Sums {
  uint32_t tmem;        // first column of the tile, this warp's lanes
  const float4* parts;  // this tile's splits, or null
  int splits, width4;   // number of them; float4 columns of one
  int row;              // in the CTA's tile
  bool any;
};
__device__ __forceinline__ void take_sums(const Sums& a, int c, float (&v)[32]) {
  if (a.parts) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0.f;
    for (int s = 0; s < a.splits; ++s) {
      const float4* q = a.parts + ((int64_t)s * a.width4 + c / 4) * kRows + a.row;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 f = __ldcg(q + i * kRows);
        v[4 * i] += f.x;
        v[4 * i + 1] += f.y;
        v[4 * i + 2] += f.z;
        v[4 * i + 3] += f.w;
      }
    }
  } else if (a.any) {
    tmem_ld32(a.tmem + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0.f;
  }
}

// The orthogonalised update of one group, in the result's type.
template <int DT>
__device__ __forceinline__ void finish_final(const Item& it, const Group& G, const Sums& a,
                                             float alpha, int64_t ld, int row0, int col, int n,
                                             int c) {
  constexpr int kSize = DT == DT_F32 ? 4 : 2, kCols = kGroupBytes / kSize;
  const float keep = it.keep, gain = it.gain * alpha;
  const bool update = it.update;
  uint8_t* base = reinterpret_cast<uint8_t*>(it.out) + (row0 * ld + col) * kSize;
  float v[32];
  for (int q = 0; q < n; q += kCols) {
    const int m = min(kCols, n - q);
    void* at = base + q * kSize;
    if (update) group_load<kSize>(G, at, ld, m);
#pragma unroll
    for (int h = 0; h < kCols / 32; ++h) {
      if (h * 32 >= m) break;
      take_sums(a, c + q + h * 32, v);
      if (update) {
        float p[32];
        row_get<DT>(G, h, p);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = fmaf(-gain, v[i], keep * p[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= alpha;
      }
      row_put<DT>(G, h, v);
    }
    group_store<kSize>(G, at, ld, m);
  }
}

// What the epilogue of one tile reads of its problem, in registers.
struct Out {
  uint8_t* out;
  const uint8_t* aux;
  const void* bias;
  int16_t* deriv;
  int64_t ld, ld_aux, ld_deriv;
  int bias_dt, act;
};

// bias, activation (and its derivative), residual: 32 columns in registers.
template <int DT, int ACT, bool DERIV>
__device__ __forceinline__ void activate_row(float (&v)[32], uint32_t (&code)[16]) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    float d0 = 0.f, d1 = 0.f;
    activate<DERIV>(ACT, v[i], &v[i], &d0);
    activate<DERIV>(ACT, v[i + 1], &v[i + 1], &d1);
    if (DERIV)
      code[i / 2] =
          (uint32_t)(uint16_t)encode_deriv(d0) | ((uint32_t)(uint16_t)encode_deriv(d1) << 16);
  }
}
template <int DT, int ACT>
__device__ __forceinline__ void finish_linear(const Out& o, const Group& G, uint32_t bias,
                                              const Sums& a, int row0, int col, int n, int c) {
  if (o.aux) group_load<2>(G, o.aux + (row0 * o.ld_aux + col) * 2, o.ld_aux, n);
  uint32_t code[2][16];
  float v[32];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h * 32 >= n) break;
    take_sums(a, c + h * 32, v);
    if (o.bias) {
      const int i = h * 32 + G.lane;
      __syncwarp();
      sts_elem<4>(bias + G.lane * 4,
                  __float_as_uint(i < n ? load_as_float(o.bias, col + i, o.bias_dt) : 0.f));
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint4 b = lds16(bias + k * 16);
        v[4 * k] += __uint_as_float(b.x);
        v[4 * k + 1] += __uint_as_float(b.y);
        v[4 * k + 2] += __uint_as_float(b.z);
        v[4 * k + 3] += __uint_as_float(b.w);
      }
    }
    if constexpr (ACT != ACT_NONE) {
      if (o.deriv) activate_row<DT, ACT, true>(v, code[h]);
      else activate_row<DT, ACT, false>(v, code[h]);
    }
    if (o.aux) {
      float r[32];
      row_get<DT>(G, h, r);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += r[i];
    }
    row_put<DT>(G, h, v);
  }
  group_store<2>(G, o.out + (row0 * o.ld + col) * 2, o.ld, n);
  if constexpr (ACT != ACT_NONE) {
    if (o.deriv) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k * 8 < n) {
          const uint32_t* q = &code[k / 4][(k % 4) * 4];
          sts16(G.piece(G.lane, k), make_uint4(q[0], q[1], q[2], q[3]));
        }
      group_store<2>(G, o.deriv + row0 * o.ld_deriv + col, o.ld_deriv, n);
    }
  }
}

// One group: rows [row0, row0 + 32) by columns [col, col + n) of the result, tile columns from c.
// DT is the type of the result (EPI_LINEAR, EPI_PLAIN); `mirror`: a symmetric result's group right
// of the diagonal block, also written transposed (a warp's 32 rows are 64 consecutive bytes).
template <int EPI, int DT>
__device__ __forceinline__ void finish(const ProductArgs& g, const Out& o, const Group& G,
                                       const Sums& a, float alpha, int row0, int col, int n,
                                       int c, bool mirror) {
  if constexpr (EPI == EPI_GRAM || EPI == EPI_POLY || EPI == EPI_APPLY) {
    float v[32];
    if constexpr (EPI == EPI_POLY)
      group_load<2>(G, o.aux + (row0 * o.ld_aux + col) * 2, o.ld_aux, n);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h * 32 >= n) break;
      take_sums(a, c + h * 32, v);
      if constexpr (EPI == EPI_POLY) {
        float x[32];
        row_get<DT_F16>(G, h, x);
        const int diag = row0 + G.lane - (col + h * 32);
#pragma unroll
        for (int i = 0; i < 32; ++i)
          v[i] = fmaf(g.c2, v[i], fmaf(g.c1, x[i], diag == i ? g.c0 : 0.f));
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= alpha;
      }
      row_put<DT_F16>(G, h, v);
      if (EPI != EPI_APPLY && mirror && G.lane < G.rows) {
        __half* t = reinterpret_cast<__half*>(o.out) + (col + h * 32) * o.ld + row0 + G.lane;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (h * 32 + i < n) t[i * o.ld] = __float2half_rn(v[i]);
      }
    }
    group_store<2>(G, o.out + (row0 * o.ld + col) * 2, o.ld, n);
  } else {
    float v[32];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h * 32 >= n) break;
      take_sums(a, c + h * 32, v);
      row_put<DT>(G, h, v);
    }
    group_store<2>(G, o.out + (row0 * o.ld + col) * 2, o.ld, n);
  }
}

template <int EPI, int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    k_product(const __grid_constant__ ProductArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kOperandSpace +
                                               kEpiWarps * (kStageOutBytes + kBiasBytes));
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_full = empty + kMaxStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile uint32_t* last_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int worker = blockIdx.x / 2, workers = gridDim.x / 2;
  const int half = g.half, halves = g.halves, stages = g.stages, buffers = g.buffers;
  const uint32_t half_bytes = (uint32_t)half * (kDepth * 2 / 2);  // one CTA's share of B
  const uint32_t stage_bytes = kTileABytes + halves * half_bytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      bar_init(&full[s], 1);
      bar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      bar_init(&acc_full[b], 1);
      bar_init(&acc_empty[b], 2 * kEpiWarps);
    }
    bar_init_fence();
  }
  if (warp == 1) tmem_alloc<2>(tmem_slot, kTmemCols);
  Unit w = locate(g, worker, 0);  // the first unit is looked up under the set-up's latency
  if (warp == 0 && elect_one()) {
    tma_prefetch(&g.p[w.p].ta);
    tma_prefetch(&g.p[w.p].tb);
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *(volatile uint32_t*)tmem_slot;

  if (warp == 0) {
    uint32_t filled = 0;  // stages filled so far
    int s = 0;
    uint32_t phase = 1;   // of "empty": the first round finds every stage free
    bool ok = true;
    const uint32_t tiles0 = smem_addr(smem);
    for (int u = worker; u < g.units && ok; u += workers) {
      if (u != worker) w = locate(g, u, w.p);
      const Problem& P = g.p[w.p];
      int k0, k1;
      split_range(P, w.split, &k0, &k1);
      const CUtensorMap *ma = &P.ta, *mb = &P.tb;
      const bool a_mn = P.a_mn, b_mn = P.b_mn;
      const int kblocks = P.kblocks;
      const int am = w.m0 + (int)rank * kRows, bn = w.n0 + (int)rank * (half / 2);
      const int za0 = w.z * P.za, zb0 = w.z * P.zb;
      const int za1 = P.za > 1, zb1 = P.zb > 1;
      for (int kb = k0; kb < k1; ++kb) {
        if (!__all_sync(0xffffffffu, bar_wait(&empty[s], phase, g.status))) {
          ok = false;
          break;
        }
        const int part = kb >= kblocks;
        const int k = (kb - part * kblocks) * kDepth;
        const int za = za0 + za1 * part, zb = zb0 + zb1 * part;
        const uint32_t a = tiles0 + s * stage_bytes, b = a + kTileABytes;
        if (elect_one()) {
          // both CTAs' bytes are counted on the first CTA's barrier
          const uint32_t bar = map_to_rank(smem_addr(&full[s]), 0);
          if (rank == 0) bar_expect_tx(&full[s], 2 * stage_bytes);
          if (a_mn) {
            tma_load<2>(ma, a, bar, am, k, za);
            tma_load<2>(ma, a + kTileABytes / 2, bar, am + 64, k, za);
          } else {
            tma_load<2>(ma, a, bar, k, am, za);
          }
          for (int h = 0; h < halves; ++h) {
            const uint32_t bh = b + h * half_bytes;
            const int n = bn + h * half;
            if (b_mn) {
              tma_load<2>(mb, bh, bar, n, k, zb);
              if (half > 128) tma_load<2>(mb, bh + 8192, bar, n + 64, k, zb);
            } else {
              tma_load<2>(mb, bh, bar, k, n, zb);
            }
          }
        }
        __syncwarp();
        ++filled;
        if (++s == stages) {
          s = 0;
          phase ^= 1;
        }
      }
    }
    // Leave no copy in flight: every stage that was filled has been read (its "empty" phase
    // completes), which the waits of a complete run establish here, each of them bounded.
    for (uint32_t i = 0; i < (uint32_t)stages && ok; ++i) {
      if (filled >= (uint32_t)stages || s < (int)filled)
        ok = __all_sync(0xffffffffu, bar_wait(&empty[s], phase, g.status));
      if (++s == stages) {
        s = 0;
        phase ^= 1;
      }
    }
    if (!ok)  // a wait ran out: let the copies that were issued land before the CTA ends
      for (const uint64_t t0 = now_ns(); now_ns() - t0 < 1000000ull;) {}
  } else if (warp == 1) {
    if (rank == 0) {
      uint32_t tile = 0, phase = 0;
      int s = 0;
      bool ok = true;
      const uint32_t tiles0 = smem_addr(smem);
      for (int u = worker; u < g.units && ok; u += workers) {
        if (u != worker) w = locate(g, u, w.p);
        const Problem& P = g.p[w.p];
        int k0, k1;
        split_range(P, w.split, &k0, &k1);
        if (k0 == k1) continue;  // an empty sum: the epilogue takes zeros
        const bool a_mn = P.a_mn, b_mn = P.b_mn;
        const uint32_t idesc = mma_idesc(g.bf16, a_mn, b_mn, kTileRows, half);
        const uint32_t step_a = mma_k_step(a_mn), step_b = mma_k_step(b_mn);
        const int buf = buffers == 2 ? tile & 1 : 0;
        const uint32_t use = buffers == 2 ? tile >> 1 : tile;
        const uint32_t d = tmem + buf * (kTmemCols / 2);
        if (!__all_sync(0xffffffffu, bar_wait(&acc_empty[buf], (use & 1) ^ 1, g.status))) break;
        tc_fence_after();
        for (int kb = k0; kb < k1; ++kb) {
          if (!__all_sync(0xffffffffu, bar_wait(&full[s], phase, g.status))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t addr = tiles0 + s * stage_bytes;
          if (elect_one()) {
            uint64_t a = mma_smem_desc(addr, a_mn);
            uint64_t b = mma_smem_desc(addr + kTileABytes, b_mn);
            if (halves == 1) {
#pragma unroll
              for (int i = 0; i < kDepth / 16; ++i, a += step_a, b += step_b)
                tc_mma<2>(d, a, b, idesc, kb > k0 || i > 0);
            } else {
              uint64_t b2 = mma_smem_desc(addr + kTileABytes + half_bytes, b_mn);
#pragma unroll
              for (int i = 0; i < kDepth / 16; ++i, a += step_a, b += step_b, b2 += step_b) {
                tc_mma_fill(d, a, b, idesc, kb > k0 || i > 0);
                tc_mma_last(d + half, a, b2, idesc, kb > k0 || i > 0);
              }
            }
            tc_commit<2>(&empty[s]);
            if (kb + 1 == k1) tc_commit<2>(&acc_full[buf]);
          }
          __syncwarp();
          if (++s == stages) {
            s = 0;
            phase ^= 1;
          }
        }
        ++tile;
      }
    }
  } else {
    const int quad = warp & 3;             // the tensor-memory lanes this warp can read
    const int turn = (warp - 2) >> 2;      // which of the quadrant's two warps
    const int r_local = quad * 32 + lane;
    const int cols = g.cols;
    Group G;
    G.s = smem_addr(smem) + (uint32_t)kOperandSpace + (warp - 2) * kStageOutBytes;
    G.lane = lane;
    const uint32_t bias = smem_addr(smem) + (uint32_t)kOperandSpace + kEpiWarps * kStageOutBytes +
                          (warp - 2) * kBiasBytes;
    uint32_t tile = 0;
    bool ok = true;  // false once a wait has run out: units pass without results, so that the
                     // block barriers of the split sums still see every warp
    for (int u = worker; u < g.units; u += workers) {
      if (u != worker) w = locate(g, u, w.p);
      const Problem& P = g.p[w.p];
      int k0, k1;
      split_range(P, w.split, &k0, &k1);
      const int buf = buffers == 2 ? tile & 1 : 0;
      const uint32_t use = buffers == 2 ? tile >> 1 : tile;
      const int row0 = w.m0 + (int)rank * kRows + quad * 32;
      const int N = P.N, splits = P.splits;
      const bool sym = P.sym;
      G.rows = max(0, min(32, P.M - row0));
      Out o;
      o.out = reinterpret_cast<uint8_t*>(P.out) + w.z * P.out_zs * 2;
      o.aux = P.aux ? reinterpret_cast<const uint8_t*>(P.aux) + w.z * P.aux_zs * 2 : nullptr;
      o.bias = P.bias;
      o.deriv = P.deriv;
      o.ld = P.ldo;
      o.ld_aux = P.ld_aux;
      o.ld_deriv = P.ld_deriv;
      o.bias_dt = P.bias_dt;
      o.act = P.act;
      const Item* item = EPI == EPI_FINAL ? P.items + w.z : nullptr;
      float alpha = g.alpha;
      if (g.unit_pow) {
        const float unit = P.scale[w.z].unit;
        alpha *= g.unit_pow == 2 ? unit * unit : unit;
      }
      if (k1 > k0 && ok) {
        ok = __all_sync(0xffffffffu, bar_wait(&acc_full[buf], use & 1, g.status));
        tc_fence_after();
      }
      const bool sums = k1 > k0 && ok;
      Sums a;
      a.tmem = tmem + buf * (kTmemCols / 2) + ((uint32_t)(quad * 32) << 16);
      a.parts = nullptr;
      a.splits = splits;
      a.width4 = cols / 4;
      a.row = r_local;
      a.any = sums;
      bool finished = ok;
      if (splits > 1) {
        // this CTA's tile of the split: [split][column / 4][row] float4
        const int64_t tile_id = (int64_t)((u - P.first) / splits) * 2 + rank;
        float4* parts = reinterpret_cast<float4*>(P.split_ws) + tile_id * splits * a.width4 * kRows;
        float4* mine = parts + (int64_t)w.split * a.width4 * kRows + r_local;
        for (int c = turn * 32; c < cols; c += 64) {
          if (w.n0 + c >= N || !sums) break;  // a split has at least one k block
          float v[32];
          tmem_ld32(a.tmem + c, v);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            __stcg(&mine[(c / 4 + i) * kRows],
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
          const bool all = ok && atomicAdd(&P.split_count[tile_id], 1u) == (uint32_t)splits - 1;
          *last_flag = all;
          if (all) P.split_count[tile_id] = 0;  // for the next launch
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
        finished = *last_flag && ok;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
        __threadfence();
        a.parts = parts;
      }
      if (finished && G.rows > 0) {
        for (int c = turn * 64; c < cols; c += 128) {
          const int col = w.n0 + c, n = min(min(64, cols - c), N - col);
          if (n <= 0) break;
          if (sym && col < w.m0) continue;  // left of the diagonal block
          if constexpr (EPI == EPI_FINAL) {
            const int dt = item->out_dt;
            if (dt == DT_BF16) finish_final<DT_BF16>(*item, G, a, alpha, N, row0, col, n, c);
            else if (dt == DT_F32) finish_final<DT_F32>(*item, G, a, alpha, N, row0, col, n, c);
            else finish_final<DT_F16>(*item, G, a, alpha, N, row0, col, n, c);
          } else if constexpr (EPI == EPI_LINEAR) {
            if (o.act == ACT_NONE)
              finish_linear<DT, ACT_NONE>(o, G, bias, a, row0, col, n, c);
            else if (o.act == ACT_RELU)
              finish_linear<DT, ACT_RELU>(o, G, bias, a, row0, col, n, c);
            else if (o.act == ACT_GELU)
              finish_linear<DT, ACT_GELU>(o, G, bias, a, row0, col, n, c);
            else if (o.act == ACT_GELU_TANH)
              finish_linear<DT, ACT_GELU_TANH>(o, G, bias, a, row0, col, n, c);
            else
              finish_linear<DT, ACT_SILU>(o, G, bias, a, row0, col, n, c);
          } else {
            finish<EPI, DT>(g, o, G, a, alpha, row0, col, n, c, sym && col >= w.m0 + kTileRows);
          }
        }
      }
      if (sums && splits == 1) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive_cluster(map_to_rank(smem_addr(&acc_empty[buf]), 0));
      }
      if (sums) ++tile;
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1) tmem_free<2>(tmem, kTmemCols);
}

}  // namespace mx
}  // namespace ta
