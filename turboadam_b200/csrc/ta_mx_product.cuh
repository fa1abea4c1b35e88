// ta_mx_product.cuh -- the tile engine of the matrix operators: one persistent,
// warp-specialised kernel for D[m][n] = epilogue(sum_k A[m][k] B[n][k]) over a
// list of products, on tcgen05 with TMA-fed 128-byte swizzled operand tiles.
//
// Why this shape. A 16-bit tensor-core product on sm_100a takes both operands from shared
// memory, whose 128 bytes per cycle serve the matrix instructions' reads and the TMA writes
// alike. A pair of SMs (cta_group::2) computes a tile of 256 rows by C columns; each SM holds 128
// rows of A and C / 2 rows of B. Per 64 k's that is 16 KB + 64 C bytes written and as many read,
// or 256 + C cycles of shared memory, against 2 C cycles of the tensor pipe: the two balance at
// C = 256, the widest tile of one instruction and the default (14336 x 4096 x 4096: 327 us,
// 1470 TFLOP/s; a pair of 128 x 128 tiles on two SMs would need 512 cycles for 256). Two
// instructions that share A over all 512 columns of tensor memory leave shared memory a quarter
// idle but no second accumulator, and measured 358 us there. Narrower tiles (down to 64 columns)
// give every pair of SMs a share of a small result. Two accumulators let a tile's epilogue run
// under the next tile's products.
//
// Roles of the 19 warps: warps 0 and 1 issue the TMA loads of A and of B, warp 2
// (of the pair's first CTA) the matrix instructions, warps 3..18 are the
// epilogue, four to each 32-row quadrant of tensor memory. They take the tile's
// 32-column chunks in turn and pass them through shared memory, so that every
// global access covers whole sectors of consecutive lines. An epilogue chunk is
// a chain of dependent instructions, some 1500 cycles: sixteen warps rather than
// eight hide twice as much of it.
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
constexpr int kFirstEpi = 3;  // first epilogue warp
constexpr int kEpiWarps = 16;
constexpr int kThreads = 32 * (kFirstEpi + kEpiWarps);
constexpr int kTmemCols = 512;
constexpr int kMaxProblems = 8;  // per launch (they travel as kernel parameters)
constexpr int kLine = 64;                   // bytes of a line of an epilogue block
constexpr int kBlockBytes = 32 * kLine;     // per epilogue warp
constexpr size_t kOperandSpace = 192 * 1024;
constexpr size_t kProductSmem = 1024 + kOperandSpace + kEpiWarps * kBlockBytes + 256;

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
  int32_t n_end;            // columns the epilogue writes: N, or whole chunks of padded lines
  int32_t kblocks;          // blocks of 64 k's in one part of the sum
  int32_t parts;            // the sum runs over this many operand pairs
  int32_t tiles_m, tiles_n, tiles;  // per matrix (tiles: on and above the diagonal, if sym)
  int32_t first;            // first work unit of this problem in the launch
  int32_t batch, splits;
  int32_t za, zb;           // z coordinate of (matrix z, part p): z * za + p * (za > 1)
  int16_t a_mn, b_mn;       // 0: K-major; 1: MN-major, 64 at a time; 2: MN-major in one copy
  int16_t sym, pad0;
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
  int32_t cols;             // tile width C
  int32_t stages;
  int32_t unit_pow;         // scale.unit enters alpha to this power (0, 1 or 2)
  float alpha, c0, c1, c2;
  uint32_t* status;
};

struct Unit {
  int p, z, m0, n0, split;
};

// First tile column of tile row i of a symmetric result: the one that holds the diagonal block's
// first column. Columns left of the diagonal block are skipped by the epilogue, those right of it
// are mirrored, in chunks of 32 columns (which divides 256 and every tile width).
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
  w.split = w.z = 0;
  if (P.splits > 1) {
    w.split = t % P.splits;
    t /= P.splits;
  }
  if (P.batch > 1) {
    w.z = t / P.tiles;
    t -= w.z * P.tiles;
  }
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
    int g0 = 0, rows = P.tiles_m;
    if (rows > 8) {
      const int group = 8 * P.tiles_n, k = t / group;
      g0 = k * 8;
      rows = min(8, rows - g0);
      t -= k * group;
    }
    j = t / rows;
    i = g0 + t - j * rows;
  }
  w.m0 = i * kTileRows;
  w.n0 = j * g.cols;
  return w;
}

// K blocks [*k0, *k1) of a split. (At most 32 splits of at most 2^25 blocks: 32 bits suffice.)
__device__ __forceinline__ void split_range(const Problem& P, int split, int* k0, int* k1) {
  const uint32_t total = (uint32_t)(P.kblocks * P.parts);
  *k0 = 0;
  *k1 = (int)total;
  if (P.splits > 1) {
    *k0 = (int)(total * (uint32_t)split / (uint32_t)P.splits);
    *k1 = (int)(total * (uint32_t)(split + 1) / (uint32_t)P.splits);
  }
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

// ---- epilogue blocks -----------------------------------------------------------
// A warp's block is 32 rows by 64 bytes of the output (32 columns of a 16-bit type, 16 of fp32).
// In registers a thread holds a stretch of one row; in global memory a row is a line. The block's
// shared-memory copy has its 16-byte pieces XORed with the row, which keeps both the row-wise
// accesses (a thread's own row) and the line-wise ones (4 threads a line) free of bank conflicts.
struct Block {
  uint32_t own;   // shared address of this thread's row, and the XOR of its pieces
  uint32_t own_x;
  uint32_t line;  // shared address of this thread's piece of line lane / 4 (and + 8, 16, 24)
  int lane;
  int rows;       // valid rows (0 .. 32)
  uint32_t base;
  __device__ __forceinline__ void init(uint32_t s, int l) {
    base = s;
    lane = l;
    own = s + l * kLine;
    own_x = ((l >> 1) & 3) << 4;
    line = s + (l >> 2) * kLine + (((l & 3) ^ ((l >> 3) & 3)) << 4);
  }
  __device__ __forceinline__ uint32_t piece(int k) const { return own + ((k << 4) ^ own_x); }
  __device__ __forceinline__ uint32_t at(int row, int byte) const {
    return base + row * kLine + ((byte & ~15) ^ (((row >> 1) & 3) << 4)) + (byte & 15);
  }
};

// Lines start on 16 bytes, and the block's columns are all there.
__device__ __forceinline__ bool whole_lines(const void* p, int64_t ld, int n, int size) {
  return n * size == kLine && (((uint32_t)(uintptr_t)p | (uint32_t)(ld * size)) & 15) == 0;
}

// p: the block's first element; n valid columns of SIZE bytes, lines ld elements apart.
template <int SIZE>
__device__ __forceinline__ void block_load(const Block& b, const uint8_t* p, int64_t ld, int n) {
  using T = typename std::conditional<SIZE == 4, uint32_t, uint16_t>::type;
  if (whole_lines(p, ld, n, SIZE)) {
    const int r0 = b.lane >> 2;
    const int64_t step = ld * (8 * SIZE);
    const uint8_t* q = p + r0 * ld * SIZE + (b.lane & 3) * 16;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i, q += step)
      v[i] = r0 + 8 * i < b.rows ? *reinterpret_cast<const uint4*>(q) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) sts16(b.line + i * 8 * kLine, v[i]);
  } else {
    const int per = 16 / SIZE * 4;  // columns of a block
    for (int e = b.lane; e < b.rows * per; e += 32)
      if (e % per < n)
        sts_elem<SIZE>(b.at(e / per, e % per * SIZE),
                       reinterpret_cast<const T*>(p)[e / per * ld + e % per]);
  }
  __syncwarp();
}
template <int SIZE>
__device__ __forceinline__ void block_store(const Block& b, uint8_t* p, int64_t ld, int n) {
  using T = typename std::conditional<SIZE == 4, uint32_t, uint16_t>::type;
  __syncwarp();
  if (whole_lines(p, ld, n, SIZE)) {
    const int r0 = b.lane >> 2;
    const int64_t step = ld * (8 * SIZE);
    uint8_t* q = p + r0 * ld * SIZE + (b.lane & 3) * 16;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lds16(b.line + i * 8 * kLine);
#pragma unroll
    for (int i = 0; i < 4; ++i, q += step)
      if (r0 + 8 * i < b.rows) *reinterpret_cast<uint4*>(q) = v[i];
  } else {
    const int per = 16 / SIZE * 4;
    for (int e = b.lane; e < b.rows * per; e += 32)
      if (e % per < n)
        reinterpret_cast<T*>(p)[e / per * ld + e % per] =
            (T)lds_elem<SIZE>(b.at(e / per, e % per * SIZE));
  }
  __syncwarp();
}
// fn(i, x) for the elements x of this thread's row: 32 of a 16-bit type or 16 of fp32.
template <int DT, typename Fn>
__device__ __forceinline__ void row_get(const Block& b, Fn fn) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint4 u = lds16(b.piece(k));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if constexpr (DT == DT_F32) {
        fn(4 * k + m, __uint_as_float(w[m]));
      } else {
        const float2 f = unpack16(w[m], DT);
        fn(8 * k + 2 * m, f.x);
        fn(8 * k + 2 * m + 1, f.y);
      }
    }
  }
}
template <int DT>
__device__ __forceinline__ void row_put(const Block& b, const float* x) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (DT == DT_F32)
      sts16(b.piece(k), make_uint4(__float_as_uint(x[4 * k]), __float_as_uint(x[4 * k + 1]),
                                   __float_as_uint(x[4 * k + 2]), __float_as_uint(x[4 * k + 3])));
    else
      sts16(b.piece(k),
            make_uint4(pack16(x[8 * k], x[8 * k + 1], DT), pack16(x[8 * k + 2], x[8 * k + 3], DT),
                       pack16(x[8 * k + 4], x[8 * k + 5], DT),
                       pack16(x[8 * k + 6], x[8 * k + 7], DT)));
  }
}

// Where a chunk's finished sums come from: tensor memory, the split workspace, or nothing (an
// empty sum).
struct Sums {
  uint32_t tmem;        // first column of the tile, this warp's lanes
  const float4* parts;  // this tile's splits, or null
  int splits, width4;   // number of them; float4 columns of one
  int row;              // in the CTA's tile
  bool any;
  int last;             // after this column's chunk the warp is done with the accumulator ...
  uint32_t done;        // ... and arrives here
};
__device__ __forceinline__ void release_sums(const Sums& a) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) bar_arrive_cluster(a.done);
}
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
    if (c == a.last) release_sums(a);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0.f;
  }
}

// What the epilogue reads of a tile's problem, in registers.
struct Out {
  uint8_t* out;
  const uint8_t* aux;
  const void* bias;
  int16_t* deriv;
  int64_t ld, ld_aux, ld_deriv;
  int bias_dt, act;
};

// A chunk of the orthogonalised update, stored or applied to the parameter.
template <int DT>
__device__ __forceinline__ void finish_final(const Item& it, const Block& b, float (&v)[32],
                                             float alpha, int64_t ld, int64_t row0, int col,
                                             int n) {
  constexpr int kSize = DT == DT_F32 ? 4 : 2, kCols = kLine / kSize;
  uint8_t* p = reinterpret_cast<uint8_t*>(it.out) + (row0 * ld + col) * kSize;
  const float keep = it.keep, gain = it.gain * alpha;
#pragma unroll
  for (int q = 0; q < 32; q += kCols) {
    const int m = min(kCols, n - q);
    if (m <= 0) break;
    float* x = v + q;
    if (it.update) {
      block_load<kSize>(b, p + q * kSize, ld, m);
      row_get<DT>(b, [&](int i, float old) { x[i] = fmaf(-gain, x[i], keep * old); });
    } else {
#pragma unroll
      for (int i = 0; i < kCols; ++i) x[i] *= alpha;
    }
    row_put<DT>(b, x);
    block_store<kSize>(b, p + q * kSize, ld, m);
  }
}

// The activation of a chunk; its derivative's codes go out 64 bytes a row, in whole sectors (the
// rows of codes are padded to whole 16-byte pieces).
template <int ACT, bool DERIV>
__device__ __forceinline__ void activate_row(float (&v)[32], int16_t* q, int n, bool row_ok) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t code[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      float d0 = 0.f, d1 = 0.f;
      activate<DERIV>(ACT, v[8 * k + 2 * m], &v[8 * k + 2 * m], &d0);
      activate<DERIV>(ACT, v[8 * k + 2 * m + 1], &v[8 * k + 2 * m + 1], &d1);
      if (DERIV)
        code[m] = (uint32_t)(uint16_t)encode_deriv(d0) | ((uint32_t)(uint16_t)encode_deriv(d1) << 16);
    }
    if (DERIV && row_ok && 8 * k < n)
      *reinterpret_cast<uint4*>(q + 8 * k) = make_uint4(code[0], code[1], code[2], code[3]);
  }
}
template <int ACT>
__device__ __forceinline__ void activate_chunk(const Out& o, const Block& b, float (&v)[32],
                                               int64_t row0, int col, int n) {
  if (o.deriv)
    activate_row<ACT, true>(v, o.deriv + (row0 + b.lane) * o.ld_deriv + col, n, b.lane < b.rows);
  else
    activate_row<ACT, false>(v, nullptr, n, false);
}
template <int DT>
__device__ __forceinline__ void finish_linear(const Out& o, const Block& b, float (&v)[32],
                                              int64_t row0, int col, int n) {
  if (o.bias) {  // lane j loads column j's, and all lanes take it from the block
    sts_elem<4>(b.base + b.lane * 4, __float_as_uint(b.lane < n ? load_as_float(o.bias, col + b.lane, o.bias_dt) : 0.f));
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint4 u = lds16(b.base + k * 16);
      v[4 * k] += __uint_as_float(u.x);
      v[4 * k + 1] += __uint_as_float(u.y);
      v[4 * k + 2] += __uint_as_float(u.z);
      v[4 * k + 3] += __uint_as_float(u.w);
    }
    __syncwarp();
  }
  if (o.act == ACT_RELU) activate_chunk<ACT_RELU>(o, b, v, row0, col, n);
  else if (o.act == ACT_GELU) activate_chunk<ACT_GELU>(o, b, v, row0, col, n);
  else if (o.act == ACT_GELU_TANH) activate_chunk<ACT_GELU_TANH>(o, b, v, row0, col, n);
  else if (o.act == ACT_SILU) activate_chunk<ACT_SILU>(o, b, v, row0, col, n);
  if (o.aux) {
    block_load<2>(b, o.aux + (row0 * o.ld_aux + col) * 2, o.ld_aux, n);
    row_get<DT>(b, [&](int i, float r) { v[i] += r; });
  }
  row_put<DT>(b, v);
  block_store<2>(b, o.out + (row0 * o.ld + col) * 2, o.ld, n);
}

// One chunk: the sums of rows [row0, row0 + 32) by columns [col, col + n) of the result. DT is
// the type of the result (EPI_LINEAR, EPI_PLAIN); `mirror`: a symmetric result's chunk right of
// the diagonal block, also written transposed (a warp's 32 rows are 64 consecutive bytes).
template <int EPI, int DT>
__device__ __forceinline__ void finish(const ProductArgs& g, const Out& o, const Item* it,
                                       const Block& b, float (&v)[32], float alpha, int64_t row0,
                                       int col, int n, bool mirror, int N) {
  if constexpr (EPI == EPI_GRAM || EPI == EPI_POLY || EPI == EPI_APPLY) {
    if constexpr (EPI == EPI_POLY) {
      block_load<2>(b, o.aux + (row0 * o.ld_aux + col) * 2, o.ld_aux, n);
      const int diag = (int)row0 + b.lane - col;
      row_get<DT_F16>(b, [&](int i, float x) {
        v[i] = fmaf(g.c2, v[i], fmaf(g.c1, x, diag == i ? g.c0 : 0.f));
      });
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= alpha;
    }
    row_put<DT_F16>(b, v);
    if (EPI != EPI_APPLY && mirror && b.lane < b.rows) {
      __half* t = reinterpret_cast<__half*>(o.out) + col * o.ld + row0 + b.lane;
#pragma unroll
      for (int i = 0; i < 32; ++i, t += o.ld)
        if (i < N - col) *t = __float2half_rn(v[i]);  // n may run into the lines' padding
    }
    block_store<2>(b, o.out + (row0 * o.ld + col) * 2, o.ld, n);
  } else if constexpr (EPI == EPI_FINAL) {
    const int dt = it->out_dt;
    if (dt == DT_BF16) finish_final<DT_BF16>(*it, b, v, alpha, N, row0, col, n);
    else if (dt == DT_F32) finish_final<DT_F32>(*it, b, v, alpha, N, row0, col, n);
    else finish_final<DT_F16>(*it, b, v, alpha, N, row0, col, n);
  } else if constexpr (EPI == EPI_LINEAR) {
    finish_linear<DT>(o, b, v, row0, col, n);
  } else {
    row_put<DT>(b, v);
    block_store<2>(b, o.out + (row0 * o.ld + col) * 2, o.ld, n);
  }
}

template <int EPI, int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    k_product(const __grid_constant__ ProductArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full =
      reinterpret_cast<uint64_t*>(smem + kOperandSpace + kEpiWarps * kBlockBytes);
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_full = empty + kMaxStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile uint32_t* last_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int worker = blockIdx.x / 2, workers = gridDim.x / 2;
  const int cols = g.cols, stages = g.stages;
  const uint32_t stage_bytes = kTileABytes + cols * (kDepth * 2 / 2);
  const uint32_t tiles0 = smem_addr(smem);

  if (warp == 0) {  // full, empty, acc_full: one arrival; acc_empty: one of each epilogue warp
    constexpr int kBars = 2 * kMaxStages + 4;
    if (lane < kBars) bar_init(&full[lane], lane < kBars - 2 ? 1 : 2 * kEpiWarps);
    bar_init_fence();
  }
  if (warp == 2) tmem_alloc(tmem_slot, kTmemCols);
  Unit w = locate(g, worker, 0);  // the first unit is looked up under the set-up's latency
  if (warp < 2 && elect_one()) tma_prefetch(warp == 0 ? &g.p[w.p].ta : &g.p[w.p].tb);
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *(volatile uint32_t*)tmem_slot;
  chain_next();
  chain_wait();

  if (warp < 2) {
    const bool is_a = warp == 0;
    const uint32_t full0 = map_to_rank(smem_addr(full), 0);  // the first CTA's barriers count both
    uint32_t filled = 0;  // stages filled so far
    int s = 0;
    uint32_t phase = 1;   // of "empty": the first round finds every stage free
    bool ok = true;
    for (int u = worker; u < g.units && ok; u += workers) {
      if (u != worker) w = locate(g, u, w.p);
      const Problem& P = g.p[w.p];
      int k0, k1;
      split_range(P, w.split, &k0, &k1);
      const CUtensorMap* map = is_a ? &P.ta : &P.tb;
      const int kind = is_a ? P.a_mn : P.b_mn, zs = is_a ? P.za : P.zb;
      const int mn = is_a ? w.m0 + (int)rank * kRows : w.n0 + (int)rank * (cols / 2);
      const int chunks = is_a ? 2 : cols / 128;
      const int kblocks = P.kblocks;
      int z = w.z * zs, k = k0 * kDepth;
      if (k0 >= kblocks) {  // the second operand pair of the sum
        k -= kblocks * kDepth;
        z += zs > 1;
      }
      for (int kb = k0; kb < k1; ++kb, k += kDepth) {
        if (kb == kblocks && kb > k0) {
          k = 0;
          z += zs > 1;
        }
        if (!__all_sync(0xffffffffu, bar_wait(&empty[s], phase, g.status))) {
          ok = false;
          break;
        }
        if (elect_one()) {
          const uint32_t bar = full0 + s * 8;
          const uint32_t dst = tiles0 + s * stage_bytes + (is_a ? 0 : kTileABytes);
          if (is_a && rank == 0) bar_expect_tx(&full[s], 2 * stage_bytes);
          if (kind == 0) {
            tma_load(map, dst, bar, k, mn, z);
          } else if (kind == 2) {
            tma_load4(map, dst, bar, k, mn >> 6, z);
          } else {
            for (int c = 0; c < chunks; ++c)
              tma_load(map, dst + c * 8192, bar, mn + c * 64, k, z);
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
  } else if (warp == 2) {
    if (rank == 0) {
      uint32_t tile = 0, phase = 0;
      int s = 0;
      bool ok = true;
      for (int u = worker; u < g.units && ok; u += workers) {
        if (u != worker) w = locate(g, u, w.p);
        const Problem& P = g.p[w.p];
        int k0, k1;
        split_range(P, w.split, &k0, &k1);
        if (k0 == k1) continue;  // an empty sum: the epilogue takes zeros
        const bool a_mn = P.a_mn, b_mn = P.b_mn;
        const uint32_t idesc = mma_idesc(g.bf16, a_mn, b_mn, kTileRows, cols);
        const uint32_t step_a = mma_k_step(a_mn), step_b = mma_k_step(b_mn);
        const int buf = tile & 1;
        const uint32_t use = tile >> 1;
        const uint32_t d = tmem + buf * (kTmemCols / 2);
        if (!__all_sync(0xffffffffu, bar_wait(&acc_empty[buf], (use & 1) ^ 1, g.status))) break;
        tc_fence_after();
        for (int kb = k0; kb < k1; ++kb) {
          if (!__all_sync(0xffffffffu, bar_wait(&full[s], phase, g.status))) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t addr = tiles0 + s * stage_bytes;
            uint64_t a = mma_smem_desc(addr, a_mn);
            uint64_t b = mma_smem_desc(addr + kTileABytes, b_mn);
#pragma unroll
            for (int i = 0; i < kDepth / 16; ++i, a += step_a, b += step_b)
              tc_mma(d, a, b, idesc, kb > k0 || i > 0);
            tc_commit(&empty[s]);
            if (kb + 1 == k1) tc_commit(&acc_full[buf]);
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
    const int quad = warp & 3;                    // the tensor-memory lanes this warp can read
    const int turn = (warp - kFirstEpi) >> 2;     // which of the quadrant's four warps
    Block b;
    b.init(tiles0 + (uint32_t)kOperandSpace + (warp - kFirstEpi) * kBlockBytes, lane);
    uint32_t tile = 0;
    bool ok = true;  // false once a wait has run out: units pass without results, so that the
                     // block barriers of the split sums still see every warp
    for (int u = worker; u < g.units; u += workers) {
      if (u != worker) w = locate(g, u, w.p);
      const Problem& P = g.p[w.p];
      int k0, k1;
      split_range(P, w.split, &k0, &k1);
      const int buf = tile & 1;
      const uint32_t use = tile >> 1;
      const int64_t row0 = w.m0 + (int)rank * kRows + quad * 32;
      const int N = P.N, n_end = P.n_end, splits = P.splits;
      const bool sym = P.sym;
      b.rows = (int)max((int64_t)0, min((int64_t)32, P.M - row0));
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
      Sums a;
      a.tmem = tmem + buf * (kTmemCols / 2) + ((uint32_t)(quad * 32) << 16);
      a.parts = nullptr;
      a.splits = splits;
      a.width4 = cols / 4;
      a.row = quad * 32 + lane;
      a.done = map_to_rank(smem_addr(&acc_empty[buf]), 0);
      // this warp's chunks: accumulator columns turn * 32 + 128 i, of which it takes those inside
      // the result and not left of a symmetric result's diagonal block
      auto wanted = [&](int c) {
        const int col = w.n0 + c;
        return col < n_end && b.rows > 0 && !(sym && col < w.m0);
      };
      a.last = -1;
      if (splits == 1)
        for (int c = turn * 32; c < cols; c += 128)
          if (wanted(c)) a.last = c;
      if (k1 > k0 && ok) {
        ok = __all_sync(0xffffffffu, bar_wait(&acc_full[buf], use & 1, g.status));
        tc_fence_after();
      }
      const bool sums = k1 > k0 && ok;
      a.any = sums;
      bool finished = ok;
      if (splits > 1) {
        // this CTA's tile of the split: [split][column / 4][row] float4
        const int64_t tile_id = (int64_t)((u - P.first) / splits) * 2 + rank;
        float4* parts = reinterpret_cast<float4*>(P.split_ws) + tile_id * splits * a.width4 * kRows;
        float4* mine = parts + (int64_t)w.split * a.width4 * kRows + a.row;
        for (int c = turn * 32; c < cols; c += 128) {
          if (!sums || !wanted(c)) continue;  // a split has at least one k block
          float v[32];
          tmem_ld32(a.tmem + c, v);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            __stcg(&mine[(c / 4 + i) * kRows],
                   make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
        }
        if (sums) release_sums(a);
        __threadfence();
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
        if (threadIdx.x == 32 * kFirstEpi) {
          const bool all = ok && atomicAdd(&P.split_count[tile_id], 1u) == (uint32_t)splits - 1;
          *last_flag = all;
          if (all) P.split_count[tile_id] = 0;  // for the next launch
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
        finished = *last_flag && ok;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
        __threadfence();
        a.parts = parts;
      } else if (sums && a.last < 0) {
        release_sums(a);
      }
      if (finished) {
        for (int c = turn * 32; c < cols; c += 128) {
          if (!wanted(c)) continue;
          const int col = w.n0 + c;
          float v[32];
          take_sums(a, c, v);
          finish<EPI, DT>(g, o, item, b, v, alpha, row0, col, min(32, n_end - col),
                          sym && col >= w.m0 + kTileRows, N);
        }
      }
      if (sums) ++tile;
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  if (warp == 2) tmem_free(tmem, kTmemCols);
}

}  // namespace mx
}  // namespace ta
