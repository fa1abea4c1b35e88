// ta_mx_product.cuh -- the tile engine of the matrix operators: one persistent,
// warp-specialised kernel for D[m][n] = epilogue(sum_k A[m][k] B[n][k]) over a
// list of products, on tcgen05 with TMA-fed 128-byte swizzled operand tiles.
//
// Why this shape. A 16-bit tensor-core product on sm_100a takes both operands from shared
// memory, whose 128 bytes per cycle serve the matrix instructions' reads and the TMA writes
// alike. A pair of SMs (cta_group::2) computes a tile of 256 rows by C columns; each SM holds 128
// rows of A and C / 2 rows of B. Per 64 k's that is 16 KB + 64 C bytes written and as many read,
// or 256 + C cycles of shared memory, against 2 C cycles of the tensor pipe: the two balance at
// C = 256, the widest tile of one instruction and the default (14336 x 4096 x 4096: 319 us,
// 1510 TFLOP/s; a pair of 128 x 128 tiles on two SMs would need 512 cycles for 256). Two
// instructions that share A over all 512 columns of tensor memory leave shared memory a quarter
// idle but no second accumulator, and measured 358 us there. Narrower tiles (down to 64 columns)
// give every pair of SMs a share of a small result. Two accumulators let a tile's epilogue run
// under the next tile's products.
//
// Roles of the 12 warps: warps 0 and 1 issue the TMA loads of A and of B, warp 2
// (of the pair's first CTA) the matrix instructions, warp 3 rests, warps 4..11
// are the epilogue, two to each 32-row quadrant of tensor memory. They take the
// tile's 32-column chunks in turn and pass them through shared memory, so that
// every global access covers whole sectors of consecutive lines. Eight warps
// leave each thread 168 registers; twelve and sixteen spilled and were slower
// (12 x 768 x 768 orthogonalised: 207, 244 and 255 us), four had too little
// under way (225 us).
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
constexpr int kFirstEpi = 4;  // first epilogue warp
constexpr int kTurns = 2;     // epilogue warps of a quadrant
constexpr int kEpiWarps = 4 * kTurns;
constexpr int kEpiStep = 32 * kTurns;  // a warp's chunks are this many columns apart
constexpr int kThreads = 32 * (kFirstEpi + kEpiWarps);
constexpr int kTmemCols = 512;
constexpr int kLine = 64;                   // bytes of a line of an epilogue block
constexpr int kBlockBytes = 32 * kLine;     // per epilogue warp
constexpr size_t kOperandSpace = 192 * 1024;
constexpr size_t kProductSmem = 1024 + kOperandSpace + kEpiWarps * kBlockBytes + 256;

// Per-matrix scale of a Newton-Schulz list: the stored fp16 input times `unit` is the
// normalised matrix (unit is NaN where the input holds a NaN or an infinity).
struct Scale {
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

// One product D[m][n] = sum_k A[m][k] B[n][k] of a launch, or of a phase of a chain: `batch`
// independent ones of one shape.
struct Problem {
  int32_t M, N;
  int32_t n_end;            // columns the epilogue writes: N, or whole chunks of padded lines
  int32_t kblocks;          // blocks of 64 k's in one part of the sum
  int32_t tiles_m, tiles_n, tiles;  // per matrix (tiles: on and above the diagonal, if sym)
  int32_t first;            // first work unit of this problem in the launch
  int32_t batch, splits;
  int16_t a_kind, b_kind;   // 0: K-major; 1: MN-major, 64 at a time; 2: MN-major in one copy
  int16_t sym;              // the result is symmetric
  int16_t a_sym, b_sym;     // the operand is (K-major; 1 or 2 of the kinds where transposed)
  int16_t pad0;
  float* split_ws;          // [unit / splits][splits][rows x columns of a CTA tile]
  uint32_t* split_count;    // zero before and after every launch
};

struct Unit {
  int p, z, m0, n0, split;
};

// A symmetric matrix is computed and stored in its upper triangle of 256 x 256 blocks only: row r
// from column r & ~255 on. Tile row i of a symmetric result starts at tile column sym_first (tile
// widths divide 256). As an operand, a block of k's left of the rows' diagonal block is read
// transposed: the element (r, k) at (k, r), MN-major where the rest of the operand is K-major.
__host__ __device__ __forceinline__ int sym_first(int i, int cols) { return i * kTileRows / cols; }

// Work unit u of the launch. Tiles of a general product run down groups of 8 tile rows, so that
// the CTAs in flight share operand tiles in L2; splits of one tile are neighbours.
template <class View>
__device__ __forceinline__ Unit locate(const View& v, int u, int p_hint) {
  Unit w;
  int p = p_hint;
  while (p + 1 < v.count() && u >= v.problem(p + 1).first) ++p;
  const Problem& P = v.problem(p);
  const int cols = v.cols();
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
      const int n = P.tiles_n - sym_first(i, cols);
      if (t < n) break;
      t -= n;
      ++i;
    }
    j = sym_first(i, cols) + t;
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
  w.n0 = j * cols;
  return w;
}

// K blocks [*k0, *k1) of a split. (At most 16 splits of at most 2^26 blocks: 32 bits suffice.)
__device__ __forceinline__ void split_range(const Problem& P, int parts, int split, int* k0,
                                            int* k1) {
  const uint32_t total = (uint32_t)(P.kblocks * parts);
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
//
// An epilogue has two warps a scheduler, so a call with branches inside (erfcf, the full forms of
// expf and of the division) leaves its latency bare: with these 8192 x 512 > 4096 takes 51, 55 and
// 61 us for SiLU, tanh-GELU and GELU, with those it took 104, 186 and 96 (32 without activation).
// The forms here have no branch, use the hardware's exponential and reciprocal (__expf,
// __fdividef), and saturate by themselves: exp(-z) = inf gives a sigmoid of 0. Relative to a sigmoid
// or a Phi they are off by a few 1e-7 where it is not small; the exponential's error grows with its
// argument, to some 1e-5 of a Phi of 1e-19 at z = -9, still 1/40 of an fp16's rounding.
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
// exp(u^2 / 2) Phi(-u) for u >= 0, Hastings' form: a polynomial in t = 1 / (1 + p u) without a
// constant term. Its coefficients are a least-maximum fit of the relative error: 4e-7 up to u = 9
// (beyond, Phi(-u) is under 1e-18).
__device__ __forceinline__ float phi_tail(float u) {
  const float t = __fdividef(1.f, fmaf(0.35f, u, 1.f));
  float q = fmaf(0.0466097929f, t, -0.192525774f);
  q = fmaf(q, t, 0.224254504f);
  q = fmaf(q, t, -0.00198693108f);
  q = fmaf(q, t, 0.147971243f);
  q = fmaf(q, t, 0.135809943f);
  q = fmaf(q, t, 0.139867052f);
  return q * t;
}
template <bool DERIV>
__device__ __forceinline__ void activate(int act, float z, float* y, float* d) {
  if (act == ACT_RELU) {
    *y = z < 0.f ? 0.f : z;  // keeps NaN
    if (DERIV) *d = z > 0.f ? 1.f : (z != z ? z : 0.f);
  } else if (act == ACT_GELU) {  // z Phi(z); derivative Phi(z) + z phi(z)
    const float e = __expf(-0.5f * z * z), tail = e * phi_tail(fabsf(z));
    const float cdf = z < 0.f ? tail : 1.f - tail;
    *y = z == -INFINITY ? 0.f : z * cdf;
    if (DERIV) *d = fabsf(z) == INFINITY ? cdf : fmaf(z * 0.39894228f, e, cdf);
  } else if (act == ACT_GELU_TANH) {  // z sigmoid(2 u), u = sqrt(2/pi) (z + 0.044715 z^3)
    const float s = sigmoid(1.59576912f * z * fmaf(0.044715f * z, z, 1.f));
    *y = z == -INFINITY ? 0.f : z * s;
    if (DERIV) {
      const float du2 = fmaf(0.214063f * z, z, 1.59576912f);
      const float t = s * (1.f - s);
      *d = t == 0.f ? s : fmaf(z * t, du2, s);
    }
  } else if (act == ACT_SILU) {  // z sigmoid(z)
    const float s = sigmoid(z);
    *y = z == -INFINITY ? 0.f : z * s;
    if (DERIV) {
      const float t = s * (1.f - s);
      *d = t == 0.f ? s : fmaf(z, t, s);
    }
  } else {
    *y = z;
    if (DERIV) *d = z != z ? z : 1.f;
  }
}

// An activation's derivative lies in (-0.13, 1.13) and is kept in 16 bits: from kLow on in steps
// of 2^-14, below in floating point of kMant mantissa bits, whose steps are no larger. So it is off
// by at most 2^-15, and relative to itself by at most 2^-9 for bf16 (down to 2^-93; beyond, by
// 2^-102) and 2^-12 for fp16 (down to 2^-13; beyond, by 2^-25, half a step of fp16's own smallest
// numbers): half of what rounding dz to the type costs next, in the activations' far negative tails
// too. (Steps of 2^-14 throughout left SiLU' 10 % off at -12 and zero from -13 on. They took as
// long in the forward pass, 75 us for 8192 x 512 > 4096 with SiLU, and 1 to 2 us less in a backward
// pass: both together 73 us against 74.5 for 9714 x 1920 > 256, 32.2 against 33.6 for 777 x 1001 >
// 1003.)
// Codes: [0, kDerivCodes) the floating ones in order, then the steps; kDerivNeg is added for a
// negative number, and what a NaN leaves in the low bits (0xffff of the one NaN that arithmetic
// gives) stands for NaN.
constexpr uint32_t kDerivCodes = 22528, kDerivNeg = 41001, kDerivNan = 0xffff;
template <int DT>
struct DerivCode {
  static constexpr int kMant = DT == DT_BF16 ? 8 : 11, kShift = 23 - kMant;
  static constexpr float kLow = DT == DT_BF16 ? 0x1p-6f : 0x1p-3f;  // 2^(kMant - 14)
  // kLow * kDown is the float whose upper bits are kDerivCodes; small ones become subnormal there
  static constexpr float kDown = DT == DT_BF16 ? 0x1p-33f : 0x1p-113f;
  static constexpr float kUp = DT == DT_BF16 ? 0x1p33f : 0x1p113f;
  // added to d * 2^14 it leaves the code in the float's low bits
  static constexpr float kAdd = 8388608.f + kDerivCodes - kLow * 16384.f;
  static constexpr uint32_t kOne = (uint32_t)(16384.f + kAdd - 8388608.f);  // of d = 1
};
// The code in the low 16 bits; what is above is to be dropped.
template <int DT>
__device__ __forceinline__ uint32_t encode_deriv(float d) {
  using C = DerivCode<DT>;
  const float m = fabsf(d);
  const uint32_t low = (__float_as_uint(m * C::kDown) + (1u << (C::kShift - 1))) >> C::kShift;
  const uint32_t high = __float_as_uint(fmaf(m, 16384.f, C::kAdd));
  uint32_t code = m < C::kLow ? low : high;
  if (d < 0.f) code += kDerivNeg;
  return code;
}
// q: 16 bits
template <int DT>
__device__ __forceinline__ float decode_deriv(uint32_t q) {
  using C = DerivCode<DT>;
  const bool neg = q >= kDerivNeg;
  const uint32_t code = neg ? q - kDerivNeg : q;
  const float low = __uint_as_float(code << C::kShift) * C::kUp;
  const float high = fmaf(__uint_as_float(0x4B000000u | code), 0x1p-14f, -C::kAdd * 0x1p-14f);
  const float m = code < kDerivCodes ? low : high;
  return q == kDerivNan ? __int_as_float(0x7fc00000) : neg ? -m : m;
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

// p: the block's first element; n valid columns of SIZE bytes, lines ld elements apart. WHOLE: its
// lines are known to be whole.
template <int SIZE, bool WHOLE = false>
__device__ __forceinline__ void block_load(const Block& b, const uint8_t* p, int64_t ld, int n) {
  using T = typename std::conditional<SIZE == 4, uint32_t, uint16_t>::type;
  if (WHOLE || whole_lines(p, ld, n, SIZE)) {
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
    constexpr int kPer = kLine / SIZE, kStep = 32 / kPer;  // columns of a block; rows at a time
    const int c = b.lane % kPer;
    const T* q = reinterpret_cast<const T*>(p) + c;
    for (int r0 = b.lane / kPer; r0 < b.rows; r0 += 8 * kStep) {
      T v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = r0 + i * kStep < b.rows && c < n ? q[(r0 + i * kStep) * ld] : (T)0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r0 + i * kStep < b.rows) sts_elem<SIZE>(b.at(r0 + i * kStep, c * SIZE), v[i]);
    }
  }
  __syncwarp();
}
template <int SIZE, bool WHOLE = false>
__device__ __forceinline__ void block_store(const Block& b, uint8_t* p, int64_t ld, int n) {
  using T = typename std::conditional<SIZE == 4, uint32_t, uint16_t>::type;
  __syncwarp();
  if (WHOLE || whole_lines(p, ld, n, SIZE)) {
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
    constexpr int kPer = kLine / SIZE, kStep = 32 / kPer;
    const int c = b.lane % kPer;
    T* q = reinterpret_cast<T*>(p) + c;
#pragma unroll 8
    for (int r = b.lane / kPer; r < b.rows; r += kStep)
      if (c < n) q[r * ld] = (T)lds_elem<SIZE>(b.at(r, c * SIZE));
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

// Where a tile goes, and what its epilogue reads.
struct Out {
  uint8_t* out;
  const uint8_t* aux;
  const void* bias;
  int16_t* deriv;
  int64_t ld, ld_aux, ld_deriv;
  int bias_dt, act;
};

__device__ __forceinline__ void epilogue_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
}

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
template <int DT, int ACT, bool DERIV>
__device__ __forceinline__ void activate_row(float (&v)[32], int16_t* q, int n, bool row_ok) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t code[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      uint32_t c[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float z = v[8 * k + 2 * m + j];
        float d = 0.f;
        activate<DERIV>(ACT, z, &v[8 * k + 2 * m + j], &d);
        if (ACT == ACT_RELU) c[j] = z > 0.f ? DerivCode<DT>::kOne : z != z ? kDerivNan : 0u;
        else c[j] = encode_deriv<DT>(d);
      }
      code[m] = __byte_perm(c[0], c[1], 0x5410);
    }
    if (DERIV && row_ok && 8 * k < n)
      *reinterpret_cast<uint4*>(q + 8 * k) = make_uint4(code[0], code[1], code[2], code[3]);
  }
}
template <int DT, int ACT>
__device__ __forceinline__ void activate_chunk(const Out& o, const Block& b, float (&v)[32],
                                               int64_t row0, int col, int n) {
  if (o.deriv)
    activate_row<DT, ACT, true>(v, o.deriv + (row0 + b.lane) * o.ld_deriv + col, n, b.lane < b.rows);
  else
    activate_row<DT, ACT, false>(v, nullptr, n, false);
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
  if (o.act == ACT_RELU) activate_chunk<DT, ACT_RELU>(o, b, v, row0, col, n);
  else if (o.act == ACT_GELU) activate_chunk<DT, ACT_GELU>(o, b, v, row0, col, n);
  else if (o.act == ACT_GELU_TANH) activate_chunk<DT, ACT_GELU_TANH>(o, b, v, row0, col, n);
  else if (o.act == ACT_SILU) activate_chunk<DT, ACT_SILU>(o, b, v, row0, col, n);
  if (o.aux) {
    block_load<2>(b, o.aux + (row0 * o.ld_aux + col) * 2, o.ld_aux, n);
    row_get<DT>(b, [&](int i, float r) { v[i] += r; });
  }
  row_put<DT>(b, v);
  block_store<2>(b, o.out + (row0 * o.ld + col) * 2, o.ld, n);
}

// One chunk of a Newton-Schulz matrix: the sums v of rows [row0, row0 + 32) by columns
// [col, col + 32), stored in fp16 as alpha v, or as the polynomial c0 I + c1 A + alpha v of
// A = aux. Its lines are padded to whole chunks: no ragged edge.
template <bool POLY>
__device__ __forceinline__ void finish_half(uint8_t* out, int64_t ld, const uint8_t* aux,
                                            int64_t ld_aux, const Block& b, float (&v)[32],
                                            float alpha, float c0, float c1, int64_t row0,
                                            int col) {
  if constexpr (POLY) {
    block_load<2, true>(b, aux + (row0 * ld_aux + col) * 2, ld_aux, 32);
    row_get<DT_F16>(b, [&](int i, float x) { v[i] = fmaf(alpha, v[i], c1 * x); });
    if (row0 == col) {  // both are multiples of 32: the diagonal is in this chunk or not
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += b.lane == i ? c0 : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= alpha;
  }
  row_put<DT_F16>(b, v);
  block_store<2, true>(b, out + (row0 * ld + col) * 2, ld, 32);
}

// ---- roles -----------------------------------------------------------------------
// A CTA's shared-memory layout and place in the launch.
struct Cta {
  uint32_t tiles0;          // shared address of the operand stages
  uint32_t full, empty;     // barriers, [kMaxStages] each
  uint32_t acc_full, acc_empty;  // [2]
  uint32_t last_flag;
  uint32_t tmem;
  uint32_t rank;            // in the pair
  int worker, workers;      // this pair, pairs
  int stages;
  uint32_t stage_bytes;
  uint32_t* status;
};

// Where a copy warp or the matrix warp stands in the ring of stages.
struct Ring {
  uint32_t count = 0;  // stages filled (or tiles computed) so far
  int s = 0;
  uint32_t phase;
  bool ok = true;      // false once a wait has run out
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
};

// Each role looks up its first unit, then passes `gate` (once, units or not), then touches memory:
// what comes before (some 1500 cycles of parameters and index arithmetic) runs while the kernel or
// phase before drains. gate() returns false if its wait ran out.

// Warp 0 (A) or 1 (B): the loads of this pair's units. Both CTAs' bytes are counted on the first
// CTA's barriers.
template <class View, class Gate>
__device__ __forceinline__ void copy_units(const View& v, const Cta& x, Ring& r, Unit w, bool is_a,
                                           Gate gate) {
  bool shut = true;
  const uint32_t full0 = map_to_rank(x.full, 0);
  const int cols = v.cols(), units = v.units();
  const uint32_t bytes = 2 * (kTileABytes + cols * kDepth);
  for (int u = x.worker; u < units && r.ok; u += x.workers) {
    if (u != x.worker) w = locate(v, u, w.p);
    const Problem& P = v.problem(w.p);
    int k0, k1;
    split_range(P, v.parts(w.p), w.split, &k0, &k1);
    const CUtensorMap* map = is_a ? v.map_a(w.p) : v.map_b(w.p);
    const int zs = is_a ? v.za(w.p) : v.zb(w.p);
    const int other = is_a ? P.a_sym : P.b_sym;  // how the transposed blocks come, if any
    const int mn = is_a ? w.m0 + (int)x.rank * kRows : w.n0 + (int)x.rank * (cols / 2);
    const int chunks = is_a ? 2 : cols / 128;
    const int kind0 = is_a ? P.a_kind : P.b_kind;
    const int diag = other ? mn & ~(kTileRows - 1) : 0;
    const CUtensorMap* map_t = other ? (is_a ? v.map_a_t(w.p) : v.map_b_t(w.p)) : map;
    const int kblocks = P.kblocks;
    int z = w.z * zs, k = k0 * kDepth;
    if (k0 >= kblocks) {  // the second operand pair of the sum
      k -= kblocks * kDepth;
      z += zs > 1;
    }
    if (shut) {
      if (elect_one()) tma_prefetch(k < diag ? map_t : map);
      __syncwarp();
      asm volatile("" ::"l"(map), "l"(map_t), "r"(kind0), "r"(mn), "r"(z), "r"(k), "r"(k1),
                   "r"(kblocks));
      shut = false;
      r.ok = gate() && r.ok;
    }
    for (int kb = k0; kb < k1 && r.ok; ++kb, k += kDepth) {
      if (kb == kblocks && kb > k0) {
        k = 0;
        z += zs > 1;
      }
      if (!__all_sync(0xffffffffu, bar_wait(x.empty + 8 * r.s, r.phase, x.status))) {
        r.ok = false;
        break;
      }
      if (elect_one()) {
        const uint32_t bar = full0 + r.s * 8;
        const uint32_t dst = x.tiles0 + r.s * x.stage_bytes + (is_a ? 0 : kTileABytes);
        if (is_a && x.rank == 0) bar_expect_tx(x.full + 8 * r.s, bytes);
        const int kind = k < diag ? other : kind0;
        const CUtensorMap* m = k < diag ? map_t : map;
        if (kind == 0) {
          tma_load(m, dst, bar, k, mn, z);
        } else if (kind == 2) {
          tma_load4(m, dst, bar, k, mn >> 6, z);
        } else {
          for (int c = 0; c < chunks; ++c)
            tma_load(m, dst + c * 8192, bar, mn + c * 64, k, z);
        }
      }
      __syncwarp();
      ++r.count;
      r.next(x.stages);
    }
  }
  if (shut) r.ok = gate() && r.ok;
}
// Leaves no copy in flight: every stage that was filled has been read (its "empty" phase
// completes), which the waits of a complete run establish here, each of them bounded.
__device__ __forceinline__ void copy_drain(const Cta& x, Ring& r) {
  for (int i = 0; i < x.stages && r.ok; ++i) {
    if (r.count >= (uint32_t)x.stages || r.s < (int)r.count)
      r.ok = __all_sync(0xffffffffu, bar_wait(x.empty + 8 * r.s, r.phase, x.status));
    r.next(x.stages);
  }
  if (!r.ok)  // a wait ran out: let the copies that were issued land before the CTA ends
    for (const uint64_t t0 = now_ns(); now_ns() - t0 < 1000000ull;) {}
}

// Warp 2 of the pair's first CTA: the matrix instructions.
template <class View>
__device__ __forceinline__ void mma_units(const View& v, const Cta& x, Ring& r, Unit w) {
  const int cols = v.cols(), units = v.units();
  for (int u = x.worker; u < units && r.ok; u += x.workers) {
    if (u != x.worker) w = locate(v, u, w.p);
    const Problem& P = v.problem(w.p);
    int k0, k1;
    split_range(P, v.parts(w.p), w.split, &k0, &k1);
    if (k0 == k1) continue;  // an empty sum: the epilogue takes zeros
    // blocks of k's up to these come transposed, in each part of the sum
    const int a_diag = P.a_kind ? 0x7fffffff : P.a_sym ? w.m0 / kDepth : 0;
    const int b_diag = P.b_kind ? 0x7fffffff : P.b_sym ? (w.n0 & ~(kTileRows - 1)) / kDepth : 0;
    int kblocks = P.kblocks;
    asm volatile("" : "+r"(kblocks));  // (read once, not in the loop)
    int k = k0 < kblocks ? k0 : k0 - kblocks;  // in its part
    const int buf = r.count & 1;
    const uint32_t d = x.tmem + buf * (kTmemCols / 2);
    if (!__all_sync(0xffffffffu,
                    bar_wait(x.acc_empty + 8 * buf, ((r.count >> 1) & 1) ^ 1, x.status))) {
      r.ok = false;
      break;
    }
    tc_fence_after();
    for (int kb = k0; kb < k1; ++kb) {
      if (!__all_sync(0xffffffffu, bar_wait(x.full + 8 * r.s, r.phase, x.status))) {
        r.ok = false;
        break;
      }
      tc_fence_after();
      const bool a_mn = k < a_diag, b_mn = k < b_diag;
      const uint32_t idesc = mma_idesc(v.bf16(), a_mn, b_mn, kTileRows, cols);
      const uint32_t step_a = mma_k_step(a_mn), step_b = mma_k_step(b_mn);
      if (elect_one()) {
        const uint32_t addr = x.tiles0 + r.s * x.stage_bytes;
        uint64_t a = mma_smem_desc(addr, a_mn);
        uint64_t b = mma_smem_desc(addr + kTileABytes, b_mn);
#pragma unroll
        for (int i = 0; i < kDepth / 16; ++i, a += step_a, b += step_b)
          tc_mma(d, a, b, idesc, kb > k0 || i > 0);
        tc_commit(x.empty + 8 * r.s);
        if (kb + 1 == k1) tc_commit(x.acc_full + 8 * buf);
      }
      __syncwarp();
      r.next(x.stages);
      if (++k == kblocks) k = 0;
    }
    ++r.count;
  }
}

// Warps 4..11: the epilogue. r.count counts tiles. Once a wait has run out, units pass without
// results, so that the block barriers of the split sums still see every warp.
template <class View, class Gate>
__device__ __forceinline__ void finish_units(const View& v, const Cta& x, Ring& r, Unit w,
                                             Block& b, Gate gate) {
  bool shut = true;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = warp & 3;                 // the tensor-memory lanes this warp can read
  const int turn = (warp - kFirstEpi) >> 2;  // which of the quadrant's warps
  const int cols = v.cols(), units = v.units();
  for (int u = x.worker; u < units; u += x.workers) {
    if (u != x.worker) w = locate(v, u, w.p);
    const Problem& P = v.problem(w.p);
    int k0, k1;
    split_range(P, v.parts(w.p), w.split, &k0, &k1);
    const int buf = r.count & 1;
    const int64_t row0 = w.m0 + (int)x.rank * kRows + quad * 32;
    const int N = P.N, n_end = P.n_end, splits = P.splits;
    const bool sym = P.sym;
    b.rows = (int)max((int64_t)0, min((int64_t)32, P.M - row0));
    const typename View::Target target = v.target(w.p, w.z);
    Sums a;
    a.tmem = x.tmem + buf * (kTmemCols / 2) + ((uint32_t)(quad * 32) << 16);
    a.parts = nullptr;
    a.splits = splits;
    a.width4 = cols / 4;
    a.row = quad * 32 + lane;
    a.done = map_to_rank(x.acc_empty + 8 * buf, 0);
    // this warp's chunks: accumulator columns turn * 32 + kEpiStep i, of which it takes those inside
    // the result and not left of a symmetric result's diagonal block
    auto wanted = [&](int c) {
      const int col = w.n0 + c;
      return col < n_end && b.rows > 0 && !(sym && col < w.m0);
    };
    a.last = -1;
    if (splits == 1)
      for (int c = turn * 32; c < cols; c += kEpiStep)
        if (wanted(c)) a.last = c;
    if (shut) {
      asm volatile("" ::"r"(a.last), "r"(n_end), "r"(splits), "r"(k0), "r"(k1), "r"(b.rows));
      target.pin();
      shut = false;
      r.ok = gate() && r.ok;
    }
    if (a.last >= 0) v.prefetch(target, b, row0, w.n0 + turn * 32, n_end);
    if (k1 > k0 && r.ok) {
      r.ok =
          __all_sync(0xffffffffu, bar_wait(x.acc_full + 8 * buf, (r.count >> 1) & 1, x.status));
      tc_fence_after();
    }
    const bool sums = k1 > k0 && r.ok;
    a.any = sums;
    bool finished = r.ok;
    if (splits > 1) {
      // this CTA's tile of the split: [split][column / 4][row] float4
      const int64_t tile_id = (int64_t)((u - P.first) / splits) * 2 + x.rank;
      float4* parts = reinterpret_cast<float4*>(P.split_ws) + tile_id * splits * a.width4 * kRows;
      float4* mine = parts + (int64_t)w.split * a.width4 * kRows + a.row;
      for (int c = turn * 32; c < cols; c += kEpiStep) {
        if (!sums || !wanted(c)) continue;  // a split has at least one k block
        float f[32];
        tmem_ld32(a.tmem + c, f);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          __stcg(&mine[(c / 4 + i) * kRows],
                 make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]));
      }
      if (sums) release_sums(a);
      __threadfence();
      epilogue_sync();
      if (threadIdx.x == 32 * kFirstEpi) {
        const bool all = r.ok && atomicAdd(&P.split_count[tile_id], 1u) == (uint32_t)splits - 1;
        sts_elem<4>(x.last_flag, all);
        if (all) P.split_count[tile_id] = 0;  // for the next launch
      }
      epilogue_sync();
      finished = lds_elem<4>(x.last_flag) && r.ok;
      epilogue_sync();
      __threadfence();
      a.parts = parts;
    } else if (sums && a.last < 0) {
      release_sums(a);
    }
    if (finished) {
      for (int c = turn * 32; c < cols; c += kEpiStep) {
        if (!wanted(c)) continue;
        const int col = w.n0 + c;
        float f[32];
        take_sums(a, c, f);
        v.finish(target, b, f, row0, col, min(32, n_end - col),
                 N);
      }
    }
    if (sums) ++r.count;
  }
  if (shut) r.ok = gate() && r.ok;
}

constexpr uint32_t kBarrierOffset = (uint32_t)kOperandSpace + kEpiWarps * kBlockBytes;

// Shared set-up of the kernels below: barriers, tensor memory, the pair's first meeting.
__device__ __forceinline__ void cta_begin(Cta& x, uint8_t* smem, int stages, uint32_t stage_bytes,
                                          uint32_t* status) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  x.tiles0 = smem_addr(smem);
  x.full = x.tiles0 + kBarrierOffset;
  x.empty = x.full + 8 * kMaxStages;
  x.acc_full = x.empty + 8 * kMaxStages;
  x.acc_empty = x.acc_full + 16;
  const uint32_t slot = x.acc_empty + 16;
  x.last_flag = slot + 4;
  x.rank = cluster_rank();
  x.worker = blockIdx.x / 2;
  x.workers = gridDim.x / 2;
  x.stages = stages;
  x.stage_bytes = stage_bytes;
  x.status = status;
  if (warp == 0) {  // full, empty, acc_full: one arrival; acc_empty: one of each epilogue warp
    constexpr int kBars = 2 * kMaxStages + 4;
    if (lane < kBars) bar_init(x.full + 8 * lane, lane < kBars - 2 ? 1 : 2 * kEpiWarps);
    bar_init_fence();
  }
  if (warp == 2) tmem_alloc(slot, kTmemCols);
}
__device__ __forceinline__ void cta_meet(Cta& x) {
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  x.tmem = lds_elem<4>(x.acc_empty + 16);
}
__device__ __forceinline__ void cta_end(const Cta& x) {
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  if ((threadIdx.x >> 5) == 2) tmem_free(x.tmem, kTmemCols);
}

// ---- the linear layer's products -------------------------------------------------
constexpr int kLinearProducts = 2;  // a layer's two gradients go in one launch
struct LinearArgs {
  CUtensorMap maps[kLinearProducts][2];
  Problem p[kLinearProducts];
  Out out[kLinearProducts];
  int32_t count, units, cols, stages;
  uint32_t* status;
};

template <bool EPILOGUE, int DT>  // with bias, activation, residual (one product); or only rounded
struct LinearView {
  struct Target {
    int p;
    __device__ __forceinline__ void pin() const {}
  };
  const LinearArgs& g;
  __device__ __forceinline__ int count() const { return EPILOGUE ? 1 : g.count; }
  __device__ __forceinline__ int units() const { return g.units; }
  __device__ __forceinline__ int cols() const { return g.cols; }
  __device__ __forceinline__ bool bf16() const { return DT == DT_BF16; }
  __device__ __forceinline__ int index(int p) const { return EPILOGUE ? 0 : p; }
  __device__ __forceinline__ const Problem& problem(int p) const { return g.p[index(p)]; }
  __device__ __forceinline__ const CUtensorMap* map_a(int p) const { return &g.maps[index(p)][0]; }
  __device__ __forceinline__ const CUtensorMap* map_b(int p) const { return &g.maps[index(p)][1]; }
  __device__ __forceinline__ const CUtensorMap* map_a_t(int) const { return nullptr; }
  __device__ __forceinline__ const CUtensorMap* map_b_t(int) const { return nullptr; }
  __device__ __forceinline__ int za(int) const { return 1; }
  __device__ __forceinline__ int zb(int) const { return 1; }
  __device__ __forceinline__ int parts(int) const { return 1; }
  __device__ __forceinline__ Target target(int p, int) const { return Target{index(p)}; }
  __device__ __forceinline__ void prefetch(const Target&, const Block&, int64_t, int, int) const {}
  __device__ __forceinline__ void finish(const Target& t, const Block& b, float (&v)[32],
                                         int64_t row0, int col, int n, int) const {
    if constexpr (EPILOGUE) {
      finish_linear<DT>(g.out[0], b, v, row0, col, n);
    } else {
      const Out& o = g.out[t.p];
      row_put<DT>(b, v);
      block_store<2>(b, o.out + (row0 * o.ld + col) * 2, o.ld, n);
    }
  }
};

template <bool EPILOGUE, int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    k_linear(const __grid_constant__ LinearArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const LinearView<EPILOGUE, DT> v{g};
  const int warp = threadIdx.x >> 5;
  Cta x;
  cta_begin(x, smem, g.stages, kTileABytes + g.cols * kDepth, g.status);
  const Unit w = locate(v, x.worker, 0);  // looked up under the set-up's latency
  cta_meet(x);
  chain_next();
  auto gate = [] {
    chain_wait();
    return true;
  };
  Ring r;
  if (warp < 2) {
    r.phase = 1;  // of "empty": the first round finds every stage free
    copy_units(v, x, r, w, warp == 0, gate);
    copy_drain(x, r);
  } else if (warp == 2) {
    r.phase = 0;
    if (x.rank == 0) mma_units(v, x, r, w);
  } else if (warp >= kFirstEpi) {
    Block b;
    b.init(x.tiles0 + (uint32_t)kOperandSpace + (warp - kFirstEpi) * kBlockBytes,
           threadIdx.x & 31);
    finish_units(v, x, r, w, b, gate);
  }
  cta_end(x);
}

}  // namespace mx
}  // namespace ta
