// ta_mx_api.cu -- host side of the matrix operators (include/turboadam_b200_matrix.h):
// argument validation, operand tensor maps, the choice of tile and split, workspace
// layout and the launch sequences.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>
#include <map>
#include <mutex>
#include <string>
#include <utility>
#include <vector>

#include "../../include/turboadam_b200_matrix.h"
#include "ta_host.h"
#include "ta_mx_chain.cuh"
#include "ta_mx_elementwise.cuh"
#include "ta_mx_few.cuh"
#include "ta_mx_product.cuh"

using namespace ta::mx;

namespace {

#define MX_CU(x)                                                                        \
  do {                                                                                  \
    cudaError_t e_ = (x);                                                               \
    if (e_ != cudaSuccess)                                                              \
      return ta_fail(TA_ERR_CUDA, std::string(#x) + ": " + cudaGetErrorString(e_));     \
  } while (0)
#define MX_OK(x)                  \
  do {                            \
    ta_status s_ = (x);           \
    if (s_ != TA_OK) return s_;   \
  } while (0)

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t up8(int64_t x) { return (x + 7) & ~(int64_t)7; }
inline int64_t up32(int64_t x) { return (x + 31) & ~(int64_t)31; }
inline size_t al256(size_t x) { return (x + 255) & ~(size_t)255; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
inline int64_t dt_bytes(int dt) { return dt == TA_F32 ? 4 : 2; }

// Elements of the type can be loaded from there (a null pointer passes).
bool typed(const void* p, int dt) { return (uintptr_t)p % dt_bytes(dt) == 0; }
ta_status check_typed(std::initializer_list<std::pair<const char*, const void*>> ps, int dt) {
  for (const auto& p : ps)
    if (!typed(p.second, dt))
      return ta_fail(TA_ERR_ALIGN, std::string(p.first) + " not aligned to its type");
  return TA_OK;
}

constexpr int64_t kMaxUnits = 0x70000000;  // work units of a launch (32-bit, with room to step)
constexpr int64_t kMaxDim = 0x7fffff00;  // every dimension (rows, columns) is held in 32 bits

constexpr int kMaxDevices = 64;

int sm_count() {  // of the current device (148 where there is none, as when sizing without a GPU)
  static std::atomic<int> known[kMaxDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 148;
  n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (n <= 0) return 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// ---- workspace -------------------------------------------------------------
// Hands out 256-byte aligned pieces; with a null base it only measures.
struct Arena {
  uint8_t* base;
  size_t used = 0;
  template <typename T>
  T* take(size_t count) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += al256(count * sizeof(T));
    return p;
  }
};

// ---- tensor maps -------------------------------------------------------------
using EncodeFn = decltype(&cuTensorMapEncodeTiled);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                         &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// The tensor-map encoder is a driver call: it needs the device's context to be current on the
// calling thread, which on a fresh thread (autograd's, say) only a runtime call makes it.
ta_status bind_device() {
  int dev = 0;
  MX_CU(cudaGetDevice(&dev));
  MX_CU(cudaSetDevice(dev));
  return TA_OK;
}

// An operand of a product: `mn` output rows (or columns) by `k`, 16-bit elements, one of the two
// contiguous; lines of the other are ld elements apart, matrices zs elements apart.
struct Operand {
  const void* p = nullptr;
  int64_t mn = 0, k = 0, ld = 0, zs = 0, z = 1;
  bool mn_major = false;
  bool sym = false;  // stored in its upper triangle of blocks
};

// How a stage of an operand is copied: 0 K-major; 1 MN-major, one copy for each chunk of 64;
// 2 MN-major in one copy, over chunks as a dimension of their own, where the lines are whole
// chunks (a chunk that ran over the end of a line would read the next one, and past the end of the
// last).
int kind_of(const Operand& o) { return !o.mn_major ? 0 : o.mn % 64 ? 1 : 2; }

// The map of an operand whose stages hold box_mn rows (or columns) of the output by 64 k's.
ta_status make_map(CUtensorMap* m, const Operand& o, bool bf16, int box_mn) {
  EncodeFn fn = encode_fn();
  if (!fn) return ta_fail(TA_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t line = (cuuint64_t)o.ld * 2;
  const cuuint64_t plane = (cuuint64_t)std::max<int64_t>(o.zs, o.ld) * 2;
  const int kind = kind_of(o);
  cuuint64_t dims[4], strides[3];
  cuuint32_t box[4] = {64, 64, 1, 1}, step[4] = {1, 1, 1, 1};
  cuuint32_t rank = 3;
  if (kind == 2) {
    rank = 4;
    dims[0] = 64;
    dims[1] = (cuuint64_t)o.k;
    dims[2] = (cuuint64_t)(o.mn / 64);
    dims[3] = (cuuint64_t)o.z;
    strides[0] = line;
    strides[1] = 128;
    strides[2] = plane;
    box[2] = (cuuint32_t)(box_mn / 64);
  } else {
    dims[0] = (cuuint64_t)(kind == 0 ? o.k : o.mn);
    dims[1] = (cuuint64_t)(kind == 0 ? o.mn : o.k);
    dims[2] = (cuuint64_t)o.z;
    strides[0] = line;
    strides[1] = plane;
    if (kind == 0) box[1] = (cuuint32_t)box_mn;
  }
  CUresult r = fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  rank, const_cast<void*>(o.p), dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return ta_fail(TA_ERR_CUDA, "cuTensorMapEncodeTiled: error " + std::to_string((int)r));
  return TA_OK;
}

// ---- products on the tile engine ---------------------------------------------------
struct Product {
  Operand a, b;
  int64_t M = 0, N = 0;
  int parts = 1;        // operand pairs the sum runs over
  bool sym = false;
  bool padded = false;  // the result's lines have room for whole chunks
  int64_t batch = 1;
};

int64_t blocks_of(const Product& p) { return cdiv(p.a.k, kDepth) * p.parts; }

int64_t tiles_of(const Product& p, int cols) {
  const int64_t m = cdiv(p.M, kTileRows), n = cdiv(p.N, cols);
  if (!p.sym) return m * n;
  int64_t t = 0;
  for (int64_t i = 0; i < m; ++i) t += n - sym_first((int)i, cols);
  return t;
}

struct Shape {
  int cols = 256;
  std::vector<int> splits;
};

// room for the split tiles of one launch
constexpr int64_t kSplitTiles = 592;                    // counters: one per CTA tile
constexpr int64_t kSplitFloats = 320ll * kRows * 256;   // partial sums

// SM cycles of a pair's tile of `cols` columns. A block of 64 k's costs what the slowest of four
// takes: the tensor pipe (2 cols), shared memory (256 + cols), the copies' issue (about 350) and,
// where the first two are close, their getting in each other's way (measured 590 cycles at 256
// columns). The epilogue, some 1500 cycles a chunk for each of four warps, is hidden behind the
// next tile's products or hides them.
double tile_cycles(double kblocks, int cols) {
  const double loop = kblocks * std::max(350.0, std::max(2.0 * cols, 256.0 + cols) + 0.15 * cols);
  const double epilogue = 1200.0 + 1500.0 * (double)cdiv(cols, 128);
  return std::max(loop, epilogue) + 0.3 * std::min(loop, epilogue);
}

// A split sum also costs its partial tiles' way through memory, and the last split's adding them
// up one after another. (With a third of this cost 64 tokens of 4096 > 4096 took 25 us instead of
// 18, 600 of 14336 > 4096 72 instead of 63 and eight GPT-2 attention matrices 252 instead of 239
// orthogonalised; with more, a 1024 x 4096 matrix 177 instead of 169.)
double unit_cycles(const Product& p, int splits, int cols) {
  return tile_cycles((double)cdiv(std::max<int64_t>(1, blocks_of(p)), splits), cols) +
         (splits > 1 ? 8000.0 + splits * 12.0 * cols : 0.0);
}

// Cycles of a launch whose pair w takes units w, w + pairs, ... of the list: the most loaded
// pair's.
double launch_cycles(const std::vector<Product>& ps, const std::vector<int>& splits, int cols,
                     int pairs) {
  if (ps.size() == 1)
    return (double)cdiv(tiles_of(ps[0], cols) * ps[0].batch * splits[0], pairs) *
           unit_cycles(ps[0], splits[0], cols);
  std::vector<double> load(pairs, 0.0);
  int64_t first = 0;
  for (size_t i = 0; i < ps.size(); ++i) {
    const int64_t n = tiles_of(ps[i], cols) * ps[i].batch * splits[i];
    const double c = unit_cycles(ps[i], splits[i], cols);
    for (int w = 0; w < pairs; ++w) load[w] += (double)(n / pairs) * c;
    for (int64_t u = 0; u < n % pairs; ++u) load[(first + u) % pairs] += c;
    first += n;
  }
  return *std::max_element(load.begin(), load.end());
}

// Tile width and splits of a launch: the lowest estimate over the widths the operands' layouts
// allow, and over some splits of its sums. Wide tiles use the tensor pipe best, narrow ones give
// every pair of SMs a share of a small result, and split sums a share of a long one. (A layer's
// gradients on 8192 tokens, 96 tiles of 36 blocks and 27 of 128: 63 us unsplit.)
Shape choose(const std::vector<Product>& ps, int pairs, bool may_split = true) {
  // MN-major (or partly transposed) operands come in whole chunks of 64 rows a CTA; the tile widths
  // of a symmetric result divide its blocks of 256
  bool chunked = false, sym = false;
  for (const Product& p : ps) {
    chunked = chunked || p.b.mn_major || p.b.sym;
    sym = sym || p.sym;
  }
  static const int kAny[] = {256, 224, 192, 160, 128, 96, 64}, kSym[] = {256, 128, 64},
                   kChunked[] = {256, 128};
  const int* widths = chunked ? kChunked : sym ? kSym : kAny;
  const int n_widths = chunked ? 2 : sym ? 3 : 7;
  Shape best;
  best.splits.assign(ps.size(), 1);
  double best_time = 1e300;
  std::vector<int> splits(ps.size());
  for (int k = 0; k < n_widths; ++k) {
    const int cols = widths[k];
    int64_t units = 0;
    double work = 0;
    for (const Product& p : ps) {
      const int64_t t = tiles_of(p, cols) * p.batch;
      units += t;
      work += (double)t * unit_cycles(p, 1, cols);
    }
    if (units == 0) return best;
    // one product: every split; a list: units of at most a share of a pair's even load
    const int tries = !may_split || units > 3 * pairs ? 1 : ps.size() == 1 ? 16 : 5;
    for (int n = 1; n <= tries; ++n) {
      int64_t tiles = 0, floats = 0;
      for (size_t i = 0; i < ps.size(); ++i) {
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(16, blocks_of(ps[i]) / 2));
        int64_t want = n;
        if (ps.size() > 1)
          want = n == 1 ? 1
                        : (int64_t)(unit_cycles(ps[i], 1, cols) * (n - 1) / (work / pairs) + 0.5);
        splits[i] = (int)std::max<int64_t>(1, std::min(want, most));
        if (splits[i] > 1) {
          const int64_t t = 2 * tiles_of(ps[i], cols) * ps[i].batch;
          tiles += t;
          floats += t * splits[i] * kRows * cols;
        }
      }
      if (tiles > kSplitTiles || floats > kSplitFloats) continue;
      const double time = launch_cycles(ps, splits, cols, pairs);
      if (time < best_time) {
        best_time = time;
        best.cols = cols;
        best.splits = splits;
      }
    }
  }
  return best;
}

// Launches a kernel of a chain: it may start its set-up while the kernel before it drains (every
// kernel of this file waits for that one before it touches global memory).
template <typename... Params, typename... Args>
ta_status launch(void (*kernel)(Params...), dim3 grid, int threads, size_t smem,
                 cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  MX_CU(cudaLaunchKernelEx(&cfg, kernel, Params(args)...));
  return TA_OK;
}

// Shared-memory limit and resident pairs of a kernel of the tile engine, found once per device. A
// die's SM count need not divide into pairs, so the pairs that fit are asked for: one that had to
// wait for another to finish would double the time of a persistent launch.
template <typename Kernel>
ta_status pairs_of(Kernel kernel, int* found, int* pairs) {  // found: [kMaxDevices], zero at first
  static std::mutex m;
  int dev = 0;
  MX_CU(cudaGetDevice(&dev));
  if (dev >= kMaxDevices) return ta_fail(TA_ERR_UNSUPPORTED, "device index over 63");
  std::lock_guard<std::mutex> lock(m);
  if (!found[dev]) {
    MX_CU(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)kProductSmem));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(sm_count() / 2 * 2));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kProductSmem;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    MX_CU(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    if (n < 1) return ta_fail(TA_ERR_CUDA, "the product kernel does not fit this device");
    found[dev] = n;
  }
  *pairs = found[dev];
  return TA_OK;
}

// The device's view of a list of products of one tile width; returns the work units.
int64_t place_products(const std::vector<Product>& ps, const Shape& shape, float* split_ws,
                       uint32_t* split_count, Problem* out, int64_t* split_tiles) {
  int64_t units = 0, floats = 0;
  *split_tiles = 0;
  for (size_t i = 0; i < ps.size(); ++i) {
    const Product& p = ps[i];
    Problem& P = out[i];
    memset(&P, 0, sizeof(P));
    P.M = (int32_t)p.M;
    P.N = (int32_t)p.N;
    P.n_end = (int32_t)(p.padded ? up32(p.N) : p.N);
    P.kblocks = (int32_t)cdiv(p.a.k, kDepth);
    P.tiles_m = (int32_t)cdiv(p.M, kTileRows);
    P.tiles_n = (int32_t)cdiv(p.N, shape.cols);
    P.tiles = (int32_t)tiles_of(p, shape.cols);
    P.first = (int32_t)units;
    P.batch = (int32_t)p.batch;
    P.splits = shape.splits[i];
    P.sym = p.sym;
    P.a_kind = (int16_t)kind_of(p.a);
    P.b_kind = (int16_t)kind_of(p.b);
    P.a_sym = p.a.sym ? (int16_t)(p.a.mn % 64 ? 1 : 2) : 0;
    P.b_sym = p.b.sym ? (int16_t)(p.b.mn % 64 ? 1 : 2) : 0;
    const int64_t tiles = tiles_of(p, shape.cols) * p.batch;
    if (P.splits > 1) {
      P.split_ws = split_ws + floats;
      P.split_count = split_count + *split_tiles;
      floats += 2 * tiles * P.splits * kRows * shape.cols;
      *split_tiles += 2 * tiles;
    }
    units += tiles * P.splits;
  }
  return units;
}

int stages_of(int cols) {
  return (int)std::min<size_t>(kMaxStages,
                               kOperandSpace / (size_t)(kTileABytes + cols * kDepth));
}

// One product with its epilogue, or up to two plain ones, in one launch. split_ws / split_count:
// kSplitFloats and kSplitTiles of them.
template <bool EPILOGUE, int DT>
ta_status run_linear(const std::vector<Product>& ps, const std::vector<Out>& outs, float* split_ws,
                     uint32_t* split_count, uint32_t* status, cudaStream_t stream) {
  static int found[kMaxDevices];
  int pairs = 0;
  MX_OK(bind_device());
  MX_OK(pairs_of(k_linear<EPILOGUE, DT>, found, &pairs));
  const Shape shape = choose(ps, pairs);
  LinearArgs g;
  memset(&g, 0, sizeof(g));
  int64_t split_tiles = 0;
  const int64_t units = place_products(ps, shape, split_ws, split_count, g.p, &split_tiles);
  if (units > kMaxUnits) return ta_fail(TA_ERR_UNSUPPORTED, "too many tiles in one call");
  if (units == 0) return TA_OK;
  for (size_t i = 0; i < ps.size(); ++i) {
    if (ps[i].a.k > 0) {
      MX_OK(make_map(&g.maps[i][0], ps[i].a, DT == DT_BF16, kRows));
      MX_OK(make_map(&g.maps[i][1], ps[i].b, DT == DT_BF16, shape.cols / 2));
    }
    g.out[i] = outs[i];
  }
  g.count = (int32_t)ps.size();
  g.units = (int32_t)units;
  g.cols = shape.cols;
  g.stages = stages_of(shape.cols);
  g.status = status;
  if (split_tiles)
    MX_CU(cudaMemsetAsync(split_count, 0, split_tiles * sizeof(uint32_t), stream));
  return launch(k_linear<EPILOGUE, DT>, dim3(2u * (unsigned)std::min<int64_t>(units, pairs)),
                kThreads, kProductSmem, stream, g);
}

// ---- orthogonalisation -----------------------------------------------------------
// Scales of the fp16 matrices: X, the Gram matrix and the polynomial are at most a few units in
// norm (the quintic keeps singular values below 1.3), so 2^10 and 2^8 leave 2^6 to 2^8 of head
// room under fp16's largest number and put elements of 2^-24 and 2^-22 on its smallest normal.
// (The product of two polynomials is at most the square of one, P A a few times A.)
constexpr float kScaleX = 1024.f, kScaleA = 1024.f, kScaleP = 256.f, kScaleT = 512.f;

// Two steps can go as a pair. With A the Gram matrix of X, P and P' the polynomials of the steps,
//   T = P A,  A' = P T  (the Gram matrix of P X, without forming P X),  Q = P' P,  X <- Q X:
// in units of a side^3 product and with r = long / short side, 3 r + 5 for two steps against
// 6 r + 2 one by one (symmetric results at half cost). The first pair acts on the input as it is
// held (16-bit inputs exactly, 32-bit ones to 22 bits, of which A sees the upper 11), so X is not
// rounded while its small singular values still drown in the error of the large ones: that leaves
// two thirds of the error (Frobenius norm against the exact iteration, on spectra that fall by 50
// within a quarter of their length over a floor: 1.0e-3 against 1.5e-3 at 768 x 768, 1.48e-3
// against 2.15e-3 at 1024 x 4096; bf16 operands would leave 2e-2). A later pair saves products only
// where r is well over 1 and there are enough of them (1024 x 4096: 175 us against 177; 2048 x
// 8192: 408 against 462; 14336 x 4096: 2209 against 2584), and rounds P and A' where X was rounded
// before: its error nears the other's as the side grows, 2.04e-3 against 1.27e-3 at 512 x 2048, 1.97e-3
// against 1.48e-3 at 1024 x 4096, 1.90e-3 against 1.65e-3 at 2048 x 8192, 1.83e-3 against 1.76e-3
// at 14336 x 4096 (in the 2-norm 4.5e-3 against 2.2e-3 at 2048 x 8192). So the later steps go in
// pairs ("deep") from a side of 2048 and r of 2 on, and one by one elsewhere. Three steps at once
// would lose 1e-2.
bool deep_pairs(int64_t side, int64_t length) { return side >= 2048 && length >= 2 * side; }

struct Class {  // matrices of one shape
  int64_t rows = 0, cols = 0, ld = 0, side = 0, lds = 0, count = 0;
  int first = 0;  // first table slot
  bool pair = false, tall = false, deep = false;
  __half *x0 = nullptr, *x1 = nullptr, *square[3] = {nullptr, nullptr, nullptr};
  int64_t xs() const { return rows * ld; }
  int64_t ss() const { return side * lds; }
};

struct OrthoPlan {
  std::vector<int> chains;  // first class of each chain
  std::vector<Class> classes;
  std::vector<std::vector<int>> members;  // tensors of each class
  int64_t items = 0;
  int64_t elems = 0;
  int64_t chunks = 0;
};

// Elements of a block of the elementwise passes: some four blocks for every SM over the whole list
// (a block's lookups and sums cost a few microseconds, its loads hide each other), at most
// kMaxChunks of a matrix.
int64_t chunk_elems(int64_t n, int64_t total) {
  const int64_t share = cdiv(total, 4 * sm_count()), least = cdiv(n, kMaxChunks);
  return cdiv(std::max<int64_t>({4096, share, least}), 2048) * 2048;
}

ta_status plan_ortho(const ta_ortho_tensor* ts, int32_t n, const ta_ortho_options* o,
                     OrthoPlan* plan) {
  if (n < 0 || (n > 0 && !ts)) return ta_fail(TA_ERR_INVALID, "null tensor list");
  if (!o || !o->coefficients) return ta_fail(TA_ERR_INVALID, "null options or coefficients");
  if (o->steps < 1 || o->steps > 32) return ta_fail(TA_ERR_INVALID, "steps must be 1 to 32");
  if (!(o->eps >= 0)) return ta_fail(TA_ERR_INVALID, "eps must not be negative");
  std::map<std::pair<std::pair<int64_t, int64_t>, bool>, int> index;
  for (int i = 0; i < n; ++i) {
    const ta_ortho_tensor& t = ts[i];
    auto bad = [&](const char* what) {
      return ta_fail(TA_ERR_INVALID, "matrix " + std::to_string(i) + ": " + what);
    };
    if (t.batch < 0 || t.rows < 0 || t.cols < 0) return bad("negative size");
    if (t.batch == 0 || t.rows == 0 || t.cols == 0) continue;
    if (t.rows > kMaxDim || t.cols > kMaxDim || t.batch > kMaxDim)
      return ta_fail(TA_ERR_UNSUPPORTED,
                     "matrix " + std::to_string(i) + ": a size is over 2^31 - 256");
    if (!t.in_dev || !t.out_dev) return bad("null pointer");
    for (int dt : {t.in_dtype, t.out_dtype, t.momentum_dev ? t.momentum_dtype : (int)TA_F32})
      if (dt != TA_F32 && dt != TA_BF16 && dt != TA_F16)
        return bad("dtypes must be TA_F32, TA_BF16 or TA_F16");
    if (!typed(t.in_dev, t.in_dtype) || !typed(t.out_dev, t.out_dtype) ||
        (t.momentum_dev && !typed(t.momentum_dev, t.momentum_dtype)))
      return ta_fail(TA_ERR_ALIGN,
                     "matrix " + std::to_string(i) + ": pointer not aligned to its type");
    const bool pair = (t.flags & TA_ORTHO_PAIR) && t.in_dtype == TA_F32;
    auto key = std::make_pair(std::make_pair(t.rows, t.cols), pair);
    auto it = index.find(key);
    if (it == index.end()) {
      it = index.emplace(key, (int)plan->classes.size()).first;
      Class c;
      c.rows = t.rows;
      c.cols = t.cols;
      c.ld = up32(t.cols);  // whole epilogue chunks
      c.tall = t.rows > t.cols;
      c.side = std::min(t.rows, t.cols);
      c.deep = deep_pairs(c.side, std::max(t.rows, t.cols));
      c.lds = up32(c.side);
      c.pair = pair;
      plan->classes.push_back(c);
      plan->members.emplace_back();
    }
    plan->classes[it->second].count += t.batch;
    plan->members[it->second].push_back(i);
  }
  // chains: up to kMaxClasses classes of one sequence of phases each
  OrthoPlan sorted;
  for (int deep = 0; deep < 2; ++deep) {
    int in_chain = kMaxClasses;
    for (size_t i = 0; i < plan->classes.size(); ++i) {
      if (plan->classes[i].deep != (deep == 1)) continue;
      if (in_chain == kMaxClasses) {
        sorted.chains.push_back((int)sorted.classes.size());
        in_chain = 0;
      }
      ++in_chain;
      sorted.classes.push_back(plan->classes[i]);
      sorted.members.push_back(plan->members[i]);
    }
  }
  *plan = sorted;
  for (const Class& c : plan->classes) plan->elems += c.count * c.rows * c.cols;
  for (Class& c : plan->classes) {
    c.first = (int)plan->items;
    plan->items += c.count;
    plan->chunks += c.count * cdiv(c.rows * c.cols, chunk_elems(c.rows * c.cols, plan->elems));
    if (plan->items > 0x7fffffff || plan->chunks > 0x7fffffff)
      return ta_fail(TA_ERR_UNSUPPORTED, "too many matrices in one call");
  }
  return TA_OK;
}

struct OrthoSpace {
  Item* table;
  Scale* scale;
  double* partial;
  uint32_t* split_count;
  uint32_t* chain;  // [chains][2]: arrivals, stop
  float* split_ws;
};

int chains_of(const OrthoPlan& plan) { return (int)plan.chains.size(); }

OrthoSpace carve_ortho(OrthoPlan* plan, Arena* a) {
  OrthoSpace s;
  s.table = a->take<Item>(plan->items);
  s.scale = a->take<Scale>(plan->items);
  s.partial = a->take<double>(plan->chunks);
  // cleared together: counters of split tiles, then two words of each chain
  s.split_count = a->take<uint32_t>(kSplitTiles + 2 * chains_of(*plan));
  s.chain = s.split_count ? s.split_count + kSplitTiles : nullptr;
  s.split_ws = a->take<float>(kSplitFloats);
  for (Class& c : plan->classes) {
    c.x0 = a->take<__half>(c.xs() * c.count * (c.pair ? 2 : 1));
    c.x1 = a->take<__half>(c.xs() * c.count);
    for (__half*& q : c.square) q = a->take<__half>(c.ss() * c.count);
  }
  return s;
}

int chain_phases(const ta_ortho_options* o, bool deep, Phase* out) {
  int n = 0;
  auto add = [&](int type, int end, int a, int b, int to, float alpha) -> Phase& {
    Phase& p = out[n++];
    memset(&p, 0, sizeof(p));
    p.type = (int8_t)type;
    p.end = (int8_t)end;
    p.a = (int8_t)a;
    p.b = (int8_t)b;
    p.out = (int8_t)to;
    p.alpha = alpha;
    return p;
  };
  int x = BUF_X0, gram = BUF_S0, poly = BUF_S0 + 1, prod = BUF_S0 + 2;
  auto polynomial = [&](int step) {
    const double* abc = o->coefficients + 3 * step;
    Phase& p = add(PH_SQUARE, END_POLY, gram, gram, poly,
                   (float)(kScaleP * abc[2] / ((double)kScaleA * kScaleA)));
    p.c0 = (float)(kScaleP * abc[0]);
    p.c1 = (float)(kScaleP * abc[1] / kScaleA);
    p.aux = (int8_t)gram;
  };
  for (int step = 0; step < o->steps;) {
    const bool first = step == 0, two = step + 1 < o->steps && (first || deep);
    add(PH_GRAM, END_SCALE, x, x, gram, first ? kScaleA : kScaleA / (kScaleX * kScaleX))
        .unit_pow = first ? 2 : 0;
    polynomial(step);
    if (two) {
      add(PH_SQUARE, END_SCALE, poly, gram, prod, kScaleT / (kScaleP * kScaleA));  // T
      add(PH_SQUARE, END_SCALE, poly, prod, gram, kScaleA / (kScaleP * kScaleT));  // A'
      std::swap(poly, prod);                                                       // P
      polynomial(step + 1);                                                        // P'
      add(PH_SQUARE, END_SCALE, poly, prod, gram, 1.f / kScaleP);                  // Q
      std::swap(poly, gram);
    }
    step += two ? 2 : 1;
    const bool last = step == o->steps;
    const int to = x == BUF_X0 ? BUF_X1 : BUF_X0;
    const float alpha = first ? 1.f / kScaleP : 1.f / (kScaleP * kScaleX);
    Phase& p = add(PH_APPLY, last ? END_FINAL : END_SCALE, poly, x, to,
                   last ? alpha : alpha * kScaleX);
    p.unit_pow = first ? 1 : 0;
    p.whole = first;
    x = to;
  }
  return n;
}

ta_status run_chain(const std::vector<Class>& classes, const ta_ortho_options* o,
                    const OrthoSpace& sp, uint32_t* words, uint32_t* status, cudaStream_t stream) {
  static int found[kMaxDevices];
  int pairs = 0;
  MX_OK(bind_device());
  MX_OK(pairs_of(k_chain, found, &pairs));
  static thread_local ChainArgs g;  // some 20 KB
  memset(&g, 0, sizeof(g));
  g.classes = (int32_t)classes.size();
  g.phases = chain_phases(o, classes[0].deep, g.phase);

  auto square = [](const Class& c, int i, bool transposed = false) {
    Operand q;
    q.p = c.square[i];
    q.mn = q.k = c.side;
    q.ld = c.lds;
    q.zs = c.ss();
    q.z = c.count;
    q.mn_major = transposed;
    q.sym = !transposed;
    return q;
  };
  // an iterate as an operand: rows x cols, row-major, so its columns are contiguous
  auto iterate = [](const Class& c, int i, bool sum_over_rows) {
    Operand q;
    q.p = i == 0 ? c.x0 : c.x1;
    q.mn = sum_over_rows ? c.cols : c.rows;
    q.k = sum_over_rows ? c.rows : c.cols;
    q.ld = c.ld;
    q.zs = c.xs();
    q.z = c.count * (i == 0 && c.pair ? 2 : 1);
    q.mn_major = sum_over_rows;
    return q;
  };
  std::vector<Product> lists[3];
  for (const Class& c : classes) {
    Product p;
    p.batch = c.count;
    p.sym = p.padded = true;
    p.M = p.N = c.side;
    p.a = p.b = iterate(c, 0, c.tall);
    lists[PH_GRAM].push_back(p);
    p.a = p.b = square(c, 0);
    lists[PH_SQUARE].push_back(p);
    p.sym = false;
    p.M = c.rows;
    p.N = c.cols;
    p.a = c.tall ? iterate(c, 0, false) : square(c, 0);
    p.b = c.tall ? square(c, 0) : iterate(c, 0, true);
    p.parts = c.pair ? 2 : 1;
    lists[PH_APPLY].push_back(p);
  }
  int64_t most = 0;
  int widest = 0;
  for (int t = 0; t < 3; ++t) {
    // an application of the first iterate may sum over two parts, the others over one: its sums
    // are not split
    const Shape shape = choose(lists[t], pairs, t != PH_APPLY);
    int64_t split_tiles = 0;
    const int64_t units =
        place_products(lists[t], shape, sp.split_ws, sp.split_count, g.p[t], &split_tiles);
    if (units > kMaxUnits) return ta_fail(TA_ERR_UNSUPPORTED, "too many tiles in one call");
    g.units[t] = (int32_t)units;
    g.cols[t] = shape.cols;
    most = std::max(most, units);
    widest = std::max(widest, shape.cols);
  }
  for (size_t i = 0; i < classes.size(); ++i) {
    const Class& c = classes[i];
    ChainClass& d = g.c[i];
    for (int x = 0; x < 2; ++x) {
      const Operand gram = iterate(c, x, c.tall), app = iterate(c, x, !c.tall);
      MX_OK(make_map(&d.maps[MAP_GRAM_A + x], gram, false, kRows));
      MX_OK(make_map(&d.maps[MAP_GRAM_B + x], gram, false, g.cols[PH_GRAM] / 2));
      MX_OK(make_map(&d.maps[MAP_APPLY_X + x], app, false,
                     c.tall ? kRows : g.cols[PH_APPLY] / 2));
    }
    for (int q = 0; q < 3; ++q) {
      MX_OK(make_map(&d.maps[MAP_SQUARE_A + q], square(c, q), false, kRows));
      MX_OK(make_map(&d.maps[MAP_SQUARE_B + q], square(c, q), false, g.cols[PH_SQUARE] / 2));
      MX_OK(make_map(&d.maps[MAP_APPLY_S + q], square(c, q), false, g.cols[PH_APPLY] / 2));
      MX_OK(make_map(&d.maps[MAP_SQUARE_A_T + q], square(c, q, true), false, kRows));
      MX_OK(make_map(&d.maps[MAP_SQUARE_B_T + q], square(c, q, true), false,
                     g.cols[PH_SQUARE] / 2));
      MX_OK(make_map(&d.maps[MAP_APPLY_S_T + q], square(c, q, true), false,
                     g.cols[PH_APPLY] / 2));
      d.buf[BUF_S0 + q] = c.square[q];
    }
    d.buf[BUF_X0] = c.x0;
    d.buf[BUF_X1] = c.x1;
    d.xs = c.xs();
    d.ss = c.ss();
    d.ld = (int32_t)c.ld;
    d.lds = (int32_t)c.lds;
    d.tall = c.tall;
    d.pair = c.pair;
    d.scale = sp.scale + c.first;
    d.items = sp.table + c.first;
  }
  g.stages = stages_of(widest);
  g.stage_bytes = kTileABytes + widest * kDepth;
  g.arrivals = words;
  g.stop = words + 1;
  g.status = status;

  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeCooperative;
  attr.val.cooperative = 1;
  cfg.gridDim = dim3(2u * (unsigned)std::min<int64_t>(most, pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kProductSmem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  MX_CU(cudaLaunchKernelEx(&cfg, k_chain, g));
  return TA_OK;
}

ta_status run_ortho(const ta_ortho_tensor* ts, const ta_ortho_options* o, OrthoPlan& plan,
                    const OrthoSpace& sp, uint32_t* status, cudaStream_t stream) {
  // the table
  std::vector<ItemSeed> seeds;
  int64_t chunk = 0;
  for (size_t k = 0; k < plan.classes.size(); ++k) {
    const Class& c = plan.classes[k];
    const int64_t n = c.rows * c.cols, ce = chunk_elems(n, plan.elems), stored = c.xs() * (c.pair ? 2 : 1);
    int64_t slot = c.first;
    for (int i : plan.members[k]) {
      const ta_ortho_tensor& t = ts[i];
      ItemSeed s;
      memset(&s, 0, sizeof(s));
      s.it.g = t.in_dev;
      s.it.mom = t.momentum_dev;
      s.it.out = t.out_dev;
      s.it.x0 = c.x0 + (slot - c.first) * stored;
      s.it.x0_lo = c.pair ? s.it.x0 + c.xs() : nullptr;
      s.it.n = n;
      s.it.cols = (int32_t)c.cols;
      s.it.ld = (int32_t)c.ld;
      s.it.chunk0 = (int32_t)chunk;
      s.it.chunks = (int32_t)cdiv(n, ce);
      s.it.chunk_elems = ce;
      s.it.keep = (float)t.keep;
      s.it.gain = (float)t.gain;
      s.it.g_dt = (int16_t)t.in_dtype;
      s.it.mom_dt = (int16_t)t.momentum_dtype;
      s.it.out_dt = (int16_t)t.out_dtype;
      s.it.update = (t.flags & TA_ORTHO_UPDATE) != 0;
      s.first = (int32_t)slot;
      s.batch = (int32_t)t.batch;
      s.elem_zs = n;
      s.x0_zs = stored;
      seeds.push_back(s);
      slot += t.batch;
      chunk += t.batch * s.it.chunks;
    }
  }
  for (size_t lo = 0; lo < seeds.size(); lo += kSeeds) {
    TableArgs ta;
    memset(&ta, 0, sizeof(ta));
    ta.count = (int32_t)std::min<size_t>(kSeeds, seeds.size() - lo);
    std::copy(seeds.begin() + lo, seeds.begin() + lo + ta.count, ta.s);
    ta.table = sp.table;
    ta.scale = sp.scale;
    ta.partial = sp.partial;
    ta.zero = sp.split_count;
    ta.zero_words = lo == 0 ? (int32_t)kSplitTiles + 2 * chains_of(plan) : 0;
    int64_t most = 1;
    for (int i = 0; i < ta.count; ++i) most = std::max<int64_t>(most, ta.s[i].batch);
    MX_OK(launch(k_table, dim3((unsigned)std::min<int64_t>(cdiv(most, kEltThreads), 64)),
                 kEltThreads, 0, stream, ta));
  }
  const float mu = (float)o->momentum;
  const int items = (int)plan.items;
  MX_OK(launch(k_norm, dim3((unsigned)chunk), kEltThreads, 0, stream, sp.table, items, mu,
               o->nesterov));
  MX_OK(launch(k_scale, dim3((unsigned)chunk), kEltThreads, 0, stream, sp.table, items, mu,
               o->nesterov, o->eps));

  for (int i = 0; i < chains_of(plan); ++i) {
    const std::vector<Class> part(
        plan.classes.begin() + plan.chains[i],
        i + 1 < chains_of(plan) ? plan.classes.begin() + plan.chains[i + 1] : plan.classes.end());
    MX_OK(run_chain(part, o, sp, sp.chain + 2 * i, status, stream));
  }
  return TA_OK;
}

// ---- linear layer ----------------------------------------------------------------
// A 16-bit matrix given by its two strides, as an operand: TMA reads it where it lies if the
// lines start on 16 bytes, else it is copied into aligned lines.
struct Lines {
  bool mn_major = false;  // the mn dimension is contiguous
  int64_t lines = 0, len = 0, stride = 0;
  bool direct = false;
};

bool lines_of(const void* p, int64_t mn, int64_t k, int64_t s_mn, int64_t s_k, Lines* l) {
  if (s_k == 1 || k <= 1) {
    l->mn_major = false;
    l->lines = mn;
    l->len = k;
    l->stride = s_mn;
  } else if (s_mn == 1 || mn <= 1) {
    l->mn_major = true;
    l->lines = k;
    l->len = mn;
    l->stride = s_k;
  } else {
    return false;
  }
  if (l->lines <= 1) l->stride = up8(l->len);
  l->direct = aligned16(p) && l->stride % 8 == 0 && l->stride >= l->len;
  return l->lines <= 1 || l->stride >= l->len;
}

// The operand, and the copy it needs first (job->rows > 0).
Operand operand_of(const void* p, int64_t mn, int64_t k, const Lines& l, uint16_t* copy,
                   CopyJob* job) {
  Operand o;
  o.mn = mn;
  o.k = k;
  o.mn_major = l.mn_major;
  o.z = 1;
  if (l.direct) {
    o.p = p;
    o.ld = l.stride;
  } else {
    o.p = copy;
    o.ld = up8(l.len);
    job->src = reinterpret_cast<const uint16_t*>(p);
    job->stride = l.stride;
    job->dst = copy;
    job->rows = (int32_t)l.lines;
    job->cols = (int32_t)l.len;
    job->ld = (int32_t)o.ld;
  }
  o.zs = o.ld * l.lines;
  return o;
}

ta_status run_copies(CopyArgs a, cudaStream_t stream) {
  if (a.job[0].rows == 0) std::swap(a.job[0], a.job[1]);
  if (a.job[0].rows == 0) return TA_OK;
  int64_t pieces = 0;
  for (const CopyJob& j : a.job) pieces = std::max(pieces, (int64_t)j.rows * (j.ld / 8));
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(pieces, kEltThreads), 16 * sm_count()), 1,
                  a.job[1].rows ? 2 : 1);
  return launch(k_copy_rows, grid, kEltThreads, 0, stream, a);
}

size_t copy_elems(const Lines& l) { return l.direct ? 0 : (size_t)(up8(l.len) * l.lines); }

bool half_type(int dt) { return dt == TA_BF16 || dt == TA_F16; }
bool any_type(int dt) { return dt == TA_F32 || half_type(dt); }

ta_status check_sizes(int64_t tokens, int64_t fan_in, int64_t fan_out) {
  if (tokens < 0 || fan_in < 0 || fan_out < 0) return ta_fail(TA_ERR_INVALID, "negative size");
  if (tokens > kMaxDim || fan_in > kMaxDim || fan_out > kMaxDim)
    return ta_fail(TA_ERR_UNSUPPORTED, "a size is over 2^31 - 256");
  return TA_OK;
}

struct LinearSpace {
  float* split_ws;
  uint32_t* split_count;
  uint16_t *xc, *wc;
};

ta_status prepare_linear(const ta_linear* op, Lines* x, Lines* w) {
  if (!op) return ta_fail(TA_ERR_INVALID, "null operator");
  MX_OK(check_sizes(op->tokens, op->fan_in, op->fan_out));
  if (!half_type(op->dtype)) return ta_fail(TA_ERR_INVALID, "dtype must be TA_BF16 or TA_F16");
  if (op->bias_dev && !any_type(op->bias_dtype))
    return ta_fail(TA_ERR_INVALID, "bias_dtype must be TA_F32, TA_BF16 or TA_F16");
  MX_OK(check_typed({{"x", op->x_dev}, {"w", op->w_dev}, {"y", op->y_dev},
                     {"residual", op->residual_dev}}, op->dtype));
  if (op->bias_dev) MX_OK(check_typed({{"bias", op->bias_dev}}, op->bias_dtype));
  if (op->activation < TA_ACT_NONE || op->activation > TA_ACT_SILU)
    return ta_fail(TA_ERR_INVALID, "unknown activation");
  if (!lines_of(op->x_dev, op->tokens, op->fan_in, op->x_strides[0], op->x_strides[1], x))
    return ta_fail(TA_ERR_INVALID, "x needs one unit stride and lines that do not overlap");
  if (!lines_of(op->w_dev, op->fan_out, op->fan_in, op->w_strides[0], op->w_strides[1], w))
    return ta_fail(TA_ERR_INVALID, "w needs one unit stride and lines that do not overlap");
  return TA_OK;
}

LinearSpace carve_linear(const Lines& x, const Lines& w, Arena* a) {
  LinearSpace s;
  s.split_count = a->take<uint32_t>(kSplitTiles);
  s.split_ws = a->take<float>(kSplitFloats);
  s.xc = a->take<uint16_t>(copy_elems(x));
  s.wc = a->take<uint16_t>(copy_elems(w));
  return s;
}

ta_status check_space(const Arena& need, void* ws, size_t bytes, const uint32_t* status) {
  if (!ws && need.used) return ta_fail(TA_ERR_INVALID, "null workspace");
  if (bytes < need.used)
    return ta_fail(TA_ERR_WORKSPACE, "workspace has " + std::to_string(bytes) + " bytes, " +
                                         std::to_string(need.used) + " are needed");
  if ((uintptr_t)ws % 256) return ta_fail(TA_ERR_ALIGN, "workspace not 256-byte aligned");
  if (!status) return ta_fail(TA_ERR_INVALID, "null status word");
  if ((uintptr_t)status % 4) return ta_fail(TA_ERR_ALIGN, "status word not 4-byte aligned");
  return TA_OK;
}

// A few rows of A, each contiguous (the elements of an MN-major one are a line apart, of a single
// row too), against all of B, read where they lie.
bool few_rows(const Product& p) {
  if (p.M < 1 || p.M > kFewMax || p.a.k < 1) return false;
  if (p.a.mn_major) return false;
  if (!aligned16(p.a.p) || (p.M > 1 && p.a.ld % 8)) return false;
  return p.b.mn_major ? p.N % 8 == 0 : p.a.k % 8 == 0;  // (B's lines start on 16 bytes)
}

template <int DT, int T>
ta_status launch_few(FewArgs& g, bool cols, int64_t room, cudaStream_t stream) {
  const int sms = sm_count();
  if (!cols) {
    // enough blocks for two on every SM, by letting warps share a sum where N is small
    g.warps_n = 8;
    while (g.warps_n > 1 && cdiv(g.N, g.warps_n * kFewRows) < 2 * sms) g.warps_n /= 2;
    return launch(k_few_rows<DT, T>, dim3((unsigned)cdiv(g.N, g.warps_n * kFewRows)), 256,
                  kFewRing, stream, g);
  }
  const int64_t blocks = cdiv(g.N, 256);
  int64_t splits = std::min<int64_t>(cdiv(4 * sms, blocks), cdiv(g.K, 32));
  splits = std::min(splits, room / ((int64_t)g.tokens * g.N));
  g.splits = (int)std::max<int64_t>(1, splits);
  MX_OK(launch(k_few_cols<DT, T>, dim3((unsigned)blocks, (unsigned)g.splits), 256, 0, stream, g));
  return launch(k_few_finish<DT>, dim3((unsigned)blocks, (unsigned)g.tokens), 256, 0, stream, g);
}

template <int DT>
ta_status run_few(const Product& p, const Out& out, float* part, int64_t room,
                  cudaStream_t stream) {
  FewArgs g;
  memset(&g, 0, sizeof(g));
  g.a = reinterpret_cast<const uint16_t*>(p.a.p);
  g.b = reinterpret_cast<const uint16_t*>(p.b.p);
  g.lda = p.a.ld;
  g.ldb = p.b.ld;
  g.tokens = (int)p.M;
  g.N = (int)p.N;
  g.K = (int)p.a.k;
  g.part = part;
  g.out = reinterpret_cast<uint16_t*>(out.out);
  g.aux = reinterpret_cast<const uint16_t*>(out.aux);
  g.bias = out.bias;
  g.deriv = out.deriv;
  g.ldo = out.ld;
  g.ld_aux = out.ld_aux;
  g.ld_deriv = out.ld_deriv;
  g.bias_dt = out.bias_dt;
  g.act = out.act;
  const bool cols = p.b.mn_major;
  if (g.tokens == 1) return launch_few<DT, 1>(g, cols, room, stream);
  if (g.tokens == 2) return launch_few<DT, 2>(g, cols, room, stream);
  return launch_few<DT, kFewMax>(g, cols, room, stream);
}

// The products of one linear call.
ta_status run_products(std::vector<Product> ps, std::vector<Out> outs, bool bf16,
                       const LinearSpace& s, uint32_t* status, cudaStream_t stream,
                       bool epilogue) {
  for (size_t i = 0; i < ps.size();) {
    if (few_rows(ps[i]) && ps[i].M * ps[i].N <= kSplitFloats) {
      MX_OK(bf16 ? run_few<DT_BF16>(ps[i], outs[i], s.split_ws, kSplitFloats, stream)
                 : run_few<DT_F16>(ps[i], outs[i], s.split_ws, kSplitFloats, stream));
      ps.erase(ps.begin() + i);
      outs.erase(outs.begin() + i);
    } else {
      ++i;
    }
  }
  if (ps.empty()) return TA_OK;
  auto run = [&](auto fn) { return fn(ps, outs, s.split_ws, s.split_count, status, stream); };
  if (epilogue) return bf16 ? run(run_linear<true, DT_BF16>) : run(run_linear<true, DT_F16>);
  return bf16 ? run(run_linear<false, DT_BF16>) : run(run_linear<false, DT_F16>);
}

struct GradLines {
  Lines dz_t, dz_o, x, w;  // dz as tokens x fan_out and as fan_out x tokens; x, w over k
  bool dw_io = false;      // dw's rows are fan_in
  bool make_dz = false;
  int64_t row_parts = 0, col_blocks = 0, col_threads = 0, ld_dz = 0;
};

ta_status prepare_grad(const ta_linear_grad* op, GradLines* g) {
  if (!op) return ta_fail(TA_ERR_INVALID, "null operator");
  MX_OK(check_sizes(op->tokens, op->fan_in, op->fan_out));
  if (!half_type(op->dtype)) return ta_fail(TA_ERR_INVALID, "dtype must be TA_BF16 or TA_F16");
  if (op->db_dev && !any_type(op->bias_dtype))
    return ta_fail(TA_ERR_INVALID, "bias_dtype must be TA_F32, TA_BF16 or TA_F16");
  MX_OK(check_typed({{"dy", op->dy_dev}, {"x", op->x_dev}, {"w", op->w_dev}, {"dx", op->dx_dev},
                     {"dw", op->dw_dev}}, op->dtype));
  if (op->db_dev) MX_OK(check_typed({{"db", op->db_dev}}, op->bias_dtype));
  const bool work = op->tokens > 0 && op->fan_out > 0;
  if (work && !op->dy_dev) return ta_fail(TA_ERR_INVALID, "null dy");
  if (op->tokens > 1 && op->dy_stride < op->fan_out)
    return ta_fail(TA_ERR_INVALID, "rows of dy overlap");
  if (op->dx_dev && op->fan_out > 0 && op->fan_in > 0 && !op->w_dev)
    return ta_fail(TA_ERR_INVALID, "dx needs w");
  if (op->dw_dev && op->tokens > 0 && op->fan_in > 0 && !op->x_dev)
    return ta_fail(TA_ERR_INVALID, "dw needs x");
  if (op->dx_dev && !lines_of(op->w_dev, op->fan_in, op->fan_out, op->w_strides[1],
                              op->w_strides[0], &g->w))
    return ta_fail(TA_ERR_INVALID, "w needs one unit stride and lines that do not overlap");
  if (op->dw_dev) {
    if (!lines_of(op->x_dev, op->fan_in, op->tokens, op->x_strides[1], op->x_strides[0], &g->x))
      return ta_fail(TA_ERR_INVALID, "x needs one unit stride and lines that do not overlap");
    Lines d;
    if (!lines_of(op->dw_dev, op->fan_out, op->fan_in, op->dw_strides[0], op->dw_strides[1], &d))
      return ta_fail(TA_ERR_INVALID, "dw needs one unit stride and lines that do not overlap");
    g->dw_io = d.mn_major;
  }
  const int64_t stride = op->tokens > 1 ? op->dy_stride : up8(op->fan_out);
  g->make_dz = op->deriv_dev || !aligned16(op->dy_dev) || stride % 8;
  g->ld_dz = g->make_dz ? up8(op->fan_out) : stride;
  // rows are split until there are some 16 blocks for every SM (8: 2 % slower at 8192 x 14336), of
  // 8 rows or more; a bias gradient's parts, which are written and read once more, end at 256 (512
  // and 1024: 2 and 7 % of a 8192 x 4096 call lost, of 8192 x 768 one 10 % gained)
  if (op->db_dev || g->make_dz) {
    const int64_t pieces = std::max<int64_t>(1, cdiv(op->fan_out, 8));
    g->col_blocks = cdiv(pieces, kEltThreads);
    g->col_threads = cdiv(cdiv(pieces, g->col_blocks), 32) * 32;
    g->row_parts = std::max<int64_t>(
        1, std::min<int64_t>({cdiv(op->tokens, 8), cdiv(16 * sm_count(), g->col_blocks),
                              (int64_t)(op->db_dev ? 256 : 32768)}));
  }
  return TA_OK;
}

struct GradSpace {
  LinearSpace lin;
  uint16_t* dz;
  float* part;
};
GradSpace carve_grad(const ta_linear_grad* op, const GradLines& g, Arena* a) {
  GradSpace s;
  s.lin = carve_linear(op->dw_dev ? g.x : Lines{false, 0, 0, 0, true},
                       op->dx_dev ? g.w : Lines{false, 0, 0, 0, true}, a);
  s.dz = a->take<uint16_t>(g.make_dz ? op->tokens * g.ld_dz : 0);
  s.part = a->take<float>(op->db_dev ? g.row_parts * op->fan_out : 0);
  return s;
}

}  // namespace

extern "C" {

size_t ta_ortho_workspace_size(const ta_ortho_tensor* tensors, int32_t n_tensors,
                               const ta_ortho_options* options) {
  try {
    ta_fail(TA_OK, "");
    OrthoPlan plan;
    if (plan_ortho(tensors, n_tensors, options, &plan) != TA_OK) return 0;
    Arena a{nullptr};
    carve_ortho(&plan, &a);
    return a.used;
  } catch (const std::exception& e) {
    ta_fail(TA_ERR_INVALID, e.what());
    return 0;
  }
}

ta_status ta_orthogonalize(const ta_ortho_tensor* tensors, int32_t n_tensors,
                           const ta_ortho_options* options, void* workspace_dev,
                           size_t workspace_bytes, uint32_t* status_dev, void* stream) {
  try {
    ta_fail(TA_OK, "");
    OrthoPlan plan;
    MX_OK(plan_ortho(tensors, n_tensors, options, &plan));
    if (plan.items == 0) return TA_OK;
    Arena need{nullptr};
    carve_ortho(&plan, &need);
    MX_OK(check_space(need, workspace_dev, workspace_bytes, status_dev));
    Arena a{reinterpret_cast<uint8_t*>(workspace_dev)};
    const OrthoSpace sp = carve_ortho(&plan, &a);
    return run_ortho(tensors, options, plan, sp, status_dev, (cudaStream_t)stream);
  } catch (const std::exception& e) {
    return ta_fail(TA_ERR_INVALID, e.what());
  }
}

size_t ta_linear_workspace_size(const ta_linear* op) {
  try {
    ta_fail(TA_OK, "");
    Lines x, w;
    if (prepare_linear(op, &x, &w) != TA_OK) return 0;
    Arena a{nullptr};
    carve_linear(x, w, &a);
    return a.used;
  } catch (const std::exception& e) {
    ta_fail(TA_ERR_INVALID, e.what());
    return 0;
  }
}

ta_status ta_linear_forward(const ta_linear* op, void* workspace_dev, size_t workspace_bytes,
                            uint32_t* status_dev, void* stream_) {
  try {
    ta_fail(TA_OK, "");
    Lines x, w;
    MX_OK(prepare_linear(op, &x, &w));
    if (op->tokens == 0 || op->fan_out == 0) return TA_OK;
    if (!op->y_dev || (op->fan_in > 0 && (!op->x_dev || !op->w_dev)))
      return ta_fail(TA_ERR_INVALID, "null pointer");
    if ((op->tokens > 1 && op->y_stride < op->fan_out) ||
        (op->residual_dev && op->tokens > 1 && op->residual_stride < 0))
      return ta_fail(TA_ERR_INVALID, "bad row stride");
    if (op->y_stride > kMaxDim || op->residual_stride > kMaxDim)
      return ta_fail(TA_ERR_UNSUPPORTED, "a row stride is over 2^31 - 256");
    if (op->deriv_dev && !aligned16(op->deriv_dev))
      return ta_fail(TA_ERR_ALIGN, "deriv not 16-byte aligned");
    Arena need{nullptr};
    carve_linear(x, w, &need);
    MX_OK(check_space(need, workspace_dev, workspace_bytes, status_dev));
    Arena a{reinterpret_cast<uint8_t*>(workspace_dev)};
    const LinearSpace s = carve_linear(x, w, &a);
    cudaStream_t stream = (cudaStream_t)stream_;
    Product p;
    if (op->fan_in > 0) {
      CopyArgs copies;
      memset(&copies, 0, sizeof(copies));
      p.a = operand_of(op->x_dev, op->tokens, op->fan_in, x, s.xc, &copies.job[0]);
      p.b = operand_of(op->w_dev, op->fan_out, op->fan_in, w, s.wc, &copies.job[1]);
      MX_OK(run_copies(copies, stream));
    }
    p.M = op->tokens;
    p.N = op->fan_out;
    Out out;
    memset(&out, 0, sizeof(out));
    out.out = reinterpret_cast<uint8_t*>(op->y_dev);
    out.ld = op->y_stride;
    out.aux = reinterpret_cast<const uint8_t*>(op->residual_dev);
    out.ld_aux = op->residual_stride;
    out.bias = op->bias_dev;
    out.bias_dt = op->bias_dtype;
    out.act = op->activation;
    out.deriv = op->deriv_dev;
    out.ld_deriv = up8(op->fan_out);
    return run_products({p}, {out}, op->dtype == TA_BF16, s, status_dev, stream, true);
  } catch (const std::exception& e) {
    return ta_fail(TA_ERR_INVALID, e.what());
  }
}

size_t ta_linear_backward_workspace_size(const ta_linear_grad* op) {
  try {
    ta_fail(TA_OK, "");
    GradLines g;
    if (prepare_grad(op, &g) != TA_OK) return 0;
    Arena a{nullptr};
    carve_grad(op, g, &a);
    return a.used;
  } catch (const std::exception& e) {
    ta_fail(TA_ERR_INVALID, e.what());
    return 0;
  }
}

ta_status ta_linear_backward(const ta_linear_grad* op, void* workspace_dev,
                             size_t workspace_bytes, uint32_t* status_dev, void* stream_) {
  try {
    ta_fail(TA_OK, "");
    GradLines g;
    MX_OK(prepare_grad(op, &g));
    if (op->deriv_dev && !aligned16(op->deriv_dev))
      return ta_fail(TA_ERR_ALIGN, "deriv not 16-byte aligned");
    Arena need{nullptr};
    carve_grad(op, g, &need);
    MX_OK(check_space(need, workspace_dev, workspace_bytes, status_dev));
    Arena a{reinterpret_cast<uint8_t*>(workspace_dev)};
    const GradSpace s = carve_grad(op, g, &a);
    cudaStream_t stream = (cudaStream_t)stream_;
    const int64_t T = op->tokens, I = op->fan_in, O = op->fan_out;
    const bool bf16 = op->dtype == TA_BF16;
    const void* dz = g.make_dz ? (const void*)s.dz : op->dy_dev;
    if (O > 0 && (g.make_dz || op->db_dev)) {
      const dim3 grid((unsigned)g.col_blocks, (unsigned)g.row_parts);
      MX_OK(launch(bf16 ? k_dz<DT_BF16> : k_dz<DT_F16>, grid, (int)g.col_threads, 0, stream,
                   reinterpret_cast<const uint16_t*>(op->dy_dev), op->dy_stride, op->deriv_dev,
                   (int)up8(O), (int)T, (int)O, g.make_dz ? s.dz : nullptr, (int)g.ld_dz,
                   op->db_dev ? s.part : nullptr));
      if (op->db_dev)
        MX_OK(launch(k_bias_grad, dim3((unsigned)cdiv(O, 32)), kEltThreads, 0, stream,
                     s.part, (int)g.row_parts, (int)O, op->db_dev, (int)op->bias_dtype));
    }
    auto result = [](void* p, int64_t ld) {
      Out out;
      memset(&out, 0, sizeof(out));
      out.out = reinterpret_cast<uint8_t*>(p);
      out.ld = ld;
      return out;
    };
    auto dz_operand = [&](bool over_tokens) {  // summed over tokens (dw) or fan_out (dx)
      Operand o;
      o.p = dz;
      o.mn = over_tokens ? O : T;
      o.k = over_tokens ? T : O;
      o.mn_major = over_tokens;
      o.ld = g.ld_dz;
      o.zs = g.ld_dz * T;
      return o;
    };
    // both products in one launch: each fills the other's last round of tiles
    std::vector<Product> ps;
    std::vector<Out> outs;
    CopyArgs copies;
    memset(&copies, 0, sizeof(copies));
    if (op->dx_dev && T > 0 && I > 0) {
      Product p;
      if (O > 0) {
        p.a = dz_operand(false);
        p.b = operand_of(op->w_dev, I, O, g.w, s.lin.wc, &copies.job[0]);
      }
      p.M = T;
      p.N = I;
      ps.push_back(p);
      outs.push_back(result(op->dx_dev, I));
    }
    if (op->dw_dev && O > 0 && I > 0) {
      Product p;
      Operand xo, zo;
      if (T > 0) {
        xo = operand_of(op->x_dev, I, T, g.x, s.lin.xc, &copies.job[1]);
        zo = dz_operand(true);
      }
      p.a = g.dw_io ? xo : zo;
      p.b = g.dw_io ? zo : xo;
      p.M = g.dw_io ? I : O;
      p.N = g.dw_io ? O : I;
      const int64_t ldo = op->dw_strides[g.dw_io ? 1 : 0];
      ps.push_back(p);
      outs.push_back(result(op->dw_dev, p.M > 1 ? ldo : p.N));
    }
    MX_OK(run_copies(copies, stream));
    if (!ps.empty()) MX_OK(run_products(ps, outs, bf16, s.lin, status_dev, stream, false));
    return TA_OK;
  } catch (const std::exception& e) {
    return ta_fail(TA_ERR_INVALID, e.what());
  }
}

}  // extern "C"
