// ta_mx_chain.cuh -- the Newton-Schulz products of a list of matrices as one
// persistent kernel: a chain of phases, each a list of symmetric or general
// products on the tile engine's roles, with a barrier over the grid between them.
//
// Why one kernel. Five steps are 16 or 17 dependent products. Launched one by one each
// paid some 10 us at these sizes for set-up, cold instructions and descriptors,
// the first loads and the tail (12 x 768 x 768: 262 us for 80 us of products).
// Here tensor memory, barriers, tensor maps and code stay, and a phase costs its
// products and a barrier. The launch is cooperative, so that every CTA is
// resident; every wait, the grid's included, ends after 2 s, and one that ran
// out ends the others through a flag.
//
// Memory between phases: results are written with ordinary stores and read by
// TMA (the async proxy) of other SMs. A CTA's epilogue threads meet, one of them
// adds to the grid's counter behind a fence; the copy warp that sees the counter
// complete acquires it and lets the CTA's other warps go, and each warp that
// reads the results fences the proxies first.
#pragma once

#include "ta_mx_product.cuh"

namespace ta {
namespace mx {

constexpr int kMaxClasses = 8;   // shapes in one chain (they travel as kernel parameters)
constexpr int kMaxPhases = 116;  // 32 steps

enum PhaseType { PH_GRAM = 0, PH_SQUARE = 1, PH_APPLY = 2 };
enum PhaseEnd { END_SCALE = 0, END_POLY = 1, END_FINAL = 2 };

// Buffers of a class: two iterates, three square matrices.
enum { BUF_X0 = 0, BUF_X1 = 1, BUF_S0 = 2, kBuffers = 5 };
// Tensor maps of a class, by role: an iterate as either operand of its Gram matrix and as the
// iterate of an application; a square matrix as either operand of a square product and as the
// right operand of an application, each also transposed (its blocks under the diagonal).
enum { MAP_GRAM_A = 0, MAP_GRAM_B = 2, MAP_APPLY_X = 4, MAP_SQUARE_A = 6, MAP_SQUARE_B = 9,
       MAP_APPLY_S = 12, MAP_SQUARE_A_T = 15, MAP_SQUARE_B_T = 18, MAP_APPLY_S_T = 21, kMaps = 24 };

struct Phase {
  int8_t type, end, a, b, out, aux;  // operands and result as buffers
  int8_t unit_pow;                   // the matrix's unit enters alpha to this power
  int8_t whole;                      // APPLY: takes both parts of a pair
  float alpha, c0, c1;
};

struct ChainClass {
  CUtensorMap maps[kMaps];
  __half* buf[kBuffers];
  int64_t xs, ss;        // elements of an iterate, of a square matrix
  int32_t ld, lds;
  int32_t tall, pair;    // pair: BUF_X0 holds two parts of each matrix
  const Scale* scale;    // [matrices]
  const Item* items;
};

struct ChainArgs {
  ChainClass c[kMaxClasses];
  Problem p[3][kMaxClasses];  // by phase type
  Phase phase[kMaxPhases];
  int32_t units[3], cols[3];
  int32_t classes, phases, stages, stage_bytes;
  uint32_t* arrivals;  // zero
  uint32_t* stop;      // zero
  uint32_t* status;
};

struct ChainView {
  struct Target {
    uint8_t* out;
    const uint8_t* aux;
    const Item* item;
    int32_t ld, ld_aux;
    float alpha;
    __device__ __forceinline__ void pin() const {
      asm volatile("" ::"l"(out), "l"(aux), "r"(ld), "r"(ld_aux), "l"(item), "f"(alpha));
    }
  };
  const ChainArgs& g;
  const Phase& ph;
  __device__ __forceinline__ int count() const { return g.classes; }
  __device__ __forceinline__ int units() const { return g.units[ph.type]; }
  __device__ __forceinline__ int cols() const { return g.cols[ph.type]; }
  __device__ __forceinline__ bool bf16() const { return false; }
  __device__ __forceinline__ const Problem& problem(int p) const { return g.p[ph.type][p]; }
  // an application's operands are (square, iterate), of a tall matrix (iterate, square)
  __device__ __forceinline__ const CUtensorMap* map_a(int p) const {
    const ChainClass& c = g.c[p];
    const int m = ph.type == PH_GRAM     ? MAP_GRAM_A + ph.a
                  : ph.type == PH_SQUARE ? MAP_SQUARE_A + ph.a - BUF_S0
                  : c.tall               ? MAP_APPLY_X + ph.b
                                         : MAP_SQUARE_A + ph.a - BUF_S0;
    return &c.maps[m];
  }
  __device__ __forceinline__ const CUtensorMap* map_b(int p) const {
    const ChainClass& c = g.c[p];
    const int m = ph.type == PH_GRAM     ? MAP_GRAM_B + ph.b
                  : ph.type == PH_SQUARE ? MAP_SQUARE_B + ph.b - BUF_S0
                  : c.tall               ? MAP_APPLY_S + ph.a - BUF_S0
                                         : MAP_APPLY_X + ph.b;
    return &c.maps[m];
  }
  __device__ __forceinline__ const CUtensorMap* map_a_t(int p) const {
    return &g.c[p].maps[MAP_SQUARE_A_T + ph.a - BUF_S0];
  }
  __device__ __forceinline__ const CUtensorMap* map_b_t(int p) const {
    return &g.c[p].maps[ph.type == PH_SQUARE ? MAP_SQUARE_B_T + ph.b - BUF_S0
                                             : MAP_APPLY_S_T + ph.a - BUF_S0];
  }
  // the first iterate's storage holds two planes of each matrix of a pair
  __device__ __forceinline__ int planes(int p, int buf) const {
    return buf == BUF_X0 && g.c[p].pair ? 2 : 1;
  }
  __device__ __forceinline__ int za(int p) const {
    if (ph.type == PH_GRAM) return planes(p, ph.a);
    return ph.type == PH_APPLY && g.c[p].tall ? planes(p, ph.b) : 1;
  }
  __device__ __forceinline__ int zb(int p) const {
    if (ph.type == PH_GRAM) return planes(p, ph.b);
    return ph.type == PH_APPLY && !g.c[p].tall ? planes(p, ph.b) : 1;
  }
  __device__ __forceinline__ int parts(int p) const {
    return ph.whole && g.c[p].pair ? 2 : 1;
  }
  __device__ __forceinline__ Target target(int p, int z) const {
    const ChainClass& c = g.c[p];
    const bool square = ph.type != PH_APPLY;
    Target t;
    t.out = nullptr;
    t.aux = nullptr;
    t.item = nullptr;
    t.ld = square ? c.lds : c.ld;
    t.ld_aux = c.lds;
    if (ph.end == END_FINAL) {
      t.item = c.items + z;
    } else {
      const int64_t zs = square ? c.ss : c.xs * planes(p, ph.out);
      t.out = reinterpret_cast<uint8_t*>(c.buf[ph.out] + z * zs);
      if (ph.end == END_POLY) t.aux = reinterpret_cast<const uint8_t*>(c.buf[ph.aux] + z * c.ss);
    }
    t.alpha = ph.alpha;
    if (ph.unit_pow) {
      const float unit = c.scale[z].unit;
      t.alpha *= ph.unit_pow == 2 ? unit * unit : unit;
    }
    return t;
  }
  // the polynomial's A: on its way into L1 while the products run
  __device__ __forceinline__ void prefetch(const Target& t, const Block& b, int64_t row0, int col,
                                           int n_end) const {
    if (ph.end == END_POLY && b.lane < b.rows && col < n_end)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(
          t.aux + ((row0 + b.lane) * t.ld_aux + col) * 2));
  }
  __device__ __forceinline__ void finish(const Target& t, const Block& b, float (&v)[32],
                                         int64_t row0, int col, int n, int N) const {
    if (ph.end == END_POLY) {
      finish_half<true>(t.out, t.ld, t.aux, t.ld_aux, b, v, t.alpha, ph.c0, ph.c1, row0, col);
    } else if (ph.end == END_SCALE) {
      finish_half<false>(t.out, t.ld, nullptr, 0, b, v, t.alpha, 0.f, 0.f, row0, col);
    } else {
      const int dt = t.item->out_dt;
      n = min(n, N - col);  // the result's lines are not padded
      if (dt == DT_BF16) finish_final<DT_BF16>(*t.item, b, v, t.alpha, N, row0, col, n);
      else if (dt == DT_F32) finish_final<DT_F32>(*t.item, b, v, t.alpha, N, row0, col, n);
      else finish_final<DT_F16>(*t.item, b, v, t.alpha, N, row0, col, n);
    }
  }
};

// Waits until `target` CTA arrivals; false after 2 s, or once any CTA has given up.
__device__ __forceinline__ bool grid_wait(const ChainArgs& g, uint32_t target) {
  const uint64_t t0 = now_ns();
  for (uint32_t n = 0;; ++n) {
    uint32_t seen;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(g.arrivals) : "memory");
    if (seen >= target) return true;
    if ((n & 63) == 63) {
      const bool stopped = *(volatile uint32_t*)g.stop != 0;
      if (stopped || now_ns() - t0 > kWaitLimitNs) {
        if (!stopped) {
          atomicOr(g.status, kStatusTimeout);
          atomicExch(g.stop, 1u);
        }
        return false;
      }
    }
  }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    k_chain(const __grid_constant__ ChainArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Cta x;
  cta_begin(x, smem, g.stages, g.stage_bytes, g.status);
  // the CTA's own barriers between phases: the first copy warp opens `go`, the second copy warp
  // answers on `passed`
  const uint32_t go = x.tiles0 + kBarrierOffset + 8 * (2 * kMaxStages + 5);
  const uint32_t passed = go + 8;
  if (threadIdx.x == 0) {
    bar_init(go, 1);
    bar_init(passed, 1);
    bar_init_fence();
  }
  cta_meet(x);
  Ring r;
  r.phase = warp < 2 ? 1 : 0;
  Block b;
  if (warp >= kFirstEpi)
    b.init(x.tiles0 + (uint32_t)kOperandSpace + (warp - kFirstEpi) * kBlockBytes, lane);
  for (int i = 0; i < g.phases; ++i) {
    const ChainView v{g, g.phase[i]};
    const Unit w = locate(v, min(x.worker, v.units() - 1), 0);
    // Between phases: the first copy warp waits for the grid and opens the CTA's barrier. A barrier
    // that opened twice would look closed to a warp that had yet to see the first time, so nobody
    // may be left behind: the epilogue warps passed the last gate before this CTA arrived at the
    // grid; the second copy warp, which has no part in that where the CTA has no unit, answers.
    auto gate = [&] {
      if (i == 0 || !r.ok) return r.ok;
      bool ok;
      if (warp == 0) {
        ok = i == 1 || __all_sync(0xffffffffu, bar_wait(passed, (i - 2) & 1, g.status));
        ok = ok && __all_sync(0xffffffffu, grid_wait(g, (uint32_t)i * gridDim.x));
        if (ok && lane == 0) bar_arrive_cluster(go);
      } else {
        ok = __all_sync(0xffffffffu, bar_wait(go, (i - 1) & 1, g.status));
        if (ok && warp == 1 && lane == 0) bar_arrive_cluster(passed);
      }
      asm volatile("fence.proxy.async.global;" ::: "memory");
      return ok;
    };
    if (warp < 2) {
      copy_units(v, x, r, w, warp == 0, gate);
    } else if (warp == 2) {
      if (x.rank == 0) mma_units(v, x, r, w);
    } else if (warp >= kFirstEpi) {
      finish_units(v, x, r, w, b, gate);
      epilogue_sync();
      if (threadIdx.x == 32 * kFirstEpi) {
        __threadfence();
        atomicAdd(g.arrivals, 1u);
      }
    }
    if (!r.ok && lane == 0) atomicExch(g.stop, 1u);
  }
  if (warp < 2) copy_drain(x, r);
  cta_end(x);
}

}  // namespace mx
}  // namespace ta
