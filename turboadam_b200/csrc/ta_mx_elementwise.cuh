// ta_mx_elementwise.cuh -- the passes around the products of the matrix
// operators: momentum and norm, scaling into fp16, the activation's gradient
// with the bias gradient, and operand copies with aligned rows.
#pragma once

#include "ta_mx_product.cuh"

namespace ta {
namespace mx {

constexpr int kEltThreads = 256;
constexpr int kMaxChunks = 1024;  // partial sums of one matrix

// ---- table ---------------------------------------------------------------------
// The items of a list travel as kernel parameters and are written to the workspace by a
// kernel, so that a call enqueues kernels only and can be captured into a CUDA graph.
struct ItemSeed {
  Item it;
  int32_t first, batch;  // table slots [first, first + batch)
  int64_t elem_zs;       // elements between the matrices of g, mom and out
  int64_t x0_zs;         // elements between the scaled matrices
};
constexpr int kSeeds = 20;
struct TableArgs {
  ItemSeed s[kSeeds];
  int32_t count;
  Item* table;
  Scale* scale;
  double* partial;
  uint32_t* zero;  // words to clear
  int32_t zero_words;
};

__device__ __forceinline__ const void* offset_dt(const void* p, int64_t elems, int dt) {
  return p ? reinterpret_cast<const uint8_t*>(p) + elems * (dt == DT_F32 ? 4 : 2) : nullptr;
}

__global__ void __launch_bounds__(kEltThreads) k_table(const __grid_constant__ TableArgs a) {
  chain_next();
  chain_wait();
  const int t = blockIdx.x * blockDim.x + threadIdx.x, stride = gridDim.x * blockDim.x;
  for (int i = t; i < a.zero_words; i += stride) a.zero[i] = 0;
  for (int k = 0; k < a.count; ++k) {
    const ItemSeed& s = a.s[k];
    for (int z = t; z < s.batch; z += stride) {
      Item it = s.it;
      it.g = offset_dt(it.g, z * s.elem_zs, it.g_dt);
      it.mom = const_cast<void*>(offset_dt(it.mom, z * s.elem_zs, it.mom_dt));
      it.out = const_cast<void*>(offset_dt(it.out, z * s.elem_zs, it.out_dt));
      it.x0 += z * s.x0_zs;
      if (it.x0_lo) it.x0_lo += z * s.x0_zs;
      it.chunk0 += z * it.chunks;
      it.partial = a.partial + it.chunk0;
      it.scale = a.scale + s.first + z;
      a.table[s.first + z] = it;
    }
  }
}

// The item whose chunks hold chunk c.
__device__ __forceinline__ const Item& find_item(const Item* table, int count, int c) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table[mid].chunk0 <= c) lo = mid;
    else hi = mid - 1;
  }
  return table[lo];
}

// Sum over the block in a fixed order; the result is valid in every thread.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double warp_sum[kEltThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0;
#pragma unroll
  for (int i = 0; i < kEltThreads / 32; ++i) s += warp_sum[i];
  __syncthreads();
  return s;
}

// stretches of a thread whose loads are under way together: 4 hold too many registers for four
// blocks an SM (12 x 768 x 768 orthogonalised: 191 us against 181), 1 and 2 measure alike
constexpr int kUnroll = 2;

struct alignas(16) F8 {
  float v[8];
};
__device__ __forceinline__ F8 load8(const void* p, int64_t i, int dt) {
  F8 r;
  if (dt == DT_F32) {
    const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    const float4 a = q[0], b = q[1];
    r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w;
    r.v[4] = b.x; r.v[5] = b.y; r.v[6] = b.z; r.v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
    float2 f;
    f = unpack16(u.x, dt); r.v[0] = f.x; r.v[1] = f.y;
    f = unpack16(u.y, dt); r.v[2] = f.x; r.v[3] = f.y;
    f = unpack16(u.z, dt); r.v[4] = f.x; r.v[5] = f.y;
    f = unpack16(u.w, dt); r.v[6] = f.x; r.v[7] = f.y;
  }
  return r;
}
__device__ __forceinline__ void store8(void* p, int64_t i, int dt, const F8& r) {
  if (dt == DT_F32) {
    float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
    q[0] = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
    q[1] = make_float4(r.v[4], r.v[5], r.v[6], r.v[7]);
  } else {
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) =
        make_uint4(pack16(r.v[0], r.v[1], dt), pack16(r.v[2], r.v[3], dt),
                   pack16(r.v[4], r.v[5], dt), pack16(r.v[6], r.v[7], dt));
  }
}
// A momentum kept in 16 bits enters the update as it is stored.
__device__ __forceinline__ float as_stored(float v, int dt) {
  if (dt == DT_BF16) return __bfloat162float(__float2bfloat16_rn(v));
  if (dt == DT_F16) return __half2float(__float2half_rn(v));
  return v;
}
__device__ __forceinline__ float direction(float g, float m, float mu, bool nesterov) {
  return nesterov ? fmaf(mu, m, (1.f - mu) * g) : m;
}
__device__ __forceinline__ bool item_vec(const Item& it) {
  return it.n % 8 == 0 && (((uintptr_t)it.g | (uintptr_t)it.mom) & 15) == 0;
}

// Momentum m <- mu m + (1 - mu) g, and a chunk's sum of squares of the update direction. Bound
// by the bytes of g and m. The squares are summed in 64 bits: gradients whose squares leave
// fp32's range keep their norm.
__global__ void __launch_bounds__(kEltThreads)
    k_norm(const Item* table, int count, float mu, int nesterov) {
  chain_next();
  chain_wait();
  const Item& it = find_item(table, count, blockIdx.x);
  const int chunk = blockIdx.x - it.chunk0;
  const int64_t e0 = chunk * it.chunk_elems, e1 = min(it.n, e0 + it.chunk_elems);
  double sum = 0;
  const bool mom = it.mom != nullptr;
  if (item_vec(it)) {
    for (int64_t i0 = e0 + threadIdx.x * 8; i0 < e1; i0 += kEltThreads * 8 * kUnroll) {
      F8 g[kUnroll], m[kUnroll];
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int64_t i = i0 + q * kEltThreads * 8;
        if (i >= e1) continue;
        g[q] = load8(it.g, i, it.g_dt);
        if (mom) m[q] = load8(it.mom, i, it.mom_dt);
      }
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int64_t i = i0 + q * kEltThreads * 8;
        if (i >= e1) continue;
        if (mom) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            m[q].v[k] = as_stored(fmaf(mu, m[q].v[k], (1.f - mu) * g[q].v[k]), it.mom_dt);
            g[q].v[k] = direction(g[q].v[k], m[q].v[k], mu, nesterov);
          }
          store8(it.mom, i, it.mom_dt, m[q]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) sum = fma((double)g[q].v[k], (double)g[q].v[k], sum);
      }
    }
  } else {
    for (int64_t i0 = e0 + threadIdx.x; i0 < e1; i0 += kEltThreads * kUnroll) {
      float u[kUnroll], m[kUnroll];
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int64_t i = i0 + q * kEltThreads;
        u[q] = i < e1 ? load_as_float(it.g, i, it.g_dt) : 0.f;
        m[q] = mom && i < e1 ? load_as_float(it.mom, i, it.mom_dt) : 0.f;
      }
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int64_t i = i0 + q * kEltThreads;
        if (i >= e1) continue;
        if (mom) {
          m[q] = as_stored(fmaf(mu, m[q], (1.f - mu) * u[q]), it.mom_dt);
          store_from_float(it.mom, i, it.mom_dt, m[q]);
          u[q] = direction(u[q], m[q], mu, nesterov);
        }
        sum = fma((double)u[q], (double)u[q], sum);
      }
    }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) it.partial[chunk] = sum;
}

// The update direction scaled by a power of two into fp16: its Frobenius norm lands in
// [2^13, 2^14), so that no element overflows and one 2^-38 of the norm still has a code. The
// scaling is exact; the division by the norm (plus eps) follows in 32 bits behind the products
// (Scale::unit). A 16-bit input enters without any rounding, a 32-bit one as a pair of fp16
// numbers where x0_lo is given (22 bits) and rounded once otherwise.
__global__ void __launch_bounds__(kEltThreads)
    k_scale(const Item* table, int count, float mu, int nesterov, double eps) {
  chain_next();
  chain_wait();
  const Item& it = find_item(table, count, blockIdx.x);
  const int chunk = blockIdx.x - it.chunk0;
  double mine = 0;
  for (int i = threadIdx.x; i < it.chunks; i += kEltThreads) mine += it.partial[i];
  const double norm = sqrt(block_sum(mine));
  float pow2 = 1.f, unit = 0.f;
  if (!(norm <= 1.7e308)) {
    unit = __int_as_float(0x7fc00000);
  } else if (norm > 0) {
    pow2 = ldexpf(1.f, max(-126, min(120, 13 - ilogb(norm))));
    unit = (float)(1.0 / ((norm + eps) * (double)pow2));
  }
  if (chunk == 0 && threadIdx.x == 0) *it.scale = Scale{unit};
  const int64_t e0 = chunk * it.chunk_elems, e1 = min(it.n, e0 + it.chunk_elems);
  const bool mom = it.mom != nullptr;
  // element i's place in the scaled matrix, whose lines are padded to ld
  auto place = [&](int64_t i) {
    if (it.cols == it.ld) return i;
    const int64_t r = it.n <= 0x7fffffff ? (int64_t)((uint32_t)i / (uint32_t)it.cols)
                                         : i / it.cols;
    return r * it.ld + (i - r * it.cols);
  };
  if (item_vec(it) && it.cols % 8 == 0) {
    for (int64_t i0 = e0 + threadIdx.x * 8; i0 < e1; i0 += kEltThreads * 8 * kUnroll) {
      F8 g[kUnroll], m[kUnroll];
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int64_t i = i0 + q * kEltThreads * 8;
        if (i >= e1) continue;
        g[q] = load8(it.g, i, it.g_dt);
        if (mom) m[q] = load8(it.mom, i, it.mom_dt);
      }
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int64_t i = i0 + q * kEltThreads * 8;
        if (i >= e1) continue;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (mom) g[q].v[k] = direction(g[q].v[k], m[q].v[k], mu, nesterov);
          g[q].v[k] *= pow2;
        }
        const int64_t at = place(i);
        store8(it.x0, at, DT_F16, g[q]);
        if (it.x0_lo) {
#pragma unroll
          for (int k = 0; k < 8; ++k) g[q].v[k] -= __half2float(__float2half_rn(g[q].v[k]));
          store8(it.x0_lo, at, DT_F16, g[q]);
        }
      }
    }
  } else {
    for (int64_t i0 = e0 + threadIdx.x; i0 < e1; i0 += kEltThreads * kUnroll) {
      float u[kUnroll], m[kUnroll];
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int64_t i = i0 + q * kEltThreads;
        u[q] = i < e1 ? load_as_float(it.g, i, it.g_dt) : 0.f;
        m[q] = mom && i < e1 ? load_as_float(it.mom, i, it.mom_dt) : 0.f;
      }
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int64_t i = i0 + q * kEltThreads;
        if (i >= e1) continue;
        if (mom) u[q] = direction(u[q], m[q], mu, nesterov);
        u[q] *= pow2;
        const int64_t at = place(i);
        const __half hi = __float2half_rn(u[q]);
        it.x0[at] = hi;
        if (it.x0_lo) it.x0_lo[at] = __float2half_rn(u[q] - __half2float(hi));
      }
    }
  }
}

// 8 elements of 16 bits that need not be aligned, zeros from the n-th on.
__device__ __forceinline__ uint4 gather8(const uint16_t* q, int n) {
  uint16_t v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = k < n ? q[k] : (uint16_t)0;
  return make_uint4(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16,
                    v[4] | (uint32_t)v[5] << 16, v[6] | (uint32_t)v[7] << 16);
}

// ---- operand copies --------------------------------------------------------------
// rows x cols 16-bit elements into rows of ld (cols rounded up to 8) elements, as TMA reads rows
// that start on 16 bytes; up to two matrices, one for each z of the grid. A thread gathers 8
// elements, all their loads under way together, for one 16-byte store.
struct CopyJob {
  const uint16_t* src;
  int64_t stride;
  uint16_t* dst;
  int32_t rows, cols, ld;
};
struct CopyArgs {
  CopyJob job[2];
};
__global__ void __launch_bounds__(kEltThreads) k_copy_rows(const __grid_constant__ CopyArgs a) {
  chain_next();
  chain_wait();
  const CopyJob& j = a.job[blockIdx.z];
  const int per = j.ld / 8, cols = j.cols;
  const int64_t pieces = (int64_t)j.rows * per, step = (int64_t)gridDim.x * kEltThreads;
  for (int64_t e = (int64_t)blockIdx.x * kEltThreads + threadIdx.x; e < pieces; e += step) {
    const int64_t r = pieces <= 0x7fffffff ? (int64_t)((uint32_t)e / (uint32_t)per) : e / per;
    const int c = (int)(e - r * per) * 8;
    *reinterpret_cast<uint4*>(j.dst + r * j.ld + c) =
        gather8(j.src + r * j.stride + c, cols - c);
  }
}

// ---- gradient of the activation, and of the bias -----------------------------------
// dz = dy act'(z), rounded to the operand type for the two products that read it; the bias
// gradient sums the unrounded dz. A thread takes 8 columns of the y-th range of rows, a block
// neighbouring threads' columns, so that its reads run along the rows (blocks of 8 rows by 256
// columns took 212 us at 8192 x 14336). What it loads stays packed until it is used: 4 rows under
// way fit the registers of enough blocks. The column sums go to part[y], which k_bias_grad adds in
// order.
constexpr int kDzRows = 4;  // rows whose loads are under way together
template <int DT>
__global__ void __launch_bounds__(kEltThreads)
    k_dz(const uint16_t* dy, int64_t dy_stride, const int16_t* deriv, int ld_deriv, int rows,
         int cols, uint16_t* dz, int ld_dz, float* part) {
  chain_next();
  chain_wait();
  const int c0 = (blockIdx.x * blockDim.x + threadIdx.x) * 8;
  if (c0 >= cols) return;
  const int r0 = (int)((int64_t)rows * blockIdx.y / gridDim.y);
  const int r1 = (int)((int64_t)rows * (blockIdx.y + 1) / gridDim.y);
  const bool vec = c0 + 8 <= cols && dy_stride % 8 == 0 && ((uintptr_t)dy & 15) == 0;
  float sum[8] = {};
  for (int r = r0; r < r1; r += kDzRows) {
    uint4 g[kDzRows], code[kDzRows];
#pragma unroll
    for (int q = 0; q < kDzRows; ++q) {
      const int row = min(r + q, r1 - 1);
      const uint16_t* at = dy + (int64_t)row * dy_stride + c0;
      g[q] = vec ? *reinterpret_cast<const uint4*>(at) : gather8(at, cols - c0);
      if (deriv)  // rows of ld_deriv (a multiple of 8) codes
        code[q] = *reinterpret_cast<const uint4*>(deriv + (int64_t)row * ld_deriv + c0);
    }
#pragma unroll
    for (int q = 0; q < kDzRows; ++q) {
      if (r + q >= r1) break;
      const uint32_t w[4] = {g[q].x, g[q].y, g[q].z, g[q].w};
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack16(w[k], DT);
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
      }
      if (deriv) {
        const uint32_t d[4] = {code[q].x, code[q].y, code[q].z, code[q].w};
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= decode_deriv<DT>(d[k >> 1] >> (16 * (k & 1)) & 0xffffu);
      }
      if (dz)  // rows of ld_dz (a multiple of 8); nothing reads the columns from cols on
        *reinterpret_cast<uint4*>(dz + (int64_t)(r + q) * ld_dz + c0) =
            make_uint4(pack16(v[0], v[1], DT), pack16(v[2], v[3], DT), pack16(v[4], v[5], DT),
                       pack16(v[6], v[7], DT));
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] += v[k];
    }
  }
  if (part) {
    float* p = part + (int64_t)blockIdx.y * cols + c0;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c0 + k < cols) p[k] = sum[k];
  }
}
// 32 columns a block, its 8 warps a share of the parts each.
__global__ void __launch_bounds__(kEltThreads)
    k_bias_grad(const float* part, int parts, int cols, void* db, int dt) {
  chain_next();
  chain_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  __shared__ float s[8][32];
  float t = 0;
  if (c < cols) {
    const int p1 = parts * (warp + 1) / 8;
#pragma unroll 8
    for (int i = parts * warp / 8; i < p1; ++i) t += part[(int64_t)i * cols + c];
  }
  s[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && c < cols) {
    t = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += s[i][lane];
    store_from_float(db, c, dt, t);
  }
}

}  // namespace mx
}  // namespace ta
