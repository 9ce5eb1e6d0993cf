// Row kernels of the feed-forward backward pass: the gradients at the pre-activations with
// their column sums (the bias gradients).
//
//   linear: dp = dout act'(p)                        gated: da = dout g act'(a), dg = dout act(a)
//
// Bound by memory: 2 bytes per element of every operand and of both parts of every gradient. A block
// owns 256 columns and a slab of rows; 32 threads cover the columns, 8 rows are worked on at once, each
// thread keeps its columns' sums in registers over the slab. 65536 x 1152 gated GELU: 193 us, 5.5 TB/s (0.83
// of the measured copy rate: the slopes and the cutting into parts take issue slots). Slab sums go to the
// workspace in FP32 and a second kernel adds them in slab order, so a sum's bits do not depend on which
// block ran first.
#include <cuda_runtime.h>

#include <type_traits>

#include "ffn.h"
#include "ffn_math.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace j1rt {

namespace {

constexpr int GC = 256;  // columns per block
constexpr int GR = 8;    // rows in flight per block

// This thread's 8 columns of one row as they are in memory. VEC: 8 neighbouring columns, 16 bytes;
// else columns lane, lane + 32, ... (coalesced 2-byte accesses, any alignment). n: the row's columns,
// 0 for a row that is not there.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const FfnMat& m, long long row, int c0, int lane, int n) {
  if constexpr (VEC) {
    const int c = c0 + lane * 8;
    return c < n ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(m.p) + row * m.ld + c)
                 : make_uint4(0u, 0u, 0u, 0u);
  } else {
    uint32_t w[4];
    const uint16_t* at = static_cast<const uint16_t*>(m.p) + row * m.ld + c0 + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (c0 + 64 * i + lane < n ? at[64 * i] : 0u) | ((c0 + 64 * i + 32 + lane < n ? at[64 * i + 32] : 0u) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <typename T>
__device__ __forceinline__ void pairs(const uint4& u, uint64_t (&v)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<T>::unpack(w[i]);
    v[i] = f2pack(f.x, f.y);
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(const FfnMat& m, long long row, int c0, int lane, int n, const uint32_t (&w)[4]) {
  uint16_t* at = static_cast<uint16_t*>(const_cast<void*>(m.p)) + row * m.ld + c0;
  if constexpr (VEC) {
    if (c0 + lane * 8 < n) *reinterpret_cast<uint4*>(at + lane * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + 32 * i + lane < n) at[32 * i + lane] = static_cast<uint16_t>(w[i >> 1] >> ((i & 1) * 16));
  }
}

// The values rounded to T, or in two parts: cut to T's bits, and what is left, rounded. Both parts have the
// value's sign and neither is 0 unless the value is (the second is 2^-24 of it at least, and T's smallest step):
// an infinite factor then gives the infinity that the value itself would, not inf - inf or 0 inf.
template <typename T>
__device__ __forceinline__ void rounded(const uint64_t (&v)[4], uint32_t (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    f2unpack(v[i], lo, hi);
    w[i] = Elem<T>::pack(lo, hi);
  }
}
template <typename T>
__device__ __forceinline__ float2 two_parts(float v) {
  const float m = fabsf(v), first = Elem<T>::cut(m != 0.f ? max_nan(m, Elem<T>::kStep) : m);
  const float left = max_nan(fmaxf(m - first, m * 0x1p-24f), Elem<T>::kStep);
  return make_float2(copysignf(first, v), copysignf(m != 0.f ? left : 0.f, v));
}
template <typename T>
__device__ __forceinline__ void two_parts(const uint64_t (&v)[4], uint32_t (&w)[4], uint32_t (&rest)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    f2unpack(v[i], lo, hi);
    const float2 a = two_parts<T>(lo), b = two_parts<T>(hi);
    w[i] = Elem<T>::pack(a.x, b.x);
    rest[i] = Elem<T>::pack(a.y, b.y);
  }
}

// da and dg (or dp) of a pair of columns, in place of dout and pre_g.
template <bool GATED, int ACT>
__device__ __forceinline__ void gradients(uint64_t& d, uint64_t p, uint64_t& q) {
  uint64_t slope = 0ull, value = 0ull;
  if constexpr (GATED || ACT != J1_ACT_NONE) act_slope<ACT>(p, slope, value);
  if constexpr (GATED) {
    const uint64_t a = mul2(mul2(d, q), slope);
    q = mul2(d, value);
    d = a;
  } else if constexpr (ACT != J1_ACT_NONE) {
    d = mul2(d, slope);
  }
}

// The largest finite magnitude of the gradients at the pre-activations, per block. FP16 has 2^-24 to 2^16, where
// dout, the activation's slope and the gate may each be small or large without the products' results being so: the
// gradients are scaled by a power of two of the call before they are rounded. It takes a pass of its own over their
// operands. Tiles of 16 rows x 256 columns, two rows per thread in flight: 65536 x 1152 gated GELU 107 us (4.2 TB/s,
// the slopes' arithmetic between the loads), 2048 x 768 linear 4.5 us; with tiles of 64 rows, four in flight, too few blocks
// had work at small sizes (the call on 2048 rows 12 us longer).
template <bool GATED, int ACT, bool VEC>
__global__ void __launch_bounds__(GC, 4) max_kernel(const FfnGrad g, int col_blocks) {
  __shared__ float red[GR];
  grid_dep_launch();
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float most = 0.f;
  grid_dep_wait();
  const int grid = gridDim.x, cols = grid % col_blocks, rows = grid / col_blocks;
  int cb = blockIdx.x % col_blocks;
#pragma unroll 1
  for (long long r0 = blockIdx.x / col_blocks * (2 * GR) + ty; r0 - ty < g.M; r0 += static_cast<long long>(rows) * (2 * GR)) {
    const int c0 = cb * GC;
    uint4 d[2], p[2], q[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long row = r0 + j * GR;
      const int n = row < g.M ? g.N : 0;
      d[j] = load8<VEC>(g.dout, row, c0, lane, n);
      p[j] = load8<VEC>(g.p0, row, c0, lane, n);
      if constexpr (GATED) q[j] = load8<VEC>(g.p1, row, c0, lane, n);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint64_t x[4], y[4], z[4];
      pairs<__half>(d[j], x);
      pairs<__half>(p[j], y);
      if constexpr (GATED) pairs<__half>(q[j], z);
      auto look = [&](uint64_t v) {
        float a, b;
        f2unpack(v, a, b);
        a = fabsf(a), b = fabsf(b);
        most = fmaxf(most, fmaxf(a <= 3e38f ? a : 0.f, b <= 3e38f ? b : 0.f));
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        gradients<GATED, ACT>(x[i], y[i], z[i]);
        look(x[i]);
        if constexpr (GATED) look(z[i]);
      }
    }
    cb += cols;
    if (cb >= col_blocks) cb -= col_blocks, r0 += 2 * GR;
  }
  most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
  if (lane == 0) red[ty] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < GR; ++i) most = fmaxf(most, red[i]);
    g.scale[1 + blockIdx.x] = most;
  }
}

// Gradients that are scaled before they are stored.
template <typename T, bool GATED, int ACT>
constexpr bool kScaled = std::is_same<T, __half>::value && ffn_two_parts(GATED, ACT);

template <typename T, bool GATED, int ACT, bool VEC>
__global__ void __launch_bounds__(GC, 3) grad_kernel(const FfnGrad g, int slab_rows, int maxima) {
  __shared__ float red[GR][GC];
  grid_dep_launch();
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c0 = blockIdx.x * GC;
  const long long r0 = static_cast<long long>(blockIdx.y) * slab_rows;
  const long long r1 = min(r0 + slab_rows, static_cast<long long>(g.M));
  uint64_t s0[4] = {}, s1[4] = {};
  grid_dep_wait();
  // VEC: the next DEPTH rows' pieces are on their way to shared memory while a row is worked on, each
  // thread reading back what it asked for itself (65536 x 1152 gated GELU, gradients in one part: 116 us; with the
  // next row in registers 141, with nothing asked for ahead 227). Otherwise the next RI rows' are in registers.
  constexpr int OPS = GATED ? 3 : ACT != J1_ACT_NONE ? 2 : 1, DEPTH = GATED ? 3 : ACT != J1_ACT_NONE ? 4 : 8;
  constexpr int RI = GATED || VEC ? 1 : 2;
  constexpr bool SCALED = kScaled<T, GATED, ACT>;
  __shared__ uint4 ring[VEC ? DEPTH * OPS * GC : 1];
  const uint32_t own = smem_u32(ring) + threadIdx.x * 16;
  uint32_t slot = 0;
  auto ask = [&](long long r) {
    const int c = c0 + lane * 8;
    const uint32_t bytes = r < r1 && c < g.N ? 16u : 0u;
    const long long row = bytes ? r : 0, col = bytes ? c : 0;  // nothing is read for 0 bytes
    auto one = [&](int op, const FfnMat& m) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(own + (slot * OPS + op) * (GC * 16)),
                   "l"(static_cast<const uint16_t*>(m.p) + row * m.ld + col), "r"(bytes)
                   : "memory");
    };
    one(0, g.dout);
    if constexpr (OPS > 1) one(1, g.p0);
    if constexpr (OPS > 2) one(2, g.p1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    slot = slot + 1 == DEPTH ? 0u : slot + 1;
  };
  uint4 d[RI], p[RI], q[RI];
  auto fetch = [&](long long r) {
    if constexpr (VEC) {
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
      const uint4* at = ring + slot * OPS * GC + threadIdx.x;
      d[0] = at[0];
      if constexpr (OPS > 1) p[0] = at[GC];
      if constexpr (OPS > 2) q[0] = at[2 * GC];
      return;
    }
#pragma unroll
    for (int j = 0; j < RI; ++j) {
      const long long row = r + j * GR;
      const int n = row < r1 ? g.N : 0;
      d[j] = load8<VEC>(g.dout, row, c0, lane, n);
      if constexpr (GATED || ACT != J1_ACT_NONE) p[j] = load8<VEC>(g.p0, row, c0, lane, n);
      if constexpr (GATED) q[j] = load8<VEC>(g.p1, row, c0, lane, n);
    }
  };
  if constexpr (VEC) {
    for (int i = 0; i < DEPTH; ++i) ask(r0 + ty + i * GR);
  } else {
    fetch(r0 + ty);
  }
  uint64_t scale = f2pack(1.f, 1.f);
  if constexpr (SCALED) {
    if (g.scale) {
      uint32_t most = 0;
      for (int i = threadIdx.x; i < maxima; i += GC) most = max(most, __float_as_uint(__ldcg(g.scale + 1 + i)));
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) red[0][ty] = __uint_as_float(most);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < GR; ++i) most = max(most, __float_as_uint(red[0][i]));
      __syncthreads();  // red is written again below
      const int e = most ? max(-100, min(100, 127 + 14 - static_cast<int>(most >> 23))) : 0;
      const float f = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      scale = f2pack(f, f);
      if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0)
        g.scale[0] = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    }
  }
  for (long long r = r0 + ty; r < r1; r += GR * RI) {
    if constexpr (VEC) fetch(r);
    uint4 d0[RI], p0[RI], q0[RI];
#pragma unroll
    for (int j = 0; j < RI; ++j) d0[j] = d[j], p0[j] = p[j], q0[j] = q[j];
    if constexpr (!VEC) fetch(r + GR * RI);
#pragma unroll
    for (int j = 0; j < RI; ++j) {
      const long long row = r + j * GR;
      const int n = row < r1 ? g.N : 0;
      uint64_t x[4], y[4], z[4];
      pairs<T>(d0[j], x);
      if constexpr (GATED || ACT != J1_ACT_NONE) pairs<T>(p0[j], y);
      if constexpr (GATED) pairs<T>(q0[j], z);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        gradients<GATED, ACT>(x[i], y[i], z[i]);
        if constexpr (GATED) s1[i] = add2(s1[i], z[i]);
        s0[i] = add2(s0[i], x[i]);
        if constexpr (SCALED) {
          x[i] = mul2(x[i], scale);
          if constexpr (GATED) z[i] = mul2(z[i], scale);
        }
      }
      auto store = [&](const FfnMat& m, const uint64_t(&v)[4]) {
        uint32_t w[4], left[4];
        if constexpr (ffn_two_parts(GATED, ACT)) {
          two_parts<T>(v, w, left);
          store8<VEC>({static_cast<const uint16_t*>(m.p) + g.lo, m.ld}, row, c0, lane, n, left);
        } else {
          rounded<T>(v, w);
        }
        store8<VEC>(m, row, c0, lane, n, w);
      };
      if (g.d0.p) store(g.d0, x);
      if constexpr (GATED) {
        if (g.d1.p) store(g.d1, z);
      }
    }
    if constexpr (VEC) ask(r + DEPTH * GR);
  }
  if constexpr (VEC) asm volatile("cp.async.wait_all;" ::: "memory");
  if (!g.partials) return;
#pragma unroll
  for (int h = 0; h < (GATED ? 2 : 1); ++h) {
    if (h) __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float lo, hi;
      f2unpack(h ? s1[i >> 1] : s0[i >> 1], lo, hi);
      red[ty][VEC ? lane * 8 + i : i * 32 + lane] = i & 1 ? hi : lo;
    }
    __syncthreads();
    const int c = c0 + static_cast<int>(threadIdx.x);
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < GR; ++k) t += red[k][threadIdx.x];
    if (gridDim.y == 1) {  // the only slab: its sums are the result
      float* sum = h ? g.sum1 : g.sum0;
      if (c < g.N && sum) sum[c] = t;
    } else if (c < g.N) {
      g.partials[(static_cast<size_t>(h) * gridDim.y + blockIdx.y) * g.N + c] = t;
    }
  }
}

// sum[c] = partials[0][c] + partials[1][c] + ... : 32 columns per block, 32 slab strides at once with
// four loads in flight each (one stride of eight and a load at a time took 10 us for 395 slabs),
// joined in a fixed order.
__global__ void __launch_bounds__(1024) slab_sum_kernel(const float* partials, int slabs, int N, float* sum0, float* sum1, int early) {
  __shared__ float red[32][33];
  grid_dep_launch();
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float* sum = blockIdx.y ? sum1 : sum0;
  const float* p = partials + static_cast<size_t>(blockIdx.y) * slabs * N;
  float t = 0.f;
  if (!early) grid_dep_wait();
  if (c < N)
    for (int s = ty; s < slabs; s += 128) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = s + 32 * i < slabs ? __ldcg(p + static_cast<size_t>(s + 32 * i) * N + c) : 0.f;
      t += (v[0] + v[1]) + (v[2] + v[3]);
    }
  red[ty][lane] = t;
  __syncthreads();
  t = red[lane][ty];  // warp ty: the 32 strides of column ty
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (lane == 0 && blockIdx.x * 32 + ty < N && sum) sum[blockIdx.x * 32 + ty] = t;
  if (early) grid_dep_wait();
}

bool vec_ok(const FfnMat& m) { return !m.p || ffn_rows16(m); }

// Copies matrices to rows on 16-byte boundaries. A thread makes 16-byte units, two at a time (two rows
// of its column, the next two's loads in flight): the two aligned pieces that hold a unit, shifted
// together. Units whose pieces would lie outside the matrix's memory, at its first and last bytes,
// are read element by element. 1003 x 1155 and 771 x 1155 together: 4.6 us (8 MB). Block (8 warps): 16 rows x 32 units, then on by gridDim.y times 16 rows.
__global__ void __launch_bounds__(256) copies_kernel(const FfnCopies c) {
  grid_dep_launch();
  const FfnCopy m = c.m[blockIdx.z];
  const int lane = threadIdx.x & 31, col = blockIdx.x * 256 + lane * 8;
  const char* lo = static_cast<const char*>(m.src.p);
  const char* hi = lo + ((static_cast<long long>(m.rows) - 1) * m.src.ld + m.cols) * 2;
  const long long step = static_cast<long long>(gridDim.y) * 16;
  grid_dep_wait();
  if (col >= m.cols) return;
  uint4 x[2], y[2];
  auto fetch = [&](long long r) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const char* a = lo + ((r + j) * m.src.ld + col) * 2;
      const char* piece = a - (reinterpret_cast<uintptr_t>(a) & 15u);
      x[j] = y[j] = make_uint4(0u, 0u, 0u, 0u);
      if (r + j < m.rows && piece >= lo && piece + 32 <= hi) {
        x[j] = *reinterpret_cast<const uint4*>(piece);
        y[j] = *reinterpret_cast<const uint4*>(piece + 16);
      }
    }
  };
  long long r = static_cast<long long>(blockIdx.y) * 16 + (threadIdx.x >> 5) * 2;
  fetch(r);
  for (; r < m.rows; r += step) {
    const uint4 x0[2] = {x[0], x[1]}, y0[2] = {y[0], y[1]};
    fetch(r + step);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (r + j >= m.rows) break;
      const char* a = lo + ((r + j) * m.src.ld + col) * 2;
      const uint32_t s = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a) & 15u);
      uint32_t w[8] = {x0[j].x, x0[j].y, x0[j].z, x0[j].w, y0[j].x, y0[j].y, y0[j].z, y0[j].w};
      if (a - s >= lo && a - s + 32 <= hi) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = s & 8 ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = s & 4 ? w[i + 1] : w[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (s & 2) * 8);
      } else {
        const uint16_t* e = reinterpret_cast<const uint16_t*>(a);
        for (int i = 0; i < 4; ++i)
          w[i] = (col + 2 * i < m.cols ? e[2 * i] : 0u) | ((col + 2 * i + 1 < m.cols ? e[2 * i + 1] : 0u) << 16);
      }
      // dst.ld is a multiple of 8: the unit lies inside the row's stride (what is behind cols is never read)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(const_cast<void*>(m.dst.p)) + (r + j) * m.dst.ld + col) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <typename T, bool GATED, int ACT>
cudaError_t load_act() {
  cudaFuncAttributes a;
  cudaError_t e = cudaFuncGetAttributes(&a, grad_kernel<T, GATED, ACT, true>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, grad_kernel<T, GATED, ACT, false>);
  if constexpr (kScaled<T, GATED, ACT>) {
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, max_kernel<GATED, ACT, true>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, max_kernel<GATED, ACT, false>);
  }
  return e;
}
template <typename T, bool GATED>
cudaError_t load_acts() {
  cudaError_t e = load_act<T, GATED, J1_ACT_NONE>();
  if (e == cudaSuccess) e = load_act<T, GATED, J1_ACT_RELU>();
  if (e == cudaSuccess) e = load_act<T, GATED, J1_ACT_GELU>();
  if (e == cudaSuccess) e = load_act<T, GATED, J1_ACT_GELU_TANH>();
  if (e == cudaSuccess) e = load_act<T, GATED, J1_ACT_SILU>();
  return e;
}

template <typename T, bool GATED, int ACT>
cudaError_t launch_grad(const FfnGrad& g, bool vec, dim3 grid, int slab_rows, cudaStream_t st) {
  int maxima = 0;
  if constexpr (kScaled<T, GATED, ACT>) {
    if (g.scale) {
      const long long tiles = (static_cast<long long>(g.M) + 2 * GR - 1) / (2 * GR) * grid.x;
      maxima = static_cast<int>(tiles < kFfnMaxBlocks ? tiles : kFfnMaxBlocks);
      const auto kern = vec ? max_kernel<GATED, ACT, true> : max_kernel<GATED, ACT, false>;
      const cudaError_t e = launch_kernel(kern, dim3(maxima), dim3(GC), 0, st, g, static_cast<int>(grid.x));
      if (e != cudaSuccess) return e;
    }
  }
  return vec ? launch_kernel(grad_kernel<T, GATED, ACT, true>, grid, dim3(GC), 0, st, g, slab_rows, maxima)
             : launch_kernel(grad_kernel<T, GATED, ACT, false>, grid, dim3(GC), 0, st, g, slab_rows, maxima);
}
template <typename T, bool GATED>
cudaError_t launch_grad(const FfnGrad& g, bool vec, dim3 grid, int slab_rows, cudaStream_t st) {
  switch (g.act) {
    case J1_ACT_NONE: return launch_grad<T, GATED, J1_ACT_NONE>(g, vec, grid, slab_rows, st);
    case J1_ACT_RELU: return launch_grad<T, GATED, J1_ACT_RELU>(g, vec, grid, slab_rows, st);
    case J1_ACT_GELU: return launch_grad<T, GATED, J1_ACT_GELU>(g, vec, grid, slab_rows, st);
    case J1_ACT_GELU_TANH: return launch_grad<T, GATED, J1_ACT_GELU_TANH>(g, vec, grid, slab_rows, st);
    default: return launch_grad<T, GATED, J1_ACT_SILU>(g, vec, grid, slab_rows, st);
  }
}

}  // namespace

cudaError_t load_ffn_rows() {
  cudaFuncAttributes a;
  cudaError_t e = cudaFuncGetAttributes(&a, copies_kernel);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, slab_sum_kernel);
  if (e == cudaSuccess) e = load_acts<__half, false>();
  if (e == cudaSuccess) e = load_acts<__half, true>();
  if (e == cudaSuccess) e = load_acts<__nv_bfloat16, false>();
  if (e == cudaSuccess) e = load_acts<__nv_bfloat16, true>();
  return e;
}

int launch_ffn_copies(const FfnCopies& c, cudaStream_t st) {
  long long rows = 1, cols = 1;
  for (int i = 0; i < c.n; ++i) {
    rows = rows > c.m[i].rows ? rows : c.m[i].rows;
    cols = cols > c.m[i].cols ? cols : c.m[i].cols;
  }
  // about eight blocks per SM over the longest matrix, each walking down its columns
  const long long bx = (cols + 255) / 256, by = (rows + 15) / 16, most = (1184 + bx - 1) / bx;
  const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>(by < most ? by : most), c.n);
  return static_cast<int>(launch_kernel(copies_kernel, grid, dim3(256), 0, st, c));
}

// About eight blocks per SM over both dimensions, at least 16 rows each (2048 x 768 x 1152 linear backward with
// gradients in one part 17.9 us, with 32 rows 18.9, with 8 18.6: more sums to add), at most 512 slabs; up to 64 rows in one
// slab, which saves the second kernel (2 us) for two more turns of the first (1 us).
int ffn_grad_slabs(int M, int N) {
  const long long cols = (static_cast<long long>(N) + GC - 1) / GC;
  long long slabs = (1184 + cols - 1) / cols;
  const long long most = M <= 64 ? 1 : (static_cast<long long>(M) + 15) / 16;
  if (slabs > most) slabs = most;
  if (slabs > 512) slabs = 512;
  return slabs < 1 ? 1 : static_cast<int>(slabs);
}

int launch_ffn_grad(const FfnGrad& g, cudaStream_t st) {
  const int slabs = ffn_grad_slabs(g.M, g.N);
  const int slab_rows = static_cast<int>((static_cast<long long>(g.M) + slabs - 1) / slabs);
  const dim3 grid((g.N + GC - 1) / GC, slabs);
  // 16-byte accesses need N itself to be a multiple of 8: elements behind a row are not ours
  const bool vec = g.N % 8 == 0 && vec_ok(g.dout) && vec_ok(g.p0) && vec_ok(g.p1) && vec_ok(g.d0) && vec_ok(g.d1);
  FfnGrad k = g;
  if (!g.sum0 && !g.sum1) k.partials = nullptr;
  cudaError_t e;
  if (g.fp16)
    e = g.gated ? launch_grad<__half, true>(k, vec, grid, slab_rows, st) : launch_grad<__half, false>(k, vec, grid, slab_rows, st);
  else
    e = g.gated ? launch_grad<__nv_bfloat16, true>(k, vec, grid, slab_rows, st)
                : launch_grad<__nv_bfloat16, false>(k, vec, grid, slab_rows, st);
  return static_cast<int>(e);
}

bool ffn_grad_sums(const FfnGrad& g) { return (g.sum0 || g.sum1) && ffn_grad_slabs(g.M, g.N) > 1; }

int launch_ffn_grad_sums(const FfnGrad& g, int early, cudaStream_t st) {
  return static_cast<int>(launch_kernel(slab_sum_kernel, dim3((g.N + 31) / 32, g.gated ? 2 : 1), dim3(1024), 0, st,
                                        static_cast<const float*>(g.partials), ffn_grad_slabs(g.M, g.N), g.N, g.sum0,
                                        g.sum1, early));
}

}  // namespace j1rt
