// Row kernels of the feed-forward backward pass: the gradients at the pre-activations with
// their column sums (the bias gradients).
//
//   linear: dp = dout act'(p)                        gated: da = dout g act'(a), dg = dout act(a)
//
// Bound by memory: 2 bytes per element and operand. A block owns 256 columns and a slab of
// rows; 32 threads cover the columns, 8 rows are in flight per block, each thread keeps its
// columns' sums in registers over the slab. Slab sums go to the workspace in FP32 and a second
// kernel adds them in slab order, so a sum's bits do not depend on which block ran first.
#include <cuda_runtime.h>

#include "ffn.h"
#include "ffn_math.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace j1rt {

namespace {

constexpr int GC = 256;  // columns per block
constexpr int GR = 8;    // rows in flight per block

// Loads / stores of this thread's 8 columns of one row. VEC: 8 neighbouring columns, 16 bytes;
// else columns lane, lane + 32, ... (coalesced 2-byte accesses, any alignment).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const FfnMat& m, long long row, int c0, int lane, int N, float (&v)[8]) {
  if constexpr (VEC) {
    const int c = c0 + lane * 8;
    const uint4 u = c < N ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(m.p) + row * m.ld + c)
                          : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<T>::unpack(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + i * 32 + lane;
      v[i] = c < N ? Elem<T>::load(m.p, row * m.ld + c) : 0.f;
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(const FfnMat& m, long long row, int c0, int lane, int N, const float (&v)[8]) {
  void* p = const_cast<void*>(m.p);
  if constexpr (VEC) {
    const int c = c0 + lane * 8;
    if (c < N) {
      uint4 u;
      u.x = Elem<T>::pack(v[0], v[1]);
      u.y = Elem<T>::pack(v[2], v[3]);
      u.z = Elem<T>::pack(v[4], v[5]);
      u.w = Elem<T>::pack(v[6], v[7]);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + row * m.ld + c) = u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + i * 32 + lane;
      if (c < N) Elem<T>::store(p, row * m.ld + c, v[i]);
    }
  }
}

template <typename T, bool GATED, int ACT, bool VEC>
__global__ void __launch_bounds__(GC) grad_kernel(const FfnGrad g, int slab_rows) {
  __shared__ float red[GR][GC];
  grid_dep_launch();
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c0 = blockIdx.x * GC;
  const long long r0 = static_cast<long long>(blockIdx.y) * slab_rows;
  const long long r1 = min(r0 + slab_rows, static_cast<long long>(g.M));
  float s0[8] = {}, s1[8] = {};
  grid_dep_wait();
  // RI rows of a thread at once, all loads before the arithmetic
  constexpr int RI = 2;
  for (long long r = r0 + ty; r < r1; r += GR * RI) {
    float d[RI][8], p[RI][8], q[RI][8];
#pragma unroll
    for (int j = 0; j < RI; ++j) {
      const long long row = r + j * GR;
      const int n = row < r1 ? g.N : 0;  // no columns of a row behind the slab
      load8<T, VEC>(g.dout, row, c0, lane, n, d[j]);
      if constexpr (GATED || ACT != J1_ACT_NONE) load8<T, VEC>(g.p0, row, c0, lane, n, p[j]);
      if constexpr (GATED) load8<T, VEC>(g.p1, row, c0, lane, n, q[j]);
    }
#pragma unroll
    for (int j = 0; j < RI; ++j) {
      const long long row = r + j * GR;
      const int n = row < r1 ? g.N : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float slope = 1.f, value = 0.f;
        if constexpr (GATED || ACT != J1_ACT_NONE) act_slope<ACT>(p[j][i], slope, value);
        if constexpr (GATED) {
          const float a = d[j][i] * q[j][i] * slope;
          q[j][i] = d[j][i] * value;
          d[j][i] = a;
          s1[i] += q[j][i];
        } else {
          d[j][i] = d[j][i] * slope;
        }
        s0[i] += d[j][i];
      }
      if (g.d0.p) store8<T, VEC>(g.d0, row, c0, lane, n, d[j]);
      if constexpr (GATED) {
        if (g.d1.p) store8<T, VEC>(g.d1, row, c0, lane, n, q[j]);
      }
    }
  }
  if (!g.partials) return;
#pragma unroll
  for (int h = 0; h < (GATED ? 2 : 1); ++h) {
    if (h) __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) red[ty][VEC ? lane * 8 + i : i * 32 + lane] = h ? s1[i] : s0[i];
    __syncthreads();
    const int c = c0 + static_cast<int>(threadIdx.x);
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < GR; ++k) t += red[k][threadIdx.x];
    if (c < g.N) g.partials[(static_cast<size_t>(h) * gridDim.y + blockIdx.y) * g.N + c] = t;
  }
}

// sum[c] = partials[0][c] + partials[1][c] + ... : 32 columns per block, 32 slab strides at once with
// four loads in flight each (one stride of eight and a load at a time took 10 us for 395 slabs),
// joined in a fixed order.
__global__ void __launch_bounds__(1024) slab_sum_kernel(const float* partials, int slabs, int N, float* sum0, float* sum1) {
  __shared__ float red[32][33];
  grid_dep_launch();
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float* sum = blockIdx.y ? sum1 : sum0;
  const float* p = partials + static_cast<size_t>(blockIdx.y) * slabs * N;
  float t = 0.f;
  grid_dep_wait();
  if (c < N)
    for (int s = ty; s < slabs; s += 128) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = s + 32 * i < slabs ? p[static_cast<size_t>(s + 32 * i) * N + c] : 0.f;
      t += (v[0] + v[1]) + (v[2] + v[3]);
    }
  red[ty][lane] = t;
  __syncthreads();
  t = red[lane][ty];  // warp ty: the 32 strides of column ty
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (lane == 0 && blockIdx.x * 32 + ty < N && sum) sum[blockIdx.x * 32 + ty] = t;
}

bool vec_ok(const FfnMat& m) { return !m.p || ffn_rows16(m); }

// Copies matrices to rows on 16-byte boundaries. A warp takes 256 columns of a row: it reads 2-byte
// elements (neighbouring lanes on neighbouring elements, any alignment), lane l keeps elements l,
// l + 32, ..., and writes pairs as words after an exchange with its neighbour, half as many stores.
// Four rows of a warp are in flight. Block (8 warps): 32 rows.
__global__ void __launch_bounds__(256) copies_kernel(const FfnCopies c) {
  grid_dep_launch();
  const FfnCopy m = c.m[blockIdx.z];
  const int lane = threadIdx.x & 31, c0 = blockIdx.x * 256;
  const long long rows = m.rows;
  grid_dep_wait();
  if (c0 >= m.cols) return;
  for (long long r = static_cast<long long>(blockIdx.y) * 32 + (threadIdx.x >> 5) * 4; r < rows; r += gridDim.y * 32ll) {
    uint32_t v[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint16_t* src = static_cast<const uint16_t*>(m.src.p) + (r + j) * m.src.ld + c0 + lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = r + j < rows && c0 + i * 32 + lane < m.cols ? src[i * 32] : 0u;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // dst.ld is a multiple of 8: the words of a row up to its stride are ours, elements behind cols stay 0
      uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(const_cast<void*>(m.dst.p)) + (r + j) * m.dst.ld + c0);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        // even lanes: word lane / 2 of columns [32 i, +32), odd lanes: of [32 (i + 1), +32)
        const uint32_t keep = lane & 1 ? v[j][i + 1] : v[j][i], give = lane & 1 ? v[j][i] : v[j][i + 1];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, give, 1);
        const uint32_t word = lane & 1 ? got | (keep << 16) : keep | (got << 16);
        const int col = (i + (lane & 1)) * 32 + (lane & ~1);
        if (r + j < rows && c0 + col < m.dst.ld) dst[col / 2] = word;
      }
    }
  }
}

template <typename T, bool GATED, int ACT>
cudaError_t launch_grad(const FfnGrad& g, bool vec, dim3 grid, int slab_rows, cudaStream_t st) {
  return vec ? launch_kernel(grad_kernel<T, GATED, ACT, true>, grid, dim3(GC), 0, st, g, slab_rows)
             : launch_kernel(grad_kernel<T, GATED, ACT, false>, grid, dim3(GC), 0, st, g, slab_rows);
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

int launch_ffn_copies(const FfnCopies& c, cudaStream_t st) {
  long long rows = 1, cols = 1;
  for (int i = 0; i < c.n; ++i) {
    rows = rows > c.m[i].rows ? rows : c.m[i].rows;
    cols = cols > c.m[i].cols ? cols : c.m[i].cols;
  }
  const long long by = (rows + 31) / 32, bx = (cols + 255) / 256;
  const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>(by < 32768 ? by : 32768), c.n);
  return static_cast<int>(launch_kernel(copies_kernel, grid, dim3(256), 0, st, c));
}

// About eight blocks per SM over both dimensions, at least 32 rows each, at most 512 slabs.
int ffn_grad_slabs(int M, int N) {
  const long long cols = (static_cast<long long>(N) + GC - 1) / GC;
  long long slabs = (1184 + cols - 1) / cols;
  const long long most = (static_cast<long long>(M) + 31) / 32;
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
  if (e != cudaSuccess || !k.partials) return static_cast<int>(e);
  return static_cast<int>(launch_kernel(slab_sum_kernel, dim3((g.N + 31) / 32, g.gated ? 2 : 1), dim3(1024), 0, st,
                                        static_cast<const float*>(k.partials), slabs, g.N, g.sum0, g.sum1));
}

}  // namespace j1rt
