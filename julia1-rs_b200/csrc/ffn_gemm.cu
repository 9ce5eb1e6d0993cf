// Matrix products of the feed-forward operators with their epilogues.
//
// out[M, N] = act(A . B + bias) (+ residual), or act(A B0^T + bias0) * (A B1^T + bias1), any
// operand order and stride. This is the plain form: 64 x 64 tiles, 16 deep, FP32 arithmetic on
// the CUDA cores, 4 x 4 results per thread.
#include <cuda_runtime.h>

#include "ffn.h"
#include "ffn_math.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace j1rt {

namespace {

constexpr int TM = 64, TN = 64, TK = 16;

__device__ __forceinline__ float act_any(int act, float p) {
  switch (act) {
    case J1_ACT_RELU: return act_value<J1_ACT_RELU>(p);
    case J1_ACT_GELU: return act_value<J1_ACT_GELU>(p);
    case J1_ACT_GELU_TANH: return act_value<J1_ACT_GELU_TANH>(p);
    case J1_ACT_SILU: return act_value<J1_ACT_SILU>(p);
  }
  return p;
}

template <typename T>
__global__ void __launch_bounds__(256) simple_kernel(const FfnGemm g) {
  __shared__ float sa[TK][TM + 1], sb[2][TK][TN + 1];
  const long long m0 = static_cast<long long>(blockIdx.y) * TM;
  const int n0 = blockIdx.x * TN;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int nb = g.gated ? 2 : 1;
  float acc[2][4][4] = {};
  grid_dep_launch();
  grid_dep_wait();
  for (int s = 0; s < g.segs; ++s)
    for (int k0 = 0; k0 < g.K; k0 += TK) {
      for (int i = threadIdx.x; i < TM * TK; i += 256) {
        // neighbouring threads along the contiguous dimension
        const int m = g.layout == FFN_TN ? i % TM : i / TK, k = g.layout == FFN_TN ? i / TM : i % TK;
        const long long r = m0 + m;
        const long long kk = k0 + k;
        sa[k][m] = r < g.M && kk < g.K
                       ? Elem<T>::load(g.a[s].p, g.layout == FFN_TN ? kk * g.a[s].ld + r : r * g.a[s].ld + kk)
                       : 0.f;
        const int n = g.layout == FFN_NT ? i / TK : i % TN, kb = g.layout == FFN_NT ? i % TK : i / TN;
        const long long c = n0 + n, kkb = k0 + kb;
        for (int h = 0; h < nb; ++h) {
          const FfnMat& b = g.b[g.gated ? h : s];
          sb[h][kb][n] = c < g.N && kkb < g.K ? Elem<T>::load(b.p, g.layout == FFN_NT ? c * b.ld + kkb : kkb * b.ld + c)
                                              : 0.f;
        }
      }
      __syncthreads();
      for (int k = 0; k < TK; ++k)
        for (int h = 0; h < nb; ++h)
          for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) acc[h][i][j] = fmaf(sa[k][ty * 4 + i], sb[h][k][tx + 16 * j], acc[h][i][j]);
      __syncthreads();
    }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      long long r = m0 + ty * 4 + i;
      const int c = n0 + tx + 16 * j;
      if (r >= g.M || c >= g.N) continue;
      float p = acc[0][i][j];
      if (g.bias[0]) p += g.bias[0][c];
      if (g.pre[0].p) Elem<T>::store(const_cast<void*>(g.pre[0].p), r * g.pre[0].ld + c, p);
      float v = act_any(g.act, p);
      if (g.gated) {
        float q = acc[1][i][j];
        if (g.bias[1]) q += g.bias[1][c];
        if (g.pre[1].p) Elem<T>::store(const_cast<void*>(g.pre[1].p), r * g.pre[1].ld + c, q);
        v *= q;
      }
      if (g.residual.p) v += Elem<T>::load(g.residual.p, r * g.residual.ld + c);
      int o = 0;
      if (r >= g.row1) {
        o = 1;
        r -= g.row1;
      } else if (r >= g.rows0) {
        continue;
      }
      Elem<T>::store(const_cast<void*>(g.out[o].p), r * g.out[o].ld + c, v);
    }
}

__device__ int g_ffn_error;

}  // namespace

cudaError_t ffn_error_word(int** p) {
  void* v = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&v, g_ffn_error);
  *p = static_cast<int*>(v);
  return e;
}

size_t ffn_partial_bytes(int, int, int) { return 0; }

int launch_ffn_gemm(const FfnGemm& g, cudaStream_t st) {
  const dim3 grid((g.N + TN - 1) / TN, (g.M + TM - 1) / TM);
  return static_cast<int>(g.fp16 ? launch_kernel(simple_kernel<__half>, grid, dim3(256), 0, st, g)
                                 : launch_kernel(simple_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, g));
}

}  // namespace j1rt
