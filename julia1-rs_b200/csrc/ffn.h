// Internal launch interface of the feed-forward operators (j1_op_linear, j1_op_gated and their
// backward passes): ffn.cpp checks arguments and plans, the .cu files launch.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/j1.h"

namespace j1rt {

// A row-major matrix of 16-bit elements: row r starts at p + r * ld elements.
struct FfnMat {
  const void* p;
  long long ld;
};
// Rows on 16-byte boundaries: what TMA and 16-byte accesses need.
inline bool ffn_rows16(const FfnMat& m) { return reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.ld % 8 == 0; }

// How the operands of out[M, N] = A . B lie in memory (K: the contraction).
enum FfnLayout : int {
  FFN_NT = 0,  // A [M, K], B [N, K]: forward
  FFN_NN = 1,  // A [M, K], B [K, N]: dx = dp . w
  FFN_TN = 2,  // A [K, M], B [K, N]: dw = dp^T . x
};

struct FfnGemm {
  int fp16;    // element type: 0 BF16, 1 FP16
  int layout;  // FfnLayout
  int gated;   // two B operands, out = act(A B0^T + bias0) * (A B1^T + bias1) (NT)
  int act;     // j1_act
  int M, N, K;
  int segs;    // out = sum over s < segs of A[s] . B[s] (NN: the two halves of a gated dx)
  int row1;    // TN: output rows >= row1 (a multiple of 32) go to out[1] from its row 0, rows in
               // [rows0, row1) nowhere; INT_MAX: all to out[0]
  int rows0;
  FfnMat a[2], b[2];
  long long lo;     // not 0: A is in two parts, the second lies lo elements behind the first
  const float* scale;  // FP16: what a sum is multiplied by before it is rounded (device memory), NULL: 1
  const float* bias[2];
  FfnMat residual;  // p NULL: none
  FfnMat out[2];    // written
  FfnMat pre[2];    // written; p NULL: not wanted
  float* partials;  // workspace of split contractions, NULL: never split
  size_t partial_bytes;
  // Kernels of one call that do not need each other run at once: a `late` kernel lets the next one start
  // only when everything before itself is complete, so an `early` one launched behind it (or behind an
  // early one) finds its inputs ready without waiting; it waits at its end instead, so that what follows
  // it still follows both.
  int early, late;
  int* err;         // device error word
  int num_sms;
};

// The operands a and b must have rows on 16-byte boundaries (ffn_rows16).
int launch_ffn_gemm(const FfnGemm& g, cudaStream_t stream);
// How it would run (see j1_selftest_ffn_plan; host arithmetic only).
void ffn_plan(const FfnGemm& g, int32_t* plan);
// Workspace that a split contraction of these sizes may take (host arithmetic only).
size_t ffn_partial_bytes(int M, int N, int K);
// Load the kernels on the current device (a lazily loaded one could not be launched first in a stream capture).
cudaError_t load_ffn_rows();
cudaError_t load_ffn_tc_bf16();
cudaError_t load_ffn_tc_fp16();
// Device address of the operators' error word on the current device.
cudaError_t ffn_error_word(int** p);

// Copies of matrices to rows on 16-byte boundaries (dst.ld a multiple of 8).
struct FfnCopy {
  FfnMat src, dst;
  int rows, cols;
};
struct FfnCopies {
  FfnCopy m[4];
  int n;
};
int launch_ffn_copies(const FfnCopies& c, cudaStream_t stream);

// Whether gradients at the pre-activations are kept in two parts. A linear layer's without activation or with ReLU
// are dout or 0: one holds them.
__host__ __device__ constexpr bool ffn_two_parts(bool gated, int act) { return gated || (act != J1_ACT_NONE && act != J1_ACT_RELU); }

// dp = dout * act'(pre) (linear), or da = dout * g * act'(a), dg = dout * act(a) (gated): the
// gradients at the pre-activations, rounded to the element type, with the column sums of the
// unrounded values. d0 (and d1) may be NULL (sums only); sums may be NULL.
struct FfnGrad {
  int fp16, gated, act;
  int M, N;
  FfnMat dout, p0, p1;  // p0: pre / pre_a (NULL p: act NONE), p1: pre_g
  FfnMat d0, d1;        // written: dp / da, dg
  float* sum0;          // [N] or NULL
  float* sum1;
  long long lo;         // in two parts: the second goes lo elements behind the first
  float* partials;      // ffn_grad_slabs(M, N) * 2 * N floats when a sum is wanted
  // FP16, NULL: as they are. d0 and d1 are multiplied by a power of two of the call that brings the
  // largest of their finite magnitudes to [2^14, 2^15); scale[0] receives its inverse, the rest is scratch.
  float* scale;         // kFfnScaleFloats
};
constexpr int kFfnMaxBlocks = 888;
constexpr int kFfnScaleFloats = 1 + kFfnMaxBlocks;
int ffn_grad_slabs(int M, int N);
int launch_ffn_grad(const FfnGrad& g, cudaStream_t stream);
// Adds the slabs' sums where there are several and a sum is wanted (ffn_grad_sums); early: see FfnGemm.
bool ffn_grad_sums(const FfnGrad& g);
int launch_ffn_grad_sums(const FfnGrad& g, int early, cudaStream_t stream);

}  // namespace j1rt
