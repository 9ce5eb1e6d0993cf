// Parameters of the tensor-core product kernel (ffn_tc.cuh) and its launchers, one translation
// unit per element type.
#pragma once
#include "ffn.h"

namespace j1rt {

struct FfnTc {
  CUtensorMap ma[4], mb[2];
  CUtensorMap mo, mp[2];    // out and pre in boxes of 32 x 32, where tma_out
  FfnMat out[2], pre[2], residual;
  const float* bias[2];
  int M, N;                 // output rows, columns
  int segs, kb_seg, kb;     // segments, 64-blocks per segment, 64-blocks in all
  int b_and;                // segment s multiplies ma[s] with mb[s & b_and]
  int act;
  int row1, rows0;          // see FfnGemm
  int m_tiles, n_tiles, tiles, group;
  int workers;              // CTAs (CG 1) or CTA pairs (CG 2) that walk the tiles; cluster splits: tiles
  int split_log2;           // log2 of:
  int split;                // CTAs of a cluster that share a tile's contraction (CG 1), else 1
  int stream_k;             // each worker takes an equal share of all tiles' blocks; FP32 pieces to partials
  int sk_q, sk_r;           // stream-K: workers per group of tiles, tiles per group
  float* partials;
  const float* scale;       // see FfnGemm
  int stages;
  int boxes;                // 32 x 32 boxes per epilogue warp
  uint32_t ring;            // shared memory of the stages
  int tma_out;              // pairs, forward: boxes are stored by TMA
  int vec_out, vec_pre, vec_res;  // rows of whole 16-byte units: 16-byte accesses
  int a_rows;               // rows of one A box (K-major A): fewer than 128 when M is smaller
  int early, late;          // see FfnGemm
  int* err;
};

// Configurations: CG (CTAs per tile pair) x BN (accumulator columns of a tile).
enum FfnCfg : int { FFN_CG2_256 = 0, FFN_CG2_192, FFN_CG1_128, FFN_CG1_64 };
int launch_ffn_tc_bf16(int cfg, int layout, int gated, FfnTc& p, cudaStream_t stream);
int launch_ffn_tc_fp16(int cfg, int layout, int gated, FfnTc& p, cudaStream_t stream);

}  // namespace j1rt
