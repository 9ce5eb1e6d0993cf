// Plans the products of the feed-forward operators: tile shape, split and tensor maps of a call.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "ffn_tc.h"
#include "kernels.h"

namespace j1rt {

namespace {

__device__ int g_ffn_error;

constexpr int kPairs = 74;                        // most CTA pairs a stream-K product uses
constexpr size_t kPieceBytes = 256 * 256 * 4;     // FP32 accumulators of a pair

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

struct Plan {
  int cfg, cg, bn, split;
  bool stream_k;
  double us;
};

// Microseconds per 64-block of a tile and CTA (or pair) and the fixed part of a tile that
// nothing hides (first loads, last epilogue).
Plan choose(const FfnGemm& g, int kb) {
  const int sms = g.num_sms;
  const auto single = [&](int cfg, int bn, double step) {
    const long long tiles = ceil_div(g.M, 128) * ceil_div(g.N, g.gated ? bn / 2 : bn);
    Plan best = {cfg, 1, bn, 1, false, 0.0};
    best.us = static_cast<double>(ceil_div(tiles, sms)) * kb * step + 1.5;
    for (int s = 2; s <= 8 && s <= kb; s *= 2) {
      const double us = static_cast<double>(ceil_div(tiles * s, sms)) * (static_cast<double>(ceil_div(kb, s)) * step + 1.5) + 1.0;
      if (us < best.us) best.split = s, best.us = us;
    }
    return best;
  };
  Plan best = single(FFN_CG1_128, 128, 0.22);
  const auto take = [&](const Plan& p) {
    if (p.us < best.us) best = p;
  };
  if (!g.gated) take(single(FFN_CG1_64, 64, 0.13));
  const auto pair = [&](int cfg, int bn, double step) {
    const long long tiles = ceil_div(g.M, 256) * ceil_div(g.N, g.gated ? bn / 2 : bn);
    const int pairs = std::max(1, std::min(kPairs, sms / 2));
    Plan p = {cfg, 2, bn, 1, false, 0.0};
    p.us = static_cast<double>(ceil_div(tiles, pairs)) * kb * step + 2.5;
    if (g.layout == FFN_TN && bn == 256 && g.partials &&
        tiles * kb < INT_MAX && tiles * kb >= pairs && (tiles + pairs) * kPieceBytes <= g.partial_bytes) {  // equal shares, then a pass over the pieces
      const double us = static_cast<double>(tiles) * kb * step / pairs + 6.0 + 0.1 * static_cast<double>(tiles + pairs) / 4;
      if (us < p.us) p.stream_k = true, p.us = us;
    }
    return p;
  };
  take(pair(FFN_CG2_256, 256, 0.40));
  if (g.layout == FFN_NT && !g.gated) take(pair(FFN_CG2_192, 192, 0.31));
  return best;
}

}  // namespace

cudaError_t ffn_error_word(int** p) {
  void* v = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&v, g_ffn_error);
  *p = static_cast<int*>(v);
  return e;
}

// Pieces of a stream-K product: one per worker and tile boundary. With more tiles than four per
// pair whole tiles balance well enough, and nothing is set aside.
size_t ffn_partial_bytes(int M, int N, int K) {
  const long long tiles = ceil_div(M, 256) * ceil_div(N, 256);
  if (tiles > 4 * kPairs || K <= 64) return 0;
  return static_cast<size_t>(tiles + kPairs) * kPieceBytes;
}

int launch_ffn_gemm(const FfnGemm& g, cudaStream_t stream) {
  FfnTc p = {};
  const int nb = g.gated ? 2 : g.segs;
  for (int i = 0; i < 2; ++i) p.out[i] = g.out[i], p.pre[i] = g.pre[i], p.bias[i] = g.bias[i];
  p.M = g.M, p.N = g.N, p.K = g.K;
  p.segs = g.segs;
  p.kb_seg = static_cast<int>(ceil_div(g.K, 64));
  if (static_cast<long long>(p.kb_seg) * g.segs > INT_MAX) return static_cast<int>(cudaErrorInvalidValue);
  p.kb = p.kb_seg * g.segs;
  const Plan plan = choose(g, p.kb);
  p.act = g.act;
  p.row1 = g.row1, p.rows0 = g.rows0;
  const long long m_tiles = ceil_div(g.M, 128 * plan.cg);
  const long long n_tiles = ceil_div(g.N, g.gated ? plan.bn / 2 : plan.bn);
  if (m_tiles * n_tiles * plan.split > INT_MAX / 64) return static_cast<int>(cudaErrorInvalidValue);
  p.m_tiles = static_cast<int>(m_tiles), p.n_tiles = static_cast<int>(n_tiles);
  p.tiles = p.m_tiles * p.n_tiles;
  p.group = 8;
  p.split = plan.split;
  for (p.split_log2 = 0; (1 << p.split_log2) < plan.split;) ++p.split_log2;
  p.stream_k = plan.stream_k;
  p.partials = g.partials;
  const int slots = plan.cg == 2 ? std::max(1, std::min(kPairs, g.num_sms / 2)) : g.num_sms;
  p.workers = plan.split > 1 ? p.tiles : plan.stream_k ? slots : std::min(p.tiles, slots);
  p.share = p.tiles * static_cast<long long>(p.kb) / p.workers;
  p.share_more = static_cast<int>(p.tiles * static_cast<long long>(p.kb) % p.workers);
  p.a_rows = plan.cg == 1 && g.layout != FFN_TN && g.M < 128 ? (g.M + 7) / 8 * 8 : 128;
  p.err = g.err;
  p.residual = g.residual;
  p.vec_res = g.residual.p && ffn_rows16(g.residual) && g.N % 8 == 0;
  const int outs = g.row1 == INT_MAX ? 1 : 2;
  p.vec_out = p.vec_pre = g.N % 8 == 0;
  for (int i = 0; i < 2; ++i) {
    if (i < outs) p.vec_out = p.vec_out && ffn_rows16(g.out[i]);
    if (g.pre[i].p) p.vec_pre = p.vec_pre && ffn_rows16(g.pre[i]);
  }
  const char* why = nullptr;
  bool ok = true;
  for (int i = 0; i < g.segs; ++i)
    ok = ok && (g.layout == FFN_TN ? make_tmap_16bit(&p.ma[i], g.fp16, g.a[i].p, g.K, g.M, g.a[i].ld, 64, 64, &why)
                                   : make_tmap_16bit(&p.ma[i], g.fp16, g.a[i].p, g.M, g.K, g.a[i].ld, 64, p.a_rows, &why));
  const uint32_t b_rows = g.layout != FFN_NT ? 64 : g.gated ? plan.bn / 2 : plan.bn / plan.cg;
  for (int i = 0; i < nb; ++i)
    ok = ok && (g.layout == FFN_NT ? make_tmap_16bit(&p.mb[i], g.fp16, g.b[i].p, g.N, g.K, g.b[i].ld, 64, b_rows, &why)
                                   : make_tmap_16bit(&p.mb[i], g.fp16, g.b[i].p, g.K, g.N, g.b[i].ld, 64, b_rows, &why));
  if (!ok) return static_cast<int>(cudaErrorInvalidValue);
  return g.fp16 ? launch_ffn_tc_fp16(plan.cfg, g.layout, g.gated, p, stream)
                : launch_ffn_tc_bf16(plan.cfg, g.layout, g.gated, p, stream);
}

}  // namespace j1rt
