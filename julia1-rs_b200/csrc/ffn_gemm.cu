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
  int sk_q, sk_r, group;  // stream-K groups; order of the tiles (tile_at)
};

// The tile shape and split with the least time by a model: microseconds per 64-block of a tile when few
// SMs work (lone: latency) and when all do (busy: single CTAs are bound by what they load through L2,
// 32 KB per 128 x 128 block against 64 KB per 256 x 256 for a pair), a launch with its epilogue (base),
// and what a cluster's exchange costs: its accumulators' rows shared out (more CTAs, fewer for each) and
// its traffic (more pieces to read). The constants are fitted to the times of 124 products (all operand
// orders and gated; 1 to 131072 rows, contractions of 64 to 131072, weights from HBM for few rows) under
// every plan: among them the plan chosen costs 0.9% more than the best one on average, 21% at most (an earlier model
// whose exchange cost the same for all rows 10%); among 124 others, most of random sizes, 4.7% and 62%, the most where a
// long M meets K below 64, whose epilogues it leaves out. Some of the first (us), best plan first:
//   768 x 768 x 1024 TN    CG 1 x 64 5.3, x 128 6.7, x 64 in clusters of two 7.1, CG 2 x 256 9.9
//   1 x 2048 x 8192        CG 1 x 128 in fours 10.6, x 64 in fours 11.7, in twos 14, in eights 16, one CTA 21-23
//   16 x 8192 x 8192       CG 1 x 128 in twos 25.0, one CTA 28.7
//   8192 x 768 x 1152      CG 2 x 192 13.3, CG 1 x 128 15.4, CG 2 x 256 15.8
//   8192 x 8192 x 2048     CG 2 x 256 186, x 192 186, CG 1 x 128 257
//   768 x 768 x 32768 TN   stream-K 47, CG 1 x 128 in twos 57
Plan choose(const FfnGemm& g, int kb) {
  const int sms = g.num_sms, pairs = std::max(1, std::min(kPairs, sms / 2));
  Plan best = {};
  best.us = 1e30;
  const auto take = [&](const Plan& p) {
    if (p.us < best.us) best = p;
  };
  struct Single {
    int cfg, bn;
    double lone, busy, few, base, split, ctas, rows, traffic;  // few: more per block when A has few rows
  };
  const auto single = [&](const Single& c) {
    const long long tiles = ceil_div(g.M, 128) * ceil_div(g.N, g.gated ? c.bn / 2 : c.bn);
    const double rows = g.layout == FFN_TN ? 1.0 : std::min<double>(g.M, 128.0) / 128.0;  // small A boxes load less
    const double quarters = g.M > 64 ? 4 : g.M > 32 ? 2 : 1;
    for (int s = 1; s <= 8 && s <= kb; s *= 2) {
      const long long ctas = tiles * s;
      // clusters of four and eight do not fill every part of the GPU
      if (s > 1 && ctas > (s == 2 ? sms : s == 4 ? sms * 7 / 8 : sms * 5 / 7)) break;
      const double load = std::min(1.0, static_cast<double>(ctas) / sms);
      const double full = c.busy * (c.bn + 128 * rows) / (c.bn + 128);
      const double step = c.lone + std::max(0.0, full - c.lone) * load + c.few * (1.0 - rows);
      double us = static_cast<double>(ceil_div(ctas, sms) * ceil_div(kb, s)) * step + c.base + (g.gated ? 0.7 : 0.0);
      if (s > 1) us += c.split + c.ctas * s + c.rows * quarters / s + c.traffic * load * s;
      take({c.cfg, 1, c.bn, s, false, us, 1, 1, 8});
    }
  };
  single({FFN_CG1_128, 128, 0.18, 0.25, 0.02, 3.4, -1.0, 0.0, 1.9, 1.0});
  if (!g.gated) single({FFN_CG1_64, 64, 0.13, 0.16, 0.055, 2.85, -0.9, 0.08, 1.5, 0.36});
  const auto pair = [&](int cfg, int bn, double lone, double busy, double base) {
    const long long tiles = ceil_div(g.M, 256) * ceil_div(g.N, g.gated ? bn / 2 : bn);
    const double load = std::min(1.0, static_cast<double>(tiles) / pairs);
    const double step = lone + (busy - lone) * load;
    take({cfg, 2, bn, 1, false, static_cast<double>(ceil_div(tiles, pairs)) * kb * step + base + (g.gated ? 0.75 : 0.0), 1, 1, 8});
    if (g.layout == FFN_TN && bn == 256 && g.partials && tiles * kb < INT_MAX && tiles * kb >= pairs &&
        (tiles + pairs) * kPieceBytes <= g.partial_bytes) {
      // q workers for every r tiles, then a pass over the pieces. Tiles of the same place in their group
      // walk the contraction together: with r dividing the tile rows, rows fastest, that is every r-th
      // row for all columns, and each of the r walks reads (rows / r + columns) x 256 columns of the
      // operands; with r dividing the tile columns the other way round.
      const long long mt = ceil_div(g.M, 256), nt = ceil_div(g.N, 256);
      for (int order = 0; order < 2; ++order)
        for (int r = 1; r <= 8; ++r) {
          const long long side = order ? nt : mt, other = order ? mt : nt, q = pairs * static_cast<long long>(r) / tiles;
          if (side % r || q < 1 || q * r * kb >= (1ll << 32)) continue;
          const double compute = static_cast<double>(tiles) * kb * 0.445 / static_cast<double>(q * (tiles / r));
          const double memory = static_cast<double>(side + r * other) * kb * (64 * 256 * 2) / 6.0e6;
          take({cfg, 2, bn, 1, true, std::max(compute, memory) + 2.1 + 0.115 * static_cast<double>(tiles + pairs),
                static_cast<int>(q), r, static_cast<int>(order ? 1 : mt)});
        }
    }
  };
  pair(FFN_CG2_256, 256, 0.28, 0.41, 4.85);
  if (g.layout == FFN_NT && !g.gated) pair(FFN_CG2_192, 192, 0.22, 0.315, 4.1);
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

void ffn_plan(const FfnGemm& g, int32_t* plan) {
  const int segs = g.lo ? 2 * g.segs : g.segs;
  const Plan p = choose(g, static_cast<int>(ceil_div(g.K, 64)) * segs);
  const int32_t v[6] = {p.cg, p.bn, p.split, p.stream_k ? p.sk_q : 0, p.sk_r, p.stream_k && p.group == 1};
  std::copy(v, v + 6, plan);
}

int launch_ffn_gemm(const FfnGemm& g, cudaStream_t stream) {
  FfnTc p = {};
  const int nb = g.gated ? 2 : g.segs;
  for (int i = 0; i < 2; ++i) p.out[i] = g.out[i], p.pre[i] = g.pre[i], p.bias[i] = g.bias[i];
  p.M = g.M, p.N = g.N;
  p.segs = g.lo ? 2 * g.segs : g.segs;
  p.b_and = g.segs - 1;
  p.kb_seg = static_cast<int>(ceil_div(g.K, 64));
  if (static_cast<long long>(p.kb_seg) * p.segs > INT_MAX) return static_cast<int>(cudaErrorInvalidValue);
  p.kb = p.kb_seg * p.segs;
  const Plan plan = choose(g, p.kb);
  p.act = g.act;
  p.row1 = g.row1, p.rows0 = g.rows0;
  const long long m_tiles = ceil_div(g.M, 128 * plan.cg);
  const long long n_tiles = ceil_div(g.N, g.gated ? plan.bn / 2 : plan.bn);
  if (m_tiles * n_tiles * plan.split > INT_MAX / 64) return static_cast<int>(cudaErrorInvalidValue);
  p.m_tiles = static_cast<int>(m_tiles), p.n_tiles = static_cast<int>(n_tiles);
  p.tiles = p.m_tiles * p.n_tiles;
  p.split = plan.split;
  for (p.split_log2 = 0; (1 << p.split_log2) < plan.split;) ++p.split_log2;
  p.stream_k = plan.stream_k;
  p.partials = g.partials;
  const int slots = plan.cg == 2 ? std::max(1, std::min(kPairs, g.num_sms / 2)) : g.num_sms;
  p.sk_q = plan.sk_q, p.sk_r = plan.sk_r;
  p.workers = plan.split > 1 ? p.tiles : plan.stream_k ? plan.sk_q * (p.tiles / plan.sk_r) : std::min(p.tiles, slots);
  p.group = plan.stream_k ? plan.group : 8;
  p.a_rows = plan.cg == 1 && g.layout != FFN_TN && g.M < 128 ? (g.M + 7) / 8 * 8 : 128;
  p.early = g.early, p.late = g.late;
  p.scale = g.scale;
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
  for (int i = 0; i < p.segs; ++i) {
    FfnMat a = g.a[i & p.b_and];
    if (i >= g.segs) a.p = static_cast<const uint16_t*>(a.p) + g.lo;
    ok = ok && (g.layout == FFN_TN ? make_tmap_16bit(&p.ma[i], g.fp16, a.p, g.K, g.M, a.ld, 64, 64, &why)
                                   : make_tmap_16bit(&p.ma[i], g.fp16, a.p, g.M, g.K, a.ld, 64, p.a_rows, &why));
  }
  const uint32_t b_rows = g.layout != FFN_NT ? 64 : g.gated ? plan.bn / 2 : plan.bn / plan.cg;
  for (int i = 0; i < nb; ++i)
    ok = ok && (g.layout == FFN_NT ? make_tmap_16bit(&p.mb[i], g.fp16, g.b[i].p, g.N, g.K, g.b[i].ld, 64, b_rows, &why)
                                   : make_tmap_16bit(&p.mb[i], g.fp16, g.b[i].p, g.K, g.N, g.b[i].ld, 64, b_rows, &why));
  // the warps' own stores where rows are not whole 16-byte units (TMA would write the unit's rest), for one
  // CTA's tiles (code that a launch of a few microseconds would fetch) and for results in two parts
  p.tma_out = plan.cg == 2 && g.layout == FFN_NT && p.vec_out && p.vec_pre;
  if (p.tma_out) {
    ok = ok && make_tmap_16bit(&p.mo, g.fp16, g.out[0].p, g.M, g.N, g.out[0].ld, 32, 32, &why);
    for (int i = 0; i < 2; ++i)
      if (g.pre[i].p) ok = ok && make_tmap_16bit(&p.mp[i], g.fp16, g.pre[i].p, g.M, g.N, g.pre[i].ld, 32, 32, &why);
  }
  if (!ok) return static_cast<int>(cudaErrorInvalidValue);
  return g.fp16 ? launch_ffn_tc_fp16(plan.cfg, g.layout, g.gated, p, stream)
                : launch_ffn_tc_bf16(plan.cfg, g.layout, g.gated, p, stream);
}

}  // namespace j1rt
