// Matrix products of the feed-forward operators on tcgen05, with their epilogues.
//
//   out[M, N] = act(A . B + bias) (+ residual), A . B over one to four operand pairs
//   out[M, N] = act(A B0^T + bias0) * (A B1^T + bias1)                            (gated)
//
// One kernel for every operand order: an operand whose contraction index is contiguous in
// memory is staged K-major (rows of 64 contraction elements, 128 bytes, 128B swizzle), one
// whose output index is contiguous MN-major (64 output elements per 128-byte row, one row per
// contraction index); tcgen05 reads either through its shared-memory descriptors, so no
// operand is transposed in memory.
//
// CG = 2: CTA pairs, 256 x BN tiles, tcgen05.mma.cta_group::2; per 256 x 256 x 64 step a CTA
//   moves 32 KB through L2 for 8.4 MFLOP, what it takes to keep the tensor cores fed.
// CG = 1: single CTAs, 128 x BN tiles, for outputs of too few 256-wide tiles to fill the GPU;
//   `split` CTAs of a cluster may share one tile's contraction, each a range of it, and add
//   their FP32 accumulators through distributed shared memory in rank order.
// Stream-K (CG = 2, weight gradients: few tiles, long contraction): q pairs take equal parts of the
//   64-blocks of r neighbouring tiles; FP32 pieces go to the workspace in the accumulator's own
//   layout and a second kernel adds a tile's pieces in order. All groups of r tiles walk the
//   contraction in step, so what one pair loads others find in L2: with one equal part of all
//   blocks per pair instead, every pair was at a place of its own, and dw of 65536 x 2304 x 768 took
//   205 us, 1.36 times a product of the same size whose tiles share their operands.
//
// Roles per CTA: warp 0 TMA producer, warp 1 TMEM allocator and MMA issuer (even CTA), then the
// epilogue warps (eight to sixteen: those of a TMEM lane quarter take its 32-column chunks in turn).
// Producer and issuer run as whole warps with one elected lane issuing: with a lane-dependent
// branch around the loop instead, an MMA step (four MMAs and a commit) took 600 cycles to issue.
// The accumulator is double buffered in TMEM, so a tile's epilogue runs under the next tile's
// products. The epilogue works on 32-column chunks, one thread per row: FP32 accumulators from
// TMEM, bias, activation, residual, one rounding, then through a swizzled 32 x 32 box in shared
// memory to the result. Pairs' forward boxes are stored by TMA where rows are whole 16-byte units
// (131072 x 1152 x 768 with GELU and saved pre-activations in 7% less time than with 16-byte stores by the warps);
// other boxes by the warps, 16 bytes a lane, or words where rows are not 16-byte aligned (8192 x 1153 x
// 768 with saved pre-activations 34 us; 47 with the alignment looked at per row instead of per lane).
//
// Code size counts: a launch of a few microseconds fetches its instructions cold, and a role's
// loop that does not fit the innermost instruction cache costs about 180 cycles per turn. So single
// CTAs work in rolled loops of 16 columns, box copies and waiting loops are out of line, and
// shared memory is addressed with 32-bit addresses throughout. Pairs, whose launches are long,
// take the 32 columns of a chunk at once for twice the independent work (131072 x 1152 x 768 with
// GELU 4% less time than by halves).
//
// Measured on one B200 (CUDA graph, inputs larger than L2): 131072 x 1152 x 768 without activation
// 183-188 us (1.26 PFLOP/s; 0.75 of the measured burst rate), with GELU 211, with GELU and saved pre-
// activations 227-236 (0.8 GB at 3.5 TB/s); 8192 x 768 x 1152 with residual 15.8 us; gated 8192 x
// 1152 x 768 21.9 us (1.32 PFLOP/s), gated 4096 x 8192 x 4096 saved 365-388 us (1.42-1.5 PFLOP/s);
// 8192 x 8192 x 8192 0.755 ms (1.46 PFLOP/s); 16 x 8192 x 8192 24.8-26.8 us (5.0-5.4 TB/s, 0.77-0.83 of
// measured); 1 x 768 x 768 4.0 us. Large products are bound by what their tiles read through L2 and by the power
// cap (tensor pipe busy 75% without activation at 32768 rows, 63% with GELU), an epilogue of
// exponentials by the latency of its chains (issue slots 54% busy), few rows by the weights' bytes, the
// smallest by launch, set-up and first loads.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "ffn_math.cuh"
#include "ffn_tc.h"
#include "kernels.h"
#include "ptx.cuh"

namespace j1rt {

namespace ffn {

constexpr int BM = 128;  // rows of a tile per CTA
constexpr int BK = 64;   // contraction elements per stage
// Epilogue warps. A linear forward tile on a pair has up to 32,768 activations per CTA, each with an
// exponential and a reciprocal: with two warps per SM sub-partition their latencies were not hidden
// (131072 x 1152 x 768 with GELU 326 us, without 182 us), with four they were (219 us then). Gated tiles
// have half of them, products without an activation none: eight warps leave room for more stages
// (gated with sixteen: 65536 x 1152 x 768 saved 206 us as with eight, 4096 x 8192 x 4096 saved 443 us
// against 384).
__host__ __device__ constexpr int epi_warps(int cg, int bn, int layout, bool gated) {
  return cg == 2 && layout == FFN_NT && !gated ? (bn == 192 ? 12 : 16) : 8;
}
constexpr uint32_t SLOT = 32 * 32 * 2;  // one 32 x 32 output box
constexpr uint32_t A_BYTES = BM * BK * 2;
constexpr uint32_t SMEM_MAX = 232448;
// bias of the chunk at hand per epilogue warp (two rows of 32 floats), barriers
constexpr uint32_t BIAS_BYTES = 2 * 32 * 4, BAR_BYTES = 256;

__host__ __device__ constexpr uint32_t b_bytes(int cg, int bn) { return static_cast<uint32_t>(bn / cg) * BK * 2; }
__host__ __device__ constexpr uint32_t tmem_cols(int bn) { return bn > 128 ? 512 : bn > 64 ? 256 : 128; }

// kind::f16 instruction descriptor (ptx.cuh idesc_bf16) with the element type as a parameter.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int m, int n, bool a_mn, bool b_mn) {
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;  // 0 f16, 1 bf16
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// True in one lane of a converged warp, always the same one.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r != 0;
}
// ---- shared-memory operations by 32-bit address
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Whether a phase is complete, without waiting.
__device__ __forceinline__ bool bar_peek(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// The same, suspending the thread for a while.
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A bounded wait of a whole warp with one outcome, as ptx.cuh's mbar_wait: after J1_WAIT_CYCLES (or
// once another role of the CTA gave up) the CTA's abort word is set, the site recorded in *err.
static __device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, uint32_t abort_word, int* err, int site) {
  const long long t0 = clock64();
  for (;;) {
    if (__all_sync(0xffffffffu, bar_try(bar, parity))) return true;
    if (__any_sync(0xffffffffu, lds32(abort_word) != 0)) return false;
    if (__any_sync(0xffffffffu, clock64() - t0 > J1_WAIT_CYCLES)) {
      if (lane_id() == 0) {
        sts32(abort_word, 1u);
        if (err) atomicCAS(err, 0, 1 | (site << 16));
      }
      __syncwarp();
      return false;
    }
  }
}
struct Waiter {
  uint32_t abort_word;
  int* err;
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity, int site) const {
    if (__all_sync(0xffffffffu, bar_peek(bar, parity))) return true;
    return wait_slow(bar, parity, abort_word, err, site);
  }
};
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  if constexpr (CG == 2)
    umma_bf16_pair(d, a, b, id, acc);
  else
    umma_bf16(d, a, b, id, acc);
}
// Arrive on the barrier at this shared address in this CTA (CG 1) or in CTA `rank` of the pair when
// this thread's MMAs are done.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar, uint32_t rank) {
  if constexpr (CG == 2)
    umma_commit_pair(mapa_shared(bar, rank));
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// One TMA box to shared address dst, completing on `bar` (CG 2: the leader's, as a cluster address).
template <int CG>
__device__ __forceinline__ void tma_box(const CUtensorMap* map, uint32_t bar, uint32_t dst, int x, int y) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
        "[%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
// 32 TMEM lanes x 16 columns.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ float4 ld_cluster(uint32_t caddr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(caddr)
               : "memory");
  return v;
}

// A worker's list of (tile, blocks [k0, k1)): whole tiles w, w + workers, ..., or its share of
// the tile-major block list (stream-K), or its range of one tile (cluster split). Everything the
// loops need is held here, in registers: after every asm statement a parameter would be read again.
struct Units {
  int tile, k0, k1;
  int kb, step, tiles;      // blocks per tile, tiles to the next one, tiles
  int group, m_tiles, n_tiles;
  int pos, end;             // stream-K: blocks [pos, end) of the list (below 2^31)

  __device__ __forceinline__ Units(const FfnTc& p, int worker, int rank) {
    kb = p.kb, step = p.workers, tiles = p.tiles;
    group = p.group, m_tiles = p.m_tiles, n_tiles = p.n_tiles;
    tile = worker, k0 = 0, k1 = kb;
    pos = end = 0;
    if (p.stream_k) {
      pos = share_begin(p, worker);
      end = share_begin(p, worker + 1);
      step = 0;
      share();
    } else if (p.split > 1) {
      const int per = (kb + p.split - 1) >> p.split_log2;  // blocks per CTA, the last ones one less
      const int full = kb - (per - 1) * p.split;
      k0 = rank * per - (rank > full ? rank - full : 0);
      k1 = k0 + per - (rank >= full ? 1 : 0);
    }
  }
  // Stream-K: every sk_q workers share sk_r neighbouring tiles in equal parts (sk_q sk_r kb < 2^32).
  static __device__ __forceinline__ int share_begin(const FfnTc& p, int worker) {
    const uint32_t q = p.sk_q, blocks = static_cast<uint32_t>(p.sk_r) * p.kb, g = static_cast<uint32_t>(worker) / q;
    return static_cast<int>(g * blocks + (worker - g * q) * blocks / q);
  }
  __device__ __forceinline__ void share() {
    tile = pos < end ? pos / kb : tiles;
    k0 = pos - tile * kb;
    k1 = min(end - pos, kb - k0) + k0;
  }
  __device__ __forceinline__ bool ok() const { return tile < tiles; }
  __device__ __forceinline__ void next() {
    tile += step;
    if (step == 0) {
      pos += k1 - k0;
      share();
    }
  }
  __device__ __forceinline__ void at(int& mt, int& nt) const;
};
// Tiles are ordered in groups of `group` tile rows, rows fastest inside a group: the tiles in
// flight share few rows of A and few columns of B, so both stay in L2.
__host__ __device__ __forceinline__ void tile_at(int tile, int group, int m_tiles, int n_tiles, int& mt, int& nt) {
  if (m_tiles == 1) {
    mt = 0, nt = tile;
    return;
  }
  const int per = group * n_tiles;
  const int first = tile / per * group;
  const int rows = m_tiles - first < group ? m_tiles - first : group;
  const int r = tile - tile / per * per;
  mt = first + r % rows;
  nt = r / rows;
}

__device__ __forceinline__ void Units::at(int& mt, int& nt) const { tile_at(tile, group, m_tiles, n_tiles, mt, nt); }

template <int ACT, int W>
__device__ __forceinline__ void act_all(uint64_t (&v)[W]) {
#pragma unroll
  for (int i = 0; i < W; ++i) v[i] = act_pair<ACT>(v[i]);
}
template <int W>
__device__ __forceinline__ void act_all(int act, uint64_t (&v)[W]) {
  switch (act) {
    case J1_ACT_RELU: act_all<J1_ACT_RELU, W>(v); break;
    case J1_ACT_GELU: act_all<J1_ACT_GELU, W>(v); break;
    case J1_ACT_GELU_TANH: act_all<J1_ACT_GELU_TANH, W>(v); break;
    case J1_ACT_SILU: act_all<J1_ACT_SILU, W>(v); break;
    default: break;
  }
}
// A pair of FP32 values rounded to two elements.
template <typename T>
__device__ __forceinline__ uint32_t pack2(uint64_t v) {
  float lo, hi;
  f2unpack(v, lo, hi);
  return Elem<T>::pack(lo, hi);
}

// 8 results of one row to m[row, col ...]: 16 bytes, or element by element up to column N.
template <typename T>
__device__ __forceinline__ void store_row8(const FfnMat& m, bool vec, long long row, int col, int N, const uint64_t (&v)[4]) {
  uint16_t* at = static_cast<uint16_t*>(const_cast<void*>(m.p)) + row * m.ld + col;
  const uint32_t w[4] = {pack2<T>(v[0]), pack2<T>(v[1]), pack2<T>(v[2]), pack2<T>(v[3])};
  if (vec) {
    *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < N) at[i] = static_cast<uint16_t>(w[i >> 1] >> ((i & 1) * 16));
  }
}

// A box to columns from col, rows from row of a map's matrix; what is behind its edges (whole 16-byte
// units) is left out.
__device__ __forceinline__ void store_box(const CUtensorMap* map, uint32_t box, int col, int row) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(box), "r"(col), "r"(row)
               : "memory");
}

// Copies a warp's box (32 rows x 32 columns, 64 bytes a row, unit u of row r at u ^ (r >> 1 & 3)) to rows
// [row, row + 32) below `rows`, columns [col, col + 32) below N of a matrix.
static __device__ __noinline__ void copy_out(uint32_t box, void* p, long long ld, int vec, int row, int rows, int col, int N) {
  const int lane = lane_id();
  __syncwarp();
  if (vec) {
    const int br = lane >> 2, bu = lane & 3;
    uint16_t* at = static_cast<uint16_t*>(p) + static_cast<long long>(row + br) * ld + col + bu * 8;
    uint4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = lds128(box + (br + 8 * i) * 64 + ((bu ^ ((br >> 1) & 3)) << 4));
    if (col + bu * 8 < N) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (row + br + 8 * i < rows) *reinterpret_cast<uint4*>(at) = w[i];
        at += 8 * ld;
      }
    }
  } else {
    // Two rows at a time, 16 lanes each. A lane's rows all start on a word or all between two: there it
    // stores the words between its own and the next (elements 2 h + 1, 2 h + 2), and the first and last
    // lane the row's first and last element. A lane reads the word behind its own as well: a shuffle in
    // this function cost the kernel a third more code.
    const int h = lane & 15, n = rows - row, left = N - col;
    const int h1 = (h + 1) & 15;
    int r = lane >> 4;
    uint16_t* at = static_cast<uint16_t*>(p) + static_cast<long long>(row + r) * ld + col;
    const bool odd = (reinterpret_cast<uintptr_t>(at) & 2u) != 0;
    const uint32_t from = box + r * 64 + (h & 3) * 4, from1 = box + r * 64 + (h1 & 3) * 4;
    const bool word = !odd || h < 15, end = odd && (h == 0 || h == 15);
    uint16_t* at_word = at + 2 * h + (odd ? 1 : 0);
    uint16_t* at_end = at + (h ? 31 : 0);
    if (left >= 32) {
#pragma unroll 1
      for (int i0 = 0; i0 < 16; i0 += 8) {
        uint32_t w[8], next[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t o = (i0 + i) * 128;
          w[i] = lds32(from + o + (((h >> 2) ^ (i & 3)) << 4));
          next[i] = lds32(from1 + o + (((h1 >> 2) ^ (i & 3)) << 4));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (r < n) {
            if (word) *reinterpret_cast<uint32_t*>(at_word) = __funnelshift_r(w[i], next[i], odd ? 16 : 0);
            if (end) *at_end = static_cast<uint16_t>(h ? w[i] >> 16 : w[i]);
          }
          r += 2;
          at_word += 2 * ld;
          at_end += 2 * ld;
        }
      }
    } else {
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const uint32_t w = lds32(from + i * 128 + (((h >> 2) ^ (i & 3)) << 4));
        if (r < n) {
          if (2 * h < left) at[2 * h] = static_cast<uint16_t>(w);
          if (2 * h + 1 < left) at[2 * h + 1] = static_cast<uint16_t>(w >> 16);
        }
        r += 2;
        at += 2 * ld;
      }
    }
  }
  __syncwarp();
}
// The other way (the residual): vec by asynchronous copies that the reader waits for.
static __device__ __noinline__ void copy_in(uint32_t box, const void* p, long long ld, int vec, int row, int rows, int col, int N) {
  const int lane = lane_id();
  if (vec) {
    const int br = lane >> 2, bu = lane & 3;
    const uint16_t* at = static_cast<const uint16_t*>(p) + static_cast<long long>(row + br) * ld + col + bu * 8;
    if (col + bu * 8 < N) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = br + 8 * i;
        if (row + r < rows) cp_async16(box + r * 64 + ((bu ^ ((r >> 1) & 3)) << 4), at);
        at += 8 * ld;
      }
    }
  } else {
    const int c = col + lane, n = min(32, rows - row);
    const uint16_t* at = static_cast<const uint16_t*>(p) + static_cast<long long>(row) * ld + c;
#pragma unroll 1
    for (int r0 = 0; r0 < n; r0 += 16) {
      uint16_t v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[i] = c < N && r0 + i < n ? *at : 0;
        at += ld;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(box + (r0 + i) * 64 + (((lane >> 3) ^ ((i >> 1) & 3)) << 4) + (lane & 7) * 2),
                     "h"(v[i])
                     : "memory");
    }
  }
}

template <typename T, int CG, int BN, int LAYOUT, bool GATED>
__global__ void __launch_bounds__(32 * (2 + epi_warps(CG, BN, LAYOUT, GATED)), 1) tc_kernel(const __grid_constant__ FfnTc p) {
  constexpr bool A_MN = LAYOUT == FFN_TN, B_MN = LAYOUT != FFN_NT;
  constexpr int EW = epi_warps(CG, BN, LAYOUT, GATED);
  constexpr int BROWS = BN / CG;             // output columns of B staged by one CTA
  constexpr int OUTW = GATED ? BN / 2 : BN;  // output columns of a tile
  constexpr uint32_t B_BYTES = b_bytes(CG, BN);
  static_assert(!(GATED && LAYOUT != FFN_NT) && OUTW % 64 == 0, "");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int stages = p.stages;
  // A boxes hold a_rows rows (128, fewer when M is smaller): an MMA still reads 128, the rows behind
  // belong to the next box or to B and only reach accumulator rows that nobody reads
  const uint32_t a_bytes = A_MN ? A_BYTES : static_cast<uint32_t>(p.a_rows) * BK * 2;
  const uint32_t sA = smem, sB = smem + stages * a_bytes;
  const uint32_t boxes = smem + p.ring;
  const uint32_t sbias = boxes + EW * p.boxes * SLOT;
  const uint32_t full = sbias + EW * BIAS_BYTES, empty = full + 64, tfull = empty + 64, tempty = tfull + 16, drain = tempty + 16;
  const uint32_t tmem_slot = drain + 8, abort_word = tmem_slot + 4;

  if (!p.late) grid_dep_launch();
  const int warp = __shfl_sync(0xffffffffu, warp_id(), 0), lane = lane_id();
  const int split = p.split;
  const int crank = CG == 2 || split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const uint32_t rank = CG == 2 ? static_cast<uint32_t>(crank) : 0u;
  const bool leader = rank == 0;
  const int worker = CG == 2 ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x) >> p.split_log2;
  const Waiter wait = {abort_word, p.err};
  uint32_t tmem_base = 0;

  if (warp == 0) {
    if (elect_one()) {
      for (int s = 0; s < stages; ++s) {
        bar_init(full + s * 8, 1);
        bar_init(empty + s * 8, 1);
      }
      for (int b = 0; b < 2; ++b) {
        bar_init(tfull + b * 8, 1);
        bar_init(tempty + b * 8, EW * CG);
      }
      bar_init(drain, 1);
      sts32(abort_word, 0u);
      fence_mbar_init();
    }
    __syncwarp();
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(tmem_cols(BN)));
      tmem_relinquish_pair();
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(tmem_cols(BN)));
      tmem_relinquish();
    }
  }
  // The list of units needs parameters only: its divisions pass while the others set up.
  Units u(p, worker, crank);
  int mt, nt;
  u.at(mt, nt);
  // Barriers initialised and TMEM allocated, in both CTAs of a pair. The producer of a single CTA
  // needs nothing from the other warps: it only arrives and starts to load.
  tc_fence_before();
  if constexpr (CG == 2) {
    cluster_sync();
  } else if (warp == 0) {
    asm volatile("bar.arrive 1, %0;" ::"n"(32 * (2 + EW)) : "memory");
  } else {
    asm volatile("bar.sync 1, %0;" ::"n"(32 * (2 + EW)) : "memory");
  }
  tc_fence_after();
  if (!p.early) grid_dep_wait();
  if (p.late) grid_dep_launch();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    const int kb_seg = p.kb_seg;
    int stage = 0, round = 0;
    uint32_t phase = 1;
    bool ok = true;
    for (; ok && u.ok(); u.next(), u.at(mt, nt)) {
      const int m0 = (mt * CG + static_cast<int>(rank)) * BM;
      const int n0 = GATED ? nt * OUTW : nt * BN + static_cast<int>(rank) * BROWS;
#pragma unroll 1
      for (int kb = u.k0; kb < u.k1; ++kb) {
        const uint32_t fb = full + stage * 8;
        if (round && !wait(empty + stage * 8, phase, 31)) {  // in the first round every stage is empty
          ok = false;
          break;
        }
        const int seg = (kb >= kb_seg ? 1 : 0) + (kb >= 2 * kb_seg ? 1 : 0) + (kb >= 3 * kb_seg ? 1 : 0);
        const int k = (kb - seg * kb_seg) * BK;
        const uint32_t da = sA + stage * a_bytes, db = sB + stage * B_BYTES;
        if (elect_one()) {
          if (leader) bar_expect(fb, CG * (a_bytes + B_BYTES));
          const uint32_t fc = CG == 2 ? mapa_shared(fb, 0) : fb;
          const CUtensorMap* ma = &p.ma[0] + seg;
          const CUtensorMap* mb = &p.mb[0] + (GATED ? static_cast<int>(rank) : seg & p.b_and);
          if constexpr (A_MN) {
            tma_box<CG>(ma, fc, da, m0, k);
            tma_box<CG>(ma, fc, da + A_BYTES / 2, m0 + 64, k);
          } else {
            tma_box<CG>(ma, fc, da, k, m0);
          }
          if constexpr (B_MN) {
#pragma unroll
            for (int c = 0; c < BROWS / 64; ++c) tma_box<CG>(mb, fc, db + c * 8192, n0 + c * 64, k);
          } else {  // gated: the tile's columns are OUTW of B0 (CTA 0), then OUTW of B1 (CTA 1)
            tma_box<CG>(mb, fc, db, k, n0);
            if constexpr (GATED && CG == 1) tma_box<CG>(mb + 1, fc, db + B_BYTES / 2, k, n0);
          }
        }
        __syncwarp();
        if (++stage == stages) {
          stage = 0;
          round = 1;
          phase ^= 1;
        }
      }
    }
    if (!ok) {
      // Unwinding after a timeout: copies in flight may complete on the other CTA's barrier,
      // so give them ample time to land before shared memory is released.
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000) __nanosleep(1000);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA)
    tmem_base = lds32(tmem_slot);
    if (leader) {
      constexpr uint32_t id = idesc<T>(BM * CG, BN, A_MN, B_MN);
      // descriptors of stage 0; a stage or a step of 16 contraction elements adds to the address
      // field (units of 16 bytes)
      const uint64_t a_desc = A_MN ? sdesc_sw128(sA, 8192, 1024) : sdesc_sw128(sA, 16, 1024);
      const uint64_t b_desc = B_MN ? sdesc_sw128(sB, 8192, 1024) : sdesc_sw128(sB, 16, 1024);
      constexpr uint32_t a_step = A_MN ? 2048 / 16 : 32 / 16, b_step = B_MN ? 2048 / 16 : 32 / 16;
      int stage = 0, acc = 0;
      uint32_t phase = 0;
      bool ok = true;
      // The test of the next stage's barrier is issued before this stage's MMAs: its latency (80
      // cycles) passes while they are issued.
      bool ready = bar_peek(full, 0);
      for (; ok && u.ok(); u.next()) {
        const int buf = acc & 1;
        if (acc >= 2) ok = wait(tempty + buf * 8, ((acc >> 1) + 1) & 1, 32);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem_base + buf * BN;
        uint32_t more = 0;  // 0: the tile's first MMA overwrites the accumulator
#pragma unroll 1
        for (int kb = u.k0; kb < u.k1; ++kb) {
          if (!__all_sync(0xffffffffu, ready) && !wait(full + stage * 8, phase, 33)) {
            ok = false;
            break;
          }
          const int next = stage + 1 == stages ? 0 : stage + 1;
          const uint32_t next_phase = next ? phase : phase ^ 1;
          ready = bar_peek(full + next * 8, next_phase);
          tc_fence_after();
          if (elect_one()) {
            const uint64_t da = a_desc + static_cast<uint32_t>(stage) * (a_bytes / 16);
            const uint64_t db = b_desc + static_cast<uint32_t>(stage) * (B_BYTES / 16);
            mma<CG>(d, da, db, id, more);
#pragma unroll
            for (int k = 1; k < BK / 16; ++k) mma<CG>(d, da + k * a_step, db + k * b_step, id, 1u);
            commit<CG>(empty + stage * 8, 0);
            if constexpr (CG == 2) commit<CG>(empty + stage * 8, 1);
          }
          __syncwarp();
          more = 1;
          stage = next;
          phase = next_phase;
        }
        if (!ok) break;
        if (elect_one()) {
          commit<CG>(tfull + buf * 8, 0);
          if constexpr (CG == 2) commit<CG>(tfull + buf * 8, 1);
        }
        __syncwarp();
        ++acc;
      }
      // Every tile's accumulators have been read (both CTAs' epilogues arrive here), or, after an
      // abort, at least every MMA has finished: TMEM may be released.
      for (int b = 0; ok && b < 2; ++b) {
        const int uses = (acc + 1 - b) / 2;
        if (uses > 0) ok = wait(tempty + b * 8, (uses - 1) & 1, 36);
      }
      if (!ok) {
        if (elect_one()) commit<CG>(drain, 0);
        __syncwarp();
        const long long t0 = clock64();
        while (!bar_try(drain, 0) && clock64() - t0 < J1_WAIT_CYCLES) {
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue warps
    const int e = warp - 2;
    const int q = warp & 3;                // TMEM lane quarter this warp may access
    constexpr int PER = EW / 4;            // warps of a quarter: they take its 32-column chunks in turn
    const int c0 = (e >> 2) * 32;
    const int M = p.M, N = p.N, act = p.act;
    const bool save = p.pre[0].p != nullptr, residual = !GATED && p.residual.p != nullptr;
    const uint32_t box = boxes + static_cast<uint32_t>(e) * p.boxes * SLOT;  // output, then pre-activations
    const uint32_t wbias = sbias + e * BIAS_BYTES;
    const uint32_t own = box + lane * 64;  // this thread's row, unit u at own + ((u ^ sw) << 4)
    const uint32_t sw = static_cast<uint32_t>((lane >> 1) & 3);
    tmem_base = lds32(tmem_slot);

    // What the chunk at (row, col) needs beside its accumulators: one column's biases per lane, loaded
    // a chunk ahead (load), then put to the warp's bias rows, and the residual to the output box, once
    // everything of the chunk before has left them (place).
    const bool bias0 = p.bias[0] != nullptr, bias1 = p.bias[1] != nullptr;
    float nb0 = 0.f, nb1 = 0.f;
    auto load = [&](int col) {
      const bool in = col + lane < N;
      if (bias0) nb0 = in ? p.bias[0][col + lane] : 0.f;
      if (GATED && bias1) nb1 = in ? p.bias[1][col + lane] : 0.f;
    };
    const bool tma = CG == 2 && LAYOUT == FFN_NT && p.tma_out;
    auto boxes_free = [&]() {  // what was stored from them has been read
      if (lane == 0) bulk_wait_read_all();
      __syncwarp();
    };
    auto place = [&](int row, int col) {
      if (tma && residual) boxes_free();
      if (bias0) sts32(wbias + lane * 4, __float_as_uint(nb0));
      if (GATED && bias1) sts32(wbias + 128 + lane * 4, __float_as_uint(nb1));
      if (residual) copy_in(box, p.residual.p, p.residual.ld, p.vec_res, row, M, col, N);
    };
    constexpr int H = CG == 2 ? 2 : 1;  // 16-column halves of a chunk in registers at a time
    auto add16 = [&](bool add, uint32_t bias, const uint32_t (&r)[H][16], uint64_t (&v)[8 * H]) {
      if (!add) {
#pragma unroll
        for (int i = 0; i < 8 * H; ++i)
          v[i] = f2pack(__uint_as_float(r[i / 8][2 * (i % 8)]), __uint_as_float(r[i / 8][2 * (i % 8) + 1]));
        return;
      }
#pragma unroll
      for (int i = 0; i < 4 * H; ++i) {
        const uint4 b = lds128(bias + i * 16);
        const uint32_t* x = &r[i / 4][4 * (i % 4)];
        v[2 * i] = add2(f2pack(__uint_as_float(x[0]), __uint_as_float(x[1])),
                        f2pack(__uint_as_float(b.x), __uint_as_float(b.y)));
        v[2 * i + 1] = add2(f2pack(__uint_as_float(x[2]), __uint_as_float(x[3])),
                            f2pack(__uint_as_float(b.z), __uint_as_float(b.w)));
      }
    };
    auto put16 = [&](uint32_t at, int j, const uint64_t (&v)[8 * H]) {  // units of this thread's row
#pragma unroll
      for (int i = 0; i < 2 * H; ++i)
        sts128(at + ((static_cast<uint32_t>(2 * j + i) ^ sw) << 4),
               make_uint4(pack2<T>(v[4 * i]), pack2<T>(v[4 * i + 1]), pack2<T>(v[4 * i + 2]), pack2<T>(v[4 * i + 3])));
    };

    // products of FP16 gradients: the power of two their operand was multiplied by is taken out here
    constexpr bool SCALED = LAYOUT != FFN_NT && std::is_same<T, __half>::value;
    uint64_t scale = 0ull;
    if constexpr (SCALED) {
      const float f = p.scale ? __ldcg(p.scale) : 1.f;
      scale = f2pack(f, f);
    }

    int acc = 0;
    bool ok = true;
    for (; ok && u.ok(); u.next(), u.at(mt, nt), ++acc) {
      const int row = (mt * CG + static_cast<int>(rank)) * BM + q * 32;  // this warp's first row
      const int n0 = nt * OUTW;
      const uint32_t buf = acc & 1;
      const bool pieces = split > 1 || p.stream_k;
      if (!pieces && row < M && c0 < OUTW && n0 + c0 < N) {
        load(n0 + c0);
        place(row, n0 + c0);
      }
      ok = wait(tfull + buf * 8, (acc >> 1) & 1, 35);
      if (!ok) break;
      tc_fence_after();
      const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BN;
      auto release = [&]() {  // the buffer has been read to the end
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2)
            mbar_arrive_remote(mapa_shared(tempty + buf * 8, 0));
          else
            bar_arrive(tempty + buf * 8);
        }
      };
      if (pieces) {
        // FP32 accumulators as they are, four columns of a row per 16 bytes, lanes side by side:
        // stream-K pieces to the workspace, a cluster's to shared memory (over the idle stages)
        constexpr int ACC = BN / PER;  // accumulator columns of this warp
        // pieces are numbered worker + tile: unique, below workers + tiles
        float4* dst = reinterpret_cast<float4*>(p.partials) +
                      (((static_cast<size_t>(worker) + u.tile) * CG + rank) * 4 + q) * (BN / 4) * 32 + lane;
        const uint32_t sdst = smem + (q * (BN / 4) * 32 + lane) * 16;
#pragma unroll 1
        for (int c = (e >> 2) * ACC; row < M && c < ((e >> 2) + 1) * ACC; c += 16) {
          uint32_t r[16];
          tmem_ld16(tb + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (split > 1)
              sts128(sdst + (c / 4 + i) * 512, make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]));
            else
              dst[(c / 4 + i) * 32] = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                                                  __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
          }
        }
        release();
        continue;
      }
      if (c0 >= OUTW) release();  // more warps than chunks
#pragma unroll 1
      for (int c = c0; c < OUTW; c += 32 * PER) {
        const int col = n0 + c;
        const bool in = row < M && col < N;
        if (in) {
          if (residual) cp_async_wait();
          __syncwarp();  // biases and residual are in place
        }
        const bool more = c + 32 * PER < OUTW && col + 32 * PER < N;
        if (more) load(col + 32 * PER);
#pragma unroll 1
        for (int j = 0; j < 2; j += H) {
          uint32_t r0[H][16], r1[H][16];
#pragma unroll
          for (int h = 0; h < H; ++h) {
            tmem_ld16(tb + c + 16 * (j + h), r0[h]);
            if constexpr (GATED) tmem_ld16(tb + BN / 2 + c + 16 * (j + h), r1[h]);
          }
          tmem_ld_wait();
          if (j + H == 2 && c + 32 * PER >= OUTW) release();
          if (!in) continue;
          if (tma) boxes_free();
          uint64_t v[8 * H];
          add16(bias0, wbias + j * 64, r0, v);
          if constexpr (SCALED) {
#pragma unroll
            for (int i = 0; i < 8 * H; ++i) v[i] = mul2(v[i], scale);
          }
          if (save) put16(own + SLOT, j, v);
          act_all<8 * H>(act, v);
          if constexpr (GATED) {
            uint64_t g[8 * H];
            add16(bias1, wbias + 128 + j * 64, r1, g);
            if (save) put16(own + 2 * SLOT, j, g);
#pragma unroll
            for (int i = 0; i < 8 * H; ++i) v[i] = mul2(v[i], g[i]);
          } else if (residual) {
#pragma unroll
            for (int i = 0; i < 2 * H; ++i) {
              const uint4 w = lds128(own + ((static_cast<uint32_t>(2 * j + i) ^ sw) << 4));
              const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int c4 = 0; c4 < 4; ++c4) {
                const float2 f = Elem<T>::unpack(x[c4]);
                v[4 * i + c4] = add2(v[4 * i + c4], f2pack(f.x, f.y));
              }
            }
          }
          put16(own, j, v);
        }
        if (!in) continue;
        if (tma) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (save) {
              store_box(&p.mp[0], box + SLOT, col, row);
              if constexpr (GATED) store_box(&p.mp[1], box + 2 * SLOT, col, row);
            }
            store_box(&p.mo, box, col, row);
            bulk_commit();
          }
          if (more) place(row, col + 32 * PER);
          continue;
        }
        if (save) {
          copy_out(box + SLOT, const_cast<void*>(p.pre[0].p), p.pre[0].ld, p.vec_pre, row, M, col, N);
          if (GATED) copy_out(box + 2 * SLOT, const_cast<void*>(p.pre[1].p), p.pre[1].ld, p.vec_pre, row, M, col, N);
        }
        const bool second = row >= p.row1;
        copy_out(box, const_cast<void*>(second ? p.out[1].p : p.out[0].p), second ? p.out[1].ld : p.out[0].ld, p.vec_out,
                 second ? row - p.row1 : row, second ? M - p.row1 : min(M, p.rows0), col, N);
        if (more) place(row, col + 32 * PER);
      }
    }
    if (tma && lane == 0) bulk_wait_all();
    if constexpr (CG == 1) {
      if (split > 1) {
        // All accumulators of the cluster are in shared memory. Units of 32 rows x 8 columns are
        // dealt to the cluster's epilogue warps; a unit's pieces are added in rank order.
        tile_at(worker, p.group, p.m_tiles, p.n_tiles, mt, nt);
        const int rows = M - mt * BM;
        const int qlog = rows > 64 ? 2 : rows > 32 ? 1 : 0;  // log2 of the quarters that may hold rows
        const int units = (OUTW / 8) << qlog;
        const int first = (e << p.split_log2) + crank;
        auto unit_bias = [&](const float* bias, int unit) {  // lane i < 8: column i
          const int c = nt * OUTW + (unit >> qlog) * 8 + lane;
          return bias && lane < 8 && unit < units && c < N ? bias[c] : 0.f;
        };
        float b0 = unit_bias(p.bias[0], first), b1 = GATED ? unit_bias(p.bias[1], first) : 0.f;
        cluster_sync();
        constexpr int FLY = 4;
        bool left = false;  // this warp has arrived for its last remote read
        if (ok) {
#pragma unroll 1
          for (int unit = first; unit < units; unit += EW << p.split_log2) {
            const int uq = unit & ((1 << qlog) - 1), c = (unit >> qlog) * 8;
            const int row = mt * BM + uq * 32 + lane, col = nt * OUTW + c;
            if (unit != first) {
              b0 = unit_bias(p.bias[0], unit);
              if (GATED) b1 = unit_bias(p.bias[1], unit);
            }
            const bool last = unit + (EW << p.split_log2) >= units;
            if (col >= N) continue;
            uint64_t v[4], g[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = g[i] = 0ull;
            const uint32_t at = smem + static_cast<uint32_t>((uq * (BN / 4) + c / 4) * 512 + lane * 16);
#pragma unroll 1
            for (int s0 = 0; s0 < split; s0 += FLY) {  // FLY CTAs' pieces in flight
              float4 x[FLY][2], y[FLY][2];
#pragma unroll
              for (int s = 0; s < FLY; ++s) {
                if (s0 + s >= split) continue;
                const uint32_t base = mapa_shared(at, s0 + s);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  x[s][i] = ld_cluster(base + i * 512);
                  if constexpr (GATED) y[s][i] = ld_cluster(base + (BN / 8 + i) * 512);
                }
              }
#pragma unroll
              for (int s = 0; s < FLY; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  if (s0 + s >= split) continue;
                  v[2 * i] = add2(v[2 * i], f2pack(x[s][i].x, x[s][i].y));
                  v[2 * i + 1] = add2(v[2 * i + 1], f2pack(x[s][i].z, x[s][i].w));
                  if constexpr (GATED) {
                    g[2 * i] = add2(g[2 * i], f2pack(y[s][i].x, y[s][i].y));
                    g[2 * i + 1] = add2(g[2 * i + 1], f2pack(y[s][i].z, y[s][i].w));
                  }
                }
            }
            if (last) {
              cluster_arrive();
              left = true;
            }
            if constexpr (SCALED) {
#pragma unroll
              for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], scale);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[i] = add2(v[i], f2pack(__shfl_sync(0xffffffffu, b0, 2 * i), __shfl_sync(0xffffffffu, b0, 2 * i + 1)));
              if constexpr (GATED)
                g[i] = add2(g[i], f2pack(__shfl_sync(0xffffffffu, b1, 2 * i), __shfl_sync(0xffffffffu, b1, 2 * i + 1)));
            }
            if (row < M) {
              if (save) store_row8<T>(p.pre[0], p.vec_pre, row, col, N, v);
              if (GATED && save) store_row8<T>(p.pre[1], p.vec_pre, row, col, N, g);
              act_all<4>(act, v);
              if constexpr (GATED) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], g[i]);
              } else if (residual) {
                const long long at_r = static_cast<long long>(row) * p.residual.ld + col;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float lo = col + 2 * i < N ? Elem<T>::load(p.residual.p, at_r + 2 * i) : 0.f;
                  const float hi = col + 2 * i + 1 < N ? Elem<T>::load(p.residual.p, at_r + 2 * i + 1) : 0.f;
                  v[i] = add2(v[i], f2pack(lo, hi));
                }
              }
              const int orow = row < p.row1 ? row : row - p.row1;
              if (row >= p.row1 || row < p.rows0)
                store_row8<T>(row < p.row1 ? p.out[0] : p.out[1], p.vec_out, orow, col, N, v);
            }
          }
        }
        if (!left) cluster_arrive();
      }
    }
  }

  // The epilogue warps end here: nothing below waits for their stores. What is left is to free
  // TMEM once they have read it, and to stay until no CTA of the cluster needs this one.
  if (warp >= 2) return;
  if constexpr (CG == 2) {
    cluster_sync();
  } else if (split > 1) {
    cluster_sync();  // meets the arrivals before the sums ...
    cluster_sync();  // ... and after them
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2)
      tmem_dealloc_pair(tmem_base, tmem_cols(BN));
    else
      tmem_dealloc(tmem_base, tmem_cols(BN));
  }
  if (p.early) grid_dep_wait();
}

// Adds the pieces of every tile of a stream-K product in order and writes the rounded result.
// Block: 32 rows x 32 columns of one tile; the pieces of a tile are consecutive workers'. Bound by the
// pieces' bytes, from L2 mostly, and by its launch: 10.8 us alone for 768 x 1152 (22 MB of pieces).
template <typename T>
__global__ void __launch_bounds__(256) pieces_kernel(const __grid_constant__ FfnTc p) {
  constexpr int CG = 2, BN = 256;
  __shared__ float box[32][33];
  grid_dep_launch();
  const int lane = threadIdx.x & 31, cg = threadIdx.x >> 5;
  const int chunk = blockIdx.x % (BN / 32), rq = (blockIdx.x / (BN / 32)) % (CG * 4), tile = blockIdx.x / (BN / 32 * CG * 4);
  int mt, nt;
  tile_at(tile, p.group, p.m_tiles, p.n_tiles, mt, nt);
  const int row = mt * CG * BM + rq * 32, col = nt * BN + chunk * 32;
  // the workers [w, end) of the tile's group whose shares meet its blocks [b0, b1)
  const int b0 = tile * p.kb, b1 = b0 + p.kb;
  int w = tile / p.sk_r * p.sk_q;
  while (Units::share_begin(p, w + 1) <= b0) ++w;
  int end = w + 1;
  while (end < p.workers && Units::share_begin(p, end) < b1) ++end;
  const float4* at = reinterpret_cast<const float4*>(p.partials) +
                     (((static_cast<size_t>(w) + tile) * CG + rq / 4) * 4 + rq % 4) * (BN / 4) * 32 + (chunk * 8 + cg) * 32 + lane;
  constexpr size_t PIECE = CG * 4 * (BN / 4) * 32;
  grid_dep_wait();
  if (row >= p.M || col >= p.N) return;
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  for (; w < end; w += 4, at += 4 * PIECE) {  // four pieces in flight
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = w + i < end ? at[i * PIECE] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t.x += x[i].x;
      t.y += x[i].y;
      t.z += x[i].z;
      t.w += x[i].w;
    }
  }
  if constexpr (std::is_same<T, __half>::value) {
    const float f = p.scale ? __ldcg(p.scale) : 1.f;
    t.x *= f, t.y *= f, t.z *= f, t.w *= f;
  }
  box[lane][cg * 4] = t.x;
  box[lane][cg * 4 + 1] = t.y;
  box[lane][cg * 4 + 2] = t.z;
  box[lane][cg * 4 + 3] = t.w;
  __syncthreads();
  int o = 0, orow = row, orows = min(p.M, p.rows0);
  if (row >= p.row1) {
    o = 1;
    orow = row - p.row1;
    orows = p.M - p.row1;
  }
  for (int r = cg; r < 32; r += 8)
    if (orow + r < orows && col + lane < p.N)
      Elem<T>::store(const_cast<void*>(p.out[o].p), static_cast<long long>(orow + r) * p.out[o].ld + col + lane, box[r][lane]);
}

template <typename T, int CG, int BN, int LAYOUT, bool GATED>
int launch_one(FfnTc& p, cudaStream_t stream) {
  constexpr int EW = epi_warps(CG, BN, LAYOUT, GATED);
  auto kern = tc_kernel<T, CG, BN, LAYOUT, GATED>;
  // no more stages than blocks a CTA will see: a small CTA can share the SM with the kernel before.
  // A cluster's CTAs leave their accumulators (BM x BN floats) over the stages.
  p.boxes = 1 + (p.pre[0].p ? (GATED ? 2 : 1) : 0);
  const uint32_t fixed = 1024 + EW * (p.boxes * SLOT + BIAS_BYTES) + BAR_BYTES;
  const uint32_t stage = (LAYOUT == FFN_TN ? BM : static_cast<uint32_t>(p.a_rows)) * BK * 2 + b_bytes(CG, BN);
  const int room = static_cast<int>((SMEM_MAX - fixed) / stage);
  const long long blocks = (static_cast<long long>(p.tiles) * p.kb + p.workers - 1) / p.workers;
  const long long mine = p.split > 1 ? (p.kb + p.split - 1) / p.split : blocks;
  p.stages = static_cast<int>(std::min<long long>(std::min(room, 8), std::max<long long>(mine, 2)));
  p.ring = std::max<uint32_t>(p.stages * stage, std::max<uint32_t>(p.split > 1 ? BM * BN * 4 : 0, A_BYTES + b_bytes(CG, BN)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(CG == 2 ? 2 * p.workers : p.workers * p.split));
  cfg.blockDim = dim3(32 * (2 + EW));
  // A CTA never waits for TMEM: two grids whose pairs or clusters held it on one SM and wanted it on
  // another would wait for each other. Whoever takes 128 of the 512 columns takes 46 KB at least, so
  // what fits an SM's 228 KB has at most four such parts (the other kernels here take more for theirs).
  constexpr uint32_t SHARE = tmem_cols(BN) / 128 * (46u << 10);
  cfg.dynamicSmemBytes = std::max(fixed + p.ring, SHARE);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG == 2 ? 2 : p.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 || p.split > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess || !p.stream_k) return static_cast<int>(e);
  return static_cast<int>(launch_kernel(pieces_kernel<T>, dim3(static_cast<unsigned>(p.tiles) * (256 / 32) * 8), dim3(256), 0,
                                        stream, p));
}

template <typename T, int LAYOUT, bool GATED>
int launch_cfg(int cfg, FfnTc& p, cudaStream_t stream) {
  switch (cfg) {
    case FFN_CG2_256: return launch_one<T, 2, 256, LAYOUT, GATED>(p, stream);
    case FFN_CG2_192:
      if constexpr (LAYOUT == FFN_NT && !GATED) return launch_one<T, 2, 192, LAYOUT, GATED>(p, stream);
      break;
    case FFN_CG1_128: return launch_one<T, 1, 128, LAYOUT, GATED>(p, stream);
    case FFN_CG1_64:
      if constexpr (!GATED) return launch_one<T, 1, 64, LAYOUT, GATED>(p, stream);
      break;
  }
  return static_cast<int>(cudaErrorInvalidValue);
}

// Loads the kernels of a layout on the current device, with their shared memory.
template <typename T, int CG, int BN, int LAYOUT, bool GATED>
cudaError_t load_one() {
  return cudaFuncSetAttribute(tc_kernel<T, CG, BN, LAYOUT, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
}
template <typename T, int LAYOUT, bool GATED>
cudaError_t load_cfg() {
  cudaError_t e = load_one<T, 2, 256, LAYOUT, GATED>();
  if (e == cudaSuccess) e = load_one<T, 1, 128, LAYOUT, GATED>();
  if constexpr (LAYOUT == FFN_NT && !GATED)
    if (e == cudaSuccess) e = load_one<T, 2, 192, LAYOUT, GATED>();
  if constexpr (!GATED)
    if (e == cudaSuccess) e = load_one<T, 1, 64, LAYOUT, GATED>();
  return e;
}
template <typename T>
cudaError_t load_tc() {
  cudaFuncAttributes a;
  cudaError_t e = cudaFuncGetAttributes(&a, pieces_kernel<T>);
  if (e == cudaSuccess) e = load_cfg<T, FFN_NT, true>();
  if (e == cudaSuccess) e = load_cfg<T, FFN_NT, false>();
  if (e == cudaSuccess) e = load_cfg<T, FFN_NN, false>();
  if (e == cudaSuccess) e = load_cfg<T, FFN_TN, false>();
  return e;
}

template <typename T>
int launch_tc(int cfg, int layout, int gated, FfnTc& p, cudaStream_t stream) {
  if (gated) return launch_cfg<T, FFN_NT, true>(cfg, p, stream);
  switch (layout) {
    case FFN_NT: return launch_cfg<T, FFN_NT, false>(cfg, p, stream);
    case FFN_NN: return launch_cfg<T, FFN_NN, false>(cfg, p, stream);
    default: return launch_cfg<T, FFN_TN, false>(cfg, p, stream);
  }
}

}  // namespace ffn

}  // namespace j1rt
