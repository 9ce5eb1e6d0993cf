// Matrix products of the feed-forward operators on tcgen05, with their epilogues.
//
//   out[M, N] = act(A . B + bias) (+ residual), A . B over one or two operand pairs
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
// Stream-K (CG = 2, weight gradients: few tiles, long contraction): every pair takes the same
//   number of 64-blocks of the tile-major list of all blocks; FP32 pieces go to the workspace
//   in the accumulator's own layout and a second kernel adds a tile's pieces in order.
//
// Roles per CTA: warp 0 TMA producer, warp 1 TMEM allocator and MMA issuer (even CTA), then the
// epilogue warps (eight: two per TMEM lane quarter, each on half of the tile's columns). GEN:
// operands whose rows do not start on 16-byte boundaries cannot be read by TMA; eight loader
// warps (and four epilogue warps) load aligned 16-byte pieces, shift them into place and store
// the boxes a TMA load would have written.
// Producer and issuer run as whole warps with one elected lane issuing: with a lane-dependent
// branch around the loop instead, an MMA step (four MMAs and a commit) took 600 cycles to issue.
// The accumulator is double buffered in TMEM, so a tile's epilogue runs under the next tile's
// products. The epilogue works on 32-column chunks, one thread per row: FP32 accumulators from
// TMEM, bias, activation, residual, one rounding, then through a swizzled 32 x 32 box in shared
// memory to coalesced 16-byte stores (element stores where rows are not 16-byte aligned).
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
constexpr int GW = 8;    // loader warps (GEN): each thread owns 4 units of A and 4 of B
__host__ __device__ constexpr int epi_warps(bool gen) { return gen ? 4 : 8; }
__host__ __device__ constexpr int threads_of(bool gen) { return 32 * (2 + epi_warps(gen) + (gen ? GW : 0)); }
constexpr uint32_t SLOT = 32 * 32 * 2;  // one 32 x 32 output box
constexpr uint32_t A_BYTES = BM * BK * 2;
constexpr uint32_t TAIL_BYTES = 8 * SLOT + 1024 /* bias */ + 256 /* barriers */;
constexpr uint32_t SMEM_MAX = 232448;

__host__ __device__ constexpr uint32_t b_bytes(int cg, int bn) { return static_cast<uint32_t>(bn / cg) * BK * 2; }
__host__ __device__ constexpr uint32_t stage_bytes(int cg, int bn) { return A_BYTES + b_bytes(cg, bn); }
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
// A bounded wait by a whole warp with one outcome.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int site) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, site));
}
// Arrivals whose writes the other CTA of the pair reads through its tensor core (GEN, CG 2).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t caddr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(caddr) : "memory");
}
__device__ __forceinline__ void fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }

template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  if constexpr (CG == 2)
    umma_bf16_pair(d, a, b, id, acc);
  else
    umma_bf16(d, a, b, id, acc);
}
// Arrive on `bar` of CTA `rank` of the pair (CG 1: of this CTA) when this thread's MMAs are done.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t rank) {
  if constexpr (CG == 2)
    umma_commit_pair(mapa_shared(smem_u32(bar), rank));
  else
    umma_commit(bar);
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
// the tile-major block list (stream-K), or its range of one tile (cluster split).
struct Units {
  int tile, k0, k1;
  long long pos, end;
};
__device__ __forceinline__ bool unit_ok(const FfnTc& p, const Units& u) {
  return p.stream_k ? u.pos < u.end : u.tile < p.tiles;
}
__device__ __forceinline__ void unit_set(const FfnTc& p, Units& u) {
  if (!p.stream_k) return;
  u.tile = static_cast<int>(u.pos / p.kb);
  u.k0 = static_cast<int>(u.pos - static_cast<long long>(u.tile) * p.kb);
  const long long left = u.end - u.pos;
  u.k1 = left < p.kb - u.k0 ? u.k0 + static_cast<int>(left) : p.kb;
}
__device__ __forceinline__ Units unit_first(const FfnTc& p, int worker, int rank) {
  Units u = {worker, 0, p.kb, 0, 0};
  if (p.stream_k) {
    const long long all = static_cast<long long>(p.tiles) * p.kb;
    u.pos = all * worker / p.workers;
    u.end = all * (worker + 1) / p.workers;
    if (u.pos < u.end) unit_set(p, u);
  } else if (p.split > 1) {
    u.k0 = static_cast<int>(static_cast<long long>(p.kb) * rank / p.split);
    u.k1 = static_cast<int>(static_cast<long long>(p.kb) * (rank + 1) / p.split);
  }
  return u;
}
__device__ __forceinline__ void unit_next(const FfnTc& p, Units& u) {
  if (p.stream_k) {
    u.pos += u.k1 - u.k0;
    if (u.pos < u.end) unit_set(p, u);
  } else {
    u.tile += p.workers;
  }
}
// Tiles are ordered in groups of `group` tile rows, rows fastest inside a group: the tiles in
// flight share few rows of A and few columns of B, so both stay in L2.
__host__ __device__ __forceinline__ void tile_at(int tile, int group, int m_tiles, int n_tiles, int& mt, int& nt) {
  const int per = group * n_tiles;
  const int first = tile / per * group;
  const int rows = m_tiles - first < group ? m_tiles - first : group;
  const int r = tile - tile / per * per;
  mt = first + r % rows;
  nt = r / rows;
}

// ---- GEN loads. A unit is 8 elements (16 bytes of a box row) from address `at`; `n` of them lie
// inside the matrix's row (n <= 0: none, all zero). The two aligned 16-byte pieces that hold it
// are loaded whole when they lie inside the matrix's memory [lo, hi), else the unit is loaded by
// elements (`slow`, only at the matrix's first and last bytes).
struct GenUnit {
  uint4 x, y;
};
__device__ __forceinline__ bool gen_load(GenUnit& g, const char* at, int n, const char* lo, const char* hi) {
  g.x = g.y = make_uint4(0u, 0u, 0u, 0u);
  if (n <= 0) return false;
  const uint32_t s = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at) & 15u);
  const char* c0 = at - s;
  if (c0 >= lo && c0 + (s ? 32 : 16) <= hi) {
    g.x = *reinterpret_cast<const uint4*>(c0);
    if (s) g.y = *reinterpret_cast<const uint4*>(c0 + 16);
    return false;
  }
  const uint16_t* e = reinterpret_cast<const uint16_t*>(at);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t l = 2 * i < n ? e[2 * i] : 0u, h = 2 * i + 1 < n ? e[2 * i + 1] : 0u;
    w[i] = l | (h << 16);
  }
  g.x = make_uint4(w[0], w[1], w[2], w[3]);
  return true;
}
// The unit's 16 bytes: the two pieces shifted by s bytes (even), elements past n zero.
__device__ __forceinline__ uint4 gen_shift(const GenUnit& g, uint32_t s, int n) {
  uint32_t w[8] = {g.x.x, g.x.y, g.x.z, g.x.w, g.y.x, g.y.y, g.y.z, g.y.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = (s & 8) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = (s & 4) ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (s & 2) * 8);
  if (n < 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (2 * i >= n) w[i] = 0u;
      else if (2 * i + 1 >= n) w[i] &= 0xffffu;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// One operand of a stage as this thread sees it: 4 units i = t + 256 j, j < 4, of 128 box rows x
// 8 units. K-major (MN false): box row = output index, units along the contraction, a step of 64
// moves 128 bytes along the row. MN-major: two chunks of 64 box rows; box row = contraction
// index, units along the output index, a step moves 64 rows. Either step keeps an address's
// offset from its 16-byte boundary, so the shift of a unit is fixed for a tile.
template <bool MN>
struct GenOperand {
  FfnMat m;
  int rows, cols, r0, c0;  // matrix extents and the tile's first row and column
  __device__ __forceinline__ void pos(int i, int k, long long& r, int& c) const {
    const int br = i >> 3, u = i & 7;
    if constexpr (MN) {
      r = k + (br & 63);
      c = c0 + (br >> 6) * 64 + u * 8;
    } else {
      r = static_cast<long long>(r0) + br;
      c = k + u * 8;
    }
  }
  __device__ __forceinline__ const char* at(long long r, int c) const {
    return static_cast<const char*>(m.p) + (r * m.ld + c) * 2;
  }
  __device__ __forceinline__ uint32_t load(GenUnit (&g)[4], int t, int k) const {
    const char* lo = static_cast<const char*>(m.p);
    const char* hi = lo + (static_cast<long long>(rows - 1) * m.ld + cols) * 2;
    uint32_t slow = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      long long r;
      int c;
      pos(t + j * GW * 32, k, r, c);
      if (gen_load(g[j], at(r, c), r < rows ? cols - c : 0, lo, hi)) slow |= 1u << j;
    }
    return slow;
  }
  // The first 64 box rows of this operand, the last 64 of `o` (units j < 2 and j >= 2).
  __device__ __forceinline__ uint32_t load2(GenUnit (&g)[4], int t, int k, const GenOperand& o) const {
    uint32_t slow = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const GenOperand& w = j < 2 ? *this : o;
      const char* lo = static_cast<const char*>(w.m.p);
      const char* hi = lo + (static_cast<long long>(rows - 1) * w.m.ld + cols) * 2;
      long long r;
      int c;
      w.pos(t + j * GW * 32, k, r, c);
      if (gen_load(g[j], w.at(r, c), r < rows ? cols - c : 0, lo, hi)) slow |= 1u << j;
    }
    return slow;
  }
  __device__ __forceinline__ void store2(const GenUnit (&g)[4], uint32_t slow, int t, int k, uint8_t* dst,
                                         const GenOperand& o) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const GenOperand& w = j < 2 ? *this : o;
      const int i = t + j * GW * 32, br = i >> 3, u = i & 7;
      long long r;
      int c;
      w.pos(i, k, r, c);
      const uint32_t s = (slow >> j) & 1 ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(w.at(r, c)) & 15u);
      *reinterpret_cast<uint4*>(dst + br * 128 + ((u ^ (br & 7)) << 4)) = gen_shift(g[j], s, cols - c);
    }
  }
  __device__ __forceinline__ void store(const GenUnit (&g)[4], uint32_t slow, int t, int k, uint8_t* dst) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = t + j * GW * 32, br = i >> 3, u = i & 7;
      long long r;
      int c;
      pos(i, k, r, c);
      const uint32_t s = (slow >> j) & 1 ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at(r, c)) & 15u);
      *reinterpret_cast<uint4*>(dst + br * 128 + ((u ^ (br & 7)) << 4)) = gen_shift(g[j], s, cols - c);
    }
  }
};

template <int ACT, int W>
__device__ __forceinline__ void act_all(float (&v)[W]) {
#pragma unroll
  for (int i = 0; i < W; i += 2) act_pair<ACT>(v[i], v[i + 1]);
}
template <int W>
__device__ __forceinline__ void act_all(int act, float (&v)[W]) {
  switch (act) {
    case J1_ACT_RELU: act_all<J1_ACT_RELU, W>(v); break;
    case J1_ACT_GELU: act_all<J1_ACT_GELU, W>(v); break;
    case J1_ACT_GELU_TANH: act_all<J1_ACT_GELU_TANH, W>(v); break;
    case J1_ACT_SILU: act_all<J1_ACT_SILU, W>(v); break;
    default: break;
  }
}

// 8 results of one row to m[row, col ...]: 16 bytes, or element by element up to column N.
template <typename T>
__device__ __forceinline__ void store_row8(const FfnMat& m, bool vec, long long row, int col, int N, const float (&v)[8]) {
  uint16_t* at = static_cast<uint16_t*>(const_cast<void*>(m.p)) + row * m.ld + col;
  const uint32_t w[4] = {Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]),
                         Elem<T>::pack(v[6], v[7])};
  if (vec) {
    *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < N) at[i] = static_cast<uint16_t>(w[i >> 1] >> ((i & 1) * 16));
  }
}

template <typename T, int CG, int BN, int LAYOUT, bool GATED, bool GEN>
__global__ void __launch_bounds__(threads_of(GEN), 1) tc_kernel(const __grid_constant__ FfnTc p) {
  constexpr bool A_MN = LAYOUT == FFN_TN, B_MN = LAYOUT != FFN_NT;
  constexpr int EW = epi_warps(GEN);
  constexpr int BROWS = BN / CG;             // output columns of B staged by one CTA
  constexpr int OUTW = GATED ? BN / 2 : BN;  // output columns of a tile
  constexpr uint32_t B_BYTES = b_bytes(CG, BN), STAGE = stage_bytes(CG, BN);
  static_assert(!(GATED && LAYOUT != FFN_NT) && !(GEN && BROWS != 128) && OUTW % 64 == 0, "");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + p.stages * A_BYTES;
  uint8_t* slots = smem + p.stages * STAGE;
  float* sbias = reinterpret_cast<float*>(slots + 8 * SLOT);
  uint64_t* full = reinterpret_cast<uint64_t*>(sbias + 8 * 32);
  uint64_t* empty = full + 8;
  uint64_t* tfull = empty + 8;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  grid_dep_launch();
  const int warp = __shfl_sync(0xffffffffu, warp_id(), 0), lane = lane_id();
  const int crank = CG == 2 || p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const uint32_t rank = CG == 2 ? static_cast<uint32_t>(crank) : 0u;
  const bool leader = rank == 0;
  const int worker = CG == 2 ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x) / p.split;
  const bool save = p.pre[0].p != nullptr;

  if (warp == 0 && elect_one()) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], GEN ? GW * CG : 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], EW * CG);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    if constexpr (!GEN) {
      tma_prefetch_desc(&p.ma[0]);
      tma_prefetch_desc(&p.mb[0]);
      if (GATED || p.segs > 1) tma_prefetch_desc(&p.mb[1]);
      if (p.segs > 1) tma_prefetch_desc(&p.ma[1]);
    }
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(tmem_slot, tmem_cols(BN));
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, tmem_cols(BN));
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (CG == 2)
    cluster_sync();  // barriers of both CTAs initialised, TMEM allocated in both
  else
    __syncthreads();
  tc_fence_after();
  grid_dep_wait();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if constexpr (!GEN) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t a_box = A_MN ? A_BYTES : static_cast<uint32_t>(p.a_rows) * BK * 2;
      for (Units u = unit_first(p, worker, crank); ok && unit_ok(p, u); unit_next(p, u)) {
        int mt, nt;
        tile_at(u.tile, p.group, p.m_tiles, p.n_tiles, mt, nt);
        const int m0 = (mt * CG + static_cast<int>(rank)) * BM;
        for (int kb = u.k0; kb < u.k1; ++kb) {
          ok = warp_wait(&empty[stage], phase ^ 1, abort_flag, p.err, 31);
          if (!ok) break;
          if (elect_one()) {
            if (leader) mbar_arrive_expect_tx(&full[stage], CG * (a_box + B_BYTES));
            const int seg = kb >= p.kb_seg ? 1 : 0;
            const int k = (kb - seg * p.kb_seg) * BK;
            uint8_t* da = sA + stage * A_BYTES;
            uint8_t* db = sB + stage * B_BYTES;
            const uint32_t fb = CG == 2 ? mapa_shared(smem_u32(&full[stage]), 0) : 0u;
            auto load = [&](const CUtensorMap* map, void* dst, int x, int y) {
              if constexpr (CG == 2)
                tma_load_2d_pair(map, fb, dst, x, y);
              else
                tma_load_2d(map, &full[stage], dst, x, y);
            };
            const CUtensorMap* ma = seg ? &p.ma[1] : &p.ma[0];
            const CUtensorMap* mb = seg ? &p.mb[1] : &p.mb[0];
            if constexpr (A_MN) {
              load(ma, da, m0, k);
              load(ma, da + A_BYTES / 2, m0 + 64, k);
            } else {
              load(ma, da, k, m0);
            }
            if constexpr (GATED) {  // the tile's columns: OUTW of B0, then OUTW of B1
              if constexpr (CG == 2) {
                load(rank ? &p.mb[1] : &p.mb[0], db, k, nt * OUTW);
              } else {
                load(&p.mb[0], db, k, nt * OUTW);
                load(&p.mb[1], db + B_BYTES / 2, k, nt * OUTW);
              }
            } else {
              const int n0 = nt * BN + static_cast<int>(rank) * BROWS;
              if constexpr (B_MN) {
#pragma unroll
                for (int c = 0; c < BROWS / 64; ++c) load(mb, db + c * 8192, n0 + c * 64, k);
              } else {
                load(mb, db, k, n0);
              }
            }
          }
          __syncwarp();
          if (++stage == p.stages) {
            stage = 0;
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
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA)
    if (leader) {
      constexpr uint32_t id = idesc<T>(BM * CG, BN, A_MN, B_MN);
      // descriptors of stage 0; a stage or a step of 16 contraction elements adds to the address
      // field (units of 16 bytes)
      const uint64_t a_desc = A_MN ? sdesc_sw128(smem_u32(sA), 8192, 1024) : sdesc_sw128(smem_u32(sA), 16, 1024);
      const uint64_t b_desc = B_MN ? sdesc_sw128(smem_u32(sB), 8192, 1024) : sdesc_sw128(smem_u32(sB), 16, 1024);
      constexpr uint32_t a_step = A_MN ? 2048 / 16 : 32 / 16, b_step = B_MN ? 2048 / 16 : 32 / 16;
      int stage = 0, acc = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (Units u = unit_first(p, worker, crank); ok && unit_ok(p, u); unit_next(p, u)) {
        const int buf = acc & 1;
        ok = warp_wait(&tempty[buf], ((acc >> 1) & 1) ^ 1, abort_flag, p.err, 32);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem_base + buf * BN;
        for (int kb = u.k0; kb < u.k1; ++kb) {
          ok = warp_wait(&full[stage], phase, abort_flag, p.err, 33);
          if (!ok) break;
          if constexpr (GEN && CG == 2) fence_cluster();
          tc_fence_after();
          if (elect_one()) {
            const uint64_t da = a_desc + static_cast<uint32_t>(stage) * (A_BYTES / 16);
            const uint64_t db = b_desc + static_cast<uint32_t>(stage) * (B_BYTES / 16);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              mma<CG>(d, da + k * a_step, db + k * b_step, id, (kb > u.k0 || k > 0) ? 1u : 0u);
            commit<CG>(&empty[stage], 0);
            if constexpr (CG == 2) commit<CG>(&empty[stage], 1);
            if (kb + 1 == u.k1) {
              commit<CG>(&tfull[buf], 0);
              if constexpr (CG == 2) commit<CG>(&tfull[buf], 1);
            }
          }
          __syncwarp();
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
        ++acc;
      }
      // All MMAs must have finished before TMEM is released.
      if (elect_one()) commit<CG>(drain, 0);
      __syncwarp();
      volatile int no_abort = 0;
      mbar_wait(drain, 0, &no_abort, nullptr, 0);
    }
  } else if (GEN && warp >= 2 + EW) {
    // ------------------------------------------------------------ loader warps (GEN)
    const int t = static_cast<int>(threadIdx.x) - 32 * (2 + EW);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    GenUnit ga[4], gb[4];
    for (Units u = unit_first(p, worker, crank); ok && unit_ok(p, u); unit_next(p, u)) {
      int mt, nt;
      tile_at(u.tile, p.group, p.m_tiles, p.n_tiles, mt, nt);
      const int m0 = (mt * CG + static_cast<int>(rank)) * BM;
      // operands of block kb; B of a single gated CTA is 64 rows of each weight
      auto seg_k = [&](int kb, int& seg) {
        seg = kb >= p.kb_seg ? 1 : 0;
        return (kb - seg * p.kb_seg) * BK;
      };
      auto op_a = [&](int seg) {
        return A_MN ? GenOperand<A_MN>{seg ? p.a[1] : p.a[0], p.K, p.M, 0, m0}
                    : GenOperand<A_MN>{seg ? p.a[1] : p.a[0], p.M, p.K, m0, 0};
      };
      auto op_b = [&](int seg) {
        if constexpr (GATED && CG == 2) return GenOperand<B_MN>{rank ? p.b[1] : p.b[0], p.N, p.K, nt * OUTW, 0};
        if constexpr (GATED && CG == 1)  // box rows 0..63 from B0, 64..127 from B1: units j < 2, j >= 2
          return GenOperand<B_MN>{seg ? p.b[1] : p.b[0], p.N, p.K, nt * OUTW - (seg ? 64 : 0), 0};
        const int n0 = nt * BN + static_cast<int>(rank) * BROWS;
        return B_MN ? GenOperand<B_MN>{seg ? p.b[1] : p.b[0], p.K, p.N, 0, n0}
                    : GenOperand<B_MN>{seg ? p.b[1] : p.b[0], p.N, p.K, n0, 0};
      };
      uint32_t slow_a = 0, slow_b = 0;
      auto load_a = [&](int kb) {
        int seg;
        const int k = seg_k(kb, seg);
        slow_a = op_a(seg).load(ga, t, k);
      };
      auto load_b = [&](int kb) {
        int seg;
        const int k = seg_k(kb, seg);
        if constexpr (GATED && CG == 1)
          slow_b = op_b(0).load2(gb, t, k, op_b(1));
        else
          slow_b = op_b(seg).load(gb, t, k);
      };
      load_a(u.k0);
      load_b(u.k0);
      for (int kb = u.k0; kb < u.k1; ++kb) {
        ok = warp_wait(&empty[stage], phase ^ 1, abort_flag, p.err, 34);
        if (!ok) break;
        int seg;
        const int k = seg_k(kb, seg);
        op_a(seg).store(ga, slow_a, t, k, sA + stage * A_BYTES);
        if (kb + 1 < u.k1) load_a(kb + 1);
        if constexpr (GATED && CG == 1)
          op_b(0).store2(gb, slow_b, t, k, sB + stage * B_BYTES, op_b(1));
        else
          op_b(seg).store(gb, slow_b, t, k, sB + stage * B_BYTES);
        if (kb + 1 < u.k1) load_b(kb + 1);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2)
            mbar_arrive_cluster(mapa_shared(smem_u32(&full[stage]), 0));
          else
            mbar_arrive(&full[stage]);
        }
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue warps
    const int e = warp - 2;
    const int q = warp & 3;              // TMEM lane quarter this warp may access
    constexpr int COLS = OUTW / (EW / 4);  // output columns of this warp
    const int c0 = (e >> 2) * COLS;
    uint8_t* box = slots + static_cast<uint32_t>(e) * SLOT;
    float* wbias = sbias + e * 32;
    const uint32_t sw = static_cast<uint32_t>((lane >> 1) & 3);
    // copying a box out (or in): rows br + 8 i, 16-byte unit bu
    const int br = lane >> 2, bu = lane & 3;
    uint4 rv[4];            // residual of the chunk to come
    float nb0 = 0.f, nb1 = 0.f;  // its biases, one column per lane

    // One box holds 32 rows x 32 columns, 64 bytes a row, unit u of row r at (u ^ (r >> 1 & 3)).
    auto put_row = [&](const float (&v)[32]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 w;
        w.x = Elem<T>::pack(v[8 * i], v[8 * i + 1]);
        w.y = Elem<T>::pack(v[8 * i + 2], v[8 * i + 3]);
        w.z = Elem<T>::pack(v[8 * i + 4], v[8 * i + 5]);
        w.w = Elem<T>::pack(v[8 * i + 6], v[8 * i + 7]);
        *reinterpret_cast<uint4*>(box + lane * 64 + ((static_cast<uint32_t>(i) ^ sw) << 4)) = w;
      }
    };
    // v through the box to rows [row, row + 32) below `rows`, columns [col, col + 32) of m.
    auto send = [&](const FfnMat& m, bool vec, int row, int rows, int col, const float (&v)[32]) {
      put_row(v);
      __syncwarp();
      if (vec) {
        uint16_t* at = static_cast<uint16_t*>(const_cast<void*>(m.p)) + static_cast<long long>(row + br) * m.ld + col + bu * 8;
        const bool in = col + bu * 8 < p.N;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = br + 8 * i;
          const uint4 w = *reinterpret_cast<const uint4*>(box + r * 64 + ((bu ^ ((r >> 1) & 3)) << 4));
          if (in && row + r < rows) *reinterpret_cast<uint4*>(at) = w;
          at += 8 * m.ld;
        }
      } else {
        const int c = col + lane, n = min(32, rows - row);
        uint16_t* at = static_cast<uint16_t*>(const_cast<void*>(m.p)) + static_cast<long long>(row) * m.ld + c;
        if (c < p.N) {
#pragma unroll 4
          for (int r = 0; r < n; ++r) {
            *at = *reinterpret_cast<const uint16_t*>(box + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
            at += m.ld;
          }
        }
      }
      __syncwarp();
    };
    auto fetch = [&](int row, int col) {  // what the chunk at (row, col) needs beside its accumulators
      nb0 = p.bias[0] && col + lane < p.N ? p.bias[0][col + lane] : 0.f;
      if constexpr (GATED) {
        nb1 = p.bias[1] && col + lane < p.N ? p.bias[1][col + lane] : 0.f;
      } else if (p.residual.p && p.vec_res) {
        const int c = col + bu * 8;
        const uint16_t* at = static_cast<const uint16_t*>(p.residual.p) + static_cast<long long>(row + br) * p.residual.ld + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          rv[i] = make_uint4(0u, 0u, 0u, 0u);
          if (row + br + 8 * i < p.M && c < p.N) rv[i] = *reinterpret_cast<const uint4*>(at);
          at += 8 * p.residual.ld;
        }
      }
    };
    auto add_bias = [&](float b, float (&v)[32]) {
      wbias[lane] = b;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 x = reinterpret_cast<const float4*>(wbias)[i];
        v[4 * i] += x.x;
        v[4 * i + 1] += x.y;
        v[4 * i + 2] += x.z;
        v[4 * i + 3] += x.w;
      }
      __syncwarp();
    };
    // Accumulators of 32 columns from `col`, row `row + lane` -> results.
    auto finish = [&](float (&v)[32], float (&g)[32], int row, int col) {
      if (p.bias[0]) add_bias(nb0, v);
      if (save) send(p.pre[0], p.vec_pre, row, p.M, col, v);
      act_all<32>(p.act, v);
      if constexpr (GATED) {
        if (p.bias[1]) add_bias(nb1, g);
        if (save) send(p.pre[1], p.vec_pre, row, p.M, col, g);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= g[i];
      } else if (p.residual.p) {
        if (p.vec_res) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = br + 8 * i;
            *reinterpret_cast<uint4*>(box + r * 64 + ((bu ^ ((r >> 1) & 3)) << 4)) = rv[i];
          }
        } else {
          const int c = col + lane, n = min(32, p.M - row);
          const uint16_t* at = static_cast<const uint16_t*>(p.residual.p) + static_cast<long long>(row) * p.residual.ld + c;
#pragma unroll 4
          for (int r = 0; r < n; ++r) {
            *reinterpret_cast<uint16_t*>(box + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2) =
                c < p.N ? *at : 0;
            at += p.residual.ld;
          }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 w = *reinterpret_cast<const uint4*>(box + lane * 64 + ((static_cast<uint32_t>(i) ^ sw) << 4));
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = Elem<T>::unpack(x[j]);
            v[8 * i + 2 * j] += f.x;
            v[8 * i + 2 * j + 1] += f.y;
          }
        }
        __syncwarp();
      }
      if (row < p.row1)
        send(p.out[0], p.vec_out, row, min(p.M, p.rows0), col, v);
      else
        send(p.out[1], p.vec_out, row - p.row1, p.M - p.row1, col, v);
    };

    int acc = 0;
    bool ok = true;
    for (Units u = unit_first(p, worker, crank); ok && unit_ok(p, u); unit_next(p, u), ++acc) {
      int mt, nt;
      tile_at(u.tile, p.group, p.m_tiles, p.n_tiles, mt, nt);
      const int row = (mt * CG + static_cast<int>(rank)) * BM + q * 32;  // this warp's first row
      const int n0 = nt * OUTW;
      const int buf = acc & 1;
      if (p.split == 1 && !p.stream_k && row < p.M && n0 + c0 < p.N) fetch(row, n0 + c0);
      ok = warp_wait(&tfull[buf], (acc >> 1) & 1, abort_flag, p.err, 35);
      if (!ok) break;
      tc_fence_after();
      const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BN;
      auto release = [&]() {  // the buffer has been read to the end
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2)
            mbar_arrive_remote(mapa_shared(smem_u32(&tempty[buf]), 0));
          else
            mbar_arrive(&tempty[buf]);
        }
      };
      if (p.split > 1 || p.stream_k) {
        // FP32 accumulators as they are, four columns of a row per 16 bytes, lanes side by side:
        // stream-K pieces to the workspace, a cluster's to shared memory (over the idle stages)
        float4* dst;
        if (p.stream_k) {
          const size_t piece = static_cast<size_t>(worker) + u.tile;  // unique and below workers + tiles
          dst = reinterpret_cast<float4*>(p.partials) + ((piece * CG + rank) * 4 + q) * (BN / 4) * 32;
        } else {
          dst = reinterpret_cast<float4*>(smem) + q * (BN / 4) * 32;
        }
        constexpr int ACC = BN / (EW / 4);  // accumulator columns of this warp
#pragma unroll 1
        for (int c = (e >> 2) * ACC; c < ((e >> 2) + 1) * ACC; c += 32) {
          uint32_t r[32];
          tmem_ld32(tb + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dst[(c / 4 + i) * 32 + lane] =
                make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]), __uint_as_float(r[4 * i + 2]),
                            __uint_as_float(r[4 * i + 3]));
        }
        release();
        continue;
      }
#pragma unroll 1
      for (int c = 0; c < COLS; c += 32) {
        uint32_t r0[32], r1[32];
        tmem_ld32(tb + c0 + c, r0);
        if constexpr (GATED) tmem_ld32(tb + BN / 2 + c0 + c, r1);
        tmem_ld_wait();
        if (c + 32 == COLS) release();
        if (row >= p.M || n0 + c0 + c >= p.N) continue;
        float v[32], g[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          v[i] = __uint_as_float(r0[i]);
          if constexpr (GATED) g[i] = __uint_as_float(r1[i]);
        }
        finish(v, g, row, n0 + c0 + c);
        if (c + 32 < COLS && n0 + c0 + c + 32 < p.N) fetch(row, n0 + c0 + c + 32);
      }
    }
    if constexpr (CG == 1) {
      if (p.split > 1) {
        // All accumulators of the cluster are in shared memory. Units of 32 rows x 8 columns are
        // dealt to the cluster's epilogue warps; a unit's pieces are added in rank order.
        cluster_sync();
        if (ok) {
          int mt, nt;
          tile_at(worker, p.group, p.m_tiles, p.n_tiles, mt, nt);
#pragma unroll 1
          for (int unit = e * p.split + crank; unit < 4 * (OUTW / 8); unit += EW * p.split) {
            const int uq = unit & 3, c = (unit >> 2) * 8;
            const int row = mt * BM + uq * 32 + lane, col = nt * OUTW + c;
            if (mt * BM + uq * 32 >= p.M || col >= p.N) continue;
            float v[8], g[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = g[i] = 0.f;
            const uint32_t at = static_cast<uint32_t>((uq * (BN / 4) + c / 4) * 512 + lane * 16);
#pragma unroll 4
            for (int s = 0; s < p.split; ++s) {
              const uint32_t base = mapa_shared(smem_u32(smem), s) + at;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float4 x = ld_cluster(base + i * 512);
                v[4 * i] += x.x;
                v[4 * i + 1] += x.y;
                v[4 * i + 2] += x.z;
                v[4 * i + 3] += x.w;
                if constexpr (GATED) {
                  const float4 y = ld_cluster(base + (BN / 8 + i) * 512);
                  g[4 * i] += y.x;
                  g[4 * i + 1] += y.y;
                  g[4 * i + 2] += y.z;
                  g[4 * i + 3] += y.w;
                }
              }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (p.bias[0] && col + i < p.N) v[i] += p.bias[0][col + i];
              if (GATED && p.bias[1] && col + i < p.N) g[i] += p.bias[1][col + i];
            }
            if (row < p.M) {
              if (save) store_row8<T>(p.pre[0], p.vec_pre, row, col, p.N, v);
              if (GATED && save) store_row8<T>(p.pre[1], p.vec_pre, row, col, p.N, g);
              act_all<8>(p.act, v);
              if constexpr (GATED) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= g[i];
              } else if (p.residual.p) {
                const long long at_r = static_cast<long long>(row) * p.residual.ld + col;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  if (col + i < p.N) v[i] += Elem<T>::load(p.residual.p, at_r + i);
              }
              const int orow = row < p.row1 ? row : row - p.row1;
              if (row >= p.row1 || row < p.rows0)
                store_row8<T>(row < p.row1 ? p.out[0] : p.out[1], p.vec_out, orow, col, p.N, v);
            }
          }
        }
      }
    }
  }
  if (CG == 1 && p.split > 1 && (warp < 2 || warp >= 2 + EW)) cluster_sync();  // meets the epilogue warps' one

  tc_fence_before();
  if (CG == 2 || p.split > 1)
    cluster_sync();  // every role of every CTA is done, the MMAs have drained
  else
    __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    if constexpr (CG == 2)
      tmem_dealloc_pair(tmem_base, tmem_cols(BN));
    else
      tmem_dealloc(tmem_base, tmem_cols(BN));
  }
}

// Adds the pieces of every tile of a stream-K product in order and writes the rounded result.
// Block: 32 rows x 32 columns of one tile; the pieces of a tile are consecutive workers'.
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
  grid_dep_wait();
  if (row >= p.M || col >= p.N) return;
  const long long all = static_cast<long long>(p.tiles) * p.kb, b0 = static_cast<long long>(tile) * p.kb, b1 = b0 + p.kb;
  // worker w holds blocks [all w / W, all (w + 1) / W): the one that holds block b0 first
  int w = static_cast<int>(b0 * p.workers / all);
  while (all * (w + 1) / p.workers <= b0) ++w;
  while (w > 0 && all * w / p.workers > b0) --w;
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  for (; w < p.workers && all * w / p.workers < b1; ++w) {
    if (all * (w + 1) / p.workers == all * w / p.workers) continue;
    const float4 x = reinterpret_cast<const float4*>(
        p.partials)[(((static_cast<size_t>(w) + tile) * CG + rq / 4) * 4 + rq % 4) * (BN / 4) * 32 + (chunk * 8 + cg) * 32 + lane];
    t.x += x.x;
    t.y += x.y;
    t.z += x.z;
    t.w += x.w;
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

template <typename T, int CG, int BN, int LAYOUT, bool GATED, bool GEN>
int launch_one(FfnTc& p, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured{0};
  auto kern = tc_kernel<T, CG, BN, LAYOUT, GATED, GEN>;
  cudaError_t e = set_smem_once(kern, SMEM_MAX, configured);
  if (e != cudaSuccess) return static_cast<int>(e);
  // no more stages than blocks a CTA will see: a small CTA can share the SM with the kernel before
  const uint32_t fixed = 1024 + TAIL_BYTES;
  const int room = static_cast<int>((SMEM_MAX - fixed) / stage_bytes(CG, BN));
  const long long blocks = (static_cast<long long>(p.tiles) * p.kb + p.workers - 1) / p.workers;
  const long long mine = p.split > 1 ? (p.kb + p.split - 1) / p.split : blocks;
  p.stages = static_cast<int>(std::min<long long>(std::min(room, 8), std::max<long long>(mine, p.split > 1 ? 4 : 2)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(CG == 2 ? 2 * p.workers : p.workers * p.split));
  cfg.blockDim = dim3(threads_of(GEN));
  cfg.dynamicSmemBytes = fixed + p.stages * stage_bytes(CG, BN);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG == 2 ? 2 : p.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 || p.split > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess || !p.stream_k) return static_cast<int>(e);
  return static_cast<int>(launch_kernel(pieces_kernel<T>, dim3(static_cast<unsigned>(p.tiles) * (256 / 32) * 8), dim3(256), 0,
                                        stream, p));
}

template <typename T, int LAYOUT, bool GATED>
int launch_cfg(int cfg, FfnTc& p, cudaStream_t stream) {
  switch (cfg) {
    case FFN_CG2_256: return launch_one<T, 2, 256, LAYOUT, GATED, false>(p, stream);
    case FFN_CG2_192:
      if constexpr (LAYOUT == FFN_NT && !GATED) return launch_one<T, 2, 192, LAYOUT, GATED, false>(p, stream);
      break;
    case FFN_CG1_128: return launch_one<T, 1, 128, LAYOUT, GATED, false>(p, stream);
    case FFN_CG1_64:
      if constexpr (!GATED) return launch_one<T, 1, 64, LAYOUT, GATED, false>(p, stream);
      break;
    case FFN_CG1_128_GEN: return launch_one<T, 1, 128, LAYOUT, GATED, true>(p, stream);
    case FFN_CG2_256_GEN: return launch_one<T, 2, 256, LAYOUT, GATED, true>(p, stream);
  }
  return static_cast<int>(cudaErrorInvalidValue);
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
