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
// Roles per CTA: warp 0 TMA producer, warp 1 TMEM allocator and MMA issuer (even CTA), warps
// 2..9 epilogue (two per TMEM lane quarter, each on half of the tile's columns). GEN: operands
// whose rows do not start on 16-byte boundaries cannot be read by TMA; six more warps load
// aligned 16-byte pieces, shift them into place and store the same swizzled boxes.
// The accumulator is double buffered in TMEM, so a tile's epilogue runs under the next tile's
// products. The epilogue works on 32-column chunks, one thread per row: FP32 accumulators from
// TMEM, bias, activation, residual, one rounding, then through a 64B-swizzled 32 x 32 box in
// shared memory by TMA store (or element stores where rows are not 16-byte aligned); nothing
// couples the warps.
#pragma once
#include <cuda_runtime.h>

#include <type_traits>

#include "ffn_math.cuh"
#include "ffn_tc.h"
#include "kernels.h"
#include "ptx.cuh"

namespace j1rt {

namespace ffn {

constexpr int BM = 128;  // rows of a tile per CTA
constexpr int BK = 64;   // contraction elements per stage
constexpr int EW = 8;    // epilogue warps
constexpr int GW = 6;    // loader warps (GEN): 16 warps in all leave 128 registers a thread
constexpr uint32_t SLOT = 32 * 32 * 2;  // one 32 x 32 output box
constexpr uint32_t A_BYTES = BM * BK * 2;
constexpr uint32_t TAIL_BYTES = 1024 /* bias */ + 256 /* barriers */;
constexpr uint32_t SMEM_MAX = 232448;

__host__ __device__ constexpr uint32_t b_bytes(int cg, int bn) { return static_cast<uint32_t>(bn / cg) * BK * 2; }
__host__ __device__ constexpr uint32_t stage_bytes(int cg, int bn) { return A_BYTES + b_bytes(cg, bn); }
// Output boxes per epilogue warp: two for the output, two per stored pre-activation.
__host__ __device__ constexpr uint32_t slot_bytes(bool gated, bool pre) {
  return EW * SLOT * (2 + (pre ? (gated ? 4 : 2) : 0));
}
__host__ __device__ constexpr uint32_t tmem_cols(int bn) { return bn > 128 ? 512 : bn > 64 ? 256 : 128; }

// kind::f16 instruction descriptor (ptx.cuh idesc_bf16) with the element type as a parameter.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int m, int n, bool a_mn, bool b_mn) {
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;  // 0 f16, 1 bf16
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

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

// ---- GEN loads: one 16-byte unit (8 elements) of row `row` from column `col` of a matrix of
// rows x cols, elements outside 0. Aligned 16-byte pieces that lie inside the matrix's memory
// are loaded whole and shifted together; the few others element by element.
__device__ __forceinline__ uint4 gen_unit(const FfnMat& m, long long row, int col, int rows, int cols, const char* lo,
                                          const char* hi) {
  if (row >= rows || col >= cols) return make_uint4(0u, 0u, 0u, 0u);
  const char* at = static_cast<const char*>(m.p) + (row * m.ld + col) * 2;
  const uint32_t s = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at) & 15u);
  const char* c0 = at - s;
  const int n = cols - col;  // elements of the unit inside the row
  uint32_t w[8];
  if (c0 >= lo && c0 + (s ? 32 : 16) <= hi) {
    const uint4 x = *reinterpret_cast<const uint4*>(c0);
    uint4 y = make_uint4(0u, 0u, 0u, 0u);
    if (s) y = *reinterpret_cast<const uint4*>(c0 + 16);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w, w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
    if (s & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (s & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (s & 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
    if (n < 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (2 * i >= n) w[i] = 0u;
        else if (2 * i + 1 >= n) w[i] &= 0xffffu;
      }
    }
  } else {
    const uint16_t* e = reinterpret_cast<const uint16_t*>(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t l = 2 * i < n ? e[2 * i] : 0u, h = 2 * i + 1 < n ? e[2 * i + 1] : 0u;
      w[i] = l | (h << 16);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// A box of `nrows` rows x 64 elements at (row0, col0) into shared memory as a 128B-swizzled TMA
// load would write it, by GW warps: unit u of row r at r * 128 + ((u ^ (r & 7)) << 4).
__device__ __forceinline__ void gen_box(const FfnMat& m, int rows, int cols, int row0, int col0, int nrows, uint8_t* dst,
                                        int t) {
  const char* lo = static_cast<const char*>(m.p);
  const char* hi = lo + (static_cast<long long>(rows - 1) * m.ld + cols) * 2;
#pragma unroll 4
  for (int i = t; i < nrows * 8; i += GW * 32) {
    const int r = i >> 3, u = i & 7;
    const uint4 v = gen_unit(m, static_cast<long long>(row0) + r, col0 + u * 8, rows, cols, lo, hi);
    *reinterpret_cast<uint4*>(dst + r * 128 + ((u ^ (r & 7)) << 4)) = v;
  }
}

template <int ACT>
__device__ __forceinline__ void act32(float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = act_value<ACT>(v[i]);
}
__device__ __forceinline__ void act32(int act, float (&v)[32]) {
  switch (act) {
    case J1_ACT_RELU: act32<J1_ACT_RELU>(v); break;
    case J1_ACT_GELU: act32<J1_ACT_GELU>(v); break;
    case J1_ACT_GELU_TANH: act32<J1_ACT_GELU_TANH>(v); break;
    case J1_ACT_SILU: act32<J1_ACT_SILU>(v); break;
    default: break;
  }
}

template <typename T, int CG, int BN, int LAYOUT, bool GATED, bool GEN>
__global__ void __launch_bounds__(32 * (2 + EW + (GEN ? GW : 0)), 1) tc_kernel(const __grid_constant__ FfnTc p) {
  constexpr bool A_MN = LAYOUT == FFN_TN, B_MN = LAYOUT != FFN_NT;
  constexpr int BROWS = BN / CG;                // output columns of B staged by one CTA
  constexpr int OUTW = GATED ? BN / 2 : BN;     // output columns of a tile
  constexpr uint32_t B_BYTES = b_bytes(CG, BN), STAGE = stage_bytes(CG, BN);
  static_assert(!(GATED && LAYOUT != FFN_NT) && !(GEN && CG != 1) && OUTW % 64 == 0, "");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + p.stages * A_BYTES;
  uint8_t* slots = smem + p.stages * STAGE;
  const bool save = p.pre[0].p != nullptr;
  float* sbias = reinterpret_cast<float*>(slots + slot_bytes(GATED, save));
  uint64_t* full = reinterpret_cast<uint64_t*>(sbias + EW * 32);
  uint64_t* empty = full + 8;
  uint64_t* tfull = empty + 8;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  grid_dep_launch();
  const int warp = warp_id(), lane = lane_id();
  const bool clustered = CG == 2 || p.split > 1;
  const int crank = clustered ? static_cast<int>(cluster_ctarank()) : 0;
  const uint32_t rank = CG == 2 ? static_cast<uint32_t>(crank) : 0u;
  const bool leader = rank == 0;
  const int worker = CG == 2 ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x) / p.split;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], GEN ? GW : 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], EW * CG);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
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
  if (clustered)
    cluster_sync();
  else
    __syncthreads();
  tc_fence_after();
  grid_dep_wait();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (!GEN && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t a_box = A_MN ? A_BYTES : static_cast<uint32_t>(p.a_rows) * BK * 2;
      for (Units u = unit_first(p, worker, crank); ok && unit_ok(p, u); unit_next(p, u)) {
        int mt, nt;
        tile_at(u.tile, p.group, p.m_tiles, p.n_tiles, mt, nt);
        const int m0 = (mt * CG + static_cast<int>(rank)) * BM;
        for (int kb = u.k0; kb < u.k1; ++kb) {
          if (!mbar_wait<true>(&empty[stage], phase ^ 1, abort_flag, p.err, 31)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(&full[stage], CG * (a_box + B_BYTES));
          const int seg = kb >= p.kb_seg ? 1 : 0;
          const int k = (kb - seg * p.kb_seg) * BK;
          uint8_t* da = sA + stage * A_BYTES;
          uint8_t* db = sB + stage * B_BYTES;
          auto load = [&](const CUtensorMap* map, void* dst, int x, int y) {
            if constexpr (CG == 2)
              tma_load_2d_pair(map, mapa_shared(smem_u32(&full[stage]), 0), dst, x, y);
            else
              tma_load_2d(map, &full[stage], dst, x, y);
          };
          if constexpr (A_MN) {
            load(&p.ma[seg], da, m0, k);
            load(&p.ma[seg], da + A_BYTES / 2, m0 + 64, k);
          } else {
            load(&p.ma[seg], da, k, m0);
          }
          if constexpr (GATED) {  // the tile's columns: OUTW of B0, then OUTW of B1
            if constexpr (CG == 2) {
              load(&p.mb[rank], db, k, nt * OUTW);
            } else {
              load(&p.mb[0], db, k, nt * OUTW);
              load(&p.mb[1], db + B_BYTES / 2, k, nt * OUTW);
            }
          } else {
            const int n0 = nt * BN + static_cast<int>(rank) * BROWS;
            if constexpr (B_MN) {
#pragma unroll
              for (int c = 0; c < BROWS / 64; ++c) load(&p.mb[seg], db + c * 8192, n0 + c * 64, k);
            } else {
              load(&p.mb[seg], db, k, n0);
            }
          }
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
    if (leader && lane == 0) {
      constexpr uint32_t id = idesc<T>(BM * CG, BN, A_MN, B_MN);
      int stage = 0, acc = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (Units u = unit_first(p, worker, crank); ok && unit_ok(p, u); unit_next(p, u)) {
        const int buf = acc & 1;
        if (!mbar_wait<true>(&tempty[buf], ((acc >> 1) & 1) ^ 1, abort_flag, p.err, 32)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + buf * BN;
        for (int kb = u.k0; kb < u.k1; ++kb) {
          if (!mbar_wait<true>(&full[stage], phase, abort_flag, p.err, 33)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + stage * A_BYTES), b0 = smem_u32(sB + stage * B_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t da = A_MN ? sdesc_sw128(a0 + k * 2048, 8192, 1024) : sdesc_sw128(a0 + k * 32, 16, 1024);
            const uint64_t db = B_MN ? sdesc_sw128(b0 + k * 2048, 8192, 1024) : sdesc_sw128(b0 + k * 32, 16, 1024);
            mma<CG>(d, da, db, id, (kb > u.k0 || k > 0) ? 1u : 0u);
          }
          commit<CG>(&empty[stage], 0);
          if constexpr (CG == 2) commit<CG>(&empty[stage], 1);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        commit<CG>(&tfull[buf], 0);
        if constexpr (CG == 2) commit<CG>(&tfull[buf], 1);
        ++acc;
      }
      // All MMAs must have finished before TMEM is released.
      commit<CG>(drain, 0);
      volatile int no_abort = 0;
      mbar_wait<true>(drain, 0, &no_abort, nullptr, 0);
    }
  } else if (GEN && warp >= 2 + EW) {
    // ------------------------------------------------------------ loader warps (GEN)
    const int t = static_cast<int>(threadIdx.x) - 32 * (2 + EW);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (Units u = unit_first(p, worker, crank); ok && unit_ok(p, u); unit_next(p, u)) {
      int mt, nt;
      tile_at(u.tile, p.group, p.m_tiles, p.n_tiles, mt, nt);
      const int m0 = mt * BM;
      for (int kb = u.k0; kb < u.k1; ++kb) {
        // one outcome per warp: the warp meets at __syncwarp below
        ok = __all_sync(0xffffffffu, mbar_wait<true>(&empty[stage], phase ^ 1, abort_flag, p.err, 34));
        if (!ok) break;
        const int seg = kb >= p.kb_seg ? 1 : 0;
        const int k = (kb - seg * p.kb_seg) * BK;
        uint8_t* da = sA + stage * A_BYTES;
        uint8_t* db = sB + stage * B_BYTES;
        if constexpr (A_MN) {
          gen_box(p.a[seg], p.K, p.M, k, m0, 64, da, t);
          gen_box(p.a[seg], p.K, p.M, k, m0 + 64, 64, da + A_BYTES / 2, t);
        } else {
          gen_box(p.a[seg], p.M, p.K, m0, k, p.a_rows, da, t);
        }
        if constexpr (GATED) {
          gen_box(p.b[0], p.N, p.K, nt * OUTW, k, OUTW, db, t);
          gen_box(p.b[1], p.N, p.K, nt * OUTW, k, OUTW, db + B_BYTES / 2, t);
        } else if constexpr (B_MN) {
#pragma unroll
          for (int c = 0; c < BROWS / 64; ++c) gen_box(p.b[seg], p.K, p.N, k, nt * BN + c * 64, 64, db + c * 8192, t);
        } else {
          gen_box(p.b[seg], p.N, p.K, nt * BN, k, BROWS, db, t);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[stage]);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..9)
    const int e = warp - 2;
    const int q = warp & 3;        // TMEM lane quarter this warp may access
    const int half = e >> 2;       // half of the tile's columns
    uint8_t* slot0 = slots + static_cast<uint32_t>(e) * SLOT;  // box b of this warp: slot0 + b * EW * SLOT
    float* wbias = sbias + e * 32;
    const uint32_t sw = static_cast<uint32_t>((lane >> 1) & 3);
    uint32_t nbox = 0;  // chunks written so far
    uint4 rv[4];        // residual of the chunk to come: rows (lane >> 2) + 8 i, unit lane & 3

    // One box holds 32 rows x 32 columns, 64 bytes a row, unit u of row r at (u ^ (r >> 1 & 3)).
    auto put_row = [&](uint8_t* box, const float (&v)[32]) {
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
    // The box to rows [row, ..) x columns [col, ..) of m: TMA clips at the matrix's edge.
    auto send = [&](const CUtensorMap* map, const FfnMat& m, bool tma, uint8_t* box, int row, int rows, int col) {
      if (tma) {
        if (lane == 0) tma_store_2d(map, box, col, row);
      } else {
        const int c = col + lane;
        if (c < p.N) {
          uint16_t* base = static_cast<uint16_t*>(const_cast<void*>(m.p)) + c;
          const int n = min(32, rows - row);
          for (int r = 0; r < n; ++r)
            base[static_cast<long long>(row + r) * m.ld] = *reinterpret_cast<const uint16_t*>(
                box + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
        }
      }
    };
    auto fetch_residual = [&](int row, int col) {
      if (!p.residual.p || !p.vec_res) return;
      const int c = col + (lane & 3) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = row + (lane >> 2) + 8 * i;
        rv[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < p.M && c < p.N)
          rv[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.residual.p) +
                                                  static_cast<long long>(r) * p.residual.ld + c);
      }
    };
    auto add_bias = [&](const float* bias, int col, float (&v)[32]) {
      if (!bias) return;
      __syncwarp();
      wbias[lane] = col + lane < p.N ? bias[col + lane] : 0.f;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 b = reinterpret_cast<const float4*>(wbias)[i];
        v[4 * i] += b.x;
        v[4 * i + 1] += b.y;
        v[4 * i + 2] += b.z;
        v[4 * i + 3] += b.w;
      }
    };
    // Accumulators of 32 columns from `col`, row `row + lane` -> results.
    auto finish = [&](float (&v)[32], float (&g)[32], int row, int col) {
      if (lane == 0) bulk_wait_read_1();  // the boxes written two chunks ago have left
      __syncwarp();
      uint8_t* box = slot0 + (nbox & 1) * (EW * SLOT);
      if constexpr (!GATED) {
        if (p.residual.p) {
          if (p.vec_res) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = (lane >> 2) + 8 * i;
              *reinterpret_cast<uint4*>(box + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4)) = rv[i];
            }
          } else {
            const int c = col + lane, n = min(32, p.M - row);
            const uint16_t* base = static_cast<const uint16_t*>(p.residual.p) + c;
            for (int r = 0; r < n; ++r)
              *reinterpret_cast<uint16_t*>(box + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2) =
                  c < p.N ? base[static_cast<long long>(row + r) * p.residual.ld] : 0;
          }
        }
      }
      add_bias(p.bias[0], col, v);
      if (save) put_row(box + 2 * EW * SLOT, v);
      act32(p.act, v);
      if constexpr (GATED) {
        add_bias(p.bias[1], col, g);
        if (save) put_row(box + 4 * EW * SLOT, g);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= g[i];
      } else if (p.residual.p) {
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
      }
      put_row(box, v);
      fence_proxy_async_smem();
      __syncwarp();
      int o = 0, orow = row, orows = min(p.M, p.rows0);
      if (row >= p.row1) {
        o = 1;
        orow = row - p.row1;
        orows = p.M - p.row1;
      }
      if (orow < orows) {
        send(&p.mout[o], p.out[o], p.tma_out, box, orow, orows, col);
        if (save) send(&p.mpre[0], p.pre[0], p.tma_pre, box + 2 * EW * SLOT, row, p.M, col);
        if (GATED && save) send(&p.mpre[1], p.pre[1], p.tma_pre, box + 4 * EW * SLOT, row, p.M, col);
      }
      if (lane == 0) bulk_commit();
      __syncwarp();
      ++nbox;
    };

    int acc = 0;
    bool ok = true;
    for (Units u = unit_first(p, worker, crank); ok && unit_ok(p, u); unit_next(p, u), ++acc) {
      int mt, nt;
      tile_at(u.tile, p.group, p.m_tiles, p.n_tiles, mt, nt);
      const int row = (mt * CG + static_cast<int>(rank)) * BM + q * 32;  // this warp's first row
      const int c0 = half * (OUTW / 2), cols = OUTW / 2;
      const int n0 = nt * OUTW;
      const int buf = acc & 1;
      if (p.split == 1 && !p.stream_k && row < p.M && n0 + c0 < p.N) fetch_residual(row, n0 + c0);
      ok = __all_sync(0xffffffffu, mbar_wait<true>(&tfull[buf], (acc >> 1) & 1, abort_flag, p.err, 35));
      if (!ok) break;
      tc_fence_after();
      const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BN;
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
#pragma unroll 1
        for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
          uint32_t r[32];
          tmem_ld32(tb + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dst[(c / 4 + i) * 32 + lane] =
                make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]), __uint_as_float(r[4 * i + 2]),
                            __uint_as_float(r[4 * i + 3]));
        }
        if (p.split > 1) break;  // one tile per cluster
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&tempty[buf]), 0));
        continue;
      }
#pragma unroll 1
      for (int c = 0; c < cols; c += 32) {
        uint32_t r0[32], r1[32];
        tmem_ld32(tb + c0 + c, r0);
        if constexpr (GATED) tmem_ld32(tb + BN / 2 + c0 + c, r1);
        tmem_ld_wait();
        if (c + 32 == cols) {  // read to the end: hand the buffer back
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2)
              mbar_arrive_remote(mapa_shared(smem_u32(&tempty[buf]), 0));
            else
              mbar_arrive(&tempty[buf]);
          }
        }
        if (row >= p.M || n0 + c0 + c >= p.N) continue;
        float v[32], g[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          v[i] = __uint_as_float(r0[i]);
          if constexpr (GATED) g[i] = __uint_as_float(r1[i]);
        }
        finish(v, g, row, n0 + c0 + c);
        if (c + 32 < cols && n0 + c0 + c + 32 < p.N) fetch_residual(row, n0 + c0 + c + 32);
      }
    }
    if (p.split > 1) {
      // all accumulators of the cluster are in shared memory; unit = (row quarter, 32 columns),
      // dealt to the CTAs in turn, one warp each; added in rank order
      cluster_sync();
      constexpr int CH = OUTW / 32;
      const int unit = e * p.split + crank;
      if (ok && unit < 4 * CH) {
        int mt, nt;
        tile_at(worker, p.group, p.m_tiles, p.n_tiles, mt, nt);
        const int uq = unit / CH, c = (unit % CH) * 32;
        const int row = mt * BM + uq * 32, col = nt * OUTW + c;
        if (row < p.M && col < p.N) {
          fetch_residual(row, col);
          float v[32], g[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = g[i] = 0.f;
          for (int s = 0; s < p.split; ++s) {
            const uint32_t base = mapa_shared(smem_u32(smem), s) + static_cast<uint32_t>((uq * (BN / 4) * 32 + lane) * 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 x = ld_cluster(base + (c / 4 + i) * 512);
              v[4 * i] += x.x;
              v[4 * i + 1] += x.y;
              v[4 * i + 2] += x.z;
              v[4 * i + 3] += x.w;
              if constexpr (GATED) {
                const float4 y = ld_cluster(base + (BN / 8 + c / 4 + i) * 512);
                g[4 * i] += y.x;
                g[4 * i + 1] += y.y;
                g[4 * i + 2] += y.z;
                g[4 * i + 3] += y.w;
              }
            }
          }
          finish(v, g, row, col);
        }
      }
    }
    if (lane == 0) bulk_wait_all();  // no store of ours may still read smem at exit
  }
  if (p.split > 1 && (warp < 2 || warp >= 2 + EW)) cluster_sync();  // meets the epilogue warps' one

  tc_fence_before();
  if (clustered)
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
  const uint32_t fixed = 1024 + slot_bytes(GATED, p.pre[0].p != nullptr) + TAIL_BYTES;
  int stages = static_cast<int>((SMEM_MAX - fixed) / stage_bytes(CG, BN));
  p.stages = stages > 8 ? 8 : stages;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(CG == 2 ? 2 * p.workers : p.workers * p.split));
  cfg.blockDim = dim3(32 * (2 + EW + (GEN ? GW : 0)));
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
