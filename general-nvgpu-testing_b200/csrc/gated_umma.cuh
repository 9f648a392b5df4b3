// The gated product of a feed-forward block as one kernel:
//
//   G = A Bg^T,  U = A Bu^T,  C = act(G) * U        A [M, K], Bg and Bu [F, K], C [M, F], fp16 or bf16
//
// A tile is 128 kCta rows by `width` columns of BOTH products.  The two weights enter one UMMA as the halves of its
// N = 2 * width rows of B: on a CTA pair (kCta = 2) the leader CTA loads `width` rows of Bg and its peer the same rows
// of Bu, which is how a cta_group::2 UMMA splits B anyway; a single CTA loads both boxes one behind the other.  So the
// main loop is that of the plain rc GEMM (gemmrc_umma.cuh) with nothing added, A is read once for both products, and
// column j of G and of U stand in TMEM columns j and width + j of the same lane: the epilogue multiplies them in
// registers and G and U never leave the SM, unless the caller wants them kept for the backward pass.  The products are
// accumulated and combined in fp32 and rounded once to the output type (three times, independently, when kept).
//
// Two variants, chosen by rows (the rule and what it measured stand beside gated_plan() in feedforward_launch.cu):
//   kCta = 2   M > 128: 256-row tiles, width 32, 64, 96 or 128, persistent grid, two TMEM accumulators, C stored by TMA.
//              4096 x 16384 x 4096 (bf16): 670 us, 1640 TFLOP/s, what cuBLAS takes for the two products alone (690 us); bound
//              by the tensor pipe (94 % active), in long runs by the power it draws (1441 TFLOP/s sustained).
//   kCta = 1   M <= 128: the call is bound by reading the weights once.  The width is whatever multiple of 8 deals F
//              to all SMs in one wave, so that every SM streams the same share of the weights through a ring of up to 16
//              stages; only the rows of A that exist are loaded.  C is small and written straight from registers.
//              One row, F = 16384, K = 4096: 44.5 us, 6.0 TB/s.  Halving the ring, so that the next launch's CTAs fit
//              beside this one's, was slower for all shapes (8192 x 4096: 25.8 -> 27.8 us).
//
// Roles: warps 0 and 6 are TMA producers, warps 1 and 7 issue UMMAs, warps 2..5 are the epilogue.
#pragma once

#include "activation.cuh"
#include "umma_common.cuh"

namespace beam {

struct GatedParams {
  CUtensorMap tm_a;       // A [M, K], box (rows per CTA) x 64, 128 B swizzle
  CUtensorMap tm_gate;    // Bg [F, K], box width x 64
  CUtensorMap tm_up;      // Bu [F, K]
  CUtensorMap tm_out[3];  // pair variant: C, G, U [M, F], store box 32 rows x 32 columns, 64 B swizzle
  void* out[3];           // C, G, U; G and U are null when they are not kept
  int m, f, k;
  int width;              // columns of F per tile
  int a_rows;             // rows of A that a CTA loads
  int stages, stage_bytes;
  int a_bytes;            // of a stage: B begins there
  int bar_offset;         // the barriers' place in shared memory, behind the ring and what else takes its place
  int m_tiles, n_tiles, group_m;
  int issuers;            // warps that issue UMMAs: 1, or 2 with an accumulator each, taking turns at the k-blocks
  int split;              // single CTAs: a cluster of this many CTAs shares each tile's contraction
  int act;
  int bf16;
  int* status;
};

constexpr int kGatedChainCols = 128;  // TMEM columns from the first issuer's accumulator to the second's

template <int kCta>
struct GatedShape {
  static constexpr int kBM = 128;
  static constexpr int kBK = 64;
  static constexpr int kABytes = kBM * kBK * 2;
  static constexpr int kMaxStages = 16;
  static constexpr int kProducers = 2;  // at most the least depth of the ring
  static constexpr int kSecondIssuer = 5 + kProducers;  // its warp
  static constexpr int kThreads = 32 * (6 + kProducers);
  static constexpr int kAccCols = 256;    // TMEM columns from one tile's accumulator to the next tile's
  static constexpr int kBufsPerWarp = 4;
  static constexpr int kStoreBufBytes = 32 * 64;
  static constexpr int kStagingBytes = kCta == 2 ? 4 * kBufsPerWarp * kStoreBufBytes : 0;
  static constexpr int kBarBytes = 512;
  static constexpr int kSmemLimit = 232448;
  static constexpr int kRingBytes = kSmemLimit - 1024 - kStagingBytes - kBarBytes;
  static_assert((2 * kMaxStages + 4) * 8 + 8 <= kBarBytes, "barrier block too small");
};

// g = act(g) * u in the first `columns` of 32 columns, a multiple of 8 (warp-uniform: a narrow tile has few).
template <int kAct>
__device__ __forceinline__ void gated_combine(uint32_t (&g)[32], const uint32_t (&u)[32], int columns) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    if (i < columns) {
#pragma unroll
      for (int q = i; q < i + 8; ++q)
        g[q] = __float_as_uint(act_value<kAct>(__uint_as_float(g[q])) * __uint_as_float(u[q]));
    }
  }
}
__device__ __forceinline__ void gated_combine(int act, uint32_t (&g)[32], const uint32_t (&u)[32], int columns) {
  switch (act) {  // warp-uniform
    case kActSilu: gated_combine<kActSilu>(g, u, columns); break;
    case kActGelu: gated_combine<kActGelu>(g, u, columns); break;
    case kActGeluTanh: gated_combine<kActGeluTanh>(g, u, columns); break;
    default: gated_combine<kActRelu>(g, u, columns); break;
  }
}

// 32 columns of both products from TMEM, the two issuers' sums added where there are two.
__device__ __forceinline__ void gated_load(const GatedParams& p, uint32_t taddr, uint32_t (&g)[32], uint32_t (&u)[32]) {
  ptx::tmem_ld_32x32(taddr, g);
  ptx::tmem_ld_32x32(taddr + p.width, u);
  ptx::tmem_ld_wait();
  if (p.issuers == 2) {
    uint32_t x[32];
    ptx::tmem_ld_32x32(taddr + kGatedChainCols, x);
    ptx::tmem_ld_wait();
#pragma unroll
    for (int q = 0; q < 32; ++q) g[q] = __float_as_uint(__uint_as_float(g[q]) + __uint_as_float(x[q]));
    ptx::tmem_ld_32x32(taddr + kGatedChainCols + p.width, x);
    ptx::tmem_ld_wait();
#pragma unroll
    for (int q = 0; q < 32; ++q) u[q] = __float_as_uint(__uint_as_float(u[q]) + __uint_as_float(x[q]));
  }
}

// One row's share of up to 32 columns, packed, straight to output `which`; columns is a multiple of 8, as is F.
__device__ __forceinline__ void gated_store_row(const GatedParams& p, int which, const uint32_t (&o)[16], int row, int col,
                                                int columns) {
  if (row >= p.m) return;
  const int valid = min(columns, p.f - col);
  uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out[which]) + (static_cast<size_t>(row) * p.f + col) * 2);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (8 * i < valid) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
}

template <int kCta>
__global__ void __launch_bounds__(GatedShape<kCta>::kThreads, 1)
    gated_umma_kernel(const __grid_constant__ GatedParams p) {
  using S = GatedShape<kCta>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t warp = ptx::warp_index();
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t cta_rank = (kCta == 2) ? ptx::cluster_ctarank() : 0u;
  const bool leader = cta_rank == 0;
  const uint32_t ctas_per_tile = kCta == 2 ? 2u : static_cast<uint32_t>(p.split);
  const uint32_t k_rank = (kCta == 1 && p.split > 1) ? ptx::cluster_ctarank() : 0u;  // which share of K is this CTA's
  const int first = static_cast<int>(blockIdx.x / ctas_per_tile);
  const int stride = static_cast<int>(gridDim.x / ctas_per_tile);
  const int tiles = p.m_tiles * p.n_tiles;
  const int all_kb = (p.k + S::kBK - 1) / S::kBK;
  const int kb_base = kCta == 2 ? 0 : all_kb * static_cast<int>(k_rank) / p.split;
  const int num_kb = kCta == 2 ? all_kb : all_kb * static_cast<int>(k_rank + 1) / p.split - kb_base;

  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
  const uint32_t staging_base = smem_base + static_cast<uint32_t>(p.stages * p.stage_bytes);  // pair variant
  const uint32_t bar_base = smem_base + static_cast<uint32_t>(p.bar_offset);
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (S::kMaxStages + s); };
  auto tmem_full_bar = [&](uint32_t a) { return bar_base + 8u * (2 * S::kMaxStages + a); };
  auto tmem_empty_bar = [&](uint32_t a) { return bar_base + 8u * (2 * S::kMaxStages + 2 + a); };
  volatile uint32_t* tmem_slot =
      reinterpret_cast<volatile uint32_t*>(smem_gen + p.bar_offset + 8 * (2 * S::kMaxStages + 4));
  volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  // Groups of group_m row tiles are walked column-major, so tiles in flight together share rows of A and of the weights.
  auto tile_at = [&](int t, int& mt, int& nt) {
    const int per_group = p.group_m * p.n_tiles;
    const int g = t / per_group;
    const int first_m = g * p.group_m;
    const int rows = min(p.group_m, p.m_tiles - first_m);
    const int r = t - g * per_group;
    mt = first_m + r % rows;
    nt = r / rows;
  };

  const uint32_t b_bytes = static_cast<uint32_t>(p.width) * 128u;
  const uint32_t stage_tx = 2u * b_bytes + static_cast<uint32_t>(kCta * p.a_rows) * 128u;
  // One CTA: the loads of k-block kb into stage s (the ring of a pair: see the producers).
  auto load_stage = [&](uint32_t s, int kb, int row_a, int row_b) {
    const uint32_t a = smem_base + s * static_cast<uint32_t>(p.stage_bytes);
    const uint32_t b = a + static_cast<uint32_t>(p.a_bytes);
    const int k0 = (kb_base + kb) * S::kBK;
    ptx::mbar_arrive_expect_tx(full_bar(s), stage_tx);
    ptx::tma_load_2d(b, &p.tm_gate, full_bar(s), k0, row_b);
    ptx::tma_load_2d(b + b_bytes, &p.tm_up, full_bar(s), k0, row_b);
    ptx::tma_load_2d(a, &p.tm_a, full_bar(s), k0, row_a);
  };
  // k-blocks whose loads one thread puts in flight before the CTA-wide set-up barrier (two stages at least are there)
  const int preloaded = kCta == 1 ? min(num_kb, 2) : 0;
  if (warp == 0) {
    if (lane < static_cast<uint32_t>(p.stages)) {
      ptx::mbar_init(full_bar(lane), 1);
      ptx::mbar_init(empty_bar(lane), 1);
    }
    if (lane < 2) {
      ptx::mbar_init(tmem_full_bar(lane), static_cast<uint32_t>(p.issuers));
      ptx::mbar_init(tmem_empty_bar(lane), 4 * kCta);  // one arrive per epilogue warp of each CTA
    }
    ptx::fence_mbar_init();
    __syncwarp();
    if (lane == 0) {
      *cta_abort = 0;
      ptx::prefetch_tensormap(&p.tm_a);
      ptx::prefetch_tensormap(&p.tm_gate);
      ptx::prefetch_tensormap(&p.tm_up);
    }
    __syncwarp();
    if constexpr (kCta == 1) {
      // The weights' first k-blocks may come into L2 while the kernel before this one finishes: a prefetch reads nothing, so
      // it does not matter whether that kernel still writes them.  16 x 8192 x 4096: 26.5 -> 25.9 us; not worth its
      // issue for narrow tiles (4 x 1024 x 2048: 7.3 -> 7.5).
      if (p.width > 32 && ptx::elect_one()) {
        for (int kb = 0; kb < min(num_kb, p.stages); ++kb) {  // one row of tiles: tile = column tile
          ptx::tma_prefetch_2d(&p.tm_gate, (kb_base + kb) * S::kBK, first * p.width);
          ptx::tma_prefetch_2d(&p.tm_up, (kb_base + kb) * S::kBK, first * p.width);
        }
      }
      __syncwarp();
      ptx::grid_dependency_wait();  // before the first global read
      if (ptx::elect_one()) {
        for (int kb = 0; kb < preloaded; ++kb) load_stage(static_cast<uint32_t>(kb), kb, 0, first * p.width);
      }
      __syncwarp();
    }
  }
  if (warp == 1) {
    ptx::tmem_alloc<kCta>(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    ptx::tmem_relinquish<kCta>();
  }
  if (kCta == 1 && p.a_bytes == S::kABytes && warp >= 2) {
    // The rows of A that do not exist are multiplied all the same: as zeros they cost little power (see the launcher).
    const uint32_t from = static_cast<uint32_t>(p.a_rows) * 128u;
    for (int s = 0; s < p.stages; ++s)
      for (uint32_t at = from + (threadIdx.x - 64u) * 16u; at < S::kABytes; at += (S::kThreads - 64u) * 16u)
        ptx::st_shared_v4(smem_base + s * static_cast<uint32_t>(p.stage_bytes) + at, 0, 0, 0, 0);
    ptx::fence_proxy_async_smem();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (kCta == 2) ptx::cluster_sync_all();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  release_next_kernel(warp);

  if (warp == 0 || (warp >= 6 && warp < S::kSecondIssuer)) {
    // ------------------------------------------------------------------ TMA producers
    ptx::grid_dependency_wait();  // before the first global read; everything else follows from these reads
    const uint32_t mine = warp == 0 ? 0u : warp - 5u;  // this warp fills every kProducers-th stage of the walk
    const uint32_t stages = static_cast<uint32_t>(p.stages);
    const CUtensorMap* tm_b = leader ? &p.tm_gate : &p.tm_up;
    int kb = static_cast<int>(mine) + (preloaded + 1 - static_cast<int>(mine)) / 2 * 2;  // its first that is not in flight yet
    uint32_t s = static_cast<uint32_t>(kb) % stages, ph = (static_cast<uint32_t>(kb) / stages) & 1u;
    for (int t = first; t < tiles; t += stride) {
      int mt, nt;
      tile_at(t, mt, nt);
      const int row_a = (mt * kCta + static_cast<int>(cta_rank)) * S::kBM;
      const int row_b = nt * p.width;
      for (; kb < num_kb; kb += S::kProducers) {
        if (!bounded_wait_converged(empty_bar(s), ph ^ 1u, cta_abort, p.status, kFaultProducerWait, lane)) break;
        if (ptx::elect_one()) {
          if constexpr (kCta == 2) {
            const uint32_t a = smem_base + s * static_cast<uint32_t>(p.stage_bytes);
            if (leader) ptx::mbar_arrive_expect_tx(full_bar(s), stage_tx);
            const uint32_t bar = ptx::mapa(full_bar(s), 0);
            ptx::tma_load_2d_pair(a, &p.tm_a, bar, kb * S::kBK, row_a);
            ptx::tma_load_2d_pair(a + static_cast<uint32_t>(p.a_bytes), tm_b, bar, kb * S::kBK, row_b);
          } else {
            load_stage(s, kb, row_a, row_b);
          }
        }
        __syncwarp();
        s += S::kProducers;
        while (s >= stages) {
          s -= stages;
          ph ^= 1u;
        }
      }
      if (kb < num_kb) break;  // a wait ran out
      kb -= num_kb;
    }
  } else if (warp == 1 || warp == S::kSecondIssuer) {
    // ------------------------------------------------------------------ MMA issuers
    // One warp needs about 380 cycles for a k-block's four UMMAs, their commit and its waits, more than the tensor pipe does
    // when N <= 128.  For those tiles two warps take turns at the k-blocks, each into an accumulator of its own (the
    // epilogue adds the two, always in the same order).  Which warp has a k-block goes by its number in the CTA's whole walk
    // and the ring is an even number of stages deep, so a stage always belongs to the same warp: a parity wait cannot mistake
    // one use of a stage for the one two uses earlier.
    const uint32_t issuers = static_cast<uint32_t>(p.issuers);
    const uint32_t mine = warp == 1 ? 0u : 1u;
    if (leader && mine < issuers) {
      const uint32_t idesc =
          ptx::umma_idesc_f16_f32(S::kBM * kCta, 2 * p.width) | (p.bf16 ? ptx::kIdescBf16Inputs : 0u);
      const uint64_t a_desc0 = ptx::umma_desc_k_sw128(smem_base);
      const uint64_t b_desc0 = ptx::umma_desc_k_sw128(smem_base + static_cast<uint32_t>(p.a_bytes));
      const uint64_t desc_stride = static_cast<uint64_t>(p.stage_bytes >> 4);
      const uint32_t stages = static_cast<uint32_t>(p.stages);
      uint32_t s = mine, ph = 0;
      int kb = static_cast<int>(mine);
      for (int t = first, j = 0; t < tiles; t += stride, ++j) {
        const uint32_t acc = static_cast<uint32_t>(j) & 1u;
        const uint32_t acc_ph = (static_cast<uint32_t>(j) >> 1) & 1u;
        if (!bounded_wait_converged(tmem_empty_bar(acc), acc_ph ^ 1u, cta_abort, p.status, kFaultMmaWaitAcc, lane)) break;
        ptx::tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * S::kAccCols + mine * kGatedChainCols;
        const int kb_first = kb;
        for (; kb < num_kb; kb += static_cast<int>(issuers)) {
          if (!bounded_wait_converged(full_bar(s), ph, cta_abort, p.status, kFaultMmaWaitFull, lane)) break;
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            ptx::umma_f16_kblock<kCta>(d_tmem, a_desc0 + s * desc_stride, b_desc0 + s * desc_stride, idesc,
                                       kb > kb_first ? 1u : 0u);
            if constexpr (kCta == 1)
              ptx::umma_commit<1>(empty_bar(s));
            else
              ptx::umma_commit_pair_both(empty_bar(s), 0x3);
          }
          __syncwarp();
          s += issuers;
          if (s >= stages) {
            s -= stages;
            ph ^= 1u;
          }
        }
        if (kb < num_kb) break;  // a wait ran out
        kb -= num_kb;
        if (ptx::elect_one()) {
          if constexpr (kCta == 1)
            ptx::umma_commit<1>(tmem_full_bar(acc));
          else
            ptx::umma_commit_pair_both(tmem_full_bar(acc), 0x3);
        }
        __syncwarp();
      }
    }
  } else if (kCta == 2 || p.split == 1) {
    // ------------------------------------------------------------------ epilogue (warps 2..5)
    const uint32_t quad = warp & 3u;  // TMEM lanes [32 quad, 32 quad + 32) are this warp's to read
    const uint32_t lead_empty0 = (kCta == 2) ? ptx::mapa(tmem_empty_bar(0), 0) : tmem_empty_bar(0);
    const bool keep = p.out[1] != nullptr;
    uint32_t stores = 0;  // bulk stores this warp has issued (selects the staging buffer)
    for (int t = first, j = 0; t < tiles; t += stride, ++j) {
      const uint32_t acc = static_cast<uint32_t>(j) & 1u;
      const uint32_t acc_ph = (static_cast<uint32_t>(j) >> 1) & 1u;
      if (!bounded_wait_warp(tmem_full_bar(acc), acc_ph, cta_abort, p.status, kFaultEpilogueWait, lane)) break;
      ptx::tc_fence_after();
      int mt, nt;
      tile_at(t, mt, nt);
      const int row0 = (mt * kCta + static_cast<int>(cta_rank)) * S::kBM + static_cast<int>(quad) * 32;
      const int col0 = nt * p.width;
      const uint32_t taddr = tmem_base + ((quad * 32u) << 16) + acc * S::kAccCols;
      const bool rows_live = row0 < p.m;  // warp-uniform
      for (int c = 0; rows_live && c < p.width && col0 + c < p.f; c += 32) {
        uint32_t g[32], u[32];
        gated_load(p, taddr + c, g, u);  // a narrow tile's last read runs into the neighbouring columns: not stored
        // Writes 32 columns of output `which`, rounded once.
        auto store = [&](const uint32_t(&v)[32], int which) {
          uint32_t o[16];
#pragma unroll
          for (int q = 0; q < 16; ++q)
            o[q] = ptx::pack_out2(__uint_as_float(v[2 * q]), __uint_as_float(v[2 * q + 1]), p.bf16);
          if constexpr (kCta == 2) {
            // `width` is a multiple of 32 here, so a box never reaches into the next tile's columns.
            const uint32_t buf =
                staging_base + (quad * S::kBufsPerWarp + stores % S::kBufsPerWarp) * S::kStoreBufBytes;
            if (stores >= S::kBufsPerWarp) {
              if (lane == 0) ptx::tma_store_wait_read<S::kBufsPerWarp - 1>();
              __syncwarp();
            }
            // Row `lane` of the box, 16-byte piece i at i ^ (lane / 2 % 4): the 64-byte swizzle, free of bank conflicts.
#pragma unroll
            for (int i = 0; i < 4; ++i)
              ptx::st_shared_v4(buf + lane * 64u + ((static_cast<uint32_t>(i) ^ ((lane >> 1) & 3u)) << 4), o[4 * i],
                                o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              ptx::tma_store_2d(&p.tm_out[which], buf, col0 + c, row0);
              ptx::tma_store_commit();
            }
            ++stores;
          } else {
            gated_store_row(p, which, o, row0 + static_cast<int>(lane), col0 + c, min(32, p.width - c));
          }
        };
        if (keep) {
          store(g, 1);
          store(u, 2);
        }
        gated_combine(p.act, g, u, kCta == 2 ? 32 : p.width - c);
        store(g, 0);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kCta == 1)
          ptx::mbar_arrive(tmem_empty_bar(acc));
        else
          ptx::mbar_arrive_cluster(lead_empty0 + 8u * acc);
      }
    }
  }

  if constexpr (kCta == 1) {
    if (p.split > 1) {
      // ---------------------------------------------------------------- a tile shared by a cluster: its epilogue
      const uint32_t split = static_cast<uint32_t>(p.split);
      const bool epilogue = warp >= 2 && warp < 6;
      const uint32_t quad = warp & 3u;
      const uint32_t row = quad * 32u + lane;
      const uint32_t taddr = tmem_base + ((quad * 32u) << 16);
      const int slice = p.width / p.split;  // columns of F that each CTA finishes, a multiple of 8
      const uint32_t groups = static_cast<uint32_t>(slice) / 2u;  // of four floats: the slice's columns of both products
      bool ready = false;
      if (epilogue) {
        ready = bounded_wait_warp(tmem_full_bar(0), 0, cta_abort, p.status, kFaultEpilogueWait, lane);
        ptx::tc_fence_after();
        ready = ready && static_cast<int>(quad * 32u) < p.m;
      }
      ptx::cluster_sync_all();  // every CTA's operands have been multiplied: the rings may be written over
      if (ready) {
        for (uint32_t to = 0; to < split; ++to) {
          if (to == k_rank) continue;
          const uint32_t there = ptx::mapa(smem_base, to);
          for (int c = 0; c < slice; c += 32) {
            uint32_t g[32], u[32];
            gated_load(p, taddr + to * slice + c, g, u);
            if (static_cast<int>(row) < p.m) {
              const uint32_t slot = exchange_slot(k_rank, to), at = static_cast<uint32_t>(c) / 4u;
              exchange_send(there, slot, groups, at, row, g, slice - c);
              exchange_send(there, slot, groups, groups / 2u + at, row, u, slice - c);
            }
          }
        }
      }
      ptx::cluster_sync_all();
      if (ready) {
        const int col0 = first * p.width + static_cast<int>(k_rank) * slice;
        for (int c = 0; c < slice && col0 + c < p.f; c += 32) {
          uint32_t g[32], u[32];
          gated_load(p, taddr + k_rank * slice + c, g, u);
          const uint32_t at = static_cast<uint32_t>(c) / 4u;
          exchange_sum(smem_base, k_rank, split, groups, at, row, g, slice - c);
          exchange_sum(smem_base, k_rank, split, groups, groups / 2u + at, row, u, slice - c);
          auto store = [&](const uint32_t(&v)[32], int which) {
            uint32_t o[16];
#pragma unroll
            for (int q = 0; q < 16; ++q)
              o[q] = ptx::pack_out2(__uint_as_float(v[2 * q]), __uint_as_float(v[2 * q + 1]), p.bf16);
            gated_store_row(p, which, o, static_cast<int>(row), col0 + c, min(32, slice - c));
          };
          if (p.out[1] != nullptr) {
            store(g, 1);
            store(u, 2);
          }
          gated_combine(p.act, g, u, slice - c);
          store(g, 0);
        }
      }
    }
  }

  // ---- teardown: bulk stores have read their staging buffers; then everyone meets and the allocating warp frees TMEM
  if (kCta == 2 && warp >= 2 && warp < 6 && lane == 0) ptx::tma_store_wait_read<0>();
  __syncwarp();
  if (*cta_abort) abort_drain_delay();
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (kCta == 2) ptx::cluster_sync_all();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<kCta>(tmem_base, 512);
  }
}

// dG = dC * U * act'(G) and dU = dC * act(G), element by element in fp32, rounded once to the operands' type: they are
// operands of the four products of the backward pass, which the tensor cores take in 16 bits.  Bound by memory: 10 bytes
// per element; 8 elements per thread keep three 16-byte loads in flight.
struct GatedSlopeParams {
  const uint4* dc;
  const uint4* gate;
  const uint4* up;
  uint4* dgate;
  uint4* dup;
  long long count8;  // groups of 8 elements
  int act;
  int bf16;
};

template <int kAct, bool kBf16>
__device__ __forceinline__ void gated_slope8(const uint4& d4, const uint4& g4, const uint4& u4, uint4& dg4, uint4& du4) {
  const uint32_t d[4] = {d4.x, d4.y, d4.z, d4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
  uint32_t dg[4], du[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 df = ptx::unpack_in2(d[i], kBf16), gf = ptx::unpack_in2(g[i], kBf16), uf = ptx::unpack_in2(u[i], kBf16);
    const float2 lo = act_value_slope<kAct>(gf.x), hi = act_value_slope<kAct>(gf.y);
    dg[i] = ptx::pack_out2(df.x * uf.x * lo.y, df.y * uf.y * hi.y, kBf16);
    du[i] = ptx::pack_out2(df.x * lo.x, df.y * hi.x, kBf16);
  }
  dg4 = make_uint4(dg[0], dg[1], dg[2], dg[3]);
  du4 = make_uint4(du[0], du[1], du[2], du[3]);
}

template <int kAct, bool kBf16>
__global__ void __launch_bounds__(256) gated_slope_kernel(const GatedSlopeParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();  // see release_next_kernel()
  const long long stride = static_cast<long long>(gridDim.x) * 256;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < p.count8; i += stride) {
    uint4 dg, du;
    gated_slope8<kAct, kBf16>(__ldcs(p.dc + i), __ldcs(p.gate + i), __ldcs(p.up + i), dg, du);
    p.dgate[i] = dg;  // read again by the products that follow: the default policy leaves them in L2 where they fit
    p.dup[i] = du;
  }
}

}  // namespace beam
