// MXFP4: quantisation, its inverse, and the product C = A B^T of two quantised matrices on the 4-bit tensor cores.
//
// A quantised [R, K] matrix (K a multiple of 32) is two arrays:
//   q       [R, K / 2] bytes, e2m1 codes, element 2 i in the low half of byte i;
//   scales  one ue8m0 byte (2^(s - 127), 255 = NaN) per 32 elements of a row, in blocks of 128 rows x 4 scales,
//           [ceil(R / 128)][ceil(K / 128)][512]: row r, scale c of a block at byte (r % 32) * 16 + (r / 32) * 4 + c.
// The scale blocks are what the tensor cores take: 512 contiguous bytes are one copy into TMEM, so the product moves
// scales like any other operand tile and no thread ever touches one.  Scales outside the matrix are 0.
#pragma once

#include "umma_common.cuh"

namespace beam {

// ------------------------------------------------------------------ quantisation
// One half-warp takes 128 elements of a row (a row of one scale block): each lane 8 elements, four lanes a scale.
//   s = floor(log2(max |x|)) - 2, at least -127: the exponent field of the largest magnitude, without a logarithm;
//   q = x 2^-s rounded to the nearest e2m1 value, ties to even; magnitudes above 6 (up to 8 by the choice of s) become 6.
// The scaling is exact in fp32.  A block with an infinity or a NaN gets the NaN scale.  Bound by memory (2 bytes in and
// 17/32 out per element) as long as the instructions per element stay few: magnitudes are compared as pairs of 16-bit integers
// (infinities and NaN order above all finite values), and a block's half-warps are laid over rows and K by shifts.
// A block of 256 threads covers 2^kb_shift blocks of K x (64 >> kb_shift) rows: its 16 half-warps lie side by side over K and then
// over rows, and each takes kMxUnits rows at equal distances, so a thread's addresses differ by constants.
struct MxUnits {
  int rows;           // rows that units are laid over (quantisation: rounded up to 128, the padding of the scales is written too)
  uint32_t kblocks;   // ceil(k / 128)
  uint32_t kb_shift;  // at most 4
  uint32_t x_blocks;  // ceil(kblocks / 2^kb_shift)
};

constexpr int kMxUnits = 4;  // units per half-warp: 16-byte loads in flight per thread

struct MxPlace {
  uint32_t row, step;   // unit i works on row + i step
  uint32_t kb, col;     // its block of K and this lane's first column
};
__device__ __forceinline__ MxPlace mx_place(const MxUnits& u) {
  const uint32_t half = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const uint32_t by = blockIdx.x / u.x_blocks, bx = blockIdx.x - by * u.x_blocks;
  MxPlace p;
  p.kb = (bx << u.kb_shift) + (half & ((1u << u.kb_shift) - 1u));
  p.step = 16u >> u.kb_shift;
  p.row = by * (kMxUnits * p.step) + (half >> u.kb_shift);
  p.col = p.kb * 128 + lane * 8;
  return p;
}
// First byte of a block's scales, and the word of a row in it.  A thread's rows lie in one group of 128.
__device__ __forceinline__ size_t mx_scale_block(const MxPlace& p, uint32_t kblocks) {
  return (static_cast<size_t>(p.row >> 7) * kblocks + p.kb) * 512;
}
__device__ __forceinline__ uint32_t mx_scale_row(uint32_t row) { return (row & 31) * 16 + ((row >> 5) & 3) * 4; }

struct MxQuantParams {
  const uint4* x;
  uint32_t* q;      // 8 codes per word
  uint8_t* scales;
  int rows, k;
  MxUnits units;
};

template <bool kBf16>
static __global__ void __launch_bounds__(256, 8) mxfp4_quantize_kernel(const MxQuantParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();  // see release_next_kernel()
  const MxPlace at = mx_place(p.units);
  const bool in_k = at.col < static_cast<uint32_t>(p.k);
  const size_t first = (static_cast<size_t>(at.row) * p.k + at.col) >> 3, step = (static_cast<size_t>(at.step) * p.k) >> 3;
  const uint4* from = p.x + first;
  uint4 x[kMxUnits];
#pragma unroll
  for (int i = 0; i < kMxUnits; ++i) {
    x[i] = make_uint4(0, 0, 0, 0);
    if (in_k && at.row + i * at.step < static_cast<uint32_t>(p.rows)) x[i] = __ldcs(from + i * step);
  }
  uint32_t* to = p.q + first;
  uint8_t* scales = p.scales + mx_scale_block(at, p.units.kblocks) + ((threadIdx.x & 15) >> 2);
  const bool writes_scale = (threadIdx.x & 3) == 0 && at.kb < p.units.kblocks;
#pragma unroll
  for (int i = 0; i < kMxUnits; ++i) {
    const uint32_t row = at.row + i * at.step;
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    uint32_t top = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
    top = max(top & 0xFFFFu, top >> 16);
    // the exponent field that the largest magnitude has in fp32; 255 for infinities and NaN, whose codes do not matter
    const uint32_t field = kBf16 ? top >> 7 : __float_as_uint(ptx::unpack_in2(top, 0).x) >> 23;
    uint32_t scale = max(field, 2u) - 2u;
    const float inv = __uint_as_float((254u - scale) << 23);  // 2^-s
    if (field == 255) scale = 255;
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = ptx::unpack_in2(w[j], kBf16);
      v[2 * j] = f.x * inv;
      v[2 * j + 1] = f.y * inv;
    }
    const uint32_t code = ptx::pack_e2m1x8(v);
    if (in_k && row < static_cast<uint32_t>(p.rows)) to[i * step] = code;
    // lanes past K hold zeros and so give the scale 0
    if (writes_scale && row < static_cast<uint32_t>(p.units.rows)) scales[mx_scale_row(row)] = static_cast<uint8_t>(scale);
  }
}

enum MxType : int { kMxFp16 = 0, kMxBf16 = 1, kMxFp32 = 2 };

// The inverse: x = q 2^s, exact in fp32 and rounded to the output type.  Same units.
template <int kType>
static __global__ void __launch_bounds__(256) mxfp4_dequantize_kernel(const uint32_t* q, const uint8_t* scales, uint4* x,
                                                                      int k, MxUnits units) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();  // see release_next_kernel()
  const MxPlace at = mx_place(units);
  if (at.col >= static_cast<uint32_t>(k)) return;
  const size_t first = (static_cast<size_t>(at.row) * k + at.col) >> 3, step = (static_cast<size_t>(at.step) * k) >> 3;
  scales += mx_scale_block(at, units.kblocks) + ((threadIdx.x & 15) >> 2);
  uint32_t code[kMxUnits], byte[kMxUnits];
#pragma unroll
  for (int i = 0; i < kMxUnits; ++i) {
    const uint32_t row = at.row + i * at.step;
    code[i] = byte[i] = 0;
    if (row < static_cast<uint32_t>(units.rows)) {
      code[i] = __ldcs(q + first + i * step);
      byte[i] = __ldcg(scales + mx_scale_row(row));  // no read-only path: the kernel ahead may have written them since this one began
    }
  }
#pragma unroll
  for (int i = 0; i < kMxUnits; ++i) {
    if (at.row + i * at.step >= static_cast<uint32_t>(units.rows)) break;
    // 2^(s - 127) in fp32: 0 is the subnormal 2^-127, 255 a NaN
    const uint32_t s = byte[i];
    const float scale = __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7FC00000u : s << 23);
    float v[8];
    ptx::unpack_e2m1x8(code[i], v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= scale;
    if constexpr (kType == kMxFp32) {
      float4* dst = reinterpret_cast<float4*>(x) + 2 * (first + i * step);
      __stcs(dst, make_float4(v[0], v[1], v[2], v[3]));
      __stcs(dst + 1, make_float4(v[4], v[5], v[6], v[7]));
    } else {
      __stcs(x + first + i * step, make_uint4(ptx::pack_out2(v[0], v[1], kType), ptx::pack_out2(v[2], v[3], kType),
                                              ptx::pack_out2(v[4], v[5], kType), ptx::pack_out2(v[6], v[7], kType)));
    }
  }
}

// ------------------------------------------------------------------ product
// C[M, N] = A B^T: 4-bit UMMAs (K = 64) with block scales, fp32 accumulation, one rounding to fp16 or bf16.
//
// A stage of the ring is 256 elements of K: 128 bytes per row, laid out by TMA with the 128-byte swizzle like any K-major
// operand, and 1 KB of scale blocks per 128 rows that a second copy brings as they are.  Per stage the issuing warp copies
// the scale blocks into TMEM and issues four UMMAs; copies and UMMAs of one thread execute in order, so nothing else
// separates them; two sets of scale columns alternate.
//
//   kCta = 2   256 x 256 tiles on a pair.  B's scales of all 256 columns are needed in both CTAs' TMEM, so both load them.
//              Two accumulators of 256 columns and the scales do not fit into 512 columns, so the accumulators overlap
//              by 64 columns: the epilogue of a tile drains that part first and hands it back, after which the next
//              tile's UMMAs may start in the other accumulator while the rest is drained.
//              What bounds it at 8192^3 (182 us, 6.0 PFLOP/s): the tensor pipe is active 81 % of the cycles; the rest is the
//              hand-back of the shared columns, some 2000 cycles for each of a pair's 14 tiles, and waits for operands.  A sixth
//              stage is worth more than a second store buffer (3 % at this size).
//   kCta = 1   M <= 128, bound by reading B: 128 rows x 64 or 128 columns (see narrow_plan() in mxfp4_launch.cu).  Only existing
//              rows of A are loaded, two issuers take turns at the stages, and clusters may share a contraction, all
//              as in gated_umma.cuh.
//
// Roles: warp 0 loads A and its scales, warp 10 B and its scales, warps 1 and 11 issue, warps 2..9 are the epilogue.
struct MxGemmParams {
  CUtensorMap tm_a;   // packed A [M, K / 2 bytes], box (rows per CTA) x 128
  CUtensorMap tm_b;   // packed B [N, K / 2 bytes], box (width / kCta) x 128
  CUtensorMap tm_sa;  // scales of A as 8-byte words [row blocks][64 ceil(K / 128)], box 1 x 128
  CUtensorMap tm_sb;  // scales of B, box 2 x 128
  CUtensorMap tm_c;   // pair: C [M, N], store box 32 rows x 32 columns, 64 B swizzle
  void* c;
  int m, n, k;
  int width;          // columns per tile
  int a_rows;         // rows of A that a CTA loads
  int stages, stage_bytes;
  int a_bytes;        // of a stage: B begins there, the scales behind B
  int bar_offset;     // the barriers' place in shared memory, behind the ring and what else takes its place
  int issuers;        // warps that issue UMMAs: 1, or 2 that take turns at the stages, an accumulator and scale columns each
  int split;          // single CTAs: a cluster of this many CTAs shares each tile's contraction
  int m_tiles, n_tiles, group_m;
  int bf16;
  int* status;
};

template <int kCta>
struct MxShape {
  static constexpr int kBK = 256;  // elements of K per stage
  static constexpr int kABytes = 128 * 128;
  static constexpr int kScaleBlocksB = kCta;  // row blocks of B's scales per tile
  static constexpr int kScaleBytes = (1 + kScaleBlocksB) * 1024;
  static constexpr int kMaxStages = 16;
  // warps: 0 and 10 producers, 1 and 11 issuers, 2..9 epilogue (two for each quarter of the lanes, taking turns at the columns)
  static constexpr int kEpilogueWarps = 8;
  static constexpr int kSecondProducer = 2 + kEpilogueWarps;
  static constexpr int kSecondIssuer = kSecondProducer + 1;
  static constexpr int kThreads = 32 * (kSecondIssuer + 1);
  static constexpr int kMaxWidth = kCta == 2 ? 256 : 128;
  static constexpr int kAccStep = kCta == 2 ? 192 : 128;  // TMEM columns from one accumulator to the other
  static constexpr int kScaleCols = kAccStep + kMaxWidth;  // first column of the scales
  static constexpr int kScaleHalf = 4 + 4 * kScaleBlocksB;  // columns of 128 elements of K
  static constexpr int kScaleSet = 2 * kScaleHalf;          // ... of a stage; an issuer alternates between two sets
  static constexpr int kStagingBytes = kCta == 2 ? kEpilogueWarps * 2048 : 0;  // a box of 32 rows x 32 columns per warp
  static constexpr int kBarBytes = 512;
  static constexpr int kSmemLimit = 232448;
  static constexpr int kRingBytes = kSmemLimit - kStagingBytes - kBarBytes;
  static_assert(kScaleCols + (3 - kCta) * 2 * kScaleSet <= 512, "accumulators and scales share 512 columns");
  static_assert((2 * kMaxStages + 4) * 8 + 8 <= kBarBytes, "barrier block too small");
};

// 32 columns of a single CTA's tile from TMEM, the two issuers' sums added where there are two.
__device__ __forceinline__ void mx_load(const MxGemmParams& p, uint32_t taddr, uint32_t (&v)[32]) {
  ptx::tmem_ld_32x32(taddr, v);
  ptx::tmem_ld_wait();
  if (p.issuers == 2) {
    uint32_t x[32];
    ptx::tmem_ld_32x32(taddr + MxShape<1>::kAccStep, x);
    ptx::tmem_ld_wait();
#pragma unroll
    for (int q = 0; q < 32; ++q) v[q] = __float_as_uint(__uint_as_float(v[q]) + __uint_as_float(x[q]));
  }
}

// One row's share of up to 32 columns, rounded, straight to C; columns is a multiple of 8, as is N.
__device__ __forceinline__ void mx_store_row(const MxGemmParams& p, const uint32_t (&v)[32], int row, int col, int columns) {
  if (row >= p.m) return;
  uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.c) + (static_cast<size_t>(row) * p.n + col) * 2);
  const int valid = min(columns, p.n - col);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (8 * i < valid) {
      uint32_t o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        o[q] = ptx::pack_out2(__uint_as_float(v[8 * i + 2 * q]), __uint_as_float(v[8 * i + 2 * q + 1]), p.bf16);
      dst[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

template <int kCta>
__global__ void __launch_bounds__(MxShape<kCta>::kThreads, 1) mxfp4_umma_kernel(const __grid_constant__ MxGemmParams p) {
  using S = MxShape<kCta>;
  extern __shared__ __align__(1024) uint8_t smem_tiles[];
  const uint32_t warp = ptx::warp_index();
  const uint32_t lane = threadIdx.x & 31;
  const int cta_rank = (kCta == 2) ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const bool leader = cta_rank == 0;
  const int ctas_per_tile = kCta == 2 ? 2 : p.split;
  const uint32_t k_rank = (kCta == 1 && p.split > 1) ? ptx::cluster_ctarank() : 0u;  // which share of K is this CTA's
  const int first = static_cast<int>(blockIdx.x) / ctas_per_tile;
  const int stride = static_cast<int>(gridDim.x) / ctas_per_tile;
  const int tiles = p.m_tiles * p.n_tiles;
  const int all_kb = (p.k + S::kBK - 1) / S::kBK;
  const int kb_base = kCta == 2 ? 0 : all_kb * static_cast<int>(k_rank) / p.split;
  const int num_kb = kCta == 2 ? all_kb : all_kb * static_cast<int>(k_rank + 1) / p.split - kb_base;

  const uint32_t smem_base = ptx::smem_u32(smem_tiles);
  const uint32_t a_bytes = static_cast<uint32_t>(p.a_bytes);
  const uint32_t b_bytes = static_cast<uint32_t>(p.width / kCta) * 128u;
  const uint32_t staging_base = smem_base + static_cast<uint32_t>(p.stages * p.stage_bytes);  // pair variant
  const uint32_t bar_base = smem_base + static_cast<uint32_t>(p.bar_offset);
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (S::kMaxStages + s); };
  auto tmem_full_bar = [&](uint32_t a) { return bar_base + 8u * (2 * S::kMaxStages + a); };
  auto tmem_empty_bar = [&](uint32_t a) { return bar_base + 8u * (2 * S::kMaxStages + 2 + a); };
  volatile uint32_t* tmem_slot =
      reinterpret_cast<volatile uint32_t*>(smem_tiles + p.bar_offset + 8 * (2 * S::kMaxStages + 4));
  volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  auto tile_at = [&](int t, int& mt, int& nt) {
    const int per_group = p.group_m * p.n_tiles;
    const int g = t / per_group;
    const int first_m = g * p.group_m;
    const int rows = min(p.group_m, p.m_tiles - first_m);
    const int r = t - g * per_group;
    mt = first_m + r % rows;
    nt = r / rows;
  };

  const uint32_t stage_tx = static_cast<uint32_t>(kCta) * (a_bytes + b_bytes + static_cast<uint32_t>(S::kScaleBytes));
  // k-blocks that one thread puts in flight before the CTA-wide set-up barrier (see gated_umma.cuh)
  const int preloaded = kCta == 1 ? min(num_kb, 2) : 0;
  // The loads of A (left) or B of k-block kb into stage s.  A's thread arms the barrier with the whole stage; B's bytes may land
  // before that (see grad_umma.cuh).
  auto load_stage = [&](bool left, uint32_t s, int kb, int block_a, int col) {
    const uint32_t a = smem_base + s * static_cast<uint32_t>(p.stage_bytes);
    const uint32_t b = a + a_bytes;
    const uint32_t sf = b + b_bytes;
    const int x = (kb_base + kb) * 128;
    if (left && leader) ptx::mbar_arrive_expect_tx(full_bar(s), stage_tx);
    if constexpr (kCta == 2) {
      const uint32_t bar = ptx::mapa(full_bar(s), 0);
      if (left) {
        ptx::tma_load_2d_pair(a, &p.tm_a, bar, x, block_a * 128);
        ptx::tma_load_2d_pair(sf, &p.tm_sa, bar, x, block_a);
      } else {
        ptx::tma_load_2d_pair(b, &p.tm_b, bar, x, col + cta_rank * 128);
        ptx::tma_load_2d_pair(sf + 1024u, &p.tm_sb, bar, x, col >> 7);
      }
    } else {
      if (left) {
        ptx::tma_load_2d(a, &p.tm_a, full_bar(s), x, block_a * 128);
        ptx::tma_load_2d(sf, &p.tm_sa, full_bar(s), x, block_a);
      } else {
        ptx::tma_load_2d(b, &p.tm_b, full_bar(s), x, col);
        ptx::tma_load_2d(sf + 1024u, &p.tm_sb, full_bar(s), x, col >> 7);
      }
    }
  };
  if (warp == 0) {
    if (lane < static_cast<uint32_t>(p.stages)) {
      ptx::mbar_init(full_bar(lane), 1);
      ptx::mbar_init(empty_bar(lane), 1);
    }
    if (lane < 2) {
      ptx::mbar_init(tmem_full_bar(lane), static_cast<uint32_t>(p.issuers));
      ptx::mbar_init(tmem_empty_bar(lane), S::kEpilogueWarps * kCta);
    }
    ptx::fence_mbar_init();
    __syncwarp();
    if (lane == 0) {
      *cta_abort = 0;
      ptx::prefetch_tensormap(&p.tm_a);
      ptx::prefetch_tensormap(&p.tm_b);
      ptx::prefetch_tensormap(&p.tm_sa);
      ptx::prefetch_tensormap(&p.tm_sb);
    }
    __syncwarp();
    if constexpr (kCta == 1) {
      // B's first stages may come into L2 while the kernel before this one finishes (see gated_umma.cuh).  Wide tiles only:
      // it takes 1 x 16384 x 8192 with its quantisation from 18.1 to 17.4 us, but adds 0.7 us to 16 x 8192 x 8192 (64-wide tiles).
      if (p.width > 64 && ptx::elect_one()) {
        for (int kb = 0; kb < min(num_kb, p.stages); ++kb)
          ptx::tma_prefetch_2d(&p.tm_b, (kb_base + kb) * 128, first * p.width);
      }
      __syncwarp();
      ptx::grid_dependency_wait();  // before the first global read
      if (ptx::elect_one()) {
        for (int kb = 0; kb < preloaded; ++kb) {
          load_stage(true, static_cast<uint32_t>(kb), kb, 0, first * p.width);
          load_stage(false, static_cast<uint32_t>(kb), kb, 0, first * p.width);
        }
      }
      __syncwarp();
    }
  }
  if (warp == 1) {
    ptx::tmem_alloc<kCta>(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    ptx::tmem_relinquish<kCta>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (kCta == 2) ptx::cluster_sync_all();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  release_next_kernel(warp);

  if (warp == 0 || warp == S::kSecondProducer) {
    // ------------------------------------------------------------------ TMA producers
    const bool left = warp == 0;
    ptx::grid_dependency_wait();  // before the first global read
    const uint32_t stages = static_cast<uint32_t>(p.stages);
    int kb = preloaded;  // at most the ring
    uint32_t s = static_cast<uint32_t>(kb) % stages, ph = static_cast<uint32_t>(kb) / stages;
    bool alive = true;
    for (int t = first; alive && t < tiles; t += stride) {
      int mt, nt;
      tile_at(t, mt, nt);
      for (; kb < num_kb; ++kb) {
        if (!bounded_wait_converged(empty_bar(s), ph ^ 1u, cta_abort, p.status, kFaultProducerWait, lane)) {
          alive = false;
          break;
        }
        if (ptx::elect_one()) load_stage(left, s, kb, mt * kCta + cta_rank, nt * p.width);
        __syncwarp();
        if (++s == stages) {
          s = 0;
          ph ^= 1u;
        }
      }
      kb = 0;
    }
  } else if (warp == 1 || warp == S::kSecondIssuer) {
    // ------------------------------------------------------------------ MMA issuers (two: see gated_umma.cuh)
    const uint32_t issuers = static_cast<uint32_t>(p.issuers);
    const uint32_t mine = warp == 1 ? 0u : 1u;
    if (leader && mine < issuers) {
      const uint32_t idesc0 = ptx::umma_idesc_mxf4(128 * kCta, p.width, 0);
      const uint32_t idesc2 = ptx::umma_idesc_mxf4(128 * kCta, p.width, 2);
      const uint64_t a_desc0 = ptx::umma_desc_k_sw128(smem_base);
      const uint64_t b_desc0 = ptx::umma_desc_k_sw128(smem_base + a_bytes);
      const uint64_t sf_desc0 = ptx::umma_desc_scales(smem_base + a_bytes + b_bytes);
      const uint64_t desc_stride = static_cast<uint64_t>(p.stage_bytes >> 4);
      const uint32_t stages = static_cast<uint32_t>(p.stages);
      const int steps = (p.k + 63) / 64 - kb_base * 4;  // UMMAs of a tile from this CTA's first k-block on
      const uint32_t scale_cols = tmem_base + S::kScaleCols + mine * 2u * S::kScaleSet;
      uint32_t s = mine, ph = 0, set = 0;
      int kb = static_cast<int>(mine);
      for (int t = first, j = 0; t < tiles; t += stride, ++j) {
        int mt, nt;
        tile_at(t, mt, nt);
        const uint32_t acc = static_cast<uint32_t>(j) & 1u;
        bool drained = true;
        if constexpr (kCta == 2) {
          // overlapping accumulators: the previous tile's shared columns must have been read
          if (j > 0)
            drained = bounded_wait_converged(tmem_empty_bar(0), static_cast<uint32_t>(j - 1) & 1u, cta_abort, p.status,
                                             kFaultMmaWaitAcc, lane);
        } else {
          drained = bounded_wait_converged(tmem_empty_bar(acc), ((static_cast<uint32_t>(j) >> 1) & 1u) ^ 1u, cta_abort,
                                           p.status, kFaultMmaWaitAcc, lane);
        }
        if (!drained) break;
        ptx::tc_fence_after();
        const uint32_t d_tmem = tmem_base + (acc + mine) * S::kAccStep;  // two issuers: one tile only, acc 0
        // a tile that starts inside a block of 128 columns starts inside that block's four TMEM columns
        const uint32_t sfb_shift = static_cast<uint32_t>(((nt * p.width) & 127) >> 5);
        const int kb_first = kb;
        for (; kb < num_kb; kb += static_cast<int>(issuers)) {
          if (!bounded_wait_converged(full_bar(s), ph, cta_abort, p.status, kFaultMmaWaitFull, lane)) break;
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            const uint64_t a = a_desc0 + s * desc_stride, b = b_desc0 + s * desc_stride, sf = sf_desc0 + s * desc_stride;
            const uint32_t sfa = scale_cols + set * S::kScaleSet, sfb = sfa + 4u;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
              ptx::tmem_cp_scales<kCta>(sfa + h * S::kScaleHalf, sf + h * (512 >> 4));
#pragma unroll
              for (uint32_t i = 0; i < S::kScaleBlocksB; ++i)
                ptx::tmem_cp_scales<kCta>(sfb + h * S::kScaleHalf + 4u * i, sf + ((1024 * (1 + i) + h * 512) >> 4));
            }
            const int live = steps - kb * 4;  // steps past K are left out: their scales may lie outside the matrix
            const uint32_t from = sfb + sfb_shift;
            ptx::umma_mxf4<kCta>(d_tmem, a, b, idesc0, sfa, from, kb > kb_first ? 1u : 0u);
            if (live > 1) ptx::umma_mxf4<kCta>(d_tmem, a + 2, b + 2, idesc2, sfa, from, 1u);
            if (live > 2)
              ptx::umma_mxf4<kCta>(d_tmem, a + 4, b + 4, idesc0, sfa + S::kScaleHalf, from + S::kScaleHalf, 1u);
            if (live > 3)
              ptx::umma_mxf4<kCta>(d_tmem, a + 6, b + 6, idesc2, sfa + S::kScaleHalf, from + S::kScaleHalf, 1u);
            if constexpr (kCta == 1)
              ptx::umma_commit<1>(empty_bar(s));
            else
              ptx::umma_commit_pair_both(empty_bar(s), 0x3);
          }
          __syncwarp();
          set ^= 1u;
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
    // ------------------------------------------------------------------ epilogue (warps 2..9)
    const uint32_t quad = warp & 3u;
    const int half = static_cast<int>(warp - 2u) >> 2;
    const uint32_t lead_empty0 = (kCta == 2) ? ptx::mapa(tmem_empty_bar(0), 0) : tmem_empty_bar(0);
    bool stored = false;  // this warp's staging buffer has been handed to a bulk store
    for (int t = first, j = 0; t < tiles; t += stride, ++j) {
      const uint32_t acc = static_cast<uint32_t>(j) & 1u;
      const uint32_t acc_ph = (static_cast<uint32_t>(j) >> 1) & 1u;
      if (!bounded_wait_warp(tmem_full_bar(acc), acc_ph, cta_abort, p.status, kFaultEpilogueWait, lane)) break;
      ptx::tc_fence_after();
      int mt, nt;
      tile_at(t, mt, nt);
      const int row0 = (mt * kCta + cta_rank) * 128 + static_cast<int>(quad) * 32;
      const uint32_t taddr = tmem_base + ((quad * 32u) << 16) + acc * S::kAccStep;
      if constexpr (kCta == 2) {
        // Columns in chunks of 64, the chunk that the other accumulator shares first: the last of an even tile, the first
        // of an odd one.  The two warps of a quarter take turns, so the first of them reads that chunk; the other's arrive
        // says that it has done with the tile before, whose accumulator the next tile goes into.
        const uint32_t buf = staging_base + (warp - 2u) * 2048u;
        auto hand_back = [&]() {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_cluster(lead_empty0);
        };
        if (half == 1) hand_back();
#pragma unroll 1
        for (int i = half; i < 4; i += 2) {
          const int c = 64 * (acc == 0 ? (i + 3) & 3 : i);
          uint32_t v[2][32];
          ptx::tmem_ld_32x32(taddr + c, v[0]);
          ptx::tmem_ld_32x32(taddr + c + 32, v[1]);
          ptx::tmem_ld_wait();
          if (i == 0) hand_back();
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            const int col = nt * 256 + c + 32 * part;
            if (row0 >= p.m || col >= p.n) continue;  // warp-uniform
            uint32_t out[16];
#pragma unroll
            for (int q = 0; q < 16; ++q)
              out[q] = ptx::pack_out2(__uint_as_float(v[part][2 * q]), __uint_as_float(v[part][2 * q + 1]), p.bf16);
            if (stored) {
              if (lane == 0) ptx::tma_store_wait_read<0>();
              __syncwarp();
            }
            // the 64-byte swizzle (see gated_umma.cuh)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              ptx::st_shared_v4(buf + lane * 64u + ((static_cast<uint32_t>(q) ^ ((lane >> 1) & 3u)) << 4), out[4 * q],
                                out[4 * q + 1], out[4 * q + 2], out[4 * q + 3]);
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              ptx::tma_store_2d(&p.tm_c, buf, col, row0);
              ptx::tma_store_commit();
            }
            stored = true;
          }
        }
      } else {
        const int col0 = nt * p.width;
        const int row = row0 + static_cast<int>(lane);
        for (int c = 32 * half; row0 < p.m && c < p.width && col0 + c < p.n; c += 64) {
          uint32_t v[32];
          mx_load(p, taddr + c, v);
          mx_store_row(p, v, row, col0 + c, 32);
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(tmem_empty_bar(acc));
      }
    }
  }

  if constexpr (kCta == 1) {
    if (p.split > 1) {
      // ---------------------------------------------------------------- a tile shared by a cluster: its epilogue
      const uint32_t split = static_cast<uint32_t>(p.split);
      const bool epilogue = warp >= 2 && warp < 2 + S::kEpilogueWarps;
      const uint32_t quad = warp & 3u;
      const int half = epilogue ? static_cast<int>(warp - 2u) >> 2 : 0;
      const uint32_t row = quad * 32u + lane;
      const uint32_t taddr = tmem_base + ((quad * 32u) << 16);
      const int slice = p.width / p.split;  // columns that each CTA finishes, a multiple of 8
      const uint32_t groups = static_cast<uint32_t>(slice) / 4u;
      bool ready = false;
      if (epilogue) {
        ready = bounded_wait_warp(tmem_full_bar(0), 0, cta_abort, p.status, kFaultEpilogueWait, lane);
        ptx::tc_fence_after();
        ready = ready && static_cast<int>(quad * 32u) < p.m;
      }
      ptx::cluster_sync_all();  // every CTA's operands have been multiplied: the rings may be written over
      if (ready) {
        int turn = 0;
        for (uint32_t to = 0; to < split; ++to) {
          if (to == k_rank) continue;
          const uint32_t there = ptx::mapa(smem_base, to);
          for (int c = 0; c < slice; c += 32) {
            if ((turn++ & 1) != half) continue;
            uint32_t v[32];
            mx_load(p, taddr + to * slice + c, v);
            if (static_cast<int>(row) < p.m)
              exchange_send(there, exchange_slot(k_rank, to), groups, static_cast<uint32_t>(c) / 4u, row, v, slice - c);
          }
        }
      }
      ptx::cluster_sync_all();
      if (ready) {
        const int col0 = first * p.width + static_cast<int>(k_rank) * slice;
        for (int c = 32 * half; c < slice && col0 + c < p.n; c += 64) {
          uint32_t v[32];
          mx_load(p, taddr + k_rank * slice + c, v);
          exchange_sum(smem_base, k_rank, split, groups, static_cast<uint32_t>(c) / 4u, row, v, slice - c);
          mx_store_row(p, v, static_cast<int>(row), col0 + c, min(32, slice - c));
        }
      }
    }
  }

  if (kCta == 2 && warp >= 2 && warp < 2 + S::kEpilogueWarps && lane == 0) ptx::tma_store_wait_read<0>();
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

}  // namespace beam
