// The gradients of rc products as one persistent kernel on CTA pairs.  For C = A B^T with A [M, K], B [N, K]:
//
//   dA = dC B        contraction over N: dC is K-major as in the rc GEMM, B runs along memory with its output columns
//   dB = dC^T A      contraction over M: both operands run along memory with their output rows and columns
//
// Nothing is transposed in memory: TMA drops 64 x 64 boxes of the operand whose contraction runs over the rows of
// memory, and the UMMA descriptors read them as M- or N-major (umma_desc_mn_sw128).  In both products the right operand
// is N-major; the left one is K-major for dA and M-major for dB.
//
// A launch carries up to three jobs (dA; dB; for the gated product dA, dBg and dBu), each with its own tensor maps, and
// the tiles of all jobs form one list: the last wave of one product is filled up by the first tiles of the next, and
// dC's rows are still in L2 when the other product reads them.  Jobs are listed longest contraction first.  A job may
// have two segments, accumulated one after the other into the same tile: dA = dG Bg + dU Bu needs no second pass.
//
// A long list is cut into launches of whole waves.  Pairs drift apart over many tiles, and what they no longer read at the same
// time comes from memory again: all gradients of 8192 x 16384 x 4096 read 10.8 GB in one launch and 5.1 GB in seven, and
// memory traffic costs clock under the power cap.  Sustained, with all waves in one launch / 14 / 7 / 4 / 2 / 1 waves per
// launch: 3806 / 3564 / 3525 / 3516 / 3534 / 3612 us; by k-blocks (see the launcher): 3512 us.
//
// A job with few tiles and a long contraction (dA of a short batch: M rows, but F or N steps) is cut into slices of its
// contraction, so that it does not keep a few pairs busy while the others are done.  A slice stores its fp32 sums as a plane of
// scratch and grad_reduce_kernel adds the planes in order (the rule stands beside plan_slices() in feedforward_launch.cu).
//
// Tiles are 256 x 256 on a cta_group::2 pair, two TMEM accumulators, fp32 throughout, rounded once at the store.
// Roles: warp 0 loads the left operand, warp 6 the right one (an N-major k-block is two boxes; one thread issuing all
// four copies of a k-block would be slower than the tensor pipe), warp 1 issues UMMAs, warps 2..5 are the epilogue.
#pragma once

#include <type_traits>

#include "umma_common.cuh"

namespace beam {

constexpr int kMaxGradJobs = 3;

struct GradJob {
  CUtensorMap tm_a[2];  // left operand of each segment: [rows, contraction], box 128 x 64, or M-major: box 64 x 64
  CUtensorMap tm_b[2];  // right operand of each segment: [contraction, columns], box 64 x 64
  CUtensorMap tm_c;     // [rows, columns], store box 32 rows x 64 columns; of a sliced job the scratch planes
                        // [slices][rows][columns] fp32, store box 32 rows x 32 columns
  int rows, cols;
  int contraction;      // of each segment
  int segments;
  int a_mn;             // the left operand is M-major
  int slices;           // of the contraction over all segments
  int m_tiles, n_tiles;
  int first_item;       // of this job in the launch's list: an item is a tile, or a slice of one
};

struct GradParams {
  GradJob job[kMaxGradJobs];
  int jobs;
  int begin, end;  // this launch's part of the list of items
  int group_m;
  int bf16;
  int* status;
};

struct GradShape {
  static constexpr int kBK = 64;
  static constexpr int kABytes = 128 * kBK * 2;
  static constexpr int kBBytes = 128 * kBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 6;
  static constexpr int kBufBytes = 32 * 128;
  static constexpr int kStagingBytes = 4 * 2 * kBufBytes;
  static constexpr int kBarBytes = 512;
  static constexpr int kSmemBytes = kStages * kStageBytes + kStagingBytes + kBarBytes + 1024;
  static constexpr int kThreads = 224;
  static_assert(kSmemBytes <= 232448, "exceeds the 227 KB of shared memory a CTA can opt in to");
};

struct GradItem {
  int mt, nt;
  int kb0, kb1;  // k-blocks, counted over all segments
  int slice;
};
__device__ __forceinline__ const GradJob& grad_item(const GradParams& p, int t, GradItem& w) {
  int i = 0;
  while (i + 1 < p.jobs && t >= p.job[i + 1].first_item) ++i;
  const GradJob& job = p.job[i];
  t -= job.first_item;
  w.slice = t % job.slices;
  t /= job.slices;
  const int per_group = p.group_m * job.n_tiles;
  const int g = t / per_group;
  const int first_m = g * p.group_m;
  const int rows = min(p.group_m, job.m_tiles - first_m);
  const int r = t - g * per_group;
  w.mt = first_m + r % rows;
  w.nt = r / rows;
  const int all = (job.contraction + GradShape::kBK - 1) / GradShape::kBK * job.segments;
  w.kb0 = all * w.slice / job.slices;
  w.kb1 = all * (w.slice + 1) / job.slices;
  return job;
}

static __global__ void __launch_bounds__(GradShape::kThreads, 1) grad_umma_kernel(const __grid_constant__ GradParams p) {
  using S = GradShape;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t warp = ptx::warp_index();
  const uint32_t lane = threadIdx.x & 31;
  const int cta_rank = static_cast<int>(ptx::cluster_ctarank());
  const bool leader = cta_rank == 0;
  const int first = p.begin + static_cast<int>(blockIdx.x >> 1);
  const int stride = static_cast<int>(gridDim.x >> 1);

  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
  const uint32_t staging_base = smem_base + S::kStages * S::kStageBytes;
  const uint32_t bar_base = staging_base + S::kStagingBytes;
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (S::kStages + s); };
  auto tmem_full_bar = [&](uint32_t a) { return bar_base + 8u * (2 * S::kStages + a); };
  auto tmem_empty_bar = [&](uint32_t a) { return bar_base + 8u * (2 * S::kStages + 2 + a); };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(
      smem_gen + S::kStages * S::kStageBytes + S::kStagingBytes + 8 * (2 * S::kStages + 4));
  volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  if (warp == 0) {
    if (lane < S::kStages) {
      ptx::mbar_init(full_bar(lane), 1);
      ptx::mbar_init(empty_bar(lane), 1);
    }
    if (lane < 2) {
      ptx::mbar_init(tmem_full_bar(lane), 1);
      ptx::mbar_init(tmem_empty_bar(lane), 8);  // one arrive per epilogue warp of each CTA
    }
    ptx::fence_mbar_init();
    if (lane == 0) *cta_abort = 0;
    __syncwarp();
  }
  if (warp == 1) {
    ptx::tmem_alloc<2>(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    ptx::tmem_relinquish<2>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync_all();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  release_next_kernel(warp);

  if (warp == 0 || warp == 6) {
    // ------------------------------------------------------------------ TMA producers
    ptx::grid_dependency_wait();  // before the first global read
    const bool left = warp == 0;
    uint32_t s = 0, ph = 0;
    bool alive = true;
    for (int t = first; alive && t < p.end; t += stride) {
      GradItem w;
      const GradJob& job = grad_item(p, t, w);
      const int row = w.mt * 256 + cta_rank * 128;
      const int col = w.nt * 256 + cta_rank * 128;
      const int num_kb = (job.contraction + S::kBK - 1) / S::kBK;
      for (int at = w.kb0; at < w.kb1; ++at) {
        const int seg = at >= num_kb ? 1 : 0;
        const int kb = at - seg * num_kb;
        const CUtensorMap* map = left ? &job.tm_a[seg] : &job.tm_b[seg];
        if (!bounded_wait_converged(empty_bar(s), ph ^ 1u, cta_abort, p.status, kFaultProducerWait, lane)) {
          alive = false;
          break;
        }
        if (ptx::elect_one()) {
          // The left producer of the leader arms the barrier with all bytes of both CTAs; bytes of the right operand that
          // land before that only make the pending count negative for a moment, the phase still needs the arrive.
          if (left && leader) ptx::mbar_arrive_expect_tx(full_bar(s), 2u * S::kStageBytes);
          const uint32_t bar = ptx::mapa(full_bar(s), 0);
          const uint32_t a = smem_base + s * S::kStageBytes;
          if (left && !job.a_mn) {
            ptx::tma_load_2d_pair(a, map, bar, kb * S::kBK, row);
          } else {
            const uint32_t dst = left ? a : a + S::kABytes;
            const int along = left ? row : col;
            ptx::tma_load_2d_pair(dst, map, bar, along, kb * S::kBK);
            ptx::tma_load_2d_pair(dst + 8192u, map, bar, along + 64, kb * S::kBK);
          }
        }
        __syncwarp();
        if (++s == S::kStages) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (leader) {
      const uint32_t idesc0 = ptx::umma_idesc_f16_f32(256, 256) | ptx::kIdescBMnMajor |
                              (p.bf16 ? ptx::kIdescBf16Inputs : 0u);
      const uint64_t a_desc_k = ptx::umma_desc_k_sw128(smem_base);
      const uint64_t a_desc_mn = ptx::umma_desc_mn_sw128(smem_base);
      const uint64_t b_desc0 = ptx::umma_desc_mn_sw128(smem_base + S::kABytes);
      constexpr uint64_t kDescStride = S::kStageBytes >> 4;
      uint32_t s = 0, ph = 0;
      bool alive = true;
      for (int t = first, j = 0; alive && t < p.end; t += stride, ++j) {
        GradItem w;
        const GradJob& job = grad_item(p, t, w);
        const uint32_t acc = static_cast<uint32_t>(j) & 1u;
        const uint32_t acc_ph = (static_cast<uint32_t>(j) >> 1) & 1u;
        if (!bounded_wait_converged(tmem_empty_bar(acc), acc_ph ^ 1u, cta_abort, p.status, kFaultMmaWaitAcc, lane)) break;
        ptx::tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * 256u;
        const uint32_t idesc = idesc0 | (job.a_mn ? ptx::kIdescAMnMajor : 0u);
        const uint64_t a_desc0 = job.a_mn ? a_desc_mn : a_desc_k;
        const uint64_t a_step = job.a_mn ? (2048 >> 4) : (32 >> 4);  // 16 steps of the contraction
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!bounded_wait_converged(full_bar(s), ph, cta_abort, p.status, kFaultMmaWaitFull, lane)) {
            alive = false;
            break;
          }
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            const uint64_t a = a_desc0 + s * kDescStride, b = b_desc0 + s * kDescStride;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
              ptx::umma_f16<2>(d_tmem, a + i * a_step, b + i * (2048 >> 4), idesc, (kb > w.kb0 || i > 0) ? 1u : 0u);
            ptx::umma_commit_pair_both(empty_bar(s), 0x3);
          }
          __syncwarp();
          if (++s == S::kStages) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (alive && ptx::elect_one()) ptx::umma_commit_pair_both(tmem_full_bar(acc), 0x3);
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue (warps 2..5)
    const uint32_t quad = warp & 3u;
    const uint32_t lead_empty0 = ptx::mapa(tmem_empty_bar(0), 0);
    uint32_t stores = 0;
    for (int t = first, j = 0; t < p.end; t += stride, ++j) {
      GradItem w;
      const GradJob& job = grad_item(p, t, w);
      const uint32_t acc = static_cast<uint32_t>(j) & 1u;
      const uint32_t acc_ph = (static_cast<uint32_t>(j) >> 1) & 1u;
      if (!bounded_wait_warp(tmem_full_bar(acc), acc_ph, cta_abort, p.status, kFaultEpilogueWait, lane)) break;
      ptx::tc_fence_after();
      const int row0 = w.mt * 256 + cta_rank * 128 + static_cast<int>(quad) * 32;
      const uint32_t taddr = tmem_base + ((quad * 32u) << 16) + acc * 256u;
      const bool sliced = job.slices > 1;
      const int step = sliced ? 32 : 64;  // columns in 128 bytes
#pragma unroll 1
      for (int c = 0; c < 256; c += step) {
        const int col = w.nt * 256 + c;
        if (row0 >= job.rows || col >= job.cols) break;  // warp-uniform
        uint32_t out[32];
        ptx::tmem_ld_32x32(taddr + c, out);
        if (!sliced) {
          uint32_t v[32];
          ptx::tmem_ld_32x32(taddr + c + 32, v);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 16; ++q)
            out[q] = ptx::pack_out2(__uint_as_float(out[2 * q]), __uint_as_float(out[2 * q + 1]), p.bf16);
#pragma unroll
          for (int q = 0; q < 16; ++q)
            out[16 + q] = ptx::pack_out2(__uint_as_float(v[2 * q]), __uint_as_float(v[2 * q + 1]), p.bf16);
        } else {
          ptx::tmem_ld_wait();
        }
        const uint32_t buf = staging_base + (quad * 2u + (stores & 1u)) * S::kBufBytes;
        if (stores >= 2) {
          if (lane == 0) ptx::tma_store_wait_read<1>();
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          ptx::st_shared_v4(buf + lane * 128u + ((static_cast<uint32_t>(i) ^ (lane & 7u)) << 4), out[4 * i],
                            out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (sliced)
            ptx::tma_store_3d(&job.tm_c, buf, col, row0, w.slice);
          else
            ptx::tma_store_2d(&job.tm_c, buf, col, row0);
          ptx::tma_store_commit();
        }
        ++stores;
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(lead_empty0 + 8u * acc);
    }
  }

  if (warp >= 2 && warp < 6 && lane == 0) ptx::tma_store_wait_all<0>();
  __syncwarp();
  if (*cta_abort) abort_drain_delay();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync_all();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<2>(tmem_base, 512);
  }
}

// Adds the planes of the sliced jobs, in the order of the slices, and rounds once.  A thread does 4 columns.  Few threads have planes
// to add, so what counts is how many loads each has in flight: four at a time take 11.1 us for the gradients of 8192 x 256 x 256, one at
// a time 13.6, eight 11.0 but up to 6 % more where planes are larger (100 x 8192 x 1024: 17.1, 18.6, 18.1).  The planes are left in L2, where
// the next call writes them again: with loads that say they are the last 16384 x 512 x 512 takes 22.9 us, without 22.2.
struct GradReduceParams {
  const float4* planes[kMaxGradJobs];
  uint2* out[kMaxGradJobs];
  long long groups[kMaxGradJobs];  // of 4 elements
  int slices[kMaxGradJobs];
  int jobs;
  int bf16;
};

static __global__ void __launch_bounds__(128) grad_reduce_kernel(const __grid_constant__ GradReduceParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();  // see release_next_kernel()
  long long at = static_cast<long long>(blockIdx.x) * 128 + threadIdx.x;
  int i = 0;
  while (i < p.jobs && at >= p.groups[i]) at -= p.groups[i++];
  if (i == p.jobs) return;
  const long long plane = p.groups[i];
  const float4* from = p.planes[i] + at;
  const int slices = p.slices[i];
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  int s = 0;
  auto add = [&](auto planes) {  // loads that do not wait for one another
    float4 v[planes.value];
#pragma unroll
    for (int u = 0; u < planes.value; ++u) v[u] = __ldcg(from + (s + u) * plane);
#pragma unroll
    for (int u = 0; u < planes.value; ++u) {
      sum.x += v[u].x; sum.y += v[u].y; sum.z += v[u].z; sum.w += v[u].w;
    }
    s += planes.value;
  };
  while (s + 4 <= slices) add(std::integral_constant<int, 4>());
  if (s + 2 <= slices) add(std::integral_constant<int, 2>());
  if (s < slices) add(std::integral_constant<int, 1>());
  p.out[i][at] = make_uint2(ptx::pack_out2(sum.x, sum.y, p.bf16), ptx::pack_out2(sum.z, sum.w, p.bf16));
}

}  // namespace beam
