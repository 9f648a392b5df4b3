// Device-side helpers shared by the UMMA kernels: bounded mbarrier waits that turn a
// would-be hang into a status code, and the status codes themselves.
#pragma once

#include "sm100_ptx.cuh"

namespace beam {

// Values written to the device status word (0 = healthy). The host maps any non-zero
// value to BEAM_ERR_DEVICE_TIMEOUT and reports the raw word through beam_device_status().
enum DeviceFault : int {
  kFaultNone = 0,
  kFaultProducerWait = 0x101,  // TMA producer gave up waiting for a free pipeline stage
  kFaultMmaWaitFull = 0x102,   // MMA issuer gave up waiting for operand bytes
  kFaultMmaWaitAcc = 0x103,    // MMA issuer gave up waiting for a drained accumulator
  kFaultEpilogueWait = 0x104,  // epilogue gave up waiting for a finished accumulator
  kFaultReduceWait = 0x105,    // split-K / LayerNorm exchange wait ran out
};

// Every spin in these kernels goes through here. A wait gives up after kWaitLimitNs of wall
// time (or at once when another role of this CTA already gave up): it raises the CTA-wide
// abort flag, records `fault` in the global status word and returns false; callers then leave
// their role loops and fall through to the common teardown, which still frees TMEM.
// The time runs from when the kernel ahead on the stream has finished (at once in a kernel that did not start early), however
// long that takes: a role may be waiting for what its CTA will only load then.
constexpr uint64_t kWaitLimitNs = 2000ull * 1000ull * 1000ull;
constexpr uint32_t kSpinSuspendNs = 4000u;

__device__ __forceinline__ bool bounded_wait(uint32_t bar, uint32_t parity, volatile int* cta_abort,
                                             int* status_word, int fault, uint64_t limit_ns = kWaitLimitNs) {
  if (ptx::mbar_try_wait(bar, parity)) return true;
  uint64_t t0 = 0;
  for (uint32_t spin = 1;; ++spin) {
    // suspended in hardware until the phase completes or kSpinSuspendNs pass: few instructions while waiting
    if (ptx::mbar_try_wait_suspend(bar, parity, kSpinSuspendNs)) return true;
    if ((spin & 0x3Fu) == 0) {
      if (*cta_abort) return false;
      if (t0 == 0) ptx::grid_dependency_wait();
      const uint64_t now = ptx::globaltimer_ns();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > limit_ns) {
        *cta_abort = 1;
        if (status_word) atomicCAS(status_word, 0, fault);
        return false;
      }
    }
  }
}

// The same wait for whole warps (the epilogue, which sleeps through a tile's main loop): only lane 0 waits, suspended
// in hardware on the barrier for up to kSuspendNs at a time instead of polling, and the rest of the warp parks at
// the shuffle.  Returns the same value in every lane.
constexpr uint32_t kSuspendNs = 50000u;

__device__ __forceinline__ bool bounded_wait_warp(uint32_t bar, uint32_t parity, volatile int* cta_abort,
                                                  int* status_word, int fault, uint32_t lane,
                                                  uint64_t limit_ns = kWaitLimitNs) {
  int ok = 1;
  if (lane == 0) {
    if (!ptx::mbar_try_wait(bar, parity)) {
      uint64_t t0 = 0;
      for (uint32_t spin = 1;; ++spin) {
        if (ptx::mbar_try_wait_suspend(bar, parity, kSuspendNs)) break;
        if ((spin & 0xFu) == 0) {
          if (*cta_abort) {
            ok = 0;
            break;
          }
          if (t0 == 0) ptx::grid_dependency_wait();
          const uint64_t now = ptx::globaltimer_ns();
          if (t0 == 0) {
            t0 = now;
          } else if (now - t0 > limit_ns) {
            *cta_abort = 1;
            if (status_word) atomicCAS(status_word, 0, fault);
            ok = 0;
            break;
          }
        }
      }
    }
  }
  ok = __shfl_sync(0xffffffffu, ok, 0);
  return ok != 0;
}

// The same wait for warps that run their loop converged (see ptx::elect_one): every lane tests once, and when the phase is not
// complete yet lane 0 waits for all.  Returns the same value in every lane.
__device__ __forceinline__ bool bounded_wait_converged(uint32_t bar, uint32_t parity, volatile int* cta_abort,
                                                       int* status_word, int fault, uint32_t lane) {
  const bool hit = ptx::mbar_try_wait(bar, parity);
  if (__all_sync(0xffffffffu, hit)) return true;
  const bool ok = bounded_wait_warp(bar, parity, cta_abort, status_word, fault, lane);
  __syncwarp();
  return ok;
}

// Lets the kernel behind this one on the stream start, called by every warp once the CTA (pair) is set up and has its TMEM.  One
// warp of the epilogue, which has nothing to do yet, waits for the kernel ahead first.  The order matters:
//   * A kernel that starts has the one before its predecessor complete behind it.  A split-K call whose caller vouches for its
//     inputs (BEAM_FLAG_INPUTS_STABLE) reads them without a wait, so this is what that promise rests on.
//   * CTAs of the kernel behind may share an SM with this one's where shared memory allows (narrow gated products take 64 KB).  Let
//     in before this CTA had its TMEM, they could take it and then wait for this grid, which would wait for them.
// Chains of 512 x 512 x 512 products: 5.78 us a call, 5.80 with the release ahead of the wait, 6.02 if every warp waits here.
__device__ __forceinline__ void release_next_kernel(uint32_t warp) {
  if (warp == 2) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
  }
}

// ---- joining the sums of a contraction that the CTAs of a cluster have split among them
// Every CTA holds the sums over its own share of K, fp32 in TMEM.  Each finishes one slice of the columns: it sends the others'
// slices into their shared memory (their rings are idle by then) and adds what arrives to its own.  What one source sends is
// [groups of 4 columns][128 rows], so consecutive lanes write consecutive 16 bytes.  `valid` of the 32 columns are moved, a
// multiple of 4.
__device__ __forceinline__ uint32_t exchange_slot(uint32_t from, uint32_t to) { return from < to ? from : from - 1; }
__device__ __forceinline__ void exchange_send(uint32_t cluster_base, uint32_t slot, uint32_t groups, uint32_t group,
                                              uint32_t row, const uint32_t (&v)[32], int valid) {
  const uint32_t at = cluster_base + ((slot * groups + group) * 128u + row) * 16u;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (4 * i < valid)
      ptx::st_cluster_f32x4(at + i * 2048u, __uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                            __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
}
// v = the sum over all ranks, in their order; `v` comes in as this rank's own share.
__device__ __forceinline__ void exchange_sum(uint32_t base, uint32_t rank, uint32_t ranks, uint32_t groups, uint32_t group,
                                             uint32_t row, uint32_t (&v)[32], int valid) {
  float sum[32];
#pragma unroll
  for (int q = 0; q < 32; ++q) sum[q] = 0.f;
  for (uint32_t from = 0; from < ranks; ++from) {
    if (from == rank) {
#pragma unroll
      for (int q = 0; q < 32; ++q) sum[q] += __uint_as_float(v[q]);
    } else {
      const uint32_t at = base + ((exchange_slot(from, rank) * groups + group) * 128u + row) * 16u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (4 * i < valid) {
          const float4 x = ptx::ld_shared_f32x4(at + i * 2048u);
          sum[4 * i] += x.x;
          sum[4 * i + 1] += x.y;
          sum[4 * i + 2] += x.z;
          sum[4 * i + 3] += x.w;
        }
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 32; ++q) v[q] = __float_as_uint(sum[q]);
}

// After an abort, give asynchronous work this CTA already issued (TMA copies into its shared
// memory, UMMAs into its TMEM) time to land before shared memory and TMEM are released.
__device__ __forceinline__ void abort_drain_delay() {
  const uint64_t t0 = ptx::globaltimer_ns();
  while (ptx::globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
}

}  // namespace beam
