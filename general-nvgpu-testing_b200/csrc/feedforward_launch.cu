// Host launchers of the gated product and of the gradients of rc products.
#include "feedforward_launch.h"

#include "gated_umma.cuh"
#include "grad_umma.cuh"
#include "launch_common.h"

namespace beam {

namespace {

struct GatedPlan {
  int ctas;       // per tile
  int width;      // columns of F per tile
  int split = 1;  // CTAs that share a tile's contraction (single-CTA tiles only)
};

// Up to 128 rows one CTA's tile holds them all and the weights are read once whatever the width, so the width only deals out F:
// the smallest multiple of 8 with which the columns take as few waves of all SMs as 128-wide tiles would.  While that
// leaves a CTA more k-blocks than bytes (a k-block takes its issuers about 0.14 us, in which an SM's share of the measured
// bandwidth is a width of 24), clusters of 2 or 4 CTAs share a tile's contraction: wider tiles over fewer k-blocks, for an exchange
// of sums at the end.  Measured, one row, us with 1 / 2 / 4 CTAs: F = 512, K = 4096 11.2 / 9.0 / 8.5; 2048, 4096 12.0 / 10.9 / 12.1; 4096, 4096 14.9 / 15.7 / 17.2;
// 1024, 8192 18.6 / 13.3 / 12.2; 1024, 2048 7.7 / 7.3 / 7.7; 512, 1024 6.0 / 6.4 / 7.2.
//
// Above, pairs work on 256 rows.  A wave of narrower tiles is shorter, but not in proportion (A is read as often, and a UMMA
// of N <= 128 is bound by its issue); measured per wave at K = 4096, in percent of a wave of 128-wide tiles: 96 columns 73 alone
// and 78 among many waves, 64 columns 60, 32 columns 55.  The width with the least total is taken, the wider of two
// that are equal: 128 for all large problems (4096 x 16384 x 4096: 681 us against 697 with 96 and 823 with 64), the narrowest
// that still takes one wave for small ones (256 x 2048 x 2048: 11.1 us with 32 against 16.2 with 128).  Pairs do not share a
// contraction, so narrow layers with a long K take a step at 129 rows: 128 / 129 / 256 rows x 512 x 8192 11.4 / 16.8 / 16.9 us,
// 1024 x 8192 12.9 / 17.2 / 17.3, 2048 x 8192 18.6 / 21.9 / 23.6, 2048 x 4096 12.0 / 11.8 / 12.2.
GatedPlan gated_plan(int m, int f, int k, const int (&fit)[4]) {
  GatedPlan plan;
  if (m <= 128) {
    plan.ctas = 1;
    const int waves = ceil_div(f, 128 * fit[0]);
    plan.width = (ceil_div(f, waves * fit[0]) + 7) / 8 * 8;
    const int num_kb = ceil_div(k, 64);
    const int split = plan.width <= 8 && num_kb >= 48 ? 4 : plan.width <= 16 && num_kb >= 32 ? 2 : 1;
    const int step = 8 * split;  // every CTA finishes a multiple of 8 columns
    const int shared_width = (ceil_div(f, fit[split / 2]) + step - 1) / step * step;
    if (split > 1 && shared_width <= 128) {
      plan.split = split;
      plan.width = shared_width;
    }
    return plan;
  }
  const int pairs = fit[3];
  plan.ctas = 2;
  const int widths[4] = {128, 96, 64, 32}, wave_cost[4] = {100, 80, 61, 55};
  long long best = 0;
  for (int i = 0; i < 4; ++i) {
    const long long tiles = static_cast<long long>(ceil_div(m, 256)) * ceil_div(f, widths[i]);
    const long long cost = (tiles + pairs - 1) / pairs * wave_cost[i];
    if (i == 0 || cost < best) {
      best = cost;
      plan.width = widths[i];
    }
  }
  return plan;
}

template <int kCta>
int launch_gated_instance(DeviceCtx* ctx, const GatedPlan& plan, int resident, const void* A, const void* Bg,
                          const void* Bu, void* C, void* G, void* U, int m, int f, int k, int activation, int bf16,
                          cudaStream_t stream) {
  using S = GatedShape<kCta>;
  GatedParams p = {};
  p.m = m;
  p.f = f;
  p.k = k;
  p.width = plan.width;
  p.act = activation;
  p.bf16 = bf16;
  p.out[0] = C;
  p.out[1] = G;
  p.out[2] = U;
  p.status = ctx->status_word;
  p.a_rows = kCta == 2 ? S::kBM : (m + 7) / 8 * 8;
  // A UMMA multiplies 128 rows of A whether they exist or not.  Wide tiles keep zeros in the missing ones: with whatever lies
  // there instead, a sustained run of one row x 16384 x 4096 is held at 1.24 GHz by the power cap (49.5 us a call, 46.8 with
  // zeros).  Narrow tiles want their shared memory for a deeper ring (1 x 4096 x 4096: 15.7 us, 16.4 with zeros).
  p.a_bytes = kCta == 1 && p.width < 48 ? p.a_rows * 128 : S::kABytes;
  p.stage_bytes = p.a_bytes + p.width * 128 * (kCta == 2 ? 1 : 2);
  p.m_tiles = ceil_div(m, S::kBM * kCta);
  p.n_tiles = ceil_div(f, p.width);
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  const int clusters = tiles < resident ? static_cast<int>(tiles) : resident;
  p.split = plan.split;
  // Two issuers for UMMAs of N <= 128; every CTA must have a k-block for each.
  p.issuers = p.width <= 64 && k > S::kBK * p.split * 2 ? 2 : 1;
  // A UMMA reads 128 rows of A whether they were loaded or not: behind the last stage there is room for them.
  const int a_slack = S::kABytes - p.a_bytes;
  p.stages = (S::kRingBytes - a_slack) / p.stage_bytes;
  if (p.stages > S::kMaxStages) p.stages = S::kMaxStages;
  if (p.issuers == 2) p.stages &= ~1;
  // 16 row tiles per group: the weights are read twice per 8192 rows.  8192 x 16384 x 4096, sustained, with 8 / 12 / 16 / 20 / 32:
  // 1588 / 1570 / 1527 / 1551 / 1660 us (cuBLAS, the two products alone: 1566).
  p.group_m = 16;
  int st = encode_tmap_2d(&p.tm_a, A, 2, m, k, k, static_cast<uint32_t>(p.a_rows), S::kBK, true);
  if (st == BEAM_OK) st = encode_tmap_2d(&p.tm_gate, Bg, 2, f, k, k, static_cast<uint32_t>(p.width), S::kBK, true);
  if (st == BEAM_OK) st = encode_tmap_2d(&p.tm_up, Bu, 2, f, k, k, static_cast<uint32_t>(p.width), S::kBK, true);
  if (kCta == 2) {
    for (int i = 0; i < 3 && st == BEAM_OK; ++i)
      if (p.out[i]) st = encode_tmap_2d_sw64(&p.tm_out[i], p.out[i], m, f, f, 32, 32);
  }
  if (st != BEAM_OK) return st;
  const int exchange = (p.split - 1) * (p.width / p.split) * 2 * 128 * 4;  // what the others of a cluster send
  p.bar_offset = p.stages * p.stage_bytes + a_slack + S::kStagingBytes;
  if (p.bar_offset < exchange) p.bar_offset = exchange;
  // CTAs that wait for one another must not share an SM with CTAs of another launch that do: each of two could hold the TMEM
  // that the other's peer waits for.  Taking all shared memory keeps such launches apart.
  const int smem = p.split > 1 ? S::kSmemLimit : p.bar_offset + S::kBarBytes + 1024;
  const int ctas = kCta * p.split;
  return launch_dependent(gated_umma_kernel<kCta>, clusters * ctas, S::kThreads, smem, ctas, stream,
                          "cudaLaunchKernelEx(gated_umma)", p);
}

int check_sizes(int m, int n, int k) {
  if (m <= 0 || n <= 0 || k <= 0) return BEAM_ERR_INVALID_ARG;
  if (k % 8 != 0 || n % 8 != 0) return BEAM_ERR_ALIGNMENT;
  // tiles are counted in 32 bits
  if (static_cast<long long>(ceil_div(m, 128)) * ceil_div(n, 8) > (1ll << 30)) return BEAM_ERR_UNSUPPORTED;
  return BEAM_OK;
}

}  // namespace

int launch_gated(const void* A, const void* Bg, const void* Bu, void* C, void* G, void* U, int m, int f, int k,
                 int activation, int bf16, cudaStream_t stream) {
  if (!A || !Bg || !Bu || !C || (G == nullptr) != (U == nullptr)) return BEAM_ERR_INVALID_ARG;
  if (activation < kActSilu || activation > kActRelu) return BEAM_ERR_INVALID_ARG;
  int st = check_sizes(m, f, k);
  if (st != BEAM_OK) return st;
  if (!aligned16(A) || !aligned16(Bg) || !aligned16(Bu) || !aligned16(C) || !aligned16(G) || !aligned16(U))
    return BEAM_ERR_ALIGNMENT;
  const size_t ab = 2ull * m * k, bb = 2ull * f * k, cb = 2ull * m * f;
  const void* outs[3] = {C, G, U};
  for (int i = 0; i < 3; ++i) {
    if (overlap(outs[i], cb, A, ab) || overlap(outs[i], cb, Bg, bb) || overlap(outs[i], cb, Bu, bb) ||
        overlap(outs[i], cb, outs[(i + 1) % 3], cb))
      return BEAM_ERR_INVALID_ARG;
  }
  DeviceCtx* ctx = current_device_ctx(&st);
  if (!ctx) return st;
  static ResidentTable table[4];
  int fit[4];  // single CTAs; clusters of 2 and 4 CTAs that share a contraction; pairs
  for (int i = 0; i < 3 && st == BEAM_OK; ++i)
    st = resident_grid(&table[i], gated_umma_kernel<1>, ctx, GatedShape<1>::kThreads, GatedShape<1>::kSmemLimit, 1 << i,
                       &fit[i]);
  if (st == BEAM_OK)
    st = resident_grid(&table[3], gated_umma_kernel<2>, ctx, GatedShape<2>::kThreads, GatedShape<2>::kSmemLimit, 2,
                       &fit[3]);
  if (st != BEAM_OK) return st;
  const GatedPlan plan = gated_plan(m, f, k, fit);
  return plan.ctas == 1 ? launch_gated_instance<1>(ctx, plan, plan.split == 1 ? fit[0] : plan.split == 2 ? fit[1] : fit[2], A,
                                                   Bg, Bu, C, G, U, m, f, k, activation, bf16, stream)
                        : launch_gated_instance<2>(ctx, plan, fit[3], A, Bg, Bu, C, G, U, m, f, k, activation, bf16, stream);
}

namespace {

// One product of a gradient launch (see GradJob).
struct JobSpec {
  const void* a[2];
  const void* b[2];
  void* c;
  int rows, cols, contraction, segments;
  bool a_mn;
  int slices = 1;

  long long tiles() const { return static_cast<long long>(ceil_div(rows, 256)) * ceil_div(cols, 256); }
  int k_blocks() const { return ceil_div(contraction, GradShape::kBK) * segments; }
  size_t plane_bytes() const { return 4ull * rows * cols; }
  size_t scratch_bytes() const { return slices > 1 ? (slices * plane_bytes() + 255) / 256 * 256 : 0; }
};

// How many slices each job's contraction is cut into: what lets the first pair finish soonest, which has an item of every round of
// the list (longest items first), plus the time to add the planes.  An item takes its k-blocks, a slice kSliceMore more (its planes
// are twice the bytes), and no less than kItemLeast, its epilogue; adding planes costs kSumLaunch and a unit per kSumBytes (all
// in units of a k-block, 0.33 us; a few more or less of each choose the same).  Planned as if all gradients were wanted,
// so that the bits of one do not depend on which others are asked for.  Measured, us, with slices of an even share of all
// k-blocks / by this rule: gated gradients of 333 x 2744 x 1000 (8 tiles of 86 k-blocks in 7 slices and 88 tiles of 6: two rounds of
// 74 pairs) 22.4 / 21.2, 1000 x 4096 x 1024 42.8 / 36.3, 129 x 11008 x 4096 120 / 95; product gradients of 8 x 8192 x 8192
// 83.1 / 65.2, 4096 x 1024 x 1024 22.8 / 19.5, 333 x 1000 x 1000 10.7 / 9.5; the worst found: 300 x 4096 x 512 11.3 / 12.1,
// 3000 x 512 x 4096 26.9 / 28.0.  32 slices: 8192 x 256 x 256 11.2 -> 11.7, 100 x 8192 x 1024 18.0 -> 18.3.
constexpr int kMaxSlices = 16, kLeastSlice = 4;  // k-blocks
constexpr float kItemLeast = 5.f, kSumLaunch = 5.f, kSumBytes = 1.3e6f, kSliceMore = 2.f;

struct PlannedJob {
  float k_blocks, plane_units;  // the latter: bytes of a plane / kSumBytes
  long long tiles;
  int slices;
};

float plan_cost(const PlannedJob* jobs, int n, int pairs) {
  float length[kMaxGradJobs], cost = 0.f, sums = 0.f;
  long long items[kMaxGradJobs], first = 0, rounds = 0;
  for (int i = 0; i < n; ++i) {
    const PlannedJob& job = jobs[i];
    float l = job.k_blocks / static_cast<float>(job.slices) + (job.slices > 1 ? kSliceMore : 0.f);
    if (l < kItemLeast) l = kItemLeast;
    int at = i;
    for (; at > 0 && length[at - 1] < l; --at) {
      length[at] = length[at - 1];
      items[at] = items[at - 1];
    }
    length[at] = l;
    items[at] = job.tiles * job.slices;
    if (job.slices > 1) sums += (static_cast<float>(job.slices) + 0.5f) * job.plane_units;  // read; half as much written
  }
  for (int i = 0; i < n; ++i) {
    first += items[i];
    const long long until = (first + pairs - 1) / pairs;
    cost += length[i] * static_cast<float>(until - rounds);
    rounds = until;
  }
  return sums > 0.f ? cost + kSumLaunch + sums : cost;
}

void plan_slices(JobSpec* jobs, int n, int pairs) {
  PlannedJob plan[kMaxGradJobs];
  for (int i = 0; i < n; ++i)
    plan[i] = {static_cast<float>(jobs[i].k_blocks()), static_cast<float>(jobs[i].plane_bytes()) / kSumBytes, jobs[i].tiles(), 1};
  float best = plan_cost(plan, n, pairs);
  for (int i = 0; i < n; ++i) {
    const int most = jobs[i].k_blocks() / kLeastSlice;
    for (int slices = 2; slices <= most && slices <= kMaxSlices; ++slices) {
      plan[i].slices = slices;
      const float cost = plan_cost(plan, n, pairs);
      if (cost < best) {
        best = cost;
        jobs[i].slices = slices;
      }
    }
    plan[i].slices = jobs[i].slices;
  }
}

int add_job(GradParams* p, const JobSpec& s, void* scratch) {
  GradJob& job = p->job[p->jobs];
  for (int i = 0; i < s.segments; ++i) {
    int st = s.a_mn ? encode_tmap_2d(&job.tm_a[i], s.a[i], 2, s.contraction, s.rows, s.rows, 64, 64, true)
                    : encode_tmap_2d(&job.tm_a[i], s.a[i], 2, s.rows, s.contraction, s.contraction, 128, 64, true);
    if (st == BEAM_OK) st = encode_tmap_2d(&job.tm_b[i], s.b[i], 2, s.contraction, s.cols, s.cols, 64, 64, true);
    if (st != BEAM_OK) return st;
  }
  const int st = s.slices > 1 ? encode_tmap_3d_f32(&job.tm_c, scratch, s.slices, s.rows, s.cols, 32, 32)
                              : encode_tmap_2d(&job.tm_c, s.c, 2, s.rows, s.cols, s.cols, 32, 64, true);
  if (st != BEAM_OK) return st;
  job.rows = s.rows;
  job.cols = s.cols;
  job.contraction = s.contraction;
  job.segments = s.segments;
  job.a_mn = s.a_mn ? 1 : 0;
  job.slices = s.slices;
  job.m_tiles = ceil_div(s.rows, 256);
  job.n_tiles = ceil_div(s.cols, 256);
  job.first_item = p->end;
  p->end += job.m_tiles * job.n_tiles * s.slices;
  ++p->jobs;
  return BEAM_OK;
}

int grad_pairs(DeviceCtx* ctx, int* pairs) {
  static ResidentTable table;
  return resident_grid(&table, grad_umma_kernel, ctx, GradShape::kThreads, GradShape::kSmemBytes, 2, pairs);
}

// The pairs that scratch sizes are computed for: the current device's, or 74 without one.
int planned_pairs() {
  int st = BEAM_OK, pairs = 0;
  DeviceCtx* ctx = current_device_ctx(&st);
  return ctx && grad_pairs(ctx, &pairs) == BEAM_OK ? pairs : 74;
}

size_t grad_scratch_bytes(const JobSpec* jobs, int n) {
  size_t bytes = 0;
  for (int i = 0; i < n; ++i) bytes += jobs[i].scratch_bytes();
  return bytes;
}

// Launches the planned jobs that have an output; `scratch` holds grad_scratch_bytes() of them.
int launch_grad(DeviceCtx* ctx, JobSpec* jobs, int n, int pairs, uint8_t* scratch, int bf16, cudaStream_t stream) {
  for (int i = 1; i < n; ++i)  // longest items first
    for (int j = i; j > 0 && jobs[j].k_blocks() / jobs[j].slices > jobs[j - 1].k_blocks() / jobs[j - 1].slices; --j) {
      const JobSpec t = jobs[j];
      jobs[j] = jobs[j - 1];
      jobs[j - 1] = t;
    }
  GradParams p = {};
  GradReduceParams r = {};
  p.bf16 = r.bf16 = bf16;
  long long groups = 0;
  for (int i = 0; i < n; ++i) {
    if (!jobs[i].c) continue;
    const int st = add_job(&p, jobs[i], scratch);
    if (st != BEAM_OK) return st;
    if (jobs[i].slices > 1) {
      r.planes[r.jobs] = reinterpret_cast<const float4*>(scratch);
      r.out[r.jobs] = static_cast<uint2*>(jobs[i].c);
      r.groups[r.jobs] = static_cast<long long>(jobs[i].rows) * (jobs[i].cols / 4);
      r.slices[r.jobs] = jobs[i].slices;
      groups += r.groups[r.jobs++];
      scratch += jobs[i].scratch_bytes();
    }
  }
  p.group_m = 8;
  p.status = ctx->status_word;
  // Launches of whole waves, each at least kLaunchKBlocks k-blocks per pair (see grad_umma.cuh); a small list is one launch.
  constexpr int kLaunchKBlocks = 1024;  // 0.33 ms at full clocks
  const int items = p.end;
  int st = BEAM_OK;
  for (p.begin = 0; p.begin < items && st == BEAM_OK; p.begin = p.end) {
    long long k_blocks = 0;
    int end = p.begin;
    for (int j = 0; end < items && k_blocks < kLaunchKBlocks; end += pairs) {
      while (j + 1 < p.jobs && end >= p.job[j + 1].first_item) ++j;
      k_blocks += ceil_div(p.job[j].contraction, GradShape::kBK) * p.job[j].segments / p.job[j].slices;
      if (k_blocks == 0) k_blocks = 1;
    }
    p.end = end < items ? end : items;
    const int clusters = p.end - p.begin < pairs ? p.end - p.begin : pairs;
    st = launch_dependent(grad_umma_kernel, clusters * 2, GradShape::kThreads, GradShape::kSmemBytes, 2, stream,
                          "cudaLaunchKernelEx(grad_umma)", p);
  }
  if (st != BEAM_OK || r.jobs == 0) return st;
  return launch_dependent(grad_reduce_kernel, static_cast<int>((groups + 127) / 128), 128, 0, 1, stream,
                          "cudaLaunchKernelEx(grad_reduce)", r);
}

size_t slope_bytes(int m, int f) { return (2ull * m * f + 255) / 256 * 256; }

template <bool kBf16>
int launch_slope(DeviceCtx* ctx, const GatedSlopeParams& p, cudaStream_t stream) {
  long long blocks = (p.count8 + 255) / 256;
  const long long most = 8ll * ctx->sm_count;  // 2048 threads on every SM
  if (blocks > most) blocks = most;
  auto run = [&](auto kernel) {
    return launch_dependent(kernel, static_cast<int>(blocks), 256, 0, 1, stream, "cudaLaunchKernelEx(gated_slope)", p);
  };
  switch (p.act) {
    case kActSilu: return run(gated_slope_kernel<kActSilu, kBf16>);
    case kActGelu: return run(gated_slope_kernel<kActGelu, kBf16>);
    case kActGeluTanh: return run(gated_slope_kernel<kActGeluTanh, kBf16>);
    default: return run(gated_slope_kernel<kActRelu, kBf16>);
  }
}

}  // namespace

namespace {

// The products of a gated backward pass and of an rc GEMM's, planned; an output that is not wanted is null.
void gated_jobs(JobSpec (&jobs)[3], const void* dG, const void* dU, const void* A, const void* Bg, const void* Bu, void* dA,
                void* dBg, void* dBu, int m, int f, int k, int pairs) {
  jobs[0] = {{dG, dU}, {Bg, Bu}, dA, m, k, f, 2, false};
  jobs[1] = {{dG, nullptr}, {A, nullptr}, dBg, f, k, m, 1, true};
  jobs[2] = {{dU, nullptr}, {A, nullptr}, dBu, f, k, m, 1, true};
  plan_slices(jobs, 3, pairs);
}

void rc_jobs(JobSpec (&jobs)[2], const void* dC, const void* A, const void* B, void* dA, void* dB, int m, int n, int k,
             int pairs) {
  jobs[0] = {{dC, nullptr}, {B, nullptr}, dA, m, k, n, 1, false};
  jobs[1] = {{dC, nullptr}, {A, nullptr}, dB, n, k, m, 1, true};
  plan_slices(jobs, 2, pairs);
}

}  // namespace

size_t gated_backward_workspace_bytes(int m, int f, int k) {
  if (check_sizes(m, f, k) != BEAM_OK || check_sizes(f, k, f) != BEAM_OK) return 0;
  JobSpec jobs[3];
  gated_jobs(jobs, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, m, f, k, planned_pairs());
  return 2 * slope_bytes(m, f) + grad_scratch_bytes(jobs, 3);
}

size_t gemmrc_backward_workspace_bytes(int m, int n, int k) {
  if (check_sizes(m, n, k) != BEAM_OK || check_sizes(n, k, n) != BEAM_OK) return 0;
  JobSpec jobs[2];
  rc_jobs(jobs, nullptr, nullptr, nullptr, nullptr, nullptr, m, n, k, planned_pairs());
  return grad_scratch_bytes(jobs, 2);
}

int launch_gated_backward(const void* dC, const void* A, const void* Bg, const void* Bu, const void* G, const void* U,
                          void* dA, void* dBg, void* dBu, int m, int f, int k, int activation, int bf16,
                          void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (!dC || !G || !U || (!dA && !dBg && !dBu)) return BEAM_ERR_INVALID_ARG;
  if (dA && (!Bg || !Bu)) return BEAM_ERR_INVALID_ARG;
  if ((dBg || dBu) && !A) return BEAM_ERR_INVALID_ARG;
  if (activation < kActSilu || activation > kActRelu) return BEAM_ERR_INVALID_ARG;
  int st = check_sizes(m, f, k);
  if (st == BEAM_OK) st = check_sizes(f, k, f);
  if (st != BEAM_OK) return st;
  const void* all[] = {dC, A, Bg, Bu, G, U, dA, dBg, dBu, workspace};
  for (const void* q : all)
    if (!aligned16(q)) return BEAM_ERR_ALIGNMENT;
  const size_t mk = 2ull * m * k, fk = 2ull * f * k, mf = 2ull * m * f;
  const size_t bytes[] = {mf, mk, fk, fk, mf, mf, mk, fk, fk, workspace_bytes};
  for (int o = 6; o < 10; ++o)
    for (int i = 0; i < o; ++i)
      if (overlap(all[o], bytes[o], all[i], bytes[i])) return BEAM_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < 2 * slope_bytes(m, f)) return BEAM_ERR_WORKSPACE;
  DeviceCtx* ctx = current_device_ctx(&st);
  if (!ctx) return st;
  int pairs = 0;
  st = grad_pairs(ctx, &pairs);
  if (st != BEAM_OK) return st;

  uint8_t* dG = static_cast<uint8_t*>(workspace);
  uint8_t* dU = dG + slope_bytes(m, f);
  JobSpec jobs[3];
  gated_jobs(jobs, dG, dU, A, Bg, Bu, dA, dBg, dBu, m, f, k, pairs);
  if (workspace_bytes < 2 * slope_bytes(m, f) + grad_scratch_bytes(jobs, 3)) return BEAM_ERR_WORKSPACE;
  GatedSlopeParams sp = {};
  sp.dc = static_cast<const uint4*>(dC);
  sp.gate = static_cast<const uint4*>(G);
  sp.up = static_cast<const uint4*>(U);
  sp.dgate = reinterpret_cast<uint4*>(dG);
  sp.dup = reinterpret_cast<uint4*>(dU);
  sp.count8 = static_cast<long long>(m) * (f / 8);
  sp.act = activation;
  st = bf16 ? launch_slope<true>(ctx, sp, stream) : launch_slope<false>(ctx, sp, stream);
  if (st != BEAM_OK) return st;
  return launch_grad(ctx, jobs, 3, pairs, dU + slope_bytes(m, f), bf16, stream);
}

int launch_gemmrc_backward(const void* dC, const void* A, const void* B, void* dA, void* dB, int m, int n, int k,
                           int bf16, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (!dC || (!dA && !dB) || (dA && !B) || (dB && !A)) return BEAM_ERR_INVALID_ARG;
  int st = check_sizes(m, n, k);
  if (st == BEAM_OK) st = check_sizes(n, k, n);
  if (st != BEAM_OK) return st;
  const void* all[] = {dC, A, B, dA, dB, workspace};
  for (const void* q : all)
    if (!aligned16(q)) return BEAM_ERR_ALIGNMENT;
  const size_t mk = 2ull * m * k, nk = 2ull * n * k, mn = 2ull * m * n;
  const size_t bytes[] = {mn, mk, nk, mk, nk, workspace_bytes};
  for (int o = 3; o < 6; ++o)
    for (int i = 0; i < o; ++i)
      if (overlap(all[o], bytes[o], all[i], bytes[i])) return BEAM_ERR_INVALID_ARG;
  DeviceCtx* ctx = current_device_ctx(&st);
  if (!ctx) return st;
  int pairs = 0;
  st = grad_pairs(ctx, &pairs);
  if (st != BEAM_OK) return st;
  JobSpec jobs[2];
  rc_jobs(jobs, dC, A, B, dA, dB, m, n, k, pairs);
  const size_t need = grad_scratch_bytes(jobs, 2);
  if (need > 0 && (!workspace || workspace_bytes < need)) return BEAM_ERR_WORKSPACE;
  return launch_grad(ctx, jobs, 2, pairs, static_cast<uint8_t*>(workspace), bf16, stream);
}

}  // namespace beam
