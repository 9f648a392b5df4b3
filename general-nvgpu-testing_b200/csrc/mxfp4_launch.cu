// Host launchers of MXFP4 quantisation and product.
#include "mxfp4_launch.h"

#include "launch_common.h"
#include "mxfp4_umma.cuh"

namespace beam {

namespace {

int check_matrix(int rows, int k) {
  if (rows <= 0 || k <= 0) return BEAM_ERR_INVALID_ARG;
  if (k % 32 != 0) return BEAM_ERR_ALIGNMENT;
  // units of 128 elements, with their padding, are counted in 32 bits
  if (static_cast<long long>(ceil_div(rows, 128)) * 128 * ceil_div(k, 128) > (1ll << 31) - 1024)
    return BEAM_ERR_UNSUPPORTED;
  return BEAM_OK;
}

size_t packed_bytes(int rows, int k) { return static_cast<size_t>(rows) * (k / 2); }

// Lays a grid of 256-thread blocks, 64 units of 128 elements each, over rows x K: as many blocks of K side by side as fit.
MxUnits lay_units(int rows, int k, int* grid) {
  MxUnits u = {};
  u.rows = rows;
  u.kblocks = static_cast<uint32_t>(ceil_div(k, 128));
  while (u.kb_shift < 4 && (1u << u.kb_shift) < u.kblocks) ++u.kb_shift;
  u.x_blocks = (u.kblocks + (1u << u.kb_shift) - 1) >> u.kb_shift;
  *grid = static_cast<int>(u.x_blocks) * ceil_div(rows, kMxUnits * 16 >> u.kb_shift);
  return u;
}

// Tiles for M <= 128.  B is read once whatever the tiles, so they only deal out N and K.  64 or 128 columns: a tile's scales start at
// the first or the third of the four TMEM columns of a scale block, and a UMMA takes scales from even columns only (a width
// of 32, which starts every other tile at an odd column, faulted with a misaligned address).  64 wherever that is one wave.
// Where SMs are left over and K is long, clusters of 2 or 4 CTAs share a tile's contraction.  Measured, one row, us with
// 1 / 2 / 4 CTAs: N = 2072, K = 8192 9.2 / 7.3 / 7.2; 1024, 4096 6.1 / 5.9 / 6.1; 4096, 4096 6.4 / 6.1; 2048, 2048 5.0 / 5.2 / 5.8; and
// with 128 columns 9.9 / 8.1 / 7.3, 6.9 / 6.5 / 6.3, 7.3 / 6.7, 5.6 / 5.6 / 5.9.
// Above 128 rows there is one form, 256 x 256 tiles on pairs over the whole of K.  It takes a step at 129 rows, since a few tiles
// leave most pairs without work: 128 / 129 / 256 rows x 2048 x 8192 7.2 / 14.5 / 14.5 us, 4096 x 4096 6.6 / 10.2 / 10.2,
// 4096 x 8192 8.7 / 14.9 / 15.1.
struct NarrowPlan {
  int width, split;
};
NarrowPlan narrow_plan(int n, int k, const int (&fit)[3]) {
  const int tiles = ceil_div(n, 64), stages = ceil_div(k, 256);
  if (tiles > fit[0]) return {128, 1};
  if (stages >= 32 && tiles <= fit[2]) return {64, 4};
  if (stages >= 16 && tiles <= fit[1]) return {64, 2};
  return {64, 1};
}

template <int kCta>
int launch_instance(DeviceCtx* ctx, const NarrowPlan& plan, int resident, const void* A, const void* sa, const void* B,
                    const void* sb, void* C, int m, int n, int k, int bf16, cudaStream_t stream) {
  using S = MxShape<kCta>;
  MxGemmParams p = {};
  p.c = C;
  p.m = m;
  p.n = n;
  p.k = k;
  p.bf16 = bf16;
  p.status = ctx->status_word;
  p.width = plan.width;
  p.split = plan.split;
  p.a_rows = kCta == 2 ? 128 : (m + 7) / 8 * 8;
  p.a_bytes = p.a_rows * 128;
  p.stage_bytes = p.a_bytes + p.width / kCta * 128 + S::kScaleBytes;
  p.m_tiles = ceil_div(m, 128 * kCta);
  p.n_tiles = ceil_div(n, p.width);
  p.group_m = 8;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  const int clusters = tiles < resident ? static_cast<int>(tiles) : resident;
  // Two issuers where a CTA has one tile, whose two accumulators take the place of the next tile's; every CTA must have a
  // stage for each.
  p.issuers = kCta == 1 && tiles <= resident && ceil_div(k, S::kBK) >= 2 * p.split ? 2 : 1;
  // A UMMA reads 128 rows of A whether they were loaded or not: behind the last stage there is room for them.
  const int a_slack = S::kABytes - p.a_bytes;
  p.stages = (S::kRingBytes - a_slack) / p.stage_bytes;
  if (p.stages > S::kMaxStages) p.stages = S::kMaxStages;
  if (p.issuers == 2) p.stages &= ~1;
  const int exchange = (p.split - 1) * (p.width / p.split) * 128 * 4;  // what the others of a cluster send
  p.bar_offset = p.stages * p.stage_bytes + a_slack + S::kStagingBytes;
  if (p.bar_offset < exchange) p.bar_offset = exchange;
  const uint64_t words = 64ull * ceil_div(k, 128);
  int st = encode_tmap_2d_u8(&p.tm_a, A, m, k / 2, static_cast<uint32_t>(p.a_rows), 128);
  if (st == BEAM_OK) st = encode_tmap_2d_u8(&p.tm_b, B, n, k / 2, static_cast<uint32_t>(p.width / kCta), 128);
  if (st == BEAM_OK) st = encode_tmap_2d_words64(&p.tm_sa, sa, ceil_div(m, 128), words, 1, 128);
  if (st == BEAM_OK) st = encode_tmap_2d_words64(&p.tm_sb, sb, ceil_div(n, 128), words, S::kScaleBlocksB, 128);
  if (st == BEAM_OK && kCta == 2) st = encode_tmap_2d_sw64(&p.tm_c, C, m, n, n, 32, 32);
  if (st != BEAM_OK) return st;
  const int ctas = kCta * p.split;
  // a cluster that shares a contraction has its SMs to itself (see feedforward_launch.cu)
  const int smem = p.split > 1 ? S::kSmemLimit : p.bar_offset + S::kBarBytes;
  return launch_dependent(mxfp4_umma_kernel<kCta>, clusters * ctas, S::kThreads, smem, ctas, stream,
                          "cudaLaunchKernelEx(mxfp4_umma)", p);
}

}  // namespace

size_t mxfp4_scales_bytes(int rows, int k) {
  if (rows <= 0 || k <= 0) return 0;
  return 512ull * ceil_div(rows, 128) * ceil_div(k, 128);
}

int launch_mxfp4_quantize(const void* x, void* q, void* scales, int rows, int k, int bf16, cudaStream_t stream) {
  if (!x || !q || !scales) return BEAM_ERR_INVALID_ARG;
  int st = check_matrix(rows, k);
  if (st != BEAM_OK) return st;
  if (!aligned16(x) || !aligned16(q) || !aligned16(scales)) return BEAM_ERR_ALIGNMENT;
  const size_t xb = 2ull * rows * k, qb = packed_bytes(rows, k), sb = mxfp4_scales_bytes(rows, k);
  if (overlap(x, xb, q, qb) || overlap(x, xb, scales, sb) || overlap(q, qb, scales, sb)) return BEAM_ERR_INVALID_ARG;
  DeviceCtx* ctx = current_device_ctx(&st);
  if (!ctx) return st;
  MxQuantParams p = {};
  int grid = 0;
  p.x = static_cast<const uint4*>(x);
  p.q = static_cast<uint32_t*>(q);
  p.scales = static_cast<uint8_t*>(scales);
  p.rows = rows;
  p.k = k;
  p.units = lay_units(ceil_div(rows, 128) * 128, k, &grid);
  return launch_dependent(bf16 ? mxfp4_quantize_kernel<true> : mxfp4_quantize_kernel<false>, grid, 256, 0, 1, stream,
                          "cudaLaunchKernelEx(mxfp4_quantize)", p);
}

int launch_mxfp4_dequantize(const void* q, const void* scales, void* x, int rows, int k, int type, cudaStream_t stream) {
  if (!x || !q || !scales) return BEAM_ERR_INVALID_ARG;
  int st = check_matrix(rows, k);
  if (st != BEAM_OK) return st;
  if (!aligned16(x) || !aligned16(q) || !aligned16(scales)) return BEAM_ERR_ALIGNMENT;
  const size_t xb = (type == kMxFp32 ? 4ull : 2ull) * rows * k;
  if (overlap(x, xb, q, packed_bytes(rows, k)) || overlap(x, xb, scales, mxfp4_scales_bytes(rows, k)))
    return BEAM_ERR_INVALID_ARG;
  DeviceCtx* ctx = current_device_ctx(&st);
  if (!ctx) return st;
  int grid = 0;
  const MxUnits u = lay_units(rows, k, &grid);
  auto kernel = type == kMxFp32   ? mxfp4_dequantize_kernel<kMxFp32>
                : type == kMxBf16 ? mxfp4_dequantize_kernel<kMxBf16>
                                  : mxfp4_dequantize_kernel<kMxFp16>;
  return launch_dependent(kernel, grid, 256, 0, 1, stream, "cudaLaunchKernelEx(mxfp4_dequantize)",
                          static_cast<const uint32_t*>(q), static_cast<const uint8_t*>(scales), static_cast<uint4*>(x), k,
                          u);
}

int launch_mxfp4_gemmrc(const void* A, const void* a_scales, const void* B, const void* b_scales, void* C, int m, int n,
                        int k, int bf16, cudaStream_t stream) {
  if (!A || !a_scales || !B || !b_scales || !C) return BEAM_ERR_INVALID_ARG;
  int st = check_matrix(m, k);
  if (st == BEAM_OK) st = check_matrix(n, k);
  if (st != BEAM_OK) return st;
  if (n % 8 != 0) return BEAM_ERR_ALIGNMENT;
  if (!aligned16(A) || !aligned16(a_scales) || !aligned16(B) || !aligned16(b_scales) || !aligned16(C))
    return BEAM_ERR_ALIGNMENT;
  if (static_cast<long long>(ceil_div(m, 128)) * ceil_div(n, 32) > (1ll << 30)) return BEAM_ERR_UNSUPPORTED;
  const size_t cb = 2ull * m * n;
  if (overlap(C, cb, A, packed_bytes(m, k)) || overlap(C, cb, B, packed_bytes(n, k)) ||
      overlap(C, cb, a_scales, mxfp4_scales_bytes(m, k)) || overlap(C, cb, b_scales, mxfp4_scales_bytes(n, k)))
    return BEAM_ERR_INVALID_ARG;
  DeviceCtx* ctx = current_device_ctx(&st);
  if (!ctx) return st;
  static ResidentTable table[4];
  int fit[3], pairs = 0;  // single CTAs; clusters of 2 and 4 CTAs that share a contraction; pairs
  if (m > 128) {
    st = resident_grid(&table[3], mxfp4_umma_kernel<2>, ctx, MxShape<2>::kThreads, MxShape<2>::kSmemLimit, 2, &pairs);
    if (st != BEAM_OK) return st;
    return launch_instance<2>(ctx, {MxShape<2>::kMaxWidth, 1}, pairs, A, a_scales, B, b_scales, C, m, n, k, bf16, stream);
  }
  for (int i = 0; i < 3; ++i) {
    st = resident_grid(&table[i], mxfp4_umma_kernel<1>, ctx, MxShape<1>::kThreads, MxShape<1>::kSmemLimit, 1 << i, &fit[i]);
    if (st != BEAM_OK) return st;
  }
  const NarrowPlan plan = narrow_plan(n, k, fit);
  return launch_instance<1>(ctx, plan, fit[plan.split / 2], A, a_scales, B, b_scales, C, m, n, k, bf16, stream);
}

}  // namespace beam
