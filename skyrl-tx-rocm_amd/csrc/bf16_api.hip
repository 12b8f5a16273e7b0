// C ABI of the operators beside the quantized path: products grouped by expert in bf16, embedding rows and their gradient,
// the norm and the clipping of adapter gradients.  Argument validation, workspace carving and kernel launches; nothing
// here synchronises, allocates or keeps state.
#include "bf16_api.h"

#include <hip/hip_runtime.h>

#include <cmath>

#include "bf16_grouped.h"
#include "embedding.h"
#include "grad_clip.h"

using namespace w8a8;

namespace {

constexpr uint32_t kMaxRows = 1u << 20;

inline bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) == 0; }
inline bool overlaps(const void* a, uint64_t an, const void* b, uint64_t bn) {
  if (!a || !b || an == 0 || bn == 0) return false;
  const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  return a0 < b0 + bn && b0 < a0 + an;
}
inline int launch_status() { return hipGetLastError() == hipSuccess ? MI355_W8A8_OK : MI355_W8A8_ERR_LAUNCH; }
inline uint64_t align256(uint64_t v) { return (v + 255u) & ~uint64_t(255); }
template <class K>
inline bool allow_lds(K kernel, uint32_t bytes) {
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == hipSuccess;
}

// ---- products grouped by expert --------------------------------------------------------------------------------------

constexpr uint32_t kGroupedTiles = MI355_W8A8_FLAG_BF16_GROUPED_TILE_256X256 | MI355_W8A8_FLAG_BF16_GROUPED_TILE_128X256 | MI355_W8A8_FLAG_BF16_GROUPED_TILE_64X128;
inline bool one_bit_at_most(uint32_t v) { return (v & (v - 1u)) == 0; }

int check_grouped_dims(uint32_t m, uint32_t k, uint32_t n, uint32_t groups) {
  if (m == 0 || k == 0 || n == 0 || groups == 0) return MI355_W8A8_ERR_SHAPE;
  if ((k & 7u) || (n & 7u)) return MI355_W8A8_ERR_UNSUPPORTED;
  // (a tile's offsets are 32 bits wide: 256 rows of either operand stay below 2^31 bytes)
  if (m > kMaxRows || k > MI355_W8A8_BF16_GROUPED_MAX_FEATURES || n > MI355_W8A8_BF16_GROUPED_MAX_FEATURES || groups > kBgMaxGroups)
    return MI355_W8A8_ERR_UNSUPPORTED;
  return MI355_W8A8_OK;
}

// most row tiles that m rows in `groups` groups can make
inline uint64_t most_row_tiles(uint32_t m, uint32_t groups, uint32_t tile) {
  const uint32_t held = groups < m ? groups : m;
  return (m + (uint64_t)(tile - 1u) * held) / tile;
}

template <int TM, int TN, int STAGES>
uint32_t grouped_lds(uint32_t groups) { return (TM + TN) * kBgDepth * 2u * STAGES + (kBgScratch + 2u * (groups + 2u)) * 4u; }
// one workgroup a CU: its stages fill the LDS
template <int TM, int TN>
uint32_t grouped_blocks(GroupedKind kind, const BgArgs& g) {
  const uint64_t n_tiles = (g.cols + TN - 1u) / TN * g.splits;
  const uint64_t tiles = n_tiles * (kind == kGroupedDw ? (uint64_t)g.groups * ((g.rows + TM - 1u) / TM) : most_row_tiles(g.m, g.groups + 1u, TM));
  return (uint32_t)(tiles < 256u ? (tiles + 7u) / 8u * 8u : 256u);
}
template <int KIND, int TM, int TN, int WM, int WN, int STAGES, int LOADERS, bool F32>
int launch_grouped_tiles(const BgArgs& g, hipStream_t s) {
  auto kernel = &bf16_grouped_kernel<KIND, TM, TN, WM, WN, STAGES, LOADERS, F32>;
  const uint32_t lds = grouped_lds<TM, TN, STAGES>(g.groups);
  if (!allow_lds(kernel, lds)) return MI355_W8A8_ERR_LAUNCH;
  hipLaunchKernelGGL(kernel, dim3(grouped_blocks<TM, TN>((GroupedKind)KIND, g)), dim3(64 * (WM * WN + LOADERS)), lds, s, g);
  return launch_status();
}
template <int TM, int TN, int WM, int WN, int STAGES, int LOADERS, bool F32>
int launch_grouped_both(const BgArgs& dx, const BgArgs& dw, hipStream_t s) {
  auto kernel = &bf16_grouped_both_kernel<TM, TN, WM, WN, STAGES, LOADERS, F32>;
  const uint32_t lds = grouped_lds<TM, TN, STAGES>(dx.groups);
  if (!allow_lds(kernel, lds)) return MI355_W8A8_ERR_LAUNCH;
  const BgBothArgs both{dx, dw, grouped_blocks<TM, TN>(kGroupedDx, dx)};
  hipLaunchKernelGGL(kernel, dim3(both.dx_blocks + grouped_blocks<TM, TN>(kGroupedDw, dw)), dim3(64 * (WM * WN + LOADERS)), lds, s, both);
  return launch_status();
}

struct GroupedPlan {
  uint32_t tile;    // one of kGroupedTiles
  uint32_t splits;  // of the contraction
  float us;         // about what it takes
};
struct GroupedSize {  // of C in tiles, and their depth in stages
  GroupedKind kind;
  uint32_t m, groups, rows, cols, depth;
  float held() const { return (float)(groups < m ? groups : m); }
  float tiles(uint32_t tm, uint32_t tn) const {
    const float row_tiles = kind == kGroupedDw ? (float)((uint64_t)groups * ((rows + tm - 1u) / tm)) : fmaxf((float)m / tm + 0.5f * held(), held());
    return row_tiles * ((cols + tn - 1u) / tn);
  }
  uint32_t stages() const { return bg_stages(kind == kGroupedDw ? (uint32_t)((float)m / held()) : depth); }
};

// Which tiles.  A call costs the rounds of its tiles on the 256 CUs times what a round takes: 4 units for 256 x 256, 2.2 for 128 x 256 and
// 1.15 for 64 x 128 (half and an eighth of the products; 32768 rows of 4096 -> 12288 in 8 groups 2640, 3000 and 6020 us).  Groups end
// in the middle of a tile, half a tile on average.  The smaller tiles have room for more stages, which is what counts where the
// weights come from memory for few rows.  us, 256 x 256 / 128 x 256 / 64 x 128, 2048 -> 1536, 128 groups of uneven sizes: forward 16384 rows 242 / 212 /
// 242, 8192 226 / 179 / 195, 512 165 / 129 / 138, 64 91 / 60 / 53, dW 16384 rows 217 / 218 / 335, 8192 172 / 178 / 269; 4096 -> 4096, 4 groups,
// 2048 rows 96 / 70 / 126; 1024 -> 1024, 8 groups, 4096 rows 27 / 19 / 19; 512 -> 512, 16 groups, 16384 rows 21 / 17 / 21.5.
// rows: of C a group (dW); depth: contraction of forward and dx.
GroupedPlan plan_grouped(GroupedKind kind, uint32_t m, uint32_t groups, uint32_t rows, uint32_t cols, uint32_t depth, uint32_t forced) {
  if (forced) return {forced, 1u, 0.0f};
  const GroupedSize size{kind, m, groups, rows, cols, depth};
  const float held = size.held();
  auto tiles = [&](uint32_t tm, uint32_t tn) { return size.tiles(tm, tn); };
  auto rounds = [](float n) { return n <= 256.0f ? 1.0f : n / 256.0f + 0.5f; };  // (how many tiles the groups make is not known, nor whether they fill the last round)
  const float small_tiles = tiles(64u, 128u), middle_tiles = tiles(128u, 256u);
  const float large = rounds(tiles(256u, 256u)) * 4.0f, middle = rounds(middle_tiles) * 2.2f, small = rounds(small_tiles) * 1.15f;
  uint32_t tile = MI355_W8A8_FLAG_BF16_GROUPED_TILE_64X128;
  float round_us = 0.47f;  // a round's time for each stage
  // (a dW of one round that is not eight stages deep is all latency and stores: 712 -> 1096, 13 groups, 1003 rows, float32 22 / 18 in the
  // smaller tiles)
  const bool shallow = kind == kGroupedDw && large == 4.0f && m / groups < 8u * kBgDepth;
  if (!shallow && large <= middle && large <= small) tile = MI355_W8A8_FLAG_BF16_GROUPED_TILE_256X256, round_us = large / 4.0f * 1.7f;
  else if (middle <= small) tile = MI355_W8A8_FLAG_BF16_GROUPED_TILE_128X256, round_us = middle / 2.2f * 0.95f;
  else round_us *= small / 1.15f;
  // Few tiles of a long contraction leave most CUs idle: then parts of it are products of their own, with float32 results
  // that a second launch adds up (4 us, and the parts written and read).  Neither is faster than the operands come from memory.  us, whole / in
  // parts: 1 row of 4096 -> 4096 27 / 14.4, 8 rows of 8952 -> 704 in 6 groups 52 / 22, 64 rows of 4096 -> 64 in 16 groups 27 / 13, dW of 272 -> 1696
  // in 4 groups of 28533 rows 78 / 57.
  const uint32_t stages = size.stages();
  const float bytes = kind == kGroupedDw ? (float)m * (rows + cols) * 2.0f : (held * cols + (float)m) * depth * 2.0f;
  const float values = kind == kGroupedDw ? (float)groups * rows * cols : (float)m * cols, memory_us = bytes / 5.0e6f;
  const float whole = fmaxf(round_us * (stages + 3.0f), memory_us);
  float best = 0.9f * whole;
  uint32_t splits = 1;
  for (uint32_t n = 2; n <= 64u && n * 2u <= stages && middle_tiles * n <= 1024.0f; ++n) {
    const float each = (float)((stages + n - 1u) / n) + 3.0f;
    const float s = ceilf(small_tiles * n / 256.0f) * 0.47f * each, m2 = ceilf(middle_tiles * n / 256.0f) * 0.95f * each;
    const float us = fmaxf(s < m2 ? s : m2, memory_us) + 4.0f + values * n * 8.0f / 5.0e6f;
    if (us >= best) continue;
    best = us;
    splits = n;
    tile = s < m2 ? MI355_W8A8_FLAG_BF16_GROUPED_TILE_64X128 : MI355_W8A8_FLAG_BF16_GROUPED_TILE_128X256;
  }
  return {tile, splits, splits > 1u ? best : whole};
}

inline uint64_t grouped_plane(GroupedKind kind, uint32_t m, uint32_t groups, uint32_t rows, uint32_t cols) {
  return kind == kGroupedDw ? (uint64_t)groups * rows * cols : (uint64_t)m * cols;
}
uint64_t grouped_workspace(GroupedKind kind, uint32_t m, uint32_t groups, uint32_t rows, uint32_t cols, uint32_t depth, uint32_t forced) {
  const GroupedPlan plan = plan_grouped(kind, m, groups, rows, cols, depth, forced);
  return plan.splits > 1u ? plan.splits * grouped_plane(kind, m, groups, rows, cols) * 4u : 0u;
}

template <int KIND, bool F32 = false>
int launch_grouped(BgArgs g, uint32_t forced, void* workspace, hipStream_t s) {
  const GroupedPlan plan = plan_grouped((GroupedKind)KIND, g.m, g.groups, g.rows, g.cols, g.depth, forced);
  g.splits = plan.splits;
  if (plan.splits > 1u) {
    void* const out = g.out;
    g.out = workspace;
    g.plane = grouped_plane((GroupedKind)KIND, g.m, g.groups, g.rows, g.cols);
    const int st = plan.tile == MI355_W8A8_FLAG_BF16_GROUPED_TILE_64X128 ? launch_grouped_tiles<KIND, 64, 128, 2, 2, 6, 4, true>(g, s)
                                                                         : launch_grouped_tiles<KIND, 128, 256, 2, 4, 3, 4, true>(g, s);
    if (st) return st;
    hipLaunchKernelGGL(bg_join_kernel<F32>, dim3((uint32_t)((g.plane / 4u + 255u) / 256u)), dim3(256), 0, s, static_cast<const float*>(workspace), out, g.plane,
                       g.splits);
    return launch_status();
  }
  if (plan.tile == MI355_W8A8_FLAG_BF16_GROUPED_TILE_256X256) return launch_grouped_tiles<KIND, 256, 256, 2, 4, 2, 0, F32>(g, s);
  if (plan.tile == MI355_W8A8_FLAG_BF16_GROUPED_TILE_128X256) return launch_grouped_tiles<KIND, 128, 256, 2, 4, 3, 4, F32>(g, s);
  return launch_grouped_tiles<KIND, 64, 128, 2, 2, 6, 4, F32>(g, s);
}

// Tiles for both gradients in one launch, or 0: with tiles of one size for both their work fills the CUs together, and it is a launch (4 us) less; a
// tile's time is that of its stages.  Not where bytes come near to bound them: reading weights and writing their gradients at once is the slower.  us, two launches /
// one: 712 -> 1096, 13 groups, 1003 rows, float32 32.3 / 23.5; 128 -> 120, 22 groups, 4051 rows 16 / 7.8; 1024 -> 1024, 8 groups, 4096 rows 41 / 31.5;
// 1576 -> 1744, 25 groups, 8260 rows 173 / 165; but 1944 -> 2072, 115 groups, 560 rows, float32 675 / 770.
uint32_t plan_grouped_both(const BgArgs& dx, const BgArgs& dw, uint32_t dw_bytes, uint32_t forced) {
  const GroupedPlan a = plan_grouped(kGroupedDx, dx.m, dx.groups, dx.rows, dx.cols, dx.depth, forced);
  const GroupedPlan b = plan_grouped(kGroupedDw, dw.m, dw.groups, dw.rows, dw.cols, dw.depth, forced);
  if (forced) return forced;
  if (a.splits > 1u || b.splits > 1u) return 0;
  const GroupedSize x{kGroupedDx, dx.m, dx.groups, dx.rows, dx.cols, dx.depth}, w{kGroupedDw, dw.m, dw.groups, dw.rows, dw.cols, dw.depth};
  const float rows = (float)dx.m * (dx.cols + dw.cols) * 2.0f, weights = (float)dx.cols * dw.cols;
  const float dx_us = (rows + x.held() * weights * 2.0f) / 5.0e6f, dw_us = (rows + w.groups * weights * dw_bytes) / 5.0e6f;
  float best = 0.97f * (fmaxf(a.us, dx_us) + fmaxf(b.us, dw_us) + 4.0f);
  uint32_t tile = 0;
  auto consider = [&](uint32_t flag, uint32_t tm, uint32_t tn, float stage_us) {
    const float each_x = (x.stages() + 3.0f) * stage_us, each_w = (w.stages() + 3.0f) * stage_us, longest = fmaxf(each_x, each_w);
    const float us = fmaxf((x.tiles(tm, tn) * each_x + w.tiles(tm, tn) * each_w) / 256.0f + 0.5f * longest, longest);
    if (us < best && dx_us + dw_us < 0.75f * us) best = us, tile = flag;
  };
  consider(MI355_W8A8_FLAG_BF16_GROUPED_TILE_256X256, 256u, 256u, 1.7f);
  consider(MI355_W8A8_FLAG_BF16_GROUPED_TILE_128X256, 128u, 256u, 0.95f);
  consider(MI355_W8A8_FLAG_BF16_GROUPED_TILE_64X128, 64u, 128u, 0.47f);
  return tile;
}
template <bool F32>
int launch_both(BgArgs dx, BgArgs dw, uint32_t tile, hipStream_t s) {
  dx.splits = dw.splits = 1;
  if (tile == MI355_W8A8_FLAG_BF16_GROUPED_TILE_256X256) return launch_grouped_both<256, 256, 2, 4, 2, 0, F32>(dx, dw, s);
  if (tile == MI355_W8A8_FLAG_BF16_GROUPED_TILE_128X256) return launch_grouped_both<128, 256, 2, 4, 3, 4, F32>(dx, dw, s);
  return launch_grouped_both<64, 128, 2, 2, 6, 4, F32>(dx, dw, s);
}

int check_grouped_workspace(const void* workspace, uint64_t given, uint64_t needed) {
  if (needed && (!workspace || given < needed)) return MI355_W8A8_ERR_WORKSPACE;
  return workspace && !aligned(workspace, 256) ? MI355_W8A8_ERR_ALIGN : MI355_W8A8_OK;
}
uint64_t grouped_bwd_workspace(uint32_t m, uint32_t k, uint32_t n, uint32_t groups, uint32_t forced, bool dx, bool dw) {  // (one after the other)
  const uint64_t a = dx ? grouped_workspace(kGroupedDx, m, groups, 0u, k, n, forced) : 0u, b = dw ? grouped_workspace(kGroupedDw, m, groups, k, n, 0u, forced) : 0u;
  return a > b ? a : b;
}

// What the two gradients' products are made of, but for the tensors.
void bwd_sizes(uint32_t m, uint32_t k, uint32_t n, uint32_t groups, BgArgs& dx, BgArgs& dw) {
  dx.m = dw.m = m;
  dx.groups = dw.groups = groups;
  dx.rows_ld = n; dx.cols_ld = n; dx.depth = n; dx.cols = k;
  dx.b_group = (uint64_t)k * n;
  dw.rows_ld = k; dw.cols_ld = n; dw.depth = 0; dw.cols = n; dw.rows = k;
  dw.out_group = (uint64_t)k * n;
}

int run_grouped(const mi355_w8a8_bf16_grouped_problem* p, hipStream_t s) {
  if (!p) return MI355_W8A8_ERR_NULL;
  if (p->struct_size != sizeof(mi355_w8a8_bf16_grouped_problem)) return MI355_W8A8_ERR_STRUCT;
  if ((p->flags & ~kGroupedTiles) || !one_bit_at_most(p->flags)) return MI355_W8A8_ERR_SHAPE;
  int st = check_grouped_dims(p->m, p->k, p->n, p->n_groups);
  if (st) return st;
  if (!p->x || !p->weight || !p->group_sizes || !p->out) return MI355_W8A8_ERR_NULL;
  if (!aligned(p->x, 16) || !aligned(p->weight, 16) || !aligned(p->out, 16) || !aligned(p->group_sizes, 4)) return MI355_W8A8_ERR_ALIGN;
  const uint64_t out_bytes = (uint64_t)p->m * p->n * 2u;
  if (overlaps(p->out, out_bytes, p->x, (uint64_t)p->m * p->k * 2u) ||
      overlaps(p->out, out_bytes, p->weight, (uint64_t)p->n_groups * p->k * p->n * 2u) ||
      overlaps(p->out, out_bytes, p->group_sizes, (uint64_t)p->n_groups * 4u))
    return MI355_W8A8_ERR_ALIAS;
  const uint64_t needed = grouped_workspace(kGroupedFwd, p->m, p->n_groups, 0u, p->n, p->k, p->flags);
  if ((st = check_grouped_workspace(p->workspace, p->workspace_bytes, needed))) return st;
  if (overlaps(p->workspace, needed, p->out, out_bytes) || overlaps(p->workspace, needed, p->x, (uint64_t)p->m * p->k * 2u) ||
      overlaps(p->workspace, needed, p->weight, (uint64_t)p->n_groups * p->k * p->n * 2u) || overlaps(p->workspace, needed, p->group_sizes, (uint64_t)p->n_groups * 4u))
    return MI355_W8A8_ERR_ALIAS;
  (void)hipGetLastError();
  BgArgs g{};
  g.a = static_cast<const uint16_t*>(p->x); g.b = static_cast<const uint16_t*>(p->weight);
  g.sizes = p->group_sizes; g.out = p->out;
  g.m = p->m; g.rows_ld = p->k; g.cols_ld = p->n; g.depth = p->k; g.cols = p->n; g.groups = p->n_groups;
  g.b_group = (uint64_t)p->k * p->n;
  return launch_grouped<kGroupedFwd>(g, p->flags, p->workspace, s);
}

int run_grouped_bwd(const mi355_w8a8_bf16_grouped_bwd_problem* p, hipStream_t s) {
  if (!p) return MI355_W8A8_ERR_NULL;
  if (p->struct_size != sizeof(mi355_w8a8_bf16_grouped_bwd_problem)) return MI355_W8A8_ERR_STRUCT;
  const uint32_t forced = p->flags & kGroupedTiles;
  if ((p->flags & ~(kGroupedTiles | MI355_W8A8_FLAG_BF16_GROUPED_DW_F32)) || !one_bit_at_most(forced)) return MI355_W8A8_ERR_SHAPE;
  int st = check_grouped_dims(p->m, p->k, p->n, p->n_groups);
  if (st) return st;
  if (!p->dy || !p->group_sizes || (!p->dx && !p->dw)) return MI355_W8A8_ERR_NULL;
  if ((p->dx && !p->weight) || (p->dw && !p->x)) return MI355_W8A8_ERR_NULL;
  if (!aligned(p->x, 16) || !aligned(p->dy, 16) || !aligned(p->weight, 16) || !aligned(p->dx, 16) || !aligned(p->dw, 16) || !aligned(p->group_sizes, 4))
    return MI355_W8A8_ERR_ALIGN;
  const bool f32 = p->flags & MI355_W8A8_FLAG_BF16_GROUPED_DW_F32;
  const uint64_t x_bytes = (uint64_t)p->m * p->k * 2u, dy_bytes = (uint64_t)p->m * p->n * 2u, sizes_bytes = (uint64_t)p->n_groups * 4u;
  const uint64_t values = (uint64_t)p->n_groups * p->k * p->n, dw_bytes = values * (f32 ? 4u : 2u);
  const uint64_t needed = grouped_bwd_workspace(p->m, p->k, p->n, p->n_groups, forced, p->dx, p->dw);
  if ((st = check_grouped_workspace(p->workspace, p->workspace_bytes, needed))) return st;
  const void* outs[3] = {p->dx, p->dw, p->workspace};
  const uint64_t bytes[3] = {x_bytes, dw_bytes, needed};
  for (int i = 0; i < 3; ++i) {
    if (overlaps(outs[i], bytes[i], p->dy, dy_bytes) || overlaps(outs[i], bytes[i], p->x, x_bytes) ||
        overlaps(outs[i], bytes[i], p->weight, values * 2u) || overlaps(outs[i], bytes[i], p->group_sizes, sizes_bytes))
      return MI355_W8A8_ERR_ALIAS;
  }
  if (overlaps(p->dx, x_bytes, p->dw, dw_bytes) || overlaps(p->workspace, needed, p->dx, x_bytes) || overlaps(p->workspace, needed, p->dw, dw_bytes)) return MI355_W8A8_ERR_ALIAS;
  (void)hipGetLastError();
  BgArgs dx{}, dw{};
  bwd_sizes(p->m, p->k, p->n, p->n_groups, dx, dw);
  dx.sizes = dw.sizes = p->group_sizes;
  dx.a = static_cast<const uint16_t*>(p->dy); dx.b = static_cast<const uint16_t*>(p->weight); dx.out = p->dx;
  dw.a = static_cast<const uint16_t*>(p->x); dw.b = static_cast<const uint16_t*>(p->dy); dw.out = p->dw;
  if (p->dx && p->dw) {
    const uint32_t tile = plan_grouped_both(dx, dw, f32 ? 4u : 2u, forced);
    if (tile) return f32 ? launch_both<true>(dx, dw, tile, s) : launch_both<false>(dx, dw, tile, s);
  }
  if (p->dx && (st = launch_grouped<kGroupedDx>(dx, forced, p->workspace, s))) return st;
  if (p->dw) st = f32 ? launch_grouped<kGroupedDw, true>(dw, forced, p->workspace, s) : launch_grouped<kGroupedDw>(dw, forced, p->workspace, s);
  return st;
}

// ---- embedding rows --------------------------------------------------------------------------------------------------

int check_embedding(const mi355_w8a8_embedding_problem* p) {
  if (!p) return MI355_W8A8_ERR_NULL;
  if (p->struct_size != sizeof(mi355_w8a8_embedding_problem)) return MI355_W8A8_ERR_STRUCT;
  if (p->flags & ~(MI355_W8A8_FLAG_EMBEDDING_F32 | MI355_W8A8_FLAG_EMBEDDING_IDS64)) return MI355_W8A8_ERR_SHAPE;
  if (p->n_tokens == 0 || p->vocab == 0 || p->width == 0) return MI355_W8A8_ERR_SHAPE;
  if (p->n_adapters == 0 && (p->adapter_indices || p->scales)) return MI355_W8A8_ERR_SHAPE;
  if (p->n_adapters > 1 && !p->adapter_indices) return MI355_W8A8_ERR_NULL;
  const uint64_t rows = (uint64_t)(p->n_adapters ? p->n_adapters : 1u) * p->vocab;
  if (p->n_tokens > kMaxRows || p->width > MI355_W8A8_EMBEDDING_MAX_WIDTH || rows > MI355_W8A8_EMBEDDING_MAX_ROWS) return MI355_W8A8_ERR_UNSUPPORTED;
  const uintptr_t id = p->flags & MI355_W8A8_FLAG_EMBEDDING_IDS64 ? 8 : 4;
  if (!p->ids) return MI355_W8A8_ERR_NULL;
  if (!aligned(p->ids, id) || !aligned(p->adapter_indices, 4) || !aligned(p->scales, 4)) return MI355_W8A8_ERR_ALIGN;
  return MI355_W8A8_OK;
}

inline uint64_t embedding_rows(const mi355_w8a8_embedding_problem* p) { return (uint64_t)(p->n_adapters ? p->n_adapters : 1u) * p->vocab; }
inline uint32_t value_bytes(const mi355_w8a8_embedding_problem* p) { return p->flags & MI355_W8A8_FLAG_EMBEDDING_F32 ? 4u : 2u; }
inline bool overlaps_indices(const mi355_w8a8_embedding_problem* p, const void* out, uint64_t bytes) {
  return overlaps(out, bytes, p->ids, (uint64_t)p->n_tokens * (p->flags & MI355_W8A8_FLAG_EMBEDDING_IDS64 ? 8u : 4u)) ||
         overlaps(out, bytes, p->adapter_indices, (uint64_t)p->n_tokens * 4u) || overlaps(out, bytes, p->scales, (uint64_t)p->n_adapters * 4u);
}

EmbedArgs embed_args(const mi355_w8a8_embedding_problem* p) {
  EmbedArgs e{};
  e.table = p->table; e.out = p->out; e.dy = p->d_out; e.ids = p->ids; e.adapters = p->adapter_indices; e.scales = p->scales;
  e.scale = p->scale; e.n = p->n_tokens; e.vocab = p->vocab; e.width = p->width; e.n_adapters = p->n_adapters ? p->n_adapters : 1u;
  e.ids64 = (p->flags & MI355_W8A8_FLAG_EMBEDDING_IDS64) != 0;
  return e;
}
inline uint32_t blocks_of(uint64_t threads) { return (uint32_t)((threads + 255u) / 256u); }

int run_embedding(const mi355_w8a8_embedding_problem* p, hipStream_t s) {
  const int st = check_embedding(p);
  if (st) return st;
  if (!p->table || !p->out) return MI355_W8A8_ERR_NULL;
  const uint32_t size = value_bytes(p);
  if (!aligned(p->table, size) || !aligned(p->out, size)) return MI355_W8A8_ERR_ALIGN;
  const uint64_t out_bytes = (uint64_t)p->n_tokens * p->width * size;
  if (overlaps(p->out, out_bytes, p->table, embedding_rows(p) * p->width * size) || overlaps_indices(p, p->out, out_bytes)) return MI355_W8A8_ERR_ALIAS;
  const EmbedArgs e = embed_args(p);
  const bool wide = p->width >= 16u / size;
  // (an axis of a launch has fewer than 2^32 threads, the widest rows of the most tokens 2^34 units)
  const uint32_t blocks = blocks_of((uint64_t)p->n_tokens * embed_units(p->width, wide ? 16u / size : 1u)), planes = (blocks + kEmbedRowBlocks - 1u) / kEmbedRowBlocks;
  const dim3 grid(planes > 1u ? kEmbedRowBlocks : blocks, planes), block(256);
  (void)hipGetLastError();
  if (size == 4u) {
    if (wide) hipLaunchKernelGGL((embed_rows_kernel<float, 4>), grid, block, 0, s, e);
    else hipLaunchKernelGGL((embed_rows_kernel<float, 1>), grid, block, 0, s, e);
  } else {
    if (wide) hipLaunchKernelGGL((embed_rows_kernel<uint16_t, 8>), grid, block, 0, s, e);
    else hipLaunchKernelGGL((embed_rows_kernel<uint16_t, 1>), grid, block, 0, s, e);
  }
  return launch_status();
}

struct EmbedLayout {
  uint32_t passes, bits, chunks, run, runs;
  uint64_t keys[2], tokens[2], notes, counts, joins, parts, total;
};

// positions of a run: enough threads to fill the chip (2048 a CU) where the rows suffice, and no more parts than that
EmbedLayout embed_layout(uint32_t n, uint64_t rows, uint32_t width, uint32_t flags) {
  EmbedLayout L{};
  uint32_t bits = 1;
  while ((rows >> bits) != 0) ++bits;  // keys up to `rows` itself
  L.passes = (bits + 10u) / 11u;
  L.bits = (bits + L.passes - 1u) / L.passes;
  L.chunks = (n + kEmbedChunk - 1u) / kEmbedChunk;
  const uint32_t vec = flags & MI355_W8A8_FLAG_EMBEDDING_F32 ? 4u : 8u;
  const uint64_t units = embed_units(width, width >= vec ? vec : 1u);
  L.run = 8;
  while (L.run < 256u && (uint64_t)n * units / (L.run * 2u) >= 524288u) L.run *= 2u;
  L.runs = (n + L.run - 1u) / L.run;
  uint64_t off = 0;
  for (int i = 0; i < 2; ++i) {
    L.keys[i] = off; off += align256((uint64_t)n * 4u);
    L.tokens[i] = off; off += align256((uint64_t)n * 4u);
  }
  L.notes = off; off += kEmbedNotes * 4u;
  L.counts = off;
  if (L.chunks > 1u) off += align256(((uint64_t)L.chunks + 1u) * (4u << L.bits));
  L.joins = off; off += align256((uint64_t)L.runs * 4u);
  L.parts = off; off += align256((uint64_t)L.runs * 2u * width * 4u);
  L.total = off;
  return L;
}

template <typename T, int V>
int launch_embed_sums(const EmbedSumArgs& a, hipStream_t s) {
  const uint32_t units = embed_units(a.e.width, V);
  const dim3 block(256);
  const dim3 grid(blocks_of((uint64_t)a.runs * (units >= 64u ? (units + 63u) / 64u * 64u : units)));
  if (units >= 64u) hipLaunchKernelGGL((embed_sum_kernel<T, V, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((embed_sum_kernel<T, V, false>), grid, block, 0, s, a);
  const int st = launch_status();
  if (st || a.runs < 2u) return st;
  constexpr int kJoin = V < 4 ? V : 4;
  const uint64_t most = ((uint64_t)a.runs * embed_units(a.e.width, kJoin) + 255u) / 256u;
  hipLaunchKernelGGL((embed_join_kernel<T, kJoin>), dim3((uint32_t)(most < 2048u ? most * 2u : 2048u + kEmbedLongs)), block, 0, s, a);
  return launch_status();
}

int run_embedding_bwd(const mi355_w8a8_embedding_problem* p, hipStream_t s) {
  int st = check_embedding(p);
  if (st) return st;
  if (!p->d_out || !p->out) return MI355_W8A8_ERR_NULL;
  const uint32_t size = value_bytes(p);
  if (!aligned(p->d_out, size) || !aligned(p->out, 16)) return MI355_W8A8_ERR_ALIGN;
  const uint64_t rows = embedding_rows(p), out_bytes = rows * p->width * size, dy_bytes = (uint64_t)p->n_tokens * p->width * size;
  const EmbedLayout L = embed_layout(p->n_tokens, rows, p->width, p->flags);
  if (!p->workspace || p->workspace_bytes < L.total) return MI355_W8A8_ERR_WORKSPACE;
  if (!aligned(p->workspace, 256)) return MI355_W8A8_ERR_ALIGN;
  if (overlaps(p->out, out_bytes, p->d_out, dy_bytes) || overlaps_indices(p, p->out, out_bytes) || overlaps(p->out, out_bytes, p->workspace, L.total) ||
      overlaps(p->workspace, L.total, p->d_out, dy_bytes) || overlaps_indices(p, p->workspace, L.total))
    return MI355_W8A8_ERR_ALIAS;
  unsigned char* ws = static_cast<unsigned char*>(p->workspace);
  auto words = [&](uint64_t off) { return reinterpret_cast<uint32_t*>(ws + off); };
  EmbedSortArgs a{};
  a.e = embed_args(p);
  a.bits = L.bits; a.passes = L.passes; a.chunks = L.chunks;
  a.notes = words(L.notes);
  // the launches that count clear a share of the gradient each (in those that place the reads would wait behind so many stores: 20 MB beside
  // 32768 tokens 12 us instead of 9), and past the caches where the
  // last one, 256 MiB, does not hold it (the rows of dy stay there then: 778 MB 193 us in all, 199 through the caches; 102 MB 26 and 23)
  const uint64_t pieces = out_bytes / 16u;
  const bool small = L.chunks == 1u;
  const uint32_t launches = small ? 1u : L.passes;
  uint32_t launched = 0, clearing = 0;
  a.stream = out_bytes > (256u << 20);
  auto share = [&] {
    const uint64_t each = pieces / launches;
    const bool last = launched + 1u == launches;
    a.clear = static_cast<uint4*>(p->out) + launched * each;
    a.clear_pieces = last ? pieces - launched * each : each;
    a.clear_rest = last ? (uint32_t)(out_bytes % 16u) : 0u;
    const uint64_t wanted = (a.clear_pieces + 1023u) / 1024u + (a.clear_rest ? 1u : 0u);
    clearing = (uint32_t)(wanted < kEmbedClearing ? wanted : kEmbedClearing);
    ++launched;
  };
  const uint32_t place_lds = (kEmbedDigits + 16u) * 4u + (32u << L.bits), small_lds = place_lds + 8192u;
  (void)hipGetLastError();
  if (small) {
    if (!allow_lds(&embed_sort_small_kernel, small_lds)) return MI355_W8A8_ERR_LAUNCH;
    a.keys_out = words(L.keys[0]); a.tokens_out = words(L.tokens[0]);
    share();
    hipLaunchKernelGGL(embed_sort_small_kernel, dim3(1u + clearing), dim3(1024), small_lds, s, a);
    if ((st = launch_status())) return st;
  } else {
    const bool scan = L.chunks > kEmbedSumChunks;
    if (!allow_lds(&embed_place_kernel<true>, place_lds) || !allow_lds(&embed_place_kernel<false>, place_lds)) return MI355_W8A8_ERR_LAUNCH;
    a.counts = words(L.counts);
    for (uint32_t pass = 0; pass < L.passes; ++pass) {
      a.keys = pass ? words(L.keys[(pass - 1u) & 1u]) : nullptr;
      a.tokens = pass ? words(L.tokens[(pass - 1u) & 1u]) : nullptr;
      a.keys_out = words(L.keys[pass & 1u]);
      a.tokens_out = words(L.tokens[pass & 1u]);
      a.shift = pass * L.bits;
      share();
      hipLaunchKernelGGL(embed_count_kernel, dim3(L.chunks + clearing), dim3(1024), 0, s, a);
      if ((st = launch_status())) return st;
      if (scan) {
        hipLaunchKernelGGL(embed_scan_kernel, dim3(1), dim3(1024), 0, s, a);
        if ((st = launch_status())) return st;
      }
      if (scan) hipLaunchKernelGGL(embed_place_kernel<true>, dim3(L.chunks), dim3(1024), place_lds, s, a);
      else hipLaunchKernelGGL(embed_place_kernel<false>, dim3(L.chunks), dim3(1024), place_lds, s, a);
      if ((st = launch_status())) return st;
    }
  }
  EmbedSumArgs b{};
  b.e = a.e;
  b.keys = a.keys_out; b.tokens = a.tokens_out;
  b.parts = reinterpret_cast<float*>(ws + L.parts);
  b.joins = words(L.joins); b.notes = a.notes;
  b.run = L.run; b.runs = L.runs;
  const bool wide = p->width >= 16u / size;
  if (size == 4u) return wide ? launch_embed_sums<float, 4>(b, s) : launch_embed_sums<float, 1>(b, s);
  return wide ? launch_embed_sums<uint16_t, 8>(b, s) : launch_embed_sums<uint16_t, 1>(b, s);
}

// ---- gradient norms and clipping -------------------------------------------------------------------------------------

// values of a piece: as few as leave the chip 2048 workgroups, at most 64 KiB, so that the last of them end soon after the first; more where the
// values of an adapter would make more than 4096 parts, since every workgroup of the scaling reads them all.  A tensor is one piece at least: thousands of
// tensors are as many parts more, and what the workgroups read together grows with the square of that.
uint32_t grad_piece_values(const mi355_w8a8_grad_tensor* t, uint32_t n, uint32_t adapters) {
  uint64_t values = 0;
  uint32_t most = 32768u, piece = 2048u;
  for (uint32_t i = 0; i < n; ++i) {
    values += t[i].count;
    if (t[i].type == MI355_W8A8_GRAD_F32) most = 16384u;
  }
  while (piece < most && values / piece * adapters > 2048u) piece *= 2u;
  while (values / piece > 4096u && piece < (1u << 28)) piece *= 2u;
  return piece;
}
inline uint64_t pieces_of(uint64_t count, uint32_t piece) { return (count + piece - 1u) / piece; }

int check_grads(const mi355_w8a8_grad_tensor* t, uint32_t n, uint32_t adapters, const float* norms, bool scale) {
  if (!t || !norms) return MI355_W8A8_ERR_NULL;
  if (n == 0 || adapters == 0) return MI355_W8A8_ERR_SHAPE;
  if (n > MI355_W8A8_GRAD_MAX_TENSORS || adapters > 65535u) return MI355_W8A8_ERR_UNSUPPORTED;
  if (!aligned(norms, 4)) return MI355_W8A8_ERR_ALIGN;
  for (uint32_t i = 0; i < n; ++i) {
    if (t[i].type > MI355_W8A8_GRAD_F32 || t[i].reserved) return MI355_W8A8_ERR_SHAPE;
    if (t[i].count == 0) continue;
    if (t[i].count > (1ull << 40) / adapters) return MI355_W8A8_ERR_UNSUPPORTED;
    if (!t[i].grad || (scale && !t[i].out)) return MI355_W8A8_ERR_NULL;
    const uint32_t size = t[i].type == MI355_W8A8_GRAD_F32 ? 4u : 2u;
    if (!aligned(t[i].grad, size) || (scale && !aligned(t[i].out, size))) return MI355_W8A8_ERR_ALIGN;
    const uint64_t bytes = t[i].count * adapters * size;
    if (overlaps(norms, adapters * 4ull, t[i].grad, bytes) || (scale && overlaps(norms, adapters * 4ull, t[i].out, bytes))) return MI355_W8A8_ERR_ALIAS;
    if (scale && t[i].out != t[i].grad && overlaps(t[i].out, bytes, t[i].grad, bytes)) return MI355_W8A8_ERR_ALIAS;
  }
  return MI355_W8A8_OK;
}

// where the table of many tensors lies behind the parts
inline uint64_t grad_parts_bytes(uint64_t pieces, uint32_t adapters) { return align256((pieces ? pieces : 1u) * adapters * 8u); }
inline uint64_t grad_table_bytes(uint32_t n) { return n > kGradShortTable ? align256((uint64_t)n * (sizeof(GradTensor) + 4u)) : 0u; }

template <uint32_t TABLE>
int launch_grads(GradArgs<TABLE>& a, uint32_t adapters, hipStream_t s) {
  hipLaunchKernelGGL(grad_norm_kernel<TABLE>, dim3(a.pieces, adapters), dim3(256), 0, s, a);
  const int st = launch_status();
  if (st) return st;
  hipLaunchKernelGGL(grad_scale_kernel<TABLE>, dim3(a.limits ? a.pieces : 1u, adapters), dim3(256), 0, s, a);
  return launch_status();
}

// entry(i, the tensor with its first piece) for every tensor that holds values
template <class Entry>
void each_grad(const mi355_w8a8_grad_tensor* t, uint32_t n, GradCall& c, Entry entry) {
  c.tensors = c.pieces = 0;
  for (uint32_t i = 0; i < n; ++i) {
    if (t[i].count == 0) continue;
    entry(c.tensors++, GradTensor{t[i].grad, t[i].out, t[i].count, c.pieces, t[i].type == MI355_W8A8_GRAD_F32});
    c.pieces += (uint32_t)pieces_of(t[i].count, c.piece);
  }
}
template <uint32_t TABLE>
int launch_grads_from_arguments(const mi355_w8a8_grad_tensor* t, uint32_t n, uint32_t adapters, const GradCall& call, hipStream_t s) {
  GradArgs<TABLE> a{};
  static_cast<GradCall&>(a) = call;
  each_grad(t, n, a, [&](uint32_t i, const GradTensor& g) { a.tensor[i] = g; });
  return launch_grads(a, adapters, s);
}
int launch_grads_from_table(const mi355_w8a8_grad_tensor* t, uint32_t n, uint32_t adapters, const GradCall& call, void* table, bool kept, hipStream_t s) {
  GradArgs<0> a{};
  static_cast<GradCall&>(a) = call;
  GradTableArgs w{};
  w.table = static_cast<GradTensor*>(table);
  w.first = reinterpret_cast<uint32_t*>(w.table + n);
  a.tensor = w.table; a.first = w.first;
  int st = MI355_W8A8_OK;
  auto write = [&] {
    if (w.tensors && !kept && !st) {
      hipLaunchKernelGGL(grad_table_kernel, dim3(1), dim3(128), 0, s, w);
      st = launch_status();
    }
    w.table += w.tensors;
    w.first += w.tensors;
    w.tensors = 0;
  };
  each_grad(t, n, a, [&](uint32_t, const GradTensor& g) {
    w.tensor[w.tensors++] = g;
    if (w.tensors == kGradTable) write();
  });
  write();
  return st ? st : launch_grads(a, adapters, s);
}

int run_grads(const mi355_w8a8_grad_tensor* t, uint32_t n, uint32_t adapters, const float* limits, float* norms, void* workspace, uint64_t workspace_bytes,
              uint32_t flags, hipStream_t s, bool scale) {
  const int st = check_grads(t, n, adapters, norms, scale);
  if (st) return st;
  if (flags & ~MI355_W8A8_FLAG_GRAD_TABLE_KEPT) return MI355_W8A8_ERR_SHAPE;
  if (scale && !limits) return MI355_W8A8_ERR_NULL;
  if (!aligned(limits, 4)) return MI355_W8A8_ERR_ALIGN;
  const uint64_t need = mi355_w8a8_grad_workspace_bytes(t, n, adapters);
  if (need == 0) return MI355_W8A8_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < need) return MI355_W8A8_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return MI355_W8A8_ERR_ALIGN;
  if (overlaps(workspace, need, norms, adapters * 4ull) || overlaps(workspace, need, limits, adapters * 4ull) ||
      overlaps(norms, adapters * 4ull, limits, limits ? adapters * 4ull : 0ull))
    return MI355_W8A8_ERR_ALIAS;
  bool any = false;
  for (uint32_t i = 0; i < n; ++i) {
    any |= t[i].count != 0;
    const uint64_t bytes = t[i].count * adapters * (t[i].type == MI355_W8A8_GRAD_F32 ? 4u : 2u);
    if (overlaps(workspace, need, t[i].grad, bytes) ||
        (scale && (overlaps(workspace, need, t[i].out, bytes) || overlaps(limits, adapters * 4ull, t[i].out, bytes))))
      return MI355_W8A8_ERR_ALIAS;
  }
  (void)hipGetLastError();
  if (!any) {  // no values: the norms are zero
    hipLaunchKernelGGL(grad_zero_norms_kernel, dim3((adapters + 255u) / 256u), dim3(256), 0, s, norms, adapters);
    return launch_status();
  }
  GradCall call{};
  call.parts = static_cast<double*>(workspace);
  call.limits = scale ? limits : nullptr;
  call.norms = norms;
  call.piece = grad_piece_values(t, n, adapters);
  if (n <= kGradShortTable) return launch_grads_from_arguments<kGradShortTable>(t, n, adapters, call, s);
  return launch_grads_from_table(t, n, adapters, call, static_cast<unsigned char*>(workspace) + need - grad_table_bytes(n),
                                 flags & MI355_W8A8_FLAG_GRAD_TABLE_KEPT, s);
}

}  // namespace

extern "C" {

uint64_t mi355_w8a8_bf16_grouped_workspace_bytes(uint32_t m, uint32_t k, uint32_t n, uint32_t n_groups, uint32_t flags) {
  return check_grouped_dims(m, k, n, n_groups) ? 0u : grouped_workspace(kGroupedFwd, m, n_groups, 0u, n, k, flags & kGroupedTiles);
}
uint64_t mi355_w8a8_bf16_grouped_bwd_workspace_bytes(uint32_t m, uint32_t k, uint32_t n, uint32_t n_groups, uint32_t flags, uint32_t want_dx,
                                                     uint32_t want_dw) {
  return check_grouped_dims(m, k, n, n_groups) ? 0u : grouped_bwd_workspace(m, k, n, n_groups, flags & kGroupedTiles, want_dx, want_dw);
}
uint32_t mi355_w8a8_bf16_grouped_bwd_joint_tile(uint32_t m, uint32_t k, uint32_t n, uint32_t n_groups, uint32_t flags) {
  if (check_grouped_dims(m, k, n, n_groups)) return 0;
  BgArgs dx{}, dw{};
  bwd_sizes(m, k, n, n_groups, dx, dw);
  return plan_grouped_both(dx, dw, flags & MI355_W8A8_FLAG_BF16_GROUPED_DW_F32 ? 4u : 2u, flags & kGroupedTiles);
}
int mi355_w8a8_bf16_grouped_v1(const mi355_w8a8_bf16_grouped_problem* problem, void* stream) {
  return run_grouped(problem, static_cast<hipStream_t>(stream));
}
int mi355_w8a8_bf16_grouped_bwd_v1(const mi355_w8a8_bf16_grouped_bwd_problem* problem, void* stream) {
  return run_grouped_bwd(problem, static_cast<hipStream_t>(stream));
}
int mi355_w8a8_embedding_v1(const mi355_w8a8_embedding_problem* problem, void* stream) {
  return run_embedding(problem, static_cast<hipStream_t>(stream));
}
uint64_t mi355_w8a8_embedding_bwd_workspace_bytes(uint32_t n_tokens, uint32_t vocab, uint32_t width, uint32_t n_adapters, uint32_t flags) {
  const uint64_t rows = (uint64_t)(n_adapters ? n_adapters : 1u) * vocab;
  if (n_tokens == 0 || rows == 0 || width == 0 || n_tokens > kMaxRows || width > MI355_W8A8_EMBEDDING_MAX_WIDTH || rows > MI355_W8A8_EMBEDDING_MAX_ROWS)
    return 0;
  return embed_layout(n_tokens, rows, width, flags).total;
}
int mi355_w8a8_embedding_bwd_v1(const mi355_w8a8_embedding_problem* problem, void* stream) {
  return run_embedding_bwd(problem, static_cast<hipStream_t>(stream));
}
uint64_t mi355_w8a8_grad_workspace_bytes(const mi355_w8a8_grad_tensor* tensors, uint32_t n_tensors, uint32_t n_adapters) {
  if (!tensors || n_tensors == 0 || n_tensors > MI355_W8A8_GRAD_MAX_TENSORS || n_adapters == 0 || n_adapters > 65535u) return 0;
  for (uint32_t i = 0; i < n_tensors; ++i)
    if (tensors[i].count > (1ull << 40) / n_adapters) return 0;
  const uint32_t piece = grad_piece_values(tensors, n_tensors, n_adapters);
  uint64_t pieces = 0;
  for (uint32_t i = 0; i < n_tensors; ++i) pieces += pieces_of(tensors[i].count, piece);
  return pieces > 0x7fffffffu ? 0u : grad_parts_bytes(pieces, n_adapters) + grad_table_bytes(n_tensors);
}
int mi355_w8a8_grad_norm_v1(const mi355_w8a8_grad_tensor* tensors, uint32_t n_tensors, uint32_t n_adapters, float* norms, void* workspace,
                            uint64_t workspace_bytes, uint32_t flags, void* stream) {
  return run_grads(tensors, n_tensors, n_adapters, nullptr, norms, workspace, workspace_bytes, flags, static_cast<hipStream_t>(stream), false);
}
int mi355_w8a8_grad_clip_v1(const mi355_w8a8_grad_tensor* tensors, uint32_t n_tensors, uint32_t n_adapters, const float* limits, float* norms,
                            void* workspace, uint64_t workspace_bytes, uint32_t flags, void* stream) {
  return run_grads(tensors, n_tensors, n_adapters, limits, norms, workspace, workspace_bytes, flags, static_cast<hipStream_t>(stream), true);
}

}  // extern "C"
