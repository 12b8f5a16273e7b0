// Products grouped by expert with ragged sizes, bf16 with float32 accumulation:
//
//   forward    out[i, n]   = sum_k x[i, k]  W[g(i), k, n]      (kGroupedFwd)
//   rows'      dx[i, k]    = sum_n dy[i, n] W[g(i), k, n]      (kGroupedDx)
//   experts'   dW[g, k, n] = sum_{i of g} x[i, k] dy[i, n]     (kGroupedDw)
//
// Group g owns group_sizes[g] rows behind those of the groups before it.  Rows behind the last group give zeros and take
// part in no sum; a group without rows has a zero dW.
//
// One kernel computes a tile C[r, c] = sum_t A[r, t] B[c, t] for all three.  What differs is which axis of an operand in
// memory is the contraction t: an operand whose rows run along t (x and dy of the first two, W of the second) is staged
// as [row][t] and read by ds_read_b128, one whose rows run along its own tile axis (W of the first, x and dy of the third) as
// [t][row] and read by ds_read_b64_tr_b16, which turns 4 x 16 values while they come out of the LDS: nothing is packed or
// transposed in memory.
//
// Fragments are those of v_mfma_f32_16x16x32_bf16: lane l holds the eight t = 8 (l / 16) .. + 7 of row l % 16.  The columns of C
// are the instruction's rows, so that a lane ends up with values of neighbouring columns: fragment j, row 4 q + v of 64 columns is
// column 32 (j / 2) + 8 q + 4 (j % 2) + v, and two fragments give the lane 16 bytes to store.
//
// Stages come by buffer_load_dwordx4 .. lds, whose range check puts zeros in the place of what lies beyond K, N or a group's rows: an
// invalid lane's offset is kOutside, past every record count.  A row of the LDS has its 16-byte units permuted by an exclusive or
// with bits of the row number (the load's lane picks the unit of memory that belongs at its place), so that a wave's read
// touches every bank equally.
#pragma once
#include "w8a8_device.h"

namespace w8a8 {

enum GroupedKind { kGroupedFwd = 0, kGroupedDx = 1, kGroupedDw = 2 };

constexpr uint32_t kBgMaxGroups = 1024;
constexpr uint32_t kOutside = 0x80000000u;     // beyond every buffer's records (at most 2^31 - 1 bytes)
constexpr uint32_t kRecords = 0x7ffffff0u;

struct BgArgs {
  const uint16_t* a;   // rows' operand: x (forward, dW) or dy (dx)
  const uint16_t* b;   // columns' operand: W, or dy (dW)
  const int32_t* sizes;
  void* out;
  uint32_t m, rows_ld, cols_ld;  // rows in all; elements between rows of a and of b
  uint32_t depth;                // contraction length of forward and dx
  uint32_t cols, rows;           // columns of C; rows of C a group (dW)
  uint32_t groups, f32;          // f32: C is float32
  uint64_t b_group, out_group;   // elements between groups of b and of C (forward, dx: of b alone)
};

typedef short v4s __attribute__((ext_vector_type(4)));

// 1 KiB to the LDS, lane l 16 bytes from base + voff to lds_addr + 16 l; lanes at kOutside give zeros.  (A statement of its own: the
// compiler drains every counter behind the builtin.)
__device__ inline void lds_buffer_load_1k(v4i rsrc, uint32_t voff, uint32_t lds_addr_uniform) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :: "v"(voff), "s"(rsrc), "s"(lds_addr_uniform) : "memory", "m0");
}
__device__ inline v4i buffer_of(const void* base_uniform) {
  const uint64_t a = reinterpret_cast<uint64_t>(base_uniform);
  v4i r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu));
  r[2] = (int)kRecords;
  r[3] = 0x00020000;  // raw, 32-bit
  return r;
}

// Where a group's rows start, and the tile a workgroup has.
struct BgPlace {
  uint32_t group, start, size;  // rows of the group; group == groups: the rows behind the last one
  uint32_t tile, tiles;         // this workgroup's place among the tiles of its group
};

// Sizes are clamped to [0, m] one by one, starts to [0, m]: whatever the array holds, no row beyond m is touched.
// per_group: tiles of a group of `size` rows.  Workgroup b of the grid takes tile (b % 8) * ceil(total / 8) + b / 8, so that the
// workgroups of one of the eight dies (which are dealt out in turn) hold tiles that follow each other and share operands
// in that die's L2.  False: no tile is left.
template <int THREADS, class PerGroup>
__device__ inline bool bg_place(const BgArgs& g, uint32_t groups_with_tail, uint32_t* lds, PerGroup per_group, BgPlace& place) {
  constexpr uint32_t kPer = (kBgMaxGroups + THREADS) / THREADS;  // groups a thread looks at, one more for the tail
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  uint32_t size[kPer], rows = 0, first = tid * kPer;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    const int s = first + i < g.groups ? g.sizes[first + i] : 0;
    size[i] = s < 0 ? 0u : ((uint32_t)s > g.m ? g.m : (uint32_t)s);
    rows += size[i];  // (at most 2^20 rows a group, 1024 groups)
  }
  // rows in front of this thread's groups
  const uint32_t incl = wave_scan(rows);
  if (lane == 63u) lds[wave] = incl;
  __syncthreads();
  uint32_t before = incl - rows;
  for (uint32_t w = 0; w < wave; ++w) before += lds[w];
  // the groups' tiles
  uint32_t start[kPer], tiles[kPer], mine = 0, at = before;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    const uint32_t gi = first + i;
    start[i] = at < g.m ? at : g.m;
    at += size[i];
    const uint32_t end = at < g.m ? at : g.m;
    size[i] = gi < g.groups ? end - start[i] : g.m - start[i];
    tiles[i] = gi < groups_with_tail ? per_group(gi, size[i]) : 0u;
    mine += tiles[i];
  }
  const uint32_t incl_t = wave_scan(mine);
  if (lane == 63u) lds[16 + wave] = incl_t;
  __syncthreads();
  uint32_t total = 0, first_tile = incl_t - mine;
#pragma unroll
  for (uint32_t w = 0; w < THREADS / 64; ++w) {
    const uint32_t n = lds[16 + w];
    first_tile += w < wave ? n : 0u;
    total += n;
  }
  const uint32_t each = (total + 7u) / 8u, in_die = blockIdx.x >> 3, wanted = (blockIdx.x & 7u) * each + in_die;
  const bool any = in_die < each && wanted < total;
  if (any) {
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      if (wanted >= first_tile && wanted < first_tile + tiles[i]) {
        lds[32] = first + i; lds[33] = start[i]; lds[34] = size[i]; lds[35] = wanted - first_tile; lds[36] = tiles[i];
      }
      first_tile += tiles[i];
    }
  }
  __syncthreads();
  if (!any) return false;
  place.group = __builtin_amdgcn_readfirstlane(lds[32]);
  place.start = __builtin_amdgcn_readfirstlane(lds[33]);
  place.size = __builtin_amdgcn_readfirstlane(lds[34]);
  place.tile = __builtin_amdgcn_readfirstlane(lds[35]);
  place.tiles = __builtin_amdgcn_readfirstlane(lds[36]);
  __syncthreads();
  return true;
}

// The unit permutations.  ALONG: the operand is staged as [T][BK] (its rows run along the contraction), else as [BK][T].
// PAIRED: the fragment's rows are those of the columns' operand (see the head).
template <bool PAIRED>
__device__ inline uint32_t bg_unit_along(uint32_t row) {  // 128-byte rows: the 16 rows of a fragment on all banks
  return PAIRED ? ((row >> 1) & 1u) | ((row >> 3) & 3u) << 1 : (row >> 1) & 7u;
}
template <bool PAIRED>
__device__ inline uint32_t bg_unit_across(uint32_t t) {  // rows of 256 bytes: four rows t of 128 bytes on all banks
  return PAIRED ? (t & 3u) << 2 : ((t & 3u) << 1) | ((t >> 3) & 1u) << 3;
}

// One operand's share of a stage: LOADS loads of 1 KiB a wave.
template <int T, int BK, bool ALONG, bool PAIRED, int WAVES>
struct BgOperand {
  static constexpr int kBytes = T * BK * 2, kLoads = kBytes / 1024 / WAVES;
  static_assert(kBytes % (1024 * WAVES) == 0, "whole loads");
  uint32_t voff[kLoads], need[kLoads];  // offset from the stage's base; the contraction index a lane needs
  uint32_t step_lo;                     // bytes between stages
  const unsigned char* base;

  // valid: rows (ALONG) or columns of the tile that exist
  __device__ inline void init(const uint16_t* first, uint32_t ld, uint32_t valid, uint32_t wave, uint32_t lane) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t off = (wave * kLoads + i) * 1024u + lane * 16u;
      if constexpr (ALONG) {
        const uint32_t row = off / (BK * 2u), unit = ((off >> 4) % (BK / 8u)) ^ (bg_unit_along<PAIRED>(row) % (BK / 8u));
        need[i] = unit * 8u;
        voff[i] = row < valid ? row * ld * 2u + unit * 16u : kOutside;
      } else {
        const uint32_t t = off / (T * 2u), unit = ((off >> 4) % (T / 8u)) ^ (bg_unit_across<PAIRED>(t) % (T / 8u));
        need[i] = t;
        voff[i] = unit * 8u < valid ? t * ld * 2u + unit * 16u : kOutside;
      }
    }
    step_lo = ALONG ? BK * 2u : BK * ld * 2u;
    base = reinterpret_cast<const unsigned char*>(first);
  }
  // left: contraction indices from the stage's start on
  __device__ inline void load(uint32_t left, uint32_t lds, uint32_t wave) {
    const v4i r = buffer_of(base);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      lds_buffer_load_1k(r, need[i] < left ? voff[i] : kOutside, __builtin_amdgcn_readfirstlane(lds + (wave * kLoads + i) * 1024u));
    base += step_lo;
  }
  // the lane's eight contraction values 32 step + 8 (lane / 16) .. of fragment f
  __device__ static inline v8bf fragment(const unsigned char* tile, uint32_t first, int f, int step, uint32_t lane) {
    const uint32_t i = lane & 15u, q = lane >> 4;
    if constexpr (ALONG) {
      const uint32_t row = first + (PAIRED ? 32u * (f >> 1) + 8u * (i >> 2) + 4u * (f & 1) + (i & 3u) : 16u * f + i);
      const uint32_t unit = (4u * step + q) ^ (bg_unit_along<PAIRED>(row) % (BK / 8u));
      return *reinterpret_cast<const v8bf*>(tile + row * (BK * 2u) + unit * 16u);
    } else {
      typedef __attribute__((address_space(3))) v4s* lds_v4s;
      const uint32_t c = i & 3u, col = first + (PAIRED ? 32u * (f >> 1) + 8u * c + 4u * (f & 1) : 16u * f + 4u * c);
      v4s h[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t t = 32u * step + 8u * q + 4u * u + (i >> 2);
        const uint32_t unit = (col >> 3) ^ (bg_unit_across<PAIRED>(t) % (T / 8u));
        h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(tile + t * (T * 2u) + unit * 16u + (col & 4u) * 2u));
      }
      typedef short v8s __attribute__((ext_vector_type(8)));
      const v8s v = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(v8bf, v);
    }
  }
};

// TM x TN tiles, WM x WN waves, stages of BK.
template <int KIND, int TM, int TN, int WM, int WN, int BK, int STAGES>
__global__ __launch_bounds__(64 * WM * WN) void bf16_grouped_kernel(BgArgs g) {
  constexpr int kWaves = WM * WN, FM = TM / WM / 16, FN = TN / WN / 16;
  static_assert(FN % 2 == 0, "a lane stores two fragments together");
  using OpA = BgOperand<TM, BK, KIND != kGroupedDw, false, kWaves>;
  using OpB = BgOperand<TN, BK, KIND == kGroupedDx, true, kWaves>;
  extern __shared__ __align__(1024) unsigned char lds[];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n_tiles = (g.cols + TN - 1u) / TN;
  BgPlace place;
  const uint32_t with_tail = KIND == kGroupedDw ? g.groups : g.groups + 1u;
  auto per_group = [&](uint32_t, uint32_t size) {
    return (KIND == kGroupedDw ? (g.rows + TM - 1u) / TM : (size + TM - 1u) / TM) * n_tiles;
  };
  if (!bg_place<64 * kWaves>(g, with_tail, reinterpret_cast<uint32_t*>(lds), per_group, place)) return;
  // the row tiles of a group in bands of eight, in a band column by column: workgroups that run side by side share both operands
  const uint32_t m_tiles = place.tiles / n_tiles, band = place.tile / (8u * n_tiles), in_band = place.tile - band * 8u * n_tiles;
  const uint32_t band_tiles = m_tiles - band * 8u < 8u ? m_tiles - band * 8u : 8u;
  const uint32_t tn = in_band / band_tiles, tm = band * 8u + in_band - tn * band_tiles;
  const uint32_t row0 = tm * TM, col0 = tn * TN;
  const uint32_t rows = (KIND == kGroupedDw ? g.rows : place.size) - row0;  // (at least one)
  const bool tail = KIND != kGroupedDw && place.group == g.groups;
  const uint32_t depth = KIND == kGroupedDw ? place.size : (tail ? 0u : g.depth);

  OpA a;
  OpB b;
  if constexpr (KIND == kGroupedDw) {
    a.init(g.a + (uint64_t)place.start * g.rows_ld + row0, g.rows_ld, rows, wave, lane);
    b.init(g.b + (uint64_t)place.start * g.cols_ld + col0, g.cols_ld, g.cols - col0, wave, lane);
  } else {
    const uint16_t* w = g.b + (uint64_t)(tail ? 0u : place.group) * g.b_group;
    a.init(g.a + (uint64_t)(place.start + row0) * g.rows_ld, g.rows_ld, rows, wave, lane);
    b.init(w + (KIND == kGroupedFwd ? (uint64_t)col0 : (uint64_t)col0 * g.cols_ld), g.cols_ld, g.cols - col0, wave, lane);
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lptr_t)lds;
  constexpr uint32_t kStage = OpA::kBytes + OpB::kBytes, kStageLoads = OpA::kLoads + OpB::kLoads;
  const uint32_t wm = wave / WN, wn = wave % WN;

  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  const uint32_t stages = (depth + BK - 1u) / BK;
  auto request = [&](uint32_t s) {
    const uint32_t at = lds0 + (s % STAGES) * kStage, left = depth - s * BK;  // (beyond the last stage: nothing is left)
    const uint32_t l = s < stages ? left : 0u;
    a.load(l, at, wave);
    b.load(l, at + OpA::kBytes, wave);
  };
  // (a request beyond the last stage reads nothing and leaves zeros: every wave counts the same loads)
  for (uint32_t s = 0; s + 1 < STAGES; ++s) request(s);
  for (uint32_t s = 0; s < stages; ++s) {
    wait_vmcnt<(STAGES - 2) * (int)kStageLoads>();
    lds_barrier();
    request(s + STAGES - 1);
    const unsigned char* at = lds + (s % STAGES) * kStage;
#pragma unroll
    for (int step = 0; step < BK / 32; ++step) {
      v8bf fa[FM], fb[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = OpB::fragment(at + OpA::kBytes, wn * (TN / WN), j, step, lane);
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = OpA::fragment(at, wm * (TM / WM), i, step, lane);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
    }
  }
  wait_vmcnt0();  // (no load into the LDS outlives the workgroup)

  const uint64_t out0 = KIND == kGroupedDw ? place.group * g.out_group : (uint64_t)place.start * g.cols;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const uint32_t r = wm * (TM / WM) + 16u * i + (lane & 15u);
    if (r >= rows) continue;
    const uint64_t at = out0 + (uint64_t)(row0 + r) * g.cols;
#pragma unroll
    for (int j = 0; j < FN; j += 2) {
      const uint32_t c = col0 + wn * (TN / WN) + 32u * (j >> 1) + 8u * (lane >> 4);
      if (c >= g.cols) continue;
      if (KIND == kGroupedDw && g.f32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(g.out) + at + c);
        p[0] = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
        p[1] = make_float4(acc[i][j + 1][0], acc[i][j + 1][1], acc[i][j + 1][2], acc[i][j + 1][3]);
      } else {
        uint4 v;  // the one rounding to bf16
        v.x = pack_bf16x2(acc[i][j][0], acc[i][j][1]);
        v.y = pack_bf16x2(acc[i][j][2], acc[i][j][3]);
        v.z = pack_bf16x2(acc[i][j + 1][0], acc[i][j + 1][1]);
        v.w = pack_bf16x2(acc[i][j + 1][2], acc[i][j + 1][3]);
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(g.out) + at + c) = v;
      }
    }
  }
}

}  // namespace w8a8
