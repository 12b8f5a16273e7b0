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
// column 32 (j / 2) + 8 q + 4 (j % 2 ^ q % 2) + v, and two fragments give the lane 16 bytes to store.  (The exclusive or puts the 8-byte
// pieces that a transposing read takes from neighbouring units into different halves of them: without it two of its rows meet on the
// same banks, a third more clocks in the LDS.)
//
// Stages come by buffer_load_dwordx4 .. lds, whose range check puts zeros in the place of what lies beyond K, N or a group's rows: an
// invalid lane's offset is kOutside, past every record count.  A row of the LDS has its 16-byte units permuted by an exclusive or
// with bits of the row number (the load's lane picks the unit of memory that belongs at its place), so that a wave's read
// touches every bank equally.
#pragma once
#include <type_traits>

#include "w8a8_device.h"

namespace w8a8 {

enum GroupedKind { kGroupedFwd = 0, kGroupedDx = 1, kGroupedDw = 2 };

constexpr uint32_t kBgMaxGroups = 1024;
constexpr uint32_t kOutside = 0x80000000u;     // beyond every buffer's records (at most 2^31 - 1 bytes)
constexpr uint32_t kRecords = 0x7ffffff0u;
constexpr int kBgDepth = 64;    // contraction indices of a stage

struct BgArgs {
  const uint16_t* a;   // rows' operand: x (forward, dW) or dy (dx)
  const uint16_t* b;   // columns' operand: W, or dy (dW)
  const int32_t* sizes;
  void* out;
  uint32_t m, rows_ld, cols_ld;  // rows in all; elements between rows of a and of b
  uint32_t depth;                // contraction length of forward and dx
  uint32_t cols, rows;           // columns of C; rows of C a group (dW)
  uint32_t groups;
  uint64_t b_group, out_group;   // elements between groups of b and of C (forward, dx: of b alone)
  uint32_t splits;               // float32 results: parts of the contraction, each with a C of its own ..
  uint64_t plane;                // .. this many elements behind the one before (1 part: C itself)
};

typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// 1 KiB to the LDS, lane l 16 bytes from base + soff + voff to lds_addr + 16 l; lanes at kOutside give zeros.  (A statement of its own:
// the compiler drains every counter behind the builtin.)
__device__ inline void lds_buffer_load_1k(v4i rsrc, uint32_t voff, uint32_t soff_uniform, uint32_t lds_addr_uniform) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
               :: "v"(voff), "s"(rsrc), "s"(soff_uniform), "s"(lds_addr_uniform) : "memory", "m0");
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

// (The offset comes in the lanes' registers alone: behind a 16-byte store with a scalar offset the compiler lets the next instruction
// write the data's registers, and the memory then got what that instruction wrote.  Without one it keeps the wait states.)
// STREAM: past the caches (non-temporal).
template <bool STREAM>
__device__ inline void buffer_store_16(v4i v, v4i rsrc, uint32_t voff) {
  void* base = reinterpret_cast<void*>((uint64_t)(uint32_t)rsrc[0] | (uint64_t)(uint32_t)rsrc[1] << 32);
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, v), __builtin_amdgcn_make_buffer_rsrc(base, 0, rsrc[2], rsrc[3]), (int)voff, 0, STREAM ? 2 : 0);
}

// (a tile without products has one stage, of zeros)
__host__ __device__ inline uint32_t bg_stages(uint32_t depth) { return depth ? (depth + kBgDepth - 1u) / kBgDepth : 1u; }

// Tables of a call in the LDS, made by every workgroup from the sizes: the first row and the first tile of every group (and of the rows
// behind the last one, which are a group of their own for the forward and dx).
struct BgTables {
  uint32_t* start;   // [groups + 2]
  uint32_t* tile;    // [groups + 2]; behind the last group: the tiles in all
};

// The die of this workgroup and the share of the tiles that it takes: the workgroups are dealt out to the eight dies in turn, a die has
// tiles that follow each other (its workgroups then share operands in its L2), and the shares cost the same.
struct BgShare { uint32_t first, end; };
constexpr uint32_t kBgScratch = 64;

// Sizes are clamped to [0, m] one by one, starts to [0, m]: whatever the array holds, no row beyond m is touched.
// tiles_of, cost_of: tiles of a group with `rows` rows (nothing behind the last of `held` groups), what each costs.  scratch: kBgScratch words.
template <int THREADS, class TilesOf, class CostOf>
__device__ inline BgShare bg_tables(const BgArgs& g, uint32_t block, uint32_t held, const BgTables& tab, uint32_t* scratch, TilesOf tiles_of, CostOf cost_of) {
  constexpr uint32_t kPer = (kBgMaxGroups + THREADS) / THREADS, kWaves = THREADS / 64;  // groups a thread looks at, one more for the rows behind them
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
  if (lane == 63u) scratch[wave] = incl;
  __syncthreads();
  uint32_t at = incl - rows;
  for (uint32_t w = 0; w < wave; ++w) at += scratch[w];
  // the groups' tiles and what they cost (64 bits: thousands of stages times millions of tiles)
  uint32_t tiles[kPer], mine = 0;
  uint64_t cost = 0;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    const uint32_t gi = first + i, start = at < g.m ? at : g.m;
    at += size[i];
    const uint32_t end = gi < g.groups && at < g.m ? at : g.m;
    size[i] = end - start;
    tiles[i] = gi < held ? tiles_of(size[i]) : 0u;
    mine += tiles[i];
    cost += (uint64_t)tiles[i] * cost_of(gi, size[i]);
    if (gi <= g.groups) tab.start[gi] = start;
  }
  uint64_t* costs = reinterpret_cast<uint64_t*>(scratch + 32);
  const uint32_t incl_t = wave_scan(mine);
  uint64_t incl_c = cost;
#pragma unroll
  for (uint32_t o = 1; o < 64u; o <<= 1) {
    const uint64_t before = __shfl_up(incl_c, o);
    if (lane >= o) incl_c += before;
  }
  if (lane == 63u) {
    scratch[16 + wave] = incl_t;
    costs[wave] = incl_c;
  }
  __syncthreads();
  uint32_t total = 0, first_tile = incl_t - mine;
  uint64_t all = 0, at_cost = incl_c - cost;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    first_tile += w < wave ? scratch[16 + w] : 0u;
    total += scratch[16 + w];
    at_cost += w < wave ? costs[w] : 0u;
    all += costs[w];
  }
  // tiles in front of the share that starts at x eighths of the cost: found by the thread whose groups hold that place
  const uint32_t die = block & 7u;
  const uint64_t from = all * die / 8u, to = all * (die + 1u) / 8u;
  if (tid == 0) {
    tab.start[g.groups + 1u] = g.m;
    tab.tile[g.groups + 1u] = total;
    scratch[12] = 0;  // (behind the rows of the at most twelve waves)
    scratch[13] = total;
  }
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    const uint64_t each = cost_of(first + i, size[i]), own = tiles[i] * each;
    if (first + i <= g.groups) tab.tile[first + i] = first_tile;
    if (die > 0u && from >= at_cost && from < at_cost + own) scratch[12] = first_tile + (uint32_t)((from - at_cost) / each);
    if (die < 7u && to >= at_cost && to < at_cost + own) scratch[13] = first_tile + (uint32_t)((to - at_cost) / each);
    first_tile += tiles[i];
    at_cost += own;
  }
  __syncthreads();
  return {(uint32_t)__builtin_amdgcn_readfirstlane(scratch[12]), (uint32_t)__builtin_amdgcn_readfirstlane(scratch[13])};
}

// The last group whose first tile is not behind `tile`: 64 places at a time, at most 17 between two of them.
__device__ inline uint32_t bg_group_of(const uint32_t* first, uint32_t groups, uint32_t tile, uint32_t lane) {
  const uint32_t step = (groups + 64u) / 64u, at = lane * step;
  const uint32_t coarse = (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(at <= groups && first[at <= groups ? at : 0u] <= tile)) - 1u;
  const uint32_t fine = coarse * step + lane;
  const bool below = lane < step && fine <= groups;
  return coarse * step + (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(below && first[below ? fine : 0u] <= tile)) - 1u;
}

// The unit permutations.  ALONG: the operand is staged as [T][BK] (its rows run along the contraction), else as [BK][T].
// PAIRED: the fragment's rows are those of the columns' operand (see the head).
template <int BK, bool PAIRED>
__device__ inline uint32_t bg_unit_along(uint32_t row) {  // rows of 64 or 128 bytes: the 16 rows of a fragment on all banks
  if (BK == 32) return PAIRED ? (row >> 3) & 3u : (row >> 2) & 3u;
  return PAIRED ? ((row >> 1) & 1u) | ((row >> 3) & 3u) << 1 : (row >> 1) & 7u;
}
template <bool PAIRED>
__device__ inline uint32_t bg_unit_across(uint32_t t) {  // rows of 256 bytes: four rows t of 128 bytes on all banks
  return PAIRED ? (t & 3u) << 2 | ((t >> 3) & 1u) : ((t & 3u) << 1) | ((t >> 3) & 1u) << 3;
}

// One operand's share of a stage: kLoads loads of 1 KiB a wave, of kPlaces rows (ALONG) or contraction indices each.  Load number
// `index` of the workgroup holds the places index * kPlaces + lane / kUnits; the permutation of a place is the exclusive or of that of its lane
// part and that of its load's, which share no bits.
template <int T, int BK, bool ALONG, bool PAIRED, int WAVES>
struct BgOperand {
  static constexpr int kBytes = T * BK * 2, kLoads = kBytes / 1024 / WAVES;
  static constexpr uint32_t kUnits = (ALONG ? BK : T) / 8u, kPlaces = 64u / kUnits;
  static_assert(kBytes % (1024 * WAVES) == 0 && BK == 64, "whole loads");
  const unsigned char* base;  // of the stage that is loaded next
  uint32_t ld_bytes, valid;   // bytes between rows in memory; rows (ALONG) or columns of the tile that exist
  uint32_t place, unit, voff; // of the lane: its place in a load, the 16-byte unit of a place of even permutation, the offset of its place

  static __device__ inline uint32_t permutation(uint32_t p) {
    if constexpr (ALONG) return bg_unit_along<BK, PAIRED>(p) % kUnits;
    else return bg_unit_across<PAIRED>(p) % kUnits;
  }
  __device__ inline void init(uint32_t ld, uint32_t lane) {
    ld_bytes = ld * 2u;
    place = lane / kUnits;
    unit = (lane % kUnits) ^ permutation(place);
    voff = place * ld_bytes;
  }
  __device__ inline void open(const uint16_t* first, uint32_t existing) {
    base = reinterpret_cast<const unsigned char*>(first);
    valid = existing;
  }
  // load i of the stage at base; left: contraction indices from there on
  __device__ inline void load(int i, uint32_t left, uint32_t lds, uint32_t wave) const {
    const uint32_t index = wave * kLoads + i, at = index * kPlaces;
    const uint32_t u = unit ^ permutation(at);
    const bool in_row = u * 8u < (ALONG ? left : valid), in_places = (int)place < (int)((ALONG ? valid : left) - at);
    lds_buffer_load_1k(buffer_of(base), in_row && in_places ? voff + u * 16u : kOutside, __builtin_amdgcn_readfirstlane(at * ld_bytes),
                       __builtin_amdgcn_readfirstlane(lds + index * 1024u));
  }
  __device__ inline void next() { base += ALONG ? BK * 2u : BK * ld_bytes; }
  // Where the lane reads, from the tile's place in the LDS, for fragment 0 of the rows or columns that begin at `first` and step 0.
  __device__ static inline uint32_t lane_place(uint32_t first, uint32_t lane) {
    const uint32_t i = lane & 15u, q = lane >> 4, c = i & 3u;
    if constexpr (ALONG) {
      const uint32_t row = first + (PAIRED ? 8u * (i >> 2) + 4u * ((i >> 2) & 1u) + c : i);
      return row * (BK * 2u) + (q ^ bg_unit_along<BK, PAIRED>(row)) * 16u;
    } else {
      const uint32_t t = 8u * q + (i >> 2), col = first + (PAIRED ? 8u * c + 4u * (c & 1u) : 4u * c);
      return t * (T * 2u) + ((col >> 3) ^ (bg_unit_across<PAIRED>(t) % (T / 8u))) * 16u + (col & 4u) * 2u;
    }
  }
  // The lane's eight contraction values 32 step + 8 (lane / 16) .. of fragment f; `at`: the tile's place and the lane's.  Fragments lie an exclusive
  // or or a constant apart (no permutation depends on f, step or the wave), so that a lane keeps one register of addresses an operand.
  __device__ static inline v8bf fragment(uint32_t at, int f, int step) {
    if constexpr (ALONG) {
      typedef __attribute__((address_space(3))) const v8bf* lds_v8bf;
      return PAIRED ? *(lds_v8bf)(uintptr_t)((at ^ (512u * (f & 1) + 64u * step)) + 4096u * (f >> 1)) : *(lds_v8bf)(uintptr_t)((at ^ (64u * step)) + 2048u * f);
    } else {
      typedef __attribute__((address_space(3))) v4s* lds_v4s;
      const uint32_t place = at ^ (PAIRED ? 64u * (f >> 1) + 8u * (f & 1) : 32u * f);
      v4s h[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(uintptr_t)(place + (32u * step + 4u * u) * (T * 2u)));
      typedef short v8s __attribute__((ext_vector_type(8)));
      const v8s v = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(v8bf, v);
    }
  }
};

// One tile of a call.
struct BgTile {
  uint32_t group, start, row0, col0, rows, depth;  // rows: of the tile's group from row0 on (at least one); start: the group's first row
  uint32_t split, first;  // part of the contraction; its first index (depth: of the part)
  uint32_t number;        // of the tile in its group (and part)
  bool empty;             // the group has no rows
};

// TM x TN tiles, WM x WN waves, STAGES stages of 64 in the LDS.  LOADERS: waves that do nothing but request the stages (0: every wave its
// share).  A wave's loads and stores return in one order, so one that waits for a stage waits for the results it stored before: with
// loaders nobody does, which is what a dW of few stages a tile is made of.  A workgroup takes tile after tile, and the stages of one follow those of
// the tile before in one stream: while a tile's results are stored the first stages of the next are on their way.
// A die's workgroups take the tiles of its share in turn.  block, blocks: of this product's workgroups (a multiple of eight).
template <int KIND, int TM, int TN, int WM, int WN, int STAGES, int LOADERS, bool F32>
__device__ __forceinline__ void bg_run(const BgArgs& g, uint32_t block, uint32_t blocks) {
  constexpr int BK = kBgDepth;
  constexpr int kWaves = WM * WN, kLoading = LOADERS ? LOADERS : kWaves, FM = TM / WM / 16, FN = TN / WN / 16;
  static_assert(FN % (F32 ? 2 : 4) == 0, "a wave stores whole lines");
  using OpA = BgOperand<TM, BK, KIND != kGroupedDw, false, kLoading>;
  using OpB = BgOperand<TN, BK, KIND == kGroupedDx, !F32, kLoading>;
  constexpr uint32_t kStage = OpA::kBytes + OpB::kBytes;
  constexpr int kLoads = OpA::kLoads + OpB::kLoads, kLoadsA = OpA::kLoads, kStores = FM * FN / (F32 ? 1 : 2);
  extern __shared__ __align__(1024) unsigned char lds[];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n_tiles = (g.cols + TN - 1u) / TN;
  BgTables tab;
  uint32_t* scratch = reinterpret_cast<uint32_t*>(lds + STAGES * kStage);  // (not in the stages: some waves load while others still read it)
  tab.start = scratch + kBgScratch;
  tab.tile = tab.start + g.groups + 2u;
  const uint32_t held = KIND == kGroupedDw ? g.groups : g.groups + 1u;
  const BgShare share = bg_tables<64 * (kWaves + LOADERS)>(
      g, block, held, tab, scratch,
      [&](uint32_t rows) { return ((KIND == kGroupedDw ? g.rows : rows) + TM - 1u) / TM * n_tiles * (F32 ? g.splits : 1u); },
      // (a tile's results take about as long to store as three of its stages to compute)
      [&](uint32_t group, uint32_t rows) {
        const uint32_t stages = bg_stages(KIND == kGroupedDw ? rows : (group < g.groups ? g.depth : 0u));
        return 3u + (F32 ? (stages + g.splits - 1u) / g.splits : stages);
      });
  const uint32_t stride = blocks >> 3, end = share.end;
  uint32_t tile = share.first + (block >> 3);
  if (tile >= end) return;

  auto describe = [&](uint32_t t) {
    BgTile d;
    d.group = __builtin_amdgcn_readfirstlane(bg_group_of(tab.tile, held, t, lane));
    d.start = __builtin_amdgcn_readfirstlane(tab.start[d.group]);
    const uint32_t size = __builtin_amdgcn_readfirstlane(tab.start[d.group + 1u]) - d.start;
    uint32_t in_group = t - __builtin_amdgcn_readfirstlane(tab.tile[d.group]);
    // the row tiles of a group in bands of eight, in a band column by column: workgroups that run side by side share both operands
    const uint32_t m_tiles = ((KIND == kGroupedDw ? g.rows : size) + TM - 1u) / TM;
    d.depth = KIND == kGroupedDw ? size : (d.group == g.groups ? 0u : g.depth);
    d.split = d.first = 0;
    if (F32 && g.splits > 1u) {  // part by part, whole stages each
      const uint32_t each = (bg_stages(d.depth) + g.splits - 1u) / g.splits * BK;
      d.split = in_group / (m_tiles * n_tiles);
      in_group -= d.split * m_tiles * n_tiles;
      d.first = d.split * each < d.depth ? d.split * each : d.depth;
      d.depth = d.depth - d.first < each ? d.depth - d.first : each;
    }
    d.number = in_group;
    d.empty = size == 0u;
    const uint32_t band = in_group / (8u * n_tiles), in_band = in_group - band * 8u * n_tiles;
    const uint32_t band_tiles = m_tiles - band * 8u < 8u ? m_tiles - band * 8u : 8u;
    const uint32_t tn = in_band / band_tiles;
    d.row0 = (band * 8u + in_band - tn * band_tiles) * TM;
    d.col0 = tn * TN;
    d.rows = (KIND == kGroupedDw ? g.rows : size) - d.row0;
    return d;
  };
  OpA a;
  OpB b;
  a.init(g.rows_ld, lane);
  b.init(g.cols_ld, lane);
  uint32_t next_tile = tile, left = 0;  // of the stage that is requested next; left: contraction indices of its tile from there on
  auto open = [&](uint32_t t) {
    const BgTile d = describe(t);
    left = d.depth;
    if constexpr (KIND == kGroupedDw) {
      a.open(g.a + (uint64_t)(d.start + d.first) * g.rows_ld + d.row0, d.rows);
      b.open(g.b + (uint64_t)(d.start + d.first) * g.cols_ld + d.col0, g.cols - d.col0);
    } else {
      const uint16_t* w = g.b + (uint64_t)(d.group == g.groups ? 0u : d.group) * g.b_group;
      a.open(g.a + (uint64_t)(d.start + d.row0) * g.rows_ld + d.first, d.rows);
      b.open(w + (KIND == kGroupedFwd ? (uint64_t)d.first * g.cols_ld + d.col0 : (uint64_t)d.col0 * g.cols_ld + d.first), g.cols - d.col0);
    }
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lptr_t)lds, loader = LOADERS ? wave - kWaves : wave;
  auto request = [&](uint32_t s, int i) {
    const uint32_t at = lds0 + (s % STAGES) * kStage;
    if (i < kLoadsA) a.load(i, left, at, loader);
    else b.load(i - kLoadsA, left, at + OpA::kBytes, loader);
  };
  auto request_all = [&](uint32_t s) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) request(s, i);
  };
  auto requested = [&] {  // on to the next stage; behind the last tile nothing is left: zeros, that every wave may count the same loads
    if (left > (uint32_t)BK) {
      left -= BK;
      a.next();
      b.next();
      return;
    }
    next_tile += stride;
    left = 0;
    if (next_tile < end) open(next_tile);
  };

  if (LOADERS && wave >= kWaves) {
    open(tile);
    for (uint32_t s = 0; s < STAGES; ++s) {
      request_all(s);
      requested();
    }
    wait_vmcnt<(STAGES - 1) * kLoads>();
    lds_barrier();
    for (uint32_t s = 0; tile < end; tile += stride) {
      for (const uint32_t last = s + bg_stages(describe(tile).depth); s < last; ++s) {
        wait_vmcnt<(STAGES - 2) * kLoads>();
        lds_barrier();
        request_all(s + STAGES);
        requested();
      }
    }
    wait_vmcnt0();  // (no load into the LDS outlives the workgroup)
    return;
  }

  const uint32_t wm = wave / WN, wn = wave % WN;
  v4f acc[FM][FN];
  v8bf fa[2][FM], fb[2][FN];
  const uint32_t place_a = lds0 + OpA::lane_place(wm * (TM / WM), lane), place_b = lds0 + OpA::kBytes + OpB::lane_place(wn * (TN / WN), lane);
  auto fetch = [&](uint32_t s, int step, int f) {  // columns' fragments first
    const uint32_t at = (s % STAGES) * kStage;
    if (f < FN) fb[step][f] = OpB::fragment(at + place_b, f, step);
    else fa[step][f - FN] = OpA::fragment(at + place_a, f - FN, step);
  };
  // Half of a stage's products, and between them, so that neither waits for the other, the fragments of the next half out of the LDS
  // and (LOAD) the requests of the stage after next.  A wave issues in order: with the reads and requests in front of
  // the products both waves of a SIMD, which the barrier holds together, left the matrix unit idle meanwhile (32768 rows of 4096 ->
  // 12288 in 8 groups 2840 us, 2660 this way, and 2600 with the addresses of OpA and OpB::fragment).
  auto half = [&](auto step_c, uint32_t s_fetch, auto load_c, uint32_t s_load, auto fresh_c) {  // FRESH: a tile's first sums
    constexpr int step = step_c.value, next = 1 - step;
    constexpr bool load = load_c.value, fresh = fresh_c.value;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l)
        if (!LOADERS && load && l * FM / kLoads == i) request(s_load, l);
#pragma unroll
      for (int f = 0; f < FM + FN; ++f)
        if (f * FM / (FM + FN) == i) fetch(s_fetch, next, f);
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[step][j], fa[step][i], fresh ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Eight neighbouring columns from two fragments, with the one rounding to bf16.  Lanes of odd lane / 16 hold the second four in the first.
  auto rounded = [&](int i, int j) {
    const bool odd = (lane >> 4) & 1u;
    const int h0 = (int)pack_bf16x2(acc[i][j][0], acc[i][j][1]), h1 = (int)pack_bf16x2(acc[i][j][2], acc[i][j][3]);
    const int k0 = (int)pack_bf16x2(acc[i][j + 1][0], acc[i][j + 1][1]), k1 = (int)pack_bf16x2(acc[i][j + 1][2], acc[i][j + 1][3]);
    return v4i{odd ? k0 : h0, odd ? k1 : h1, odd ? h0 : k0, odd ? h1 : k1};
  };
  // Every wave stores the same number of times, lanes outside the tile's rows or columns beyond the buffer's end.  A lane holds 16
  // bytes of either half of a row's 128-byte line; lanes eight rows apart exchange one, and an instruction stores eight whole lines.
  auto store = [&](const BgTile& d) {
    constexpr uint32_t size = F32 ? 4u : 2u, kLine = 128u / size;
    const uint64_t at = (KIND == kGroupedDw ? d.group * g.out_group : (uint64_t)d.start * g.cols) + (uint64_t)d.row0 * g.cols + d.col0 +
                        (F32 ? d.split * g.plane : 0u);
    const v4i out = buffer_of(static_cast<unsigned char*>(g.out) + at * size);
    // A dW is larger than the caches and leaves x and dy there no room: it is streamed where its rows are whole lines (us, streamed /
    // not, 768 -> 2048, 128 groups, 32768 rows: bf16 171 / 207, float32 210 / 275; parts of lines are not joined on that way: 712 ->
    // 1096, 13 groups, 1003 rows, float32 28 / 23 when it was tried).
    const bool stream = KIND == kGroupedDw && g.cols * size % 128u == 0u && !(F32 && g.splits > 1u);
    uint32_t own = lane;
    asm volatile("" : "+v"(own));  // (offsets are made anew for every tile: kept over the products they would be spilled)
    const bool high = own & 8u;
    const uint32_t row = own & 7u, col = (own >> 4) * (16u / size) + (high ? kLine / 2u : 0u), voff = (row * g.cols + col) * size;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const uint32_t r0 = wm * (TM / WM) + 16u * i;
#pragma unroll
      for (uint32_t c0 = 0; c0 < TN / WN; c0 += kLine) {
        v4i x, y;  // the halves of the line
        if constexpr (F32) {
          x = __builtin_bit_cast(v4i, acc[i][c0 / 16u]);
          y = __builtin_bit_cast(v4i, acc[i][c0 / 16u + 1u]);
        } else {
          x = rounded(i, c0 / 16u);
          y = rounded(i, c0 / 16u + 2u);
        }
        v4i mine, theirs;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          mine[v] = high ? y[v] : x[v];
          theirs[v] = __builtin_amdgcn_update_dpp(0, high ? x[v] : y[v], 0x128, 0xf, 0xf, false);  // row_ror:8
        }
        v4i upper, lower;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          upper[v] = high ? theirs[v] : mine[v];
          lower[v] = high ? mine[v] : theirs[v];
        }
        const uint32_t c = wn * (TN / WN) + c0, to = voff + (r0 * g.cols + c) * size;
        const bool in_cols = (int)col < (int)(g.cols - d.col0 - c);
        const uint32_t to_upper = in_cols && (int)row < (int)(d.rows - r0) ? to : kOutside;
        const uint32_t to_lower = in_cols && (int)row < (int)(d.rows - r0 - 8u) ? to + 8u * g.cols * size : kOutside;
        if (stream) {
          buffer_store_16<true>(upper, out, to_upper);
          buffer_store_16<true>(lower, out, to_lower);
        } else {
          buffer_store_16<false>(upper, out, to_upper);
          buffer_store_16<false>(lower, out, to_lower);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // The dW of a group without rows is one stretch of zeros (whole lines: K and N are multiples of 8), a tile's share of it as many bytes as a
  // tile holds: the same stores, but line after line (1616 -> 10504, 56 of 78 groups empty, 756 us -> 540).
  auto clear = [&](const BgTile& d) {
    constexpr uint32_t size = F32 ? 4u : 2u;
    const uint64_t all = (uint64_t)g.rows * g.cols * size, from = (uint64_t)d.number * (TM * TN * size);
    const uint64_t left_bytes = from < all ? all - from : 0u;
    const uint32_t held_bytes = left_bytes < TM * TN * size ? (uint32_t)left_bytes : TM * TN * size;
    const v4i out = buffer_of(static_cast<unsigned char*>(g.out) + (d.group * g.out_group + (F32 ? d.split * g.plane : 0u)) * size + from);
    const bool stream = !(F32 && g.splits > 1u);
    uint32_t own = lane;
    asm volatile("" : "+v"(own));
#pragma nounroll
    for (uint32_t i = 0; i < kStores; ++i) {
      const uint32_t at = (wave * kStores + i) * 1024u + own * 16u;
      if (stream) buffer_store_16<true>(v4i{0, 0, 0, 0}, out, at < held_bytes ? at : kOutside);
      else buffer_store_16<false>(v4i{0, 0, 0, 0}, out, at < held_bytes ? at : kOutside);
    }
  };

  constexpr std::integral_constant<int, 0> first{};
  constexpr std::integral_constant<int, 1> second{};
  if constexpr (!LOADERS) {
    open(tile);
    for (uint32_t s = 0; s < STAGES; ++s) {
      request_all(s);
      requested();
    }
    wait_vmcnt<(STAGES - 1) * kLoads>();
  }
  lds_barrier();
#pragma unroll
  for (int f = 0; f < FM + FN; ++f) fetch(0, 0, f);
  bool stored = false;   // the stores of the tile before are the newest of what is on its way
  for (uint32_t s = 0; tile < end; tile += stride) {
    const BgTile d = describe(tile);
    const uint32_t last = s + bg_stages(d.depth);
    for (bool fresh = true; s < last; ++s, fresh = false) {
      if (fresh) half(first, s, std::false_type{}, 0u, std::true_type{});
      else half(first, s, std::false_type{}, 0u, std::false_type{});
      // the one barrier of a stage: behind it the next stage has arrived for every wave, and nobody reads this one any more
      if constexpr (!LOADERS) {
        if (stored) wait_vmcnt<(STAGES - 2) * kLoads + kStores>();
        else wait_vmcnt<(STAGES - 2) * kLoads>();
        stored = false;
      }
      lds_barrier();
      half(second, s + 1u, std::true_type{}, s + STAGES, std::false_type{});
      if constexpr (!LOADERS) requested();
    }
    if (KIND == kGroupedDw && d.empty) clear(d);
    else store(d);
    stored = true;
  }
  if constexpr (!LOADERS) wait_vmcnt0();
}

template <int KIND, int TM, int TN, int WM, int WN, int STAGES, int LOADERS = 0, bool F32 = false>
__global__ __launch_bounds__(64 * (WM * WN + LOADERS)) void bf16_grouped_kernel(BgArgs g) {
  bg_run<KIND, TM, TN, WM, WN, STAGES, LOADERS, F32>(g, blockIdx.x, gridDim.x);
}

// Both gradients in one launch: dx by the first dx_blocks workgroups, dW by the others, which begin where dx leaves CUs or is done.
struct BgBothArgs { BgArgs dx, dw; uint32_t dx_blocks; };
template <int TM, int TN, int WM, int WN, int STAGES, int LOADERS, bool F32>
__global__ __launch_bounds__(64 * (WM * WN + LOADERS)) void bf16_grouped_both_kernel(BgBothArgs g) {
  if (blockIdx.x < g.dx_blocks) bg_run<kGroupedDx, TM, TN, WM, WN, STAGES, LOADERS, false>(g.dx, blockIdx.x, g.dx_blocks);
  else bg_run<kGroupedDw, TM, TN, WM, WN, STAGES, LOADERS, F32>(g.dw, blockIdx.x - g.dx_blocks, gridDim.x - g.dx_blocks);
}

// The parts of a split contraction: C = their sum in order, with the one rounding.  A thread four values of C.
template <bool F32>
__global__ __launch_bounds__(256) void bg_join_kernel(const float* parts, void* out, uint64_t plane, uint32_t splits) {
  const uint64_t i = ((uint64_t)blockIdx.x * 256u + threadIdx.x) * 4u;
  if (i >= plane) return;
  float4 sum = *reinterpret_cast<const float4*>(parts + i);
#pragma unroll 8
  for (uint32_t s = 1; s < splits; ++s) {
    const float4 p = *reinterpret_cast<const float4*>(parts + s * plane + i);
    sum.x += p.x; sum.y += p.y; sum.z += p.z; sum.w += p.w;
  }
  if constexpr (F32) *reinterpret_cast<float4*>(static_cast<float*>(out) + i) = sum;
  else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
}

}  // namespace w8a8
