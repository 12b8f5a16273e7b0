// Rows of an embedding table, scaled, and the table's gradient by sorted tokens.
//
//   forward    out[t]   = scale(t) * table[row(t)]           row(t) = adapter(t) * vocab + id(t)
//   backward   grad[v]  = scale(v) * sum_{t: row(t) = v} dy[t]   every row of the table is written, zeros where no token names it
//
// A plain table is one adapter with one scale.  An id outside [0, vocab), or an adapter outside [0, adapters), names no row: the
// forward gives zeros, the backward leaves the token out.
//
//   embed_rows_kernel          a thread per unit of the output
//   embed_sort_small_kernel    up to 1024 tokens: a stable radix sort of the rows' numbers in one launch
//   embed_count_kernel, embed_scan_kernel, embed_place_kernel   more of them: for each digit a launch that counts, while other workgroups
//                              clear a share of the gradient, and one that places the keys (and a scan of the counts between them
//                              where there are many chunks)
//   embed_sum_kernel           a thread per (run of positions of the sorted order, unit of a row): the sums of the rows that begin
//                              and end inside a run are written, the others' parts are left in the workspace
//   embed_join_kernel          rows that reach over several runs: their parts
//
// Sums are float32 in a fixed order of the tokens: the same bits at every call.
#pragma once
#include "w8a8_device.h"

namespace w8a8 {

struct EmbedArgs {
  const void* table;       // forward
  void* out;               // forward: [n, width]; backward: the table's gradient
  const void* dy;          // backward
  const void* ids;         // int32 or int64 [n]
  const int32_t* adapters; // int32 [n] or null
  const float* scales;     // f32 [n_adapters], or null: `scale`
  float scale;
  uint32_t n, vocab, width, n_adapters, ids64;
};

// row of token t, or n_adapters * vocab where there is none
__device__ inline uint32_t embed_row(const EmbedArgs& e, uint32_t t) {
  const uint32_t none = e.n_adapters * e.vocab;
  uint64_t id;
  if (e.ids64) id = (uint64_t)static_cast<const int64_t*>(e.ids)[t];
  else id = (uint64_t)(int64_t)static_cast<const int32_t*>(e.ids)[t];
  if (id >= e.vocab) return none;
  if (!e.adapters) return (uint32_t)id;
  const uint32_t a = (uint32_t)e.adapters[t];
  return a < e.n_adapters ? a * e.vocab + (uint32_t)id : none;
}

// A unit is V values of a row: 16 bytes wherever they begin (the loads and stores need no alignment beyond the values'), the last one of a row
// drawn back to the row's end, so that two threads may write the same values there; one value where a row has fewer.  (Values one by
// one for widths that are no multiple of 8: 5498 rows of 3415 bf16 values summed in 21 us, 10 this way.)
__host__ __device__ inline uint32_t embed_units(uint32_t width, uint32_t v) { return (width + v - 1u) / v; }
__device__ inline uint32_t embed_start(uint32_t u, uint32_t width, uint32_t v) { return u * v + v <= width ? u * v : width - v; }

typedef uint32_t v4u_at_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t v2u_at_2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float v4f_at_4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T, int V> struct EmbedUnit;
template <> struct EmbedUnit<uint16_t, 8> {
  static __device__ inline void load(const void* p, float (&f)[8]) {
    const v4u_at_2 r = *static_cast<const v4u_at_2*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ inline void store(void* p, const float (&f)[8]) {
    *static_cast<v4u_at_2*>(p) = v4u_at_2{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
  }
};
template <> struct EmbedUnit<uint16_t, 4> {  // (of the join, which reads float32 values)
  static __device__ inline void store(void* p, const float (&f)[4]) { *static_cast<v2u_at_2*>(p) = v2u_at_2{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])}; }
};
template <> struct EmbedUnit<uint16_t, 1> {
  static __device__ inline void load(const void* p, float (&f)[1]) { f[0] = bf16_bits_to_f32(*static_cast<const uint16_t*>(p)); }
  static __device__ inline void store(void* p, const float (&f)[1]) { *static_cast<uint16_t*>(p) = (uint16_t)f32_to_bf16_bits(f[0]); }
};
template <> struct EmbedUnit<float, 4> {
  static __device__ inline void load(const void* p, float (&f)[4]) {
    const v4f_at_4 r = *static_cast<const v4f_at_4*>(p);
    f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w;
  }
  static __device__ inline void store(void* p, const float (&f)[4]) { *static_cast<v4f_at_4*>(p) = v4f_at_4{f[0], f[1], f[2], f[3]}; }
};
template <> struct EmbedUnit<float, 1> {
  static __device__ inline void load(const void* p, float (&f)[1]) { f[0] = *static_cast<const float*>(p); }
  static __device__ inline void store(void* p, const float (&f)[1]) { *static_cast<float*>(p) = f[0]; }
};

constexpr uint32_t kEmbedRowBlocks = 1u << 20;  // workgroups along the first axis
template <typename T, int V>
__global__ __launch_bounds__(256) void embed_rows_kernel(EmbedArgs e) {
  const uint32_t units = embed_units(e.width, V);
  const uint64_t i = ((uint64_t)blockIdx.y * kEmbedRowBlocks + blockIdx.x) * 256u + threadIdx.x;
  const uint32_t t = (uint32_t)(i / units), at = embed_start((uint32_t)(i - (uint64_t)t * units), e.width, V);
  if (t >= e.n) return;
  const uint32_t row = embed_row(e, t);
  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = 0.0f;
  if (row < e.n_adapters * e.vocab) {
    const float s = e.scales ? e.scales[row / e.vocab] : e.scale;
    EmbedUnit<T, V>::load(static_cast<const T*>(e.table) + (uint64_t)row * e.width + at, f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] *= s;
  }
  EmbedUnit<T, V>::store(static_cast<T*>(e.out) + (uint64_t)t * e.width + at, f);
}

// ---------------------------------------------------------------------------------------
constexpr uint32_t kEmbedChunk = 1024;      // keys a workgroup places
constexpr uint32_t kEmbedDigits = 2048;     // most values of one digit
constexpr uint32_t kEmbedSumChunks = 64;    // up to here a workgroup adds up the chunks' counts for itself
constexpr uint32_t kEmbedNotes = 64;        // words in front of the counts; the first: rows of many parts
constexpr uint32_t kEmbedShort = 8;         // parts that a thread of the join adds up by itself
constexpr uint32_t kEmbedLongs = 1024;      // most workgroups for the rows of more

struct EmbedSortArgs {
  EmbedArgs e;
  const uint32_t* keys;     // null: the first pass, from the ids
  const uint32_t* tokens;
  uint32_t* keys_out;
  uint32_t* tokens_out;
  uint32_t* counts;         // [chunks + 1][digits] of this pass: keys of a chunk with a digit; behind a scan the keys in front of them
  uint32_t* notes;          // [kEmbedNotes]
  uint32_t shift, bits, chunks, passes;
  uint32_t stream;          // the gradient is larger than the caches: it is cleared past them
  uint4* clear;             // the share of the gradient that this launch clears, in 16-byte pieces, and the bytes behind the last one
  uint64_t clear_pieces;
  uint32_t clear_rest;
};

__device__ inline uint32_t embed_key(const EmbedSortArgs& a, uint32_t p) { return a.keys ? a.keys[p] : embed_row(a.e, p); }

// The first 256 threads of each of at most 256 workgroups, 16 bytes after 16 bytes all over the share: so few write 6.9 TB/s (past the
// caches 6.4), four times the threads 6.2 (5.6).
constexpr uint32_t kEmbedClearing = 256;
__device__ inline void embed_clear(const EmbedSortArgs& a, uint32_t block, uint32_t blocks) {
  if (threadIdx.x >= 256u) return;
  const uint64_t step = (uint64_t)blocks * 256u;
  const v4u_at_2 zeros = {0u, 0u, 0u, 0u};
  v4u_at_2* const clear = reinterpret_cast<v4u_at_2*>(a.clear);
  if (a.stream) {
    for (uint64_t i = (uint64_t)block * 256u + threadIdx.x; i < a.clear_pieces; i += step) __builtin_nontemporal_store(zeros, clear + i);
  } else {
    for (uint64_t i = (uint64_t)block * 256u + threadIdx.x; i < a.clear_pieces; i += step) clear[i] = zeros;
  }
  if (block == 0 && threadIdx.x < a.clear_rest) reinterpret_cast<unsigned char*>(a.clear + a.clear_pieces)[threadIdx.x] = 0;
}

// Keys of a chunk in front of this thread's with the same digit: in earlier waves, and in earlier lanes of its wave.  A wave finds the
// lanes that share a digit with one ballot a bit.  wave_cnt: [16][digits].
__device__ inline uint32_t embed_rank(uint32_t d, bool valid, uint32_t digits, uint16_t* wave_cnt) {
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  for (uint32_t i = tid; i < 2u * digits; i += 1024u) reinterpret_cast<uint4*>(wave_cnt)[i] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  unsigned long long same = __builtin_amdgcn_ballot_w64(valid);
  for (uint32_t bit = 1u; bit < digits; bit <<= 1) {
    const bool one = d & bit;
    const unsigned long long ones = __builtin_amdgcn_ballot_w64(one);
    same &= one ? ones : ~ones;
  }
  const uint32_t in_wave = (uint32_t)__builtin_popcountll(same & ((1ull << lane) - 1ull));
  if (valid && in_wave == 0) wave_cnt[wave * digits + d] = (uint16_t)__builtin_popcountll(same);
  __syncthreads();
  uint32_t rank = in_wave;
#pragma unroll
  for (uint32_t w = 0; w < 16; ++w) {
    const uint32_t c = wave_cnt[w * digits + d];
    rank += w < wave ? c : 0u;
  }
  return rank;
}

// exclusive prefix over values 2 tid, 2 tid + 1 of the workgroup's 1024 threads
__device__ inline void embed_prefix(uint32_t (&v)[2], uint32_t* waves) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t own = v[0] + v[1], incl = wave_scan(own);
  if (lane == 63u) waves[wave] = incl;
  __syncthreads();
  uint32_t before = incl - own;
#pragma unroll
  for (uint32_t w = 0; w < 16; ++w) before += w < wave ? waves[w] : 0u;
  v[1] = before + v[0];
  v[0] = before;
}

// Up to one chunk of keys: all passes in the LDS, in one launch.
__global__ __launch_bounds__(1024) void embed_sort_small_kernel(EmbedSortArgs a) {
  extern __shared__ __align__(16) unsigned char lds[];
  if (blockIdx.x >= 1u) return embed_clear(a, blockIdx.x - 1u, gridDim.x - 1u);
  uint32_t* all = reinterpret_cast<uint32_t*>(lds);   // keys of a digit, then those of smaller ones
  uint32_t* waves = all + kEmbedDigits;
  uint32_t* moved = waves + 16;                       // [2][1024] keys and tokens in their new order
  uint16_t* wave_cnt = reinterpret_cast<uint16_t*>(moved + 2048);
  const uint32_t tid = threadIdx.x, digits = 1u << a.bits;
  if (tid < kEmbedNotes) a.notes[tid] = 0;
  const bool valid = tid < a.e.n;
  uint32_t key = valid ? embed_row(a.e, tid) : 0u, token = tid;
  for (uint32_t pass = 0; pass < a.passes; ++pass) {
    const uint32_t d = (key >> (pass * a.bits)) & (digits - 1u);
    all[tid] = all[tid + 1024u] = 0;
    const uint32_t rank = embed_rank(d, valid, digits, wave_cnt);  // (its barriers: all is clear, the keys are read)
    if (valid) atomicAdd(&all[d], 1u);
    __syncthreads();
    uint32_t v[2] = {all[2 * tid], all[2 * tid + 1]};
    embed_prefix(v, waves);
    all[2 * tid] = v[0];
    all[2 * tid + 1] = v[1];
    __syncthreads();
    if (valid) {
      const uint32_t at = all[d] + rank;
      moved[at] = key;
      moved[1024u + at] = token;
    }
    __syncthreads();
    key = moved[tid];
    token = moved[1024u + tid];
  }
  if (valid) {
    a.keys_out[tid] = key;
    a.tokens_out[tid] = token;
  }
}

// A pass' digits, chunk by chunk.  (Counted by the launch that places the digit before, with an atomic a key, that launch takes as much
// longer as this one costs: 13 us for 8.6.)
__global__ __launch_bounds__(1024) void embed_count_kernel(EmbedSortArgs a) {
  __shared__ uint32_t cnt[kEmbedDigits];
  if (blockIdx.x >= a.chunks) return embed_clear(a, blockIdx.x - a.chunks, gridDim.x - a.chunks);
  const uint32_t tid = threadIdx.x, chunk = blockIdx.x, digits = 1u << a.bits;
  if (chunk == 0 && tid < kEmbedNotes) a.notes[tid] = 0;
  cnt[tid] = cnt[tid + 1024u] = 0;
  __syncthreads();
  const uint32_t p = chunk * kEmbedChunk + tid;
  if (p < a.e.n) atomicAdd(&cnt[(embed_key(a, p) >> a.shift) & (digits - 1u)], 1u);
  __syncthreads();
  for (uint32_t i = tid; i < digits; i += 1024u) a.counts[((uint64_t)chunk << a.bits) + i] = cnt[i];
}
// Many chunks: their counts become the keys of the digit in earlier chunks, and behind them the keys of smaller digits.
__global__ __launch_bounds__(1024) void embed_scan_kernel(EmbedSortArgs a) {
  __shared__ uint32_t waves[16];
  const uint32_t tid = threadIdx.x, digits = 1u << a.bits;
  uint32_t v[2] = {0u, 0u};
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h) {
    const uint32_t d = 2u * tid + h;
    if (d >= digits) continue;
    uint32_t run = 0;
#pragma unroll 16
    for (uint32_t c = 0; c < a.chunks; ++c) {
      const uint32_t t = a.counts[((uint64_t)c << a.bits) + d];
      a.counts[((uint64_t)c << a.bits) + d] = run;
      run += t;
    }
    v[h] = run;
  }
  embed_prefix(v, waves);
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h)
    if (2u * tid + h < digits) a.counts[((uint64_t)a.chunks << a.bits) + 2u * tid + h] = v[h];
}
// Every key to its place.
template <bool SCANNED>
__global__ __launch_bounds__(1024) void embed_place_kernel(EmbedSortArgs a) {
  extern __shared__ __align__(16) unsigned char lds[];
  uint32_t* first = reinterpret_cast<uint32_t*>(lds);
  uint32_t* waves = first + kEmbedDigits;
  uint16_t* wave_cnt = reinterpret_cast<uint16_t*>(waves + 16);
  const uint32_t tid = threadIdx.x, chunk = blockIdx.x, digits = 1u << a.bits;
  const uint32_t p = chunk * kEmbedChunk + tid;
  const bool valid = p < a.e.n;
  const uint32_t key = valid ? embed_key(a, p) : 0u, d = (key >> a.shift) & (digits - 1u);
  if (SCANNED) {
    for (uint32_t i = tid; i < digits; i += 1024u)
      first[i] = a.counts[((uint64_t)a.chunks << a.bits) + i] + a.counts[((uint64_t)chunk << a.bits) + i];
  } else {
    uint32_t v[2] = {0u, 0u}, earlier[2] = {0u, 0u};
    if (2u * tid < digits) {
      const uint2* row = reinterpret_cast<const uint2*>(a.counts) + tid;
#pragma unroll 16
      for (uint32_t c = 0; c < a.chunks; ++c) {
        const uint2 t = row[(uint64_t)c << (a.bits - 1u)];
        v[0] += t.x;
        v[1] += t.y;
        earlier[0] += c < chunk ? t.x : 0u;
        earlier[1] += c < chunk ? t.y : 0u;
      }
    }
    embed_prefix(v, waves);
    first[2 * tid] = v[0] + earlier[0];
    first[2 * tid + 1] = v[1] + earlier[1];
  }
  const uint32_t rank = embed_rank(d, valid, digits, wave_cnt);  // (behind its barriers `first` is whole)
  if (!valid) return;
  const uint32_t at = first[d] + rank;
  a.keys_out[at] = key;
  a.tokens_out[at] = a.keys ? a.tokens[p] : p;
}

// ---------------------------------------------------------------------------------------
struct EmbedSumArgs {
  EmbedArgs e;
  const uint32_t* keys;    // [n], sorted
  const uint32_t* tokens;
  float* parts;            // [runs][2][width]: of a row that reaches into the run, of one that begins in it and reaches out
  uint32_t* joins;         // [runs] runs whose last row begins in them and has more than kEmbedShort parts, in any order
  uint32_t* notes;         // the first: how many
  uint32_t run, runs;      // positions of a run
};

__device__ inline float embed_scale(const EmbedArgs& e, uint32_t row) { return e.scales ? e.scales[row / e.vocab] : e.scale; }

// Sums of unit u of run r's rows, from value `first` of theirs on.  WIDE: the run is the wave's, so that its keys and tokens come by scalar loads.
template <typename T, int V, bool WIDE>
__device__ inline void embed_sum_run(const EmbedSumArgs& a, uint32_t r, uint32_t u) {
  const uint32_t none = a.e.n_adapters * a.e.vocab;
  const uint32_t p0 = r * a.run, p1 = p0 + a.run < a.e.n ? p0 + a.run : a.e.n;
  const uint32_t first = embed_start(u, a.e.width, V);
  const T* dy = static_cast<const T*>(a.e.dy) + first;
  T* out = static_cast<T*>(a.e.out) + first;
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.0f;
  const uint32_t behind = p1 < a.e.n ? a.keys[p1] : none + 1u;
  bool from_before = p0 > 0 && a.keys[p0 - 1u] == a.keys[p0];
  // eight positions at a time: their rows are on the way together
  for (uint32_t p = p0; p < p1; p += 8u) {
    uint32_t k[9], t[8];
    float f[8][V];
#pragma unroll
    for (uint32_t x = 0; x < 8; ++x) {
      const uint32_t at = p + x < p1 ? p + x : p1 - 1u;
      k[x] = a.keys[at];
      t[x] = a.tokens[at];
    }
    k[8] = p + 8u < p1 ? a.keys[p + 8u] : behind;
#pragma unroll
    for (uint32_t x = 0; x < 8; ++x) EmbedUnit<T, V>::load(dy + (uint64_t)t[x] * a.e.width, f[x]);
#pragma unroll
    for (uint32_t x = 0; x < 8; ++x) {
      if (p + x >= p1) break;
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += f[x][j];
      const bool last = p + x + 1u == p1;
      const uint32_t next = last ? behind : k[x + 1];
      if (next == k[x] && !last) continue;
      if (k[x] < none) {
        if (from_before || next == k[x]) {
          float* part = a.parts + ((uint64_t)r * 2u + (from_before ? 0u : 1u)) * a.e.width + first;
#pragma unroll
          for (int j = 0; j < V; ++j) part[j] = sum[j];
          if (!from_before && u == 0) {
            const uint64_t far = (uint64_t)(r + kEmbedShort) * a.run;
            if (far < a.e.n && a.keys[far] == k[x]) a.joins[atomicAdd(a.notes, 1u)] = r;
          }
        } else {
          const float s = embed_scale(a.e, k[x]);
#pragma unroll
          for (int j = 0; j < V; ++j) sum[j] *= s;
          EmbedUnit<T, V>::store(out + (uint64_t)k[x] * a.e.width, sum);
        }
      }
      from_before = false;
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    }
  }
}

template <typename T, int V, bool WIDE>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedSumArgs a) {
  const uint32_t units = embed_units(a.e.width, V);
  if (WIDE) {  // a wave: 64 units of one run
    const uint32_t waves = (units + 63u) / 64u, w = __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6));
    const uint32_t r = w / waves, u = (w - r * waves) * 64u + (threadIdx.x & 63u);
    if (r < a.runs && u < units) embed_sum_run<T, V, true>(a, r, u);
  } else {
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint32_t r = (uint32_t)(i / units), u = (uint32_t)(i - (uint64_t)r * units);
    if (r < a.runs) embed_sum_run<T, V, false>(a, r, u);
  }
}

// The rows that reach over several runs.  Few parts: a thread adds up its unit's, all requested together.  Many: a workgroup takes
// four units, each of a unit's 64 threads a 64th of the parts, then theirs pairwise.  (A thread for every row walks the 160
// parts of a padding word one after the other, 33 us; a workgroup for every row with two parts is 28 us of dependent loads; sixteen threads
// a unit are 19 us for a row of 630 parts, 64 of them 8.)
template <typename T, int V>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedSumArgs a) {
  __shared__ float lds[4][4][V];
  const uint32_t units = embed_units(a.e.width, V);
  const uint32_t longs = gridDim.x < 2u * kEmbedLongs ? gridDim.x / 2u : kEmbedLongs;  // the first workgroups: rows of many parts
  for (uint64_t i = (uint64_t)(blockIdx.x - longs) * 256u + threadIdx.x; blockIdx.x >= longs && i < (uint64_t)(a.runs - 1u) * units;
       i += (uint64_t)(gridDim.x - longs) * 256u) {
    const uint32_t r = (uint32_t)(i / units), first = embed_start((uint32_t)(i - (uint64_t)r * units), a.e.width, V);
    const uint32_t end = (r + 1u) * a.run, key = a.keys[end], last = a.keys[end - 1u];  // (a run follows: this one is whole)
    const uint32_t before = r ? a.keys[r * a.run - 1u] : key + 1u;
    const uint64_t far = (uint64_t)(r + kEmbedShort) * a.run;
    if (last != key || before == key || key >= a.e.n_adapters * a.e.vocab || (far < a.e.n && a.keys[far] == key)) continue;
    float f[kEmbedShort][V];
#pragma unroll
    for (uint32_t x = 0; x < kEmbedShort; ++x) {
      const uint64_t at = (uint64_t)(r + x) * a.run;
      const bool held = x < 2u || (at < a.e.n && a.keys[at] == key);
      const float* part = a.parts + ((uint64_t)(r + x) * 2u + (x == 0 ? 1u : 0u)) * a.e.width + first;
#pragma unroll
      for (int j = 0; j < V; ++j) f[x][j] = held ? part[j] : 0.0f;
    }
    float sum[V];
    const float s = embed_scale(a.e, key);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      sum[j] = f[0][j];
#pragma unroll
      for (uint32_t x = 1; x < kEmbedShort; ++x) sum[j] += f[x][j];
      sum[j] *= s;
    }
    EmbedUnit<T, V>::store(static_cast<T*>(a.e.out) + (uint64_t)key * a.e.width + first, sum);
  }
  if (blockIdx.x >= longs) return;
  const uint32_t groups = (units + 3u) / 4u, lane = threadIdx.x & 3u, share = threadIdx.x >> 2;
  const uint64_t todo = (uint64_t)a.notes[0] * groups;
  for (uint64_t i = blockIdx.x; i < todo; i += longs) {
    const uint32_t r = a.joins[i / groups], u = (uint32_t)(i % groups) * 4u + lane, first = embed_start(u < units ? u : units - 1u, a.e.width, V);
    const uint32_t key = a.keys[(r + 1u) * a.run];
    // its parts: the run's own and those of the runs that begin with the row, which follow each other: 256 places of the rest, then one by
    // one between two of them (at most 2^17 runs)
    uint32_t parts = 1u;
    for (uint32_t step = (a.runs - r + 255u) / 256u; step; step = step > 1u ? (step + 255u) / 256u : 0u) {
      const uint64_t place = (uint64_t)r + parts + (uint64_t)(threadIdx.x + 1u) * step - 1u;
      parts += (uint32_t)__syncthreads_count(place < a.runs && a.keys[place * a.run] == key) * step;
    }
    const uint32_t each = (parts + 63u) / 64u, from = share * each, to = from + each < parts ? from + each : parts;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
#pragma unroll 8
    for (uint32_t x = from; x < to; ++x) {
      const float* part = a.parts + ((uint64_t)(r + x) * 2u + (x == 0 ? 1u : 0u)) * a.e.width + first;
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += part[j];
    }
    // the sixteen shares of a wave, then the four waves
#pragma unroll
    for (uint32_t o = 4; o < 64u; o <<= 1)
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += __shfl_xor(sum[j], o);
    if ((threadIdx.x & 63u) < 4u)
#pragma unroll
      for (int j = 0; j < V; ++j) lds[threadIdx.x >> 6][lane][j] = sum[j];
    __syncthreads();
    if (share == 0 && u < units) {
#pragma unroll
      for (uint32_t y = 1; y < 4; ++y)
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += lds[y][lane][j];
      const float s = embed_scale(a.e, key);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] *= s;
      EmbedUnit<T, V>::store(static_cast<T*>(a.e.out) + (uint64_t)key * a.e.width + first, sum);
    }
    __syncthreads();
  }
}

}  // namespace w8a8
