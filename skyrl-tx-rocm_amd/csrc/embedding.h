// Rows of an embedding table, scaled, and the table's gradient by sorted tokens.
//
//   forward    out[t]   = scale(t) * table[row(t)]           row(t) = adapter(t) * vocab + id(t)
//   backward   grad[v]  = scale(v) * sum_{t: row(t) = v} dy[t]   every row of the table is written, zeros where no token names it
//
// A plain table is one adapter with one scale.  An id outside [0, vocab), or an adapter outside [0, adapters), names no row: the
// forward gives zeros, the backward leaves the token out.
//
//   embed_rows_kernel          a thread per 16 bytes of the output
//   embed_sort_kernel          one stable pass of a radix sort of the rows' numbers; its other workgroups clear the gradient
//   embed_sum_kernel           a thread per (run of positions of the sorted order, 16 bytes of a row): the sums of the rows that begin
//                              and end inside a run are written, the others' parts are left in the workspace
//   embed_join_kernel          rows that reach over several runs: their parts in order
//
// Sums are float32 in the order of the tokens: the same bits at every call.
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

// V values of a row at a time: 16 bytes where rows and pointers allow, else one value.
template <typename T, int V> struct EmbedUnit;
template <> struct EmbedUnit<uint16_t, 8> {
  static __device__ inline void load(const void* p, float (&f)[8]) {
    const uint4 r = *static_cast<const uint4*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ inline void store(void* p, const float (&f)[8]) {
    *static_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <> struct EmbedUnit<uint16_t, 1> {
  static __device__ inline void load(const void* p, float (&f)[1]) { f[0] = bf16_bits_to_f32(*static_cast<const uint16_t*>(p)); }
  static __device__ inline void store(void* p, const float (&f)[1]) { *static_cast<uint16_t*>(p) = (uint16_t)f32_to_bf16_bits(f[0]); }
};
template <> struct EmbedUnit<float, 4> {
  static __device__ inline void load(const void* p, float (&f)[4]) {
    const float4 r = *static_cast<const float4*>(p);
    f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w;
  }
  static __device__ inline void store(void* p, const float (&f)[4]) { *static_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct EmbedUnit<float, 1> {
  static __device__ inline void load(const void* p, float (&f)[1]) { f[0] = *static_cast<const float*>(p); }
  static __device__ inline void store(void* p, const float (&f)[1]) { *static_cast<float*>(p) = f[0]; }
};

template <typename T, int V>
__global__ __launch_bounds__(256) void embed_rows_kernel(EmbedArgs e) {
  const uint32_t units = e.width / V;
  const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  const uint32_t t = (uint32_t)(i / units), u = (uint32_t)(i - (uint64_t)t * units);
  if (t >= e.n) return;
  const uint32_t row = embed_row(e, t);
  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = 0.0f;
  if (row < e.n_adapters * e.vocab) {
    const float s = e.scales ? e.scales[row / e.vocab] : e.scale;
    EmbedUnit<T, V>::load(static_cast<const T*>(e.table) + (uint64_t)row * e.width + u * V, f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] *= s;
  }
  EmbedUnit<T, V>::store(static_cast<T*>(e.out) + (uint64_t)t * e.width + u * V, f);
}

// ---------------------------------------------------------------------------------------
constexpr uint32_t kEmbedChunk = 1024;      // keys a workgroup places
constexpr uint32_t kEmbedDigits = 2048;     // most values of one digit
constexpr uint32_t kEmbedSortChunks = 64;   // up to here a workgroup counts all keys for itself

struct EmbedSortArgs {
  EmbedArgs e;
  const uint32_t* keys;     // null: the first pass, from the ids
  const uint32_t* tokens;
  uint32_t* keys_out;
  uint32_t* tokens_out;
  uint32_t* counts;         // [chunks][digits], where the counting has launches of its own
  uint32_t shift, digits, chunks;
  uint4* clear;             // the share of the gradient that this launch clears, in 16-byte pieces, and the bytes behind the last one
  uint64_t clear_pieces;
  uint32_t clear_rest;
};

__device__ inline uint32_t embed_key(const EmbedSortArgs& a, uint32_t p) { return a.keys ? a.keys[p] : embed_row(a.e, p); }

__device__ inline void embed_clear(const EmbedSortArgs& a, uint32_t block, uint32_t blocks) {
  const uint64_t step = (uint64_t)blocks * 1024u;
  for (uint64_t i = (uint64_t)block * 1024u + threadIdx.x; i < a.clear_pieces; i += step) a.clear[i] = make_uint4(0u, 0u, 0u, 0u);
  if (block == 0 && threadIdx.x < a.clear_rest) reinterpret_cast<unsigned char*>(a.clear + a.clear_pieces)[threadIdx.x] = 0;
}

// Place of a key: keys of smaller digits, keys of its digit in earlier chunks (both in first[digit]), in earlier waves of its
// chunk, in earlier lanes of its wave.  A wave finds the lanes that share a digit with one ballot a bit.
__device__ inline void embed_place(const EmbedSortArgs& a, uint32_t chunk, const uint32_t* first, uint16_t* wave_cnt) {
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t words = 16u * a.digits / 2u;
  for (uint32_t i = tid; i < words; i += 1024u) reinterpret_cast<uint32_t*>(wave_cnt)[i] = 0;
  __syncthreads();
  const uint32_t p = chunk * kEmbedChunk + tid;
  const bool valid = p < a.e.n;
  const uint32_t key = valid ? embed_key(a, p) : 0u, d = (key >> a.shift) & (a.digits - 1u);
  unsigned long long same = __builtin_amdgcn_ballot_w64(valid);
  for (uint32_t bit = 1u; bit < a.digits; bit <<= 1) {
    const bool one = d & bit;
    const unsigned long long ones = __builtin_amdgcn_ballot_w64(one);
    same &= one ? ones : ~ones;
  }
  const uint32_t rank = (uint32_t)__builtin_popcountll(same & ((1ull << lane) - 1ull));
  if (valid && rank == 0) wave_cnt[wave * a.digits + d] = (uint16_t)__builtin_popcountll(same);
  __syncthreads();
  if (!valid) return;
  uint32_t at = first[d] + rank;
#pragma unroll
  for (uint32_t w = 0; w < 16; ++w) {
    const uint32_t c = wave_cnt[w * a.digits + d];
    at += w < wave ? c : 0u;
  }
  a.keys_out[at] = key;
  a.tokens_out[at] = a.keys ? a.tokens[p] : p;
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

// The whole pass in one launch: every chunk's workgroup counts all keys, those of earlier chunks apart.  Workgroups behind the
// chunks clear their share of the gradient meanwhile.
__global__ __launch_bounds__(1024) void embed_sort_kernel(EmbedSortArgs a) {
  extern __shared__ __align__(16) unsigned char lds[];
  if (blockIdx.x >= a.chunks) return embed_clear(a, blockIdx.x - a.chunks, gridDim.x - a.chunks);
  uint32_t* all = reinterpret_cast<uint32_t*>(lds);   // keys of a digit; then the first place of this chunk's
  uint32_t* earlier = all + kEmbedDigits;
  uint32_t* waves = earlier + kEmbedDigits;
  uint16_t* wave_cnt = reinterpret_cast<uint16_t*>(waves + 16);
  const uint32_t tid = threadIdx.x, chunk = blockIdx.x;
  for (uint32_t i = tid; i < kEmbedDigits; i += 1024u) all[i] = earlier[i] = 0;
  __syncthreads();
#pragma unroll 4
  for (uint32_t c = 0; c < a.chunks; ++c) {
    const uint32_t p = c * kEmbedChunk + tid;
    const uint32_t d = (embed_key(a, p < a.e.n ? p : a.e.n - 1u) >> a.shift) & (a.digits - 1u);
    if (p < a.e.n) {
      atomicAdd(&all[d], 1u);
      if (c < chunk) atomicAdd(&earlier[d], 1u);
    }
  }
  __syncthreads();
  uint32_t v[2] = {all[2 * tid], all[2 * tid + 1]};
  embed_prefix(v, waves);
  all[2 * tid] = v[0] + earlier[2 * tid];
  all[2 * tid + 1] = v[1] + earlier[2 * tid + 1];
  __syncthreads();
  embed_place(a, chunk, all, wave_cnt);
}

// The same in three launches for more chunks: counts of every chunk, their prefix over the chunks, the places.
__global__ __launch_bounds__(1024) void embed_count_kernel(EmbedSortArgs a) {
  __shared__ uint32_t cnt[kEmbedDigits];
  if (blockIdx.x >= a.chunks) return embed_clear(a, blockIdx.x - a.chunks, gridDim.x - a.chunks);
  const uint32_t tid = threadIdx.x, chunk = blockIdx.x;
  for (uint32_t i = tid; i < kEmbedDigits; i += 1024u) cnt[i] = 0;
  __syncthreads();
  const uint32_t p = chunk * kEmbedChunk + tid;
  if (p < a.e.n) atomicAdd(&cnt[(embed_key(a, p) >> a.shift) & (a.digits - 1u)], 1u);
  __syncthreads();
  for (uint32_t i = tid; i < a.digits; i += 1024u) a.counts[(uint64_t)chunk * a.digits + i] = cnt[i];
}
__global__ __launch_bounds__(1024) void embed_scan_kernel(EmbedSortArgs a) {
  __shared__ uint32_t waves[16];
  const uint32_t tid = threadIdx.x;
  uint32_t v[2] = {0u, 0u};
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h) {
    const uint32_t d = 2u * tid + h;
    if (d >= a.digits) continue;
    uint32_t run = 0;
#pragma unroll 8
    for (uint32_t c = 0; c < a.chunks; ++c) {
      const uint32_t t = a.counts[(uint64_t)c * a.digits + d];
      a.counts[(uint64_t)c * a.digits + d] = run;
      run += t;
    }
    v[h] = run;
  }
  embed_prefix(v, waves);
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h)
    if (2u * tid + h < a.digits) a.counts[(uint64_t)a.chunks * a.digits + 2u * tid + h] = v[h];
}
__global__ __launch_bounds__(1024) void embed_place_kernel(EmbedSortArgs a) {
  extern __shared__ __align__(16) unsigned char lds[];
  uint32_t* first = reinterpret_cast<uint32_t*>(lds);
  uint16_t* wave_cnt = reinterpret_cast<uint16_t*>(first + kEmbedDigits);
  for (uint32_t i = threadIdx.x; i < a.digits; i += 1024u)
    first[i] = a.counts[(uint64_t)a.chunks * a.digits + i] + a.counts[(uint64_t)blockIdx.x * a.digits + i];
  __syncthreads();
  embed_place(a, blockIdx.x, first, wave_cnt);
}

// ---------------------------------------------------------------------------------------
struct EmbedSumArgs {
  EmbedArgs e;
  const uint32_t* keys;    // [n], sorted
  const uint32_t* tokens;
  float* parts;            // [runs][2][width]: of a row that reaches into the run, of one that begins in it and reaches out
  uint32_t run, runs;      // positions of a run
};

__device__ inline float embed_scale(const EmbedArgs& e, uint32_t row) { return e.scales ? e.scales[row / e.vocab] : e.scale; }

template <typename T, int V>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedSumArgs a) {
  const uint32_t units = a.e.width / V;
  const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  const uint32_t r = (uint32_t)(i / units), u = (uint32_t)(i - (uint64_t)r * units);
  if (r >= a.runs) return;
  const uint32_t none = a.e.n_adapters * a.e.vocab;
  const uint32_t p0 = r * a.run, p1 = p0 + a.run < a.e.n ? p0 + a.run : a.e.n;
  const T* dy = static_cast<const T*>(a.e.dy);
  T* out = static_cast<T*>(a.e.out);
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.0f;
  uint32_t key = a.keys[p0];
  bool from_before = p0 > 0 && a.keys[p0 - 1u] == key;
  // eight positions at a time: their rows are on the way together
  for (uint32_t p = p0; p < p1; p += 8u) {
    uint32_t k[9];
    float f[8][V];
#pragma unroll
    for (uint32_t x = 0; x < 8; ++x) {
      const uint32_t at = p + x < p1 ? p + x : p1 - 1u;
      k[x] = a.keys[at];
      EmbedUnit<T, V>::load(dy + (uint64_t)a.tokens[at] * a.e.width + u * V, f[x]);
    }
    k[8] = p + 8u < a.e.n ? a.keys[p + 8u] : none + 1u;
#pragma unroll
    for (uint32_t x = 0; x < 8; ++x) {
      if (p + x >= p1) break;
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += f[x][j];
      const bool last = p + x + 1u == p1;
      const uint32_t next = last ? (p1 < a.e.n ? a.keys[p1] : none + 1u) : k[x + 1];
      if (next == k[x] && !last) continue;
      if (k[x] < none) {
        if (from_before || next == k[x]) {
          float* part = a.parts + ((uint64_t)r * 2u + (from_before ? 0u : 1u)) * a.e.width + u * V;
#pragma unroll
          for (int j = 0; j < V; ++j) part[j] = sum[j];
        } else {
          const float s = embed_scale(a.e, k[x]);
#pragma unroll
          for (int j = 0; j < V; ++j) sum[j] *= s;
          EmbedUnit<T, V>::store(out + (uint64_t)k[x] * a.e.width + u * V, sum);
        }
      }
      from_before = false;
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    }
  }
}

// Run r's last row, where it begins in r and goes on behind it: its part there and one of every run that it reaches into.
template <typename T, int V>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedSumArgs a) {
  const uint32_t units = a.e.width / V;
  const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  const uint32_t r = (uint32_t)(i / units), u = (uint32_t)(i - (uint64_t)r * units);
  if (r + 1u >= a.runs) return;
  const uint32_t p0 = r * a.run, end = p0 + a.run;  // (a run follows: this one is whole)
  const uint32_t key = a.keys[end];
  if (a.keys[end - 1u] != key || key >= a.e.n_adapters * a.e.vocab) return;
  if (p0 > 0 && a.keys[p0 - 1u] == key) return;  // begins earlier
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = a.parts[((uint64_t)r * 2u + 1u) * a.e.width + u * V + j];
  // last position of the row, by bisection: lo holds the key, hi does not
  uint32_t lo = end, hi = a.e.n;
  while (hi - lo > 1u) {
    const uint32_t mid = lo + (hi - lo) / 2u;
    if (a.keys[mid] == key) lo = mid; else hi = mid;
  }
  const uint32_t last = lo / a.run;
#pragma unroll 8
  for (uint32_t x = r + 1u; x <= last; ++x) {
    const float* part = a.parts + (uint64_t)x * 2u * a.e.width + u * V;
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] += part[j];
  }
  const float s = embed_scale(a.e, key);
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] *= s;
  EmbedUnit<T, V>::store(static_cast<T*>(a.e.out) + (uint64_t)key * a.e.width + u * V, sum);
}

}  // namespace w8a8
