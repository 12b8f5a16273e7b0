// The global norm over many gradient tensors, one for each adapter (the leading axis of every tensor), and the gradients scaled
// down to that adapter's limit:
//
//   norm[a] = sqrt(sum over tensors and their elements of adapter a of g^2)
//   out     = g * (norm[a] > limit[a] ? limit[a] / norm[a] : 1)
//
// Bound by memory: the gradients are read twice (the norm has to be known before the first value can be written) and written once.
// Squares and sums are double: a square of a float32 is exact there and neither over- nor underflows, and the parts are added in
// one order, so the same gradients give the same bits.
//
//   grad_norm_kernel   a workgroup per piece of one tensor's adapter: the sum of its squares
//   grad_scale_kernel  a workgroup per piece: the parts of its adapter added up, then the piece scaled
//
// Up to kGradShortTable tensors come in the kernels' arguments.  More lie in a table in the workspace, written by launches whose arguments they
// are (grad_table_kernel, 120 a launch) once for all calls on it: two launches for any number of tensors.  Norm and scaling of 204 tensors
// of 2.6 MB in all 19.1 us as two launches each with the tensors as arguments, 9.5 so; 64 of 24 KB 8.6 and 7.2 us (4 KiB of arguments take
// their time), where the table has to be written first 7.3 and 8.5.
#pragma once
#include "w8a8_device.h"

namespace w8a8 {

constexpr uint32_t kGradTable = 120, kGradShortTable = 16;

struct GradTensor {
  const void* grad;
  void* out;
  uint64_t count;         // values of one adapter
  uint32_t first_piece;   // among the pieces of one adapter
  uint32_t f32;
};
struct GradCall {
  double* parts;          // [adapters][pieces]
  const float* limits;    // [adapters]
  float* norms;           // [adapters]
  uint32_t tensors, pieces;  // pieces of one adapter
  uint32_t piece;         // values of a piece
};
template <uint32_t TABLE> struct GradArgs : GradCall { GradTensor tensor[TABLE]; };
template <> struct GradArgs<0> : GradCall {
  const GradTensor* tensor;  // [tensors]
  const uint32_t* first;     // [tensors] their first pieces
};

struct GradTableArgs {
  GradTensor tensor[kGradTable];
  GradTensor* table;
  uint32_t* first;
  uint32_t tensors;
};
__global__ __launch_bounds__(128) void grad_table_kernel(GradTableArgs a) {
  if (threadIdx.x >= a.tensors) return;
  a.table[threadIdx.x] = a.tensor[threadIdx.x];
  a.first[threadIdx.x] = a.tensor[threadIdx.x].first_piece;
}

typedef uint32_t v4whole __attribute__((ext_vector_type(4)));
typedef uint32_t v4unaligned __attribute__((ext_vector_type(4), aligned(2)));  // (out may lie at another offset from 16 than grad)
// (pointers out of a table are to any memory for the compiler: its flat accesses look at the LDS too)
template <typename T>
__device__ inline __attribute__((address_space(1))) T* in_memory(T* p) { return (__attribute__((address_space(1))) T*)p; }

struct GradPiece { const GradTensor* t; uint64_t at; uint32_t count; };  // at: first value, in the whole tensor

template <uint32_t TABLE>
__device__ inline GradPiece grad_piece(const GradArgs<TABLE>& a, uint32_t adapter, uint32_t piece) {
  uint32_t lo = 0, hi = a.tensors;  // the last tensor whose first piece is not behind this one
  if constexpr (TABLE == 0) {  // 64 places at a time
    while (hi - lo > 1u) {
      const uint32_t step = (hi - lo + 63u) / 64u, mid = lo + (threadIdx.x & 63u) * step;
      const uint32_t in = (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(mid < hi && a.first[mid < hi ? mid : lo] <= piece));
      lo = __builtin_amdgcn_readfirstlane(lo + (in - 1u) * step);
      hi = lo + step < hi ? lo + step : hi;
    }
  } else {
    while (hi - lo > 1u) {
      const uint32_t mid = (lo + hi) / 2u;
      if (a.tensor[mid].first_piece <= piece) lo = mid; else hi = mid;
    }
  }
  GradPiece p;
  p.t = &a.tensor[lo];
  const uint64_t from = (uint64_t)(piece - p.t->first_piece) * a.piece, left = p.t->count - from;
  p.at = adapter * p.t->count + from;
  p.count = left < a.piece ? (uint32_t)left : a.piece;
  return p;
}

// f(index, 16 bytes' values, how many): the piece in whole 16-byte units behind the values in front of the first one
template <typename T> struct GradUnit;
template <> struct GradUnit<uint16_t> {
  static constexpr uint32_t kN = 8;
  static __device__ inline float one(uint16_t v) { return bf16_bits_to_f32(v); }
  static __device__ inline uint16_t back(float v) { return (uint16_t)f32_to_bf16_bits(v); }
  static __device__ inline void open(const uint4& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ inline uint4 close(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <> struct GradUnit<float> {
  static constexpr uint32_t kN = 4;
  static __device__ inline float one(float v) { return v; }
  static __device__ inline float back(float v) { return v; }
  static __device__ inline void open(const uint4& r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  static __device__ inline uint4 close(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

template <typename T>
__device__ inline double grad_squares(const GradPiece& p) {
  constexpr uint32_t N = GradUnit<T>::kN;
  const auto* g = in_memory(static_cast<const T*>(p.t->grad) + p.at);
  const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(g) & 15u) / sizeof(T);
  const uint32_t head = off ? (N - off < p.count ? N - off : p.count) : 0u, units = (p.count - head) / N;
  double sum = 0.0;
  auto add = [&](float v) { sum = __builtin_fma((double)v, (double)v, sum); };
  if (threadIdx.x < head) add(GradUnit<T>::one(g[threadIdx.x]));
  const auto* u = reinterpret_cast<const __attribute__((address_space(1))) v4whole*>(g + head);
  for (uint32_t i = threadIdx.x; i < units; i += 1024u) {
    v4whole r[4];
#pragma unroll
    for (uint32_t x = 0; x < 4; ++x) r[x] = i + x * 256u < units ? u[i + x * 256u] : v4whole{0u, 0u, 0u, 0u};
#pragma unroll
    for (uint32_t x = 0; x < 4; ++x) {
      float f[N];
      GradUnit<T>::open(make_uint4(r[x][0], r[x][1], r[x][2], r[x][3]), f);
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) add(f[j]);
    }
  }
  const uint32_t done = head + units * N;
  if (threadIdx.x < p.count - done) add(GradUnit<T>::one(g[done + threadIdx.x]));
  return sum;
}

__device__ inline double grad_block_sum(double v) {
  __shared__ double waves[4];
  v = wave_sum(v);
  if ((threadIdx.x & 63u) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  const double s = (waves[0] + waves[1]) + (waves[2] + waves[3]);
  __syncthreads();
  return s;
}

template <uint32_t TABLE>
__global__ __launch_bounds__(256) void grad_norm_kernel(GradArgs<TABLE> a) {
  const uint32_t adapter = blockIdx.y, piece = blockIdx.x;
  const GradPiece p = grad_piece(a, adapter, piece);
  const double s = grad_block_sum(p.t->f32 ? grad_squares<float>(p) : grad_squares<uint16_t>(p));
  if (threadIdx.x == 0) a.parts[(uint64_t)adapter * a.pieces + piece] = s;
}

template <typename T>
__device__ inline void grad_scale(const GradPiece& p, float factor) {
  constexpr uint32_t N = GradUnit<T>::kN;
  if (factor == 1.0f && p.t->grad == p.t->out) return;
  const auto* g = in_memory(static_cast<const T*>(p.t->grad) + p.at);
  auto* o = in_memory(static_cast<T*>(p.t->out) + p.at);
  const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(g) & 15u) / sizeof(T);
  const uint32_t head = off ? (N - off < p.count ? N - off : p.count) : 0u, units = (p.count - head) / N;
  if (threadIdx.x < head) o[threadIdx.x] = GradUnit<T>::back(GradUnit<T>::one(g[threadIdx.x]) * factor);
  const auto* u = reinterpret_cast<const __attribute__((address_space(1))) v4whole*>(g + head);
  auto* w = reinterpret_cast<__attribute__((address_space(1))) v4unaligned*>(o + head);
  for (uint32_t i = threadIdx.x; i < units; i += 1024u) {
    v4whole r[4];
#pragma unroll
    for (uint32_t x = 0; x < 4; ++x) r[x] = i + x * 256u < units ? u[i + x * 256u] : v4whole{0u, 0u, 0u, 0u};
#pragma unroll
    for (uint32_t x = 0; x < 4; ++x) {
      float f[N];
      GradUnit<T>::open(make_uint4(r[x][0], r[x][1], r[x][2], r[x][3]), f);
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) f[j] *= factor;
      const uint4 v = GradUnit<T>::close(f);
      // past the caches, which the next norm's reads would have to wait for: 32 tensors of 838 MB in all 234 us, 211 so
      if (i + x * 256u < units) __builtin_nontemporal_store(v4unaligned{v.x, v.y, v.z, v.w}, w + i + x * 256u);
    }
  }
  const uint32_t done = head + units * N;
  if (threadIdx.x < p.count - done) o[done + threadIdx.x] = GradUnit<T>::back(GradUnit<T>::one(g[done + threadIdx.x]) * factor);
}

template <uint32_t TABLE>
__global__ __launch_bounds__(256) void grad_scale_kernel(GradArgs<TABLE> a) {
  // from the last piece to the first: what the norm read last is in the caches yet
  const uint32_t adapter = gridDim.y - 1u - blockIdx.y, piece = gridDim.x - 1u - blockIdx.x;
  double s = 0.0;
  for (uint32_t i = threadIdx.x; i < a.pieces; i += 256u) s += a.parts[(uint64_t)adapter * a.pieces + i];
  const double norm = sqrt(grad_block_sum(s));
  if (piece == 0 && threadIdx.x == 0) a.norms[adapter] = (float)norm;
  if (!a.limits) return;
  const float given = a.limits[adapter];
  const double limit = given < 0.0f ? 0.0 : (double)given;
  const float factor = norm > limit ? (float)(limit / norm) : 1.0f;  // (where either is no number the gradients stay as they are)
  const GradPiece p = grad_piece(a, adapter, piece);
  if (p.t->f32) grad_scale<float>(p, factor); else grad_scale<uint16_t>(p, factor);
}

__global__ __launch_bounds__(256) void grad_zero_norms_kernel(float* norms, uint32_t n) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i < n) norms[i] = 0.0f;
}

}  // namespace w8a8
