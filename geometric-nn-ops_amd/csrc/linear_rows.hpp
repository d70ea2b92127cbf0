// What the kernels that keep a weight in LDS and walk over many rows share: the rows' way between memory and the products'
// order, and the sums' start.
#pragma once

#include <type_traits>

#include "linear_common.hpp"

namespace gnn {
namespace lin {

constexpr int RS_LDS = 144 << 10;         // the weight and the bias, beside 2 KB a wave
constexpr int64_t RS_MIN_ROWS = 1 << 15;  // below, filling LDS costs more than it saves

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// `at`: a byte offset that is the same for the whole wave
__device__ __forceinline__ u32x4_t buffer_load16(__amdgpu_buffer_rsrc_t r, uint32_t off, int at = 0) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, off, at, 0);
}
// Stores take their whole offset from a vector register: behind a 16-byte store whose scalar offset is a
// register the compiler takes no wait state before it reuses the data's registers, and the last lanes of
// every 16 then stored the next store's address instead of their first dword.

// Global accesses whose neighbouring lanes lie in different rows move 16 bytes a request and hold the memory
// pipeline up (128 -> 512 over 512^2 rows: 100 us with the stores alone that way, 39 us is what the bytes
// take). So a wave moves 32 x 64-byte tiles with 4 lanes a row ("memory order": access i of two, lane -> row
// 16 i + lane / 4, chunk lane % 4) and turns them into or from the products' order (lane -> row lane % 32,
// chunks 2 t + lane / 32) through 2 KB of LDS of its own, its chunks swizzled too. A wave's LDS
// accesses stay in order: no wait is needed beyond the data's own.
constexpr int TURN = 2048;
struct Turn {
  unsigned char* to_rows[2];  // products' order, t = 0, 1
  unsigned char* to_mem[2];   // memory order, i = 0, 1
  __device__ __forceinline__ Turn(unsigned char* tile, int lane) {
    const int r = lane & 31, g = lane >> 5;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      to_rows[k] = tile + r * 64 + (((2 * k + g) ^ chunk_swizzle<64>(r)) << 4);
      const int m = 16 * k + (lane >> 2);
      to_mem[k] = tile + m * 64 + (((lane & 3) ^ chunk_swizzle<64>(m)) << 4);
    }
  }
  __device__ __forceinline__ static void put(unsigned char* const (&at)[2], const u32x4_t (&v)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) *reinterpret_cast<u32x4_t*>(at[k]) = v[k];
  }
  __device__ __forceinline__ static void get(unsigned char* const (&at)[2], u32x4_t (&v)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) v[k] = *reinterpret_cast<const u32x4_t*>(at[k]);
  }
};

// Descriptor of rows m0 .. m0 + 31 of a tensor of `cols` columns (none of them where m0 is past the end)
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, int64_t m0, int64_t M, int64_t ld, int cols) {
  const int64_t n = min((int64_t)32, M - m0);
  const int range = n > 0 ? (int)(((n - 1) * ld + cols) * sizeof(T)) : 0;
  return buffer_rsrc((const T*)base + (n > 0 ? m0 * ld : 0), range);
}

template <typename T>
__device__ __forceinline__ f32x8 to8(u32x4_t v) {
  return TypeOps<T>::to_f32(__builtin_bit_cast(typename TypeOps<T>::V8, v));
}

// The 32 x 32 sums start from the bias
__device__ __forceinline__ f32x16 bias_tile(const float* bias, int g) {
  f32x16 acc;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f32x4 b = *reinterpret_cast<const f32x4*>(bias + 16 * (q / 2) + 8 * g + 4 * (q % 2));
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[4 * q + i] = b[i];
  }
  return acc;
}

// f(an activation as a constant)
template <typename F>
inline __host__ __device__ void with_activation(int act, F f) {
  switch (act) {
    case GNN_ACT_RELU: f(std::integral_constant<int, GNN_ACT_RELU>()); break;
    case GNN_ACT_GELU: f(std::integral_constant<int, GNN_ACT_GELU>()); break;
    case GNN_ACT_SILU: f(std::integral_constant<int, GNN_ACT_SILU>()); break;
    case GNN_ACT_SIGMOID: f(std::integral_constant<int, GNN_ACT_SIGMOID>()); break;
    default: f(std::integral_constant<int, GNN_ACT_NONE>()); break;
  }
}

// Byte offsets of a lane's two accesses of a tile in memory order; `left` columns from the lane's chunk on:
// tiles at column c are there where c < left
struct MemOrder {
  uint32_t off[2];
  int left;
  __device__ __forceinline__ MemOrder(int64_t ld, int cols, int lane) : left(cols - 8 * (lane & 3)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) off[i] = (uint32_t)((16 * i + (lane >> 2)) * ld + 8 * (lane & 3)) * 2;
  }
  __device__ __forceinline__ void load(u32x4_t (&v)[2], __amdgpu_buffer_rsrc_t r, int col) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) v[i] = buffer_load16(r, col < left ? off[i] : BUFFER_OOB, 2 * col);
  }
  __device__ __forceinline__ void store(const u32x4_t (&v)[2], __amdgpu_buffer_rsrc_t r, int col) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) buffer_store(v[i], r, col < left ? off[i] + 2 * col : BUFFER_OOB);
  }
};

}  // namespace lin
}  // namespace gnn
