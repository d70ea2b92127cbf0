// What the kernels of attention over states of another length share: the shapes, a tile of rows in LDS and its
// fragments, and the keys that a mask leaves.
//
// The queries of the heads that share a key head are the rows of one product: row r of the U G rows of (batch, key
// head) is query r / G of head hk G + r % G, so that K and V are read once for all of them.
#pragma once

#include "gnn_common.hpp"
#include "gnn_internal.hpp"

namespace gnn {
namespace cross {

constexpr float LOG2E = 1.4426950408889634f;

// Up to so many keys 16-bit operands made here, p and dQ's dS, are multiplied in two parts, 2^-17 exact: few terms cancel, and
// their roundings do not: of 3 keys, where P (dP - Delta) is a small difference, gradients were off by 2.5 times the one
// rounding at the end, of 64 and more by 1.4. One tile of keys costs nothing that shows.
constexpr int FINE = 64;

struct Shape {
  int B, U, V, H, Hk, G, D;
  int rows;  // U G
};

// 8 elements at any element's address
template <typename T>
__device__ __forceinline__ typename TypeOps<T>::V8 load8_at(const T* p) {
  typedef typename TypeOps<T>::V8 V8;
  typedef V8 VU __attribute__((aligned(sizeof(T))));
  return *(const __attribute__((address_space(1))) VU*)p;
}
// 16 bytes at any element's address
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ u32x4 load16_at(const T* p) {
  typedef u32x4 VU __attribute__((aligned(2)));
  return *(const __attribute__((address_space(1))) VU*)p;
}
// 4 elements at any element's address, the first `left` of them
template <typename T>
__device__ __forceinline__ f32x4 load4_at(const T* p, int left) {
  typedef typename TypeOps<T>::V4 V4;
  typedef V4 VU __attribute__((aligned(sizeof(T))));
  if (left >= 4) {
    const V4 v = *(const __attribute__((address_space(1))) VU*)p;
    return TypeOps<T>::to_f32(v);
  }
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = e < left ? TypeOps<T>::to_f32(p[e]) : 0.f;
  return v;
}
template <typename T>
__device__ __forceinline__ void store4_at(T* p, const f32x4& v, int left) {
  typedef typename TypeOps<T>::V4 V4;
  typedef V4 VU __attribute__((aligned(sizeof(T))));
  const V4 o = TypeOps<T>::from_f32(v);
  if (left >= 4) {
    *(__attribute__((address_space(1))) VU*)p = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) p[e] = o[e];
}

// A row's biases of the keys that a lane holds of a half tile, 8 q + 4 g + (0 .. 3) from `key0` on, on their way while
// the products run: where the half tile is known to be WHOLE, no load is in a branch. Keys past V: zeros.
template <typename T>
struct HalfBias {
  typedef typename TypeOps<T>::V4 V4;
  V4 f[4];
  template <bool WHOLE>
  __device__ __forceinline__ void load(const T* row, int key0, int V, int g) {
    typedef V4 VU __attribute__((aligned(sizeof(T))));
    if (WHOLE || key0 + 32 <= V) {  // uniform
#pragma unroll
      for (int q = 0; q < 4; ++q) f[q] = *(const __attribute__((address_space(1))) VU*)(row + key0 + 8 * q + 4 * g);
      return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int key = key0 + 8 * q + 4 * g;
      f[q] = TypeOps<T>::from_f32(key < V ? load4_at(row + key, V - key) : f32x4{0.f, 0.f, 0.f, 0.f});
    }
  }
  __device__ __forceinline__ f32x4 at(int q) const { return TypeOps<T>::to_f32(f[q]); }
};

// Rows of DP elements in LDS, laid out so that the reads hit no bank twice: fragments of 32 rows (8 consecutive elements
// a lane), turned ones (8 rows of one column a lane), or both. LDS serves 16 lanes' 16 bytes, and 32 lanes' 8, at once.
//   BY_ROWS     a pitch of an odd number of 16-byte chunks: 16 rows' chunk c lie on different banks;
//   BY_COLUMNS  a pitch of 64 (or 192) bytes modulo 256: 4 rows' 64 bytes do; fp32: 4 rows further on is 128 bytes on;
//   BOTH        a pitch of a power of two with the chunks in chunk_swizzle's order, which costs exclusive-ors for addresses
//               that are one register and constants in the other two.
enum Layout { BOTH, BY_ROWS, BY_COLUMNS };

template <typename T, int DP, Layout LAYOUT = BOTH>
struct RowTile {
  static constexpr int BYTES = DP * (int)sizeof(T);
  static constexpr int PITCH = LAYOUT == BY_ROWS                       ? BYTES + 16
                               : LAYOUT == BY_COLUMNS && sizeof(T) == 4 ? BYTES + 32
                               : LAYOUT == BY_COLUMNS                   ? (BYTES % 128 == 64 ? BYTES : BYTES + 64)
                               : BYTES <= 64                            ? 64
                               : BYTES <= 128                           ? 128
                               : BYTES <= 256                           ? 256
                                                                        : 512;
  static constexpr int CPR = BYTES / 16;            // chunks a row
  static constexpr int EPC = 16 / (int)sizeof(T);   // elements a chunk
  typedef typename TypeOps<T>::V8 V8;
  typedef typename TypeOps<T>::V4 V4;
  static __device__ __forceinline__ int at(int row, int chunk) {
    if constexpr (LAYOUT == BOTH) return row * PITCH + ((chunk ^ chunk_swizzle<(PITCH < 256 ? PITCH : 256)>(row)) << 4);
    return row * PITCH + (chunk << 4);
  }
  // elements 16 kk + 8 g .. + 7 of a row
  static __device__ __forceinline__ V8 row8(const unsigned char* tile, int row, int kk, int g) {
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const V8*>(tile + at(row, 2 * kk + g));
    } else {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(tile + at(row, 4 * kk + 2 * g));
      const f32x4 hi = *reinterpret_cast<const f32x4*>(tile + at(row, 4 * kk + 2 * g + 1));
      return V8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  }
  // column 32 cc + lane % 32 of the rows row0 + 16 kk + 8 (e / 4) + 4 g + e % 4: the order in which a 32x32
  // accumulator holds its rows. 16-bit: ds_read_b64_tr_b16 hands the 16 lanes of a group a block of 4 rows x 16
  // columns turned.
  static __device__ __forceinline__ V8 turned8(const unsigned char* tile, int row0, int kk, int cc, int lane) {
    const int g = lane >> 5;
    V8 f;
    if constexpr (sizeof(T) == 2) {
      typedef short v4i16 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) v4i16 lds_v4i16;
      const int r16 = lane & 15, col = 32 * cc + 16 * ((lane >> 4) & 1) + 4 * (r16 & 3);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned char* p = tile + at(row0 + 16 * kk + 8 * h + 4 * g + (r16 >> 2), col >> 3) + 2 * (col & 7);
        const V4 x = __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                (lds_v4i16*)(__attribute__((address_space(3))) const unsigned char*)p));
#pragma unroll
        for (int e = 0; e < 4; ++e) f[4 * h + e] = x[e];
      }
    } else {
      const int col = 32 * cc + (lane & 31);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        f[e] = *reinterpret_cast<const float*>(tile + at(row0 + 16 * kk + 8 * (e >> 2) + 4 * g + (e & 3), col >> 2) +
                                               4 * (col & 3));
    }
    return f;
  }
};

// ROWS rows of a tensor on their way to LDS through registers: chunk i of a thread is row(i), elements col(i) .. A
// thread's first row and column are the same for every tile, its other rows whole steps further on: where all ROWS rows
// exist the addresses are a uniform base each and one 32-bit offset (the host keeps 64 rows below 2^31 bytes).
template <typename T, int DP, int ROWS, int NT>
struct Staged {
  typedef RowTile<T, DP> Tile;
  static constexpr int N = ROWS * Tile::CPR / NT;
  static constexpr bool EVEN = NT % Tile::CPR == 0;  // every chunk of a thread is in the same column
  static constexpr int STEP = NT / Tile::CPR;        // rows from one chunk to the next, where EVEN
  static_assert(N * NT == ROWS * Tile::CPR, "chunks a thread");
  u32x4 reg[N];
  static __device__ __forceinline__ int row(int i, int tid) { return EVEN ? tid / Tile::CPR + i * STEP : (tid + i * NT) / Tile::CPR; }
  static __device__ __forceinline__ int chunk(int i, int tid) { return EVEN ? tid % Tile::CPR : (tid + i * NT) % Tile::CPR; }
  // the thread's index where it is rarely needed: opaque, so that what follows from it is not kept in registers
  static __device__ __forceinline__ int rare_tid() {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    return tid;
  }
  // rows first .. first + ROWS - 1 of `end` rows, those past the last one its copies; columns past D read column 0
  __device__ __forceinline__ void load_rows(const T* base, int64_t stride, int first, int end, int D) {
    if (EVEN && first + ROWS <= end) {  // uniform
      const int c = chunk(0, threadIdx.x) * Tile::EPC;
      const uint32_t lane = (uint32_t)((int)threadIdx.x / Tile::CPR * (int)stride + (c < D ? c : 0)) * (uint32_t)sizeof(T);
      const T* tile = base + first * stride;
#pragma unroll
      for (int i = 0; i < N; ++i) reg[i] = load16_at((const T*)((const char*)(tile + i * STEP * stride) + lane));
      return;
    }
    load(base, D, [&](int r) { return (int64_t)min(first + r, end - 1) * stride; });
  }
  // rows first .. of the `end` rows of G heads that share a key head: row r is token r / G, head r % G, `token` and `head`
  // elements apart; those past the last one its copies
  __device__ __forceinline__ void load_heads(const T* base, int64_t token, int64_t head, int G, int first, int end, int D) {
    if (EVEN && first + ROWS <= end && STEP % G == 0) {  // uniform; first is a multiple of ROWS, and so of STEP
      const int c = chunk(0, threadIdx.x) * Tile::EPC, r = row(0, threadIdx.x);
      const uint32_t lane = (uint32_t)(r / G * (int)token + r % G * (int)head + (c < D ? c : 0)) * (uint32_t)sizeof(T);
      const T* tile = base + first / G * token;
#pragma unroll
      for (int i = 0; i < N; ++i) reg[i] = load16_at((const T*)((const char*)(tile + i * (STEP / G) * token) + lane));
      return;
    }
    load(base, D, [&](int r) {
      const int at = min(first + r, end - 1);
      return at / G * token + at % G * head;
    });
  }
  // row r from base + offset(r): always a readable row
  template <typename Offset>
  __device__ __forceinline__ void load(const T* base, int D, Offset offset) {
    const int tid = rare_tid();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = chunk(i, tid) * Tile::EPC;
      reg[i] = load16_at(base + offset(row(i, tid)) + (c < D ? c : 0));
    }
  }
  // whole rows of D = DP elements, into a tile of any layout
  template <typename To = Tile>
  __device__ __forceinline__ void store(unsigned char* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      *reinterpret_cast<u32x4*>(tile + To::at(row(i, threadIdx.x), chunk(i, threadIdx.x))) = reg[i];
  }
  // rows for which `keep` is false, and columns past D, are zeros
  template <typename To = Tile, typename Keep>
  __device__ __forceinline__ void store(unsigned char* tile, int D, Keep keep) const {
    const int tid = rare_tid();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t ok = chunk(i, tid) * Tile::EPC < D && keep(row(i, tid)) ? ~0u : 0u;
      *reinterpret_cast<u32x4*>(tile + To::at(row(i, tid), chunk(i, tid))) = reg[i] & u32x4{ok, ok, ok, ok};
    }
  }
};

// Bit j of the result: key `key0 + j` is below V and kept. The same for the whole wave.
__device__ __forceinline__ uint64_t live_keys(const uint8_t* mask, int64_t stride, int key0, int V) {
  const int left = V - key0;
  uint64_t live = left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
  if (mask && live) live &= __ballot(mask[(int64_t)min(key0 + (int)(threadIdx.x & 63), V - 1) * stride] != 0);
  return live;
}

// The first and one past the last kept key of [k0, k1), found by all threads of a workgroup; first >= end where there
// is none. `found`: two ints of LDS. Padded sequences end early, and a tile of theirs that is not visited costs nothing.
template <int NT>
__device__ __forceinline__ void live_range(const uint8_t* mask, int64_t stride, int& k0, int& k1, int* found) {
  if (threadIdx.x == 0) found[0] = k1, found[1] = k0;
  __syncthreads();
  constexpr int AT_ONCE = 8;
  int first = k1, last = k0;
  for (int base = k0 + (int)threadIdx.x; base < k1; base += NT * AT_ONCE) {
    uint8_t m[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) m[i] = mask[(int64_t)min(base + i * NT, k1 - 1) * stride];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
      if (m[i] && base + i * NT < k1) first = min(first, base + i * NT), last = max(last, base + i * NT + 1);
  }
  if (first < last) atomicMin(&found[0], first), atomicMax(&found[1], last);
  __syncthreads();
  k0 = found[0], k1 = found[1];
}

// Fragment kk of an accumulator: its 8 elements 8 kk .. as T
template <typename T>
__device__ __forceinline__ typename TypeOps<T>::V8 acc_frag(const f32x16& a, int kk) {
  const f32x8 x = {a[8 * kk + 0], a[8 * kk + 1], a[8 * kk + 2], a[8 * kk + 3],
                   a[8 * kk + 4], a[8 * kk + 5], a[8 * kk + 6], a[8 * kk + 7]};
  return TypeOps<T>::from_f32(x);
}
// what its rounding to f left
template <typename T>
__device__ __forceinline__ typename TypeOps<T>::V8 low_frag(const f32x16& a, int kk, const typename TypeOps<T>::V8& f) {
  const f32x8 x = {a[8 * kk + 0], a[8 * kk + 1], a[8 * kk + 2], a[8 * kk + 3],
                   a[8 * kk + 4], a[8 * kk + 5], a[8 * kk + 6], a[8 * kk + 7]};
  return TypeOps<T>::from_f32(x - TypeOps<T>::to_f32(f));
}
__device__ __forceinline__ void fill(f32x16& a, float x) {
#pragma unroll
  for (int i = 0; i < 16; ++i) a[i] = x;
}
__device__ __forceinline__ void clear(f32x16& a) { fill(a, 0.f); }
// maximum and sum over the lane pair (l, l ^ 32) without a trip through LDS
__device__ __forceinline__ float pair_top(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// row of element i of an accumulator in lane group g
__device__ __forceinline__ int acc_row(int i, int g) { return 8 * (i / 4) + 4 * g + i % 4; }

}  // namespace cross
}  // namespace gnn
