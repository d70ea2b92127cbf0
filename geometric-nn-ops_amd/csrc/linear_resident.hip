// The linear layer of fused_linear.hip for many rows and a weight that fits LDS (16-bit types): the layers of
// a pair transition and the projections around it, which HBM bounds (128 -> 512 over 512^2 pixels: 336 MB
// against 34 GFLOP).
//
// A workgroup of 8 waves loads the weight into LDS once, rows padded to whole 32x32 tiles with zeros and
// their 16-byte chunks in chunk_swizzle's order, and stays. From there
// on every wave works alone, without a barrier: it takes 32 rows at a time (the next ones on their way while it
// works on these) and multiplies. The products
// are transposed, as in linear_kernel: a lane ends up with 8 consecutive outputs of one row. Rows and columns
// past the end are dropped by the range of the buffer descriptors, so that no load or store sits in a branch
// and the counters' waits stay exact.
// 512^2 x 128 -> 512, bf16, relu: 74 us (4.5 TB/s; the tiles of linear_kernel 192); 384^2 rows: without an
// activation 40, silu 54, gelu 77; 384^2 x 512 -> 128 with a residual 62 (3.7 TB/s).
//
// Two forms, by what a wave's registers hold: `rows` (I <= 256) the rows' fragments, going over the outputs
// 32 at a time; `outputs` (O <= 128) the sums of all outputs, going over the contraction 128 at a time.
#include <algorithm>
#include <type_traits>

#include "linear_common.hpp"

namespace gnn {

namespace {

using namespace lin;

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

// W [O][I] (or, transposed, W[n][k] at k ld + n) into rows of rowb bytes, in tiles of 32 in tile_output's order,
// zeros past I and O; then the bias. As it is stored, the weight comes by global_load_lds, all of it in flight
// at once (through registers, four loads at a time, this took 10 us more of a 128 KB weight).
// SW: the rows' bytes, or 256 for any multiple
template <typename T, int NT, int SW>
__device__ __forceinline__ void fill_weight(unsigned char* smem, const LinArgs& a, bool transposed, int rows, int rowb) {
  typedef typename TypeOps<T>::V8 V8;
  const int cpr = rowb / 16;
  const T* w = (const T*)a.w;
  if (!transposed) {
    const int lane = threadIdx.x & 63;
    for (int e0 = (threadIdx.x >> 6) * 64; e0 < rows * cpr; e0 += NT) {  // 1 KB an instruction
      const uint32_t e = e0 + lane, r = e / (uint32_t)cpr, c = (e - r * cpr) ^ chunk_swizzle<SW>(r);
      const int n = (r & ~31) + tile_output(r & 31);
      const void* src = n < a.O && 8 * (int)c < a.I ? (const void*)(w + (int64_t)n * a.w_ld + 8 * c) : (const void*)zero_chunk;
      __builtin_amdgcn_global_load_lds(src, (lds_void_t*)(smem + 16 * e0), 16, 0, 0);
    }
  } else {
    const uint32_t K = 8 * cpr;
#pragma unroll 4
    for (uint32_t e = threadIdx.x; e < (uint32_t)rows / 8 * K; e += NT) {
      const int k = e % K, n = e / K * 8;
      V8 v = zero8<T>();
      if (k < a.I && n < a.O) v = load8(w + (int64_t)k * a.w_ld + n);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = ((n + i) & ~31) + tile_row((n + i) & 31);
        *reinterpret_cast<T*>(smem + r * rowb + (((k >> 3) ^ chunk_swizzle<SW>(r)) << 4) + 2 * (k & 7)) = v[i];
      }
    }
  }
  float* bias = (float*)(smem + rows * rowb);
  for (int n = threadIdx.x; n < rows; n += NT) bias[n] = a.bias && n < a.O ? (float)((const T*)a.bias)[n] : 0.f;
  __builtin_amdgcn_s_waitcnt(0x070);  // the DMA and the bias have landed: vmcnt(0) lgkmcnt(0)
}

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

// What becomes of z: act(z), act(z) + side, or side * act'(z)
enum Epilogue { EPI_ACT, EPI_ADD, EPI_DZ };

// 8 consecutive outputs as their 16 bytes
template <typename T, int EPI, int ACT>
__device__ __forceinline__ u32x4_t finish16(f32x8 z, u32x4_t side) {
  if constexpr (EPI == EPI_DZ)
    slope_all<false, ACT>(z);
  else
    activate_all<false, ACT>(z);
  if constexpr (EPI == EPI_ADD) z += to8<T>(side);
  if constexpr (EPI == EPI_DZ) z *= to8<T>(side);
  return __builtin_bit_cast(u32x4_t, TypeOps<T>::from_f32(z));
}
// f(an activation as a constant)
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
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

// KS: 16-element steps of the contraction held in registers
template <typename T, int KS, int EPI, int ACT, int NT>
__global__ __launch_bounds__(NT, NT / 256) void linear_rows_kernel(const LinArgs a, int transposed) {
  typedef typename TypeOps<T>::V8 V8;
  constexpr bool SIDE = EPI != EPI_ACT;
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int ROWB = 32 * KS;
  const int nb = (a.O + 31) / 32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
  unsigned char* const weight = smem + NT / 64 * TURN;
  fill_weight<T, NT, ROWB>(weight, a, transposed, 64 * ((nb + 1) / 2), ROWB);
  const float* bias = (const float*)(weight + 64 * ((nb + 1) / 2) * ROWB);
  __syncthreads();
  const Turn turn(smem + wave * TURN, lane);
  const MemOrder xm(a.x_ld, a.I, lane), sm(a.side_ld, a.O, lane), om(a.out_ld, a.O, lane);
  const int64_t groups = (a.M + 31) / 32, step = (int64_t)gridDim.x * (NT / 64);
  auto load_rows = [&](u32x4_t (&x)[KS / 2][2], int64_t grp) {
    const auto r = rows_rsrc<T>(a.x, grp * 32, a.M, a.x_ld, a.I);
#pragma unroll
    for (int p = 0; p < KS / 2; ++p) xm.load(x[p], r, 32 * p);
  };
  const unsigned char* wrow[KS];
#pragma unroll
  for (int kk = 0; kk < KS; ++kk) wrow[kk] = weight + l32 * ROWB + (((2 * kk + g) ^ chunk_swizzle<ROWB>(l32)) << 4);
  // The products of a tile run beside the epilogue of the one before it (of the last rows' last tile, where a
  // wave goes on to new rows): tile() starts a tile's sums, finish() ends the ones before.
  u32x4_t next[KS / 2][2], x[KS / 2][2];
  auto turn_rows = [&]() {
#pragma unroll
    for (int p = 0; p < KS / 2; ++p) {
      Turn::put(turn.to_mem, next[p]);
      Turn::get(turn.to_rows, x[p]);
    }
  };
  auto tile = [&](int y) {
    f32x16 acc = bias_tile(bias + 32 * y, g);
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
      Mma<T, PREC_NATIVE>::step(acc, *reinterpret_cast<const V8*>(wrow[kk] + y * 32 * ROWB),
                                __builtin_bit_cast(V8, x[kk / 2][kk % 2]));
    return acc;
  };
  auto finish = [&](const f32x16& acc, const u32x4_t (&side)[2], u32x4_t (&o)[2]) {
    u32x4_t s[2];
    if (SIDE) {
      Turn::put(turn.to_mem, side);
      Turn::get(turn.to_rows, s);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) o[t] = finish16<T, EPI, ACT>(outputs8(acc, t), s[t]);
    Turn::put(turn.to_rows, o);
    Turn::get(turn.to_mem, o);
  };
  int64_t grp = (int64_t)blockIdx.x * (NT / 64) + wave;
  // rows of 16 steps take 64 registers: theirs are not loaded ahead
  constexpr bool AHEAD = KS <= 8;
  load_rows(next, grp);
  turn_rows();
  if (AHEAD) load_rows(next, grp + step);
  f32x16 acc = tile(0);
  for (; grp < groups; grp += step) {
    const auto srs = rows_rsrc<T>(a.side, grp * 32, a.M, a.side_ld, a.O);
    const auto ors = rows_rsrc<T>(a.out, grp * 32, a.M, a.out_ld, a.O);
    u32x4_t side[2][2][2];  // of this pair of tiles and the next
    auto load_side = [&](u32x4_t (&s)[2][2], int y) {
      sm.load(s[0], srs, 32 * y);
      sm.load(s[1], srs, 32 * (y + 1));
    };
    // tiles by twos, whose 128-byte lines are stored at once
    auto pair = [&](int y, u32x4_t (&s)[2][2]) {
      u32x4_t o[2][2];
      f32x16 ahead = tile(y + 1);  // zeros past the last: the weight's rows are padded to pairs
      finish(acc, s[0], o[0]);
      acc = ahead;
      if (y + 2 < nb) {
        ahead = tile(y + 2);
      } else {
        if (!AHEAD) load_rows(next, grp + step);
        turn_rows();
        if (AHEAD) load_rows(next, grp + 2 * step);
        ahead = tile(0);
      }
      finish(acc, s[1], o[1]);
      acc = ahead;
      om.store(o[0], ors, 32 * y);
      om.store(o[1], ors, 32 * (y + 1));
      if (SIDE) load_side(s, y + 4);
    };
    if (SIDE) {
      load_side(side[0], 0);
      load_side(side[1], 2);
    }
    for (int y = 0; y < nb; y += 4) {
      pair(y, side[0]);
      if (y + 2 < nb) pair(y + 2, side[1]);
    }
  }
}

// The activation's gradient and the input's in one pass: dz = dy act'(z) is written for the weight's gradient,
// and goes on from the registers into dx = dz W. A tile of dz, 8 consecutive outputs a lane, is an operand
// fragment of that product as it stands; W's columns for it come from the same LDS image by ds_read_b64_tr_b16
// (4 rows of 16 columns each), the columns in tile_output's order again. Beside dz kept and read back, this
// saves the read of dz and a launch.
template <typename T, int KS, int ACT, int NT>
__global__ __launch_bounds__(NT, NT / 256) void linear_rows_bwd_kernel(const LinArgs a, int) {
  typedef typename TypeOps<T>::V8 V8;
  typedef typename TypeOps<T>::V4 V4;
  typedef short v4i16 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4i16 lds_v4i16;
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int ROWB = 32 * KS, KB = KS / 2;
  const int nb = (a.O + 31) / 32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
  unsigned char* const weight = smem + NT / 64 * TURN;
  fill_weight<T, NT, ROWB>(weight, a, false, 64 * ((nb + 1) / 2), ROWB);
  const float* bias = (const float*)(weight + 64 * ((nb + 1) / 2) * ROWB);
  __syncthreads();
  const Turn turn(smem + wave * TURN, lane);
  const MemOrder xm(a.x_ld, a.I, lane), sm(a.side_ld, a.O, lane), om(a.out_ld, a.O, lane), dm(a.dx_ld, a.I, lane);
  const int64_t groups = (a.M + 31) / 32, step = (int64_t)gridDim.x * (NT / 64);
  const unsigned char* wrow[KS];
#pragma unroll
  for (int kk = 0; kk < KS; ++kk) wrow[kk] = weight + l32 * ROWB + (((2 * kk + g) ^ chunk_swizzle<ROWB>(l32)) << 4);
  // transposed reads: row 4 g + q (and 8 further), 4 columns of the 32 of block kb
  const unsigned char* wcol[2][KB];
  {
    const int row = 4 * g + ((lane & 15) >> 2), m = lane & 3;
    const int col = 16 * ((lane >> 4) & 1) + 4 * (2 * (m & 1) + (m >> 1));
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        wcol[b][kb] = weight + (row + 8 * b) * ROWB + (((4 * kb + (col >> 3)) ^ chunk_swizzle<ROWB>(row + 8 * b)) << 4) +
                      2 * (col & 7);
  }
  auto column8 = [&](int kb, int row) {
    V4 v[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
      v[b] = __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                        (lds_v4i16*)(__attribute__((address_space(3))) const unsigned char*)(
                                            wcol[b][kb] + row * ROWB)));
    return __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto load_rows = [&](u32x4_t (&x)[KS / 2][2], int64_t grp) {
    const auto r = rows_rsrc<T>(a.x, grp * 32, a.M, a.x_ld, a.I);
#pragma unroll
    for (int p = 0; p < KS / 2; ++p) xm.load(x[p], r, 32 * p);
  };
  u32x4_t x[KS / 2][2];
  auto turn_rows = [&]() {
#pragma unroll
    for (int p = 0; p < KS / 2; ++p) {
      Turn::put(turn.to_mem, x[p]);
      Turn::get(turn.to_rows, x[p]);
    }
  };
  auto tile = [&](int y) {
    f32x16 acc = bias_tile(bias + 32 * y, g);
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
      Mma<T, PREC_NATIVE>::step(acc, *reinterpret_cast<const V8*>(wrow[kk] + y * 32 * ROWB),
                                __builtin_bit_cast(V8, x[kk / 2][kk % 2]));
    return acc;
  };
  // Beside the sums of dx, no registers are left for the next rows or for two tiles at once: holding them
  // spilled up to 232 bytes a lane (147456 x 128 -> 512, bf16: 133 us with the next rows, 102 with two tiles, 96
  // without either)
  for (int64_t grp = (int64_t)blockIdx.x * (NT / 64) + wave; grp < groups; grp += step) {
    load_rows(x, grp);
    turn_rows();
    const auto srs = rows_rsrc<T>(a.side, grp * 32, a.M, a.side_ld, a.O);
    const auto ors = rows_rsrc<T>(a.out, grp * 32, a.M, a.out_ld, a.O);
    const auto drs = rows_rsrc<T>(a.dx, grp * 32, a.M, a.dx_ld, a.I);
    f32x16 dx[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) dx[kb][r] = 0.f;
    u32x4_t side[2][2];
    auto load_side = [&](u32x4_t (&s)[2][2], int y) {
      sm.load(s[0], srs, 32 * y);
      sm.load(s[1], srs, 32 * (y + 1));
    };
    auto finish = [&](const f32x16& z, const u32x4_t (&side)[2], u32x4_t (&o)[2], int y) {
      u32x4_t s[2];
      Turn::put(turn.to_mem, side);
      Turn::get(turn.to_rows, s);
#pragma unroll
      for (int t = 0; t < 2; ++t) o[t] = finish16<T, EPI_DZ, ACT>(outputs8(z, t), s[t]);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          Mma<T, PREC_NATIVE>::step(dx[kb], column8(kb, 32 * y + 16 * t), __builtin_bit_cast(V8, o[t]));
      Turn::put(turn.to_rows, o);
      Turn::get(turn.to_mem, o);
    };
    auto pair = [&](int y, u32x4_t (&s)[2][2]) {
      u32x4_t o[2][2];
      finish(tile(y), s[0], o[0], y);
      finish(tile(y + 1), s[1], o[1], y + 1);
      om.store(o[0], ors, 32 * y);
      om.store(o[1], ors, 32 * (y + 1));
      load_side(s, y + 2);
    };
    load_side(side, 0);
    for (int y = 0; y < nb; y += 2) pair(y, side);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      u32x4_t o[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) o[t] = finish16<T, EPI_ACT, GNN_ACT_NONE>(outputs8(dx[kb], t), o[t]);
      Turn::put(turn.to_rows, o);
      Turn::get(turn.to_mem, o);
      dm.store(o, drs, 32 * kb);
    }
  }
}

// YB: 32-output tiles whose sums a wave holds; the contraction in steps of 128
template <typename T, int YB, int EPI, int NT>
__global__ __launch_bounds__(NT, NT / 256) void linear_outputs_kernel(const LinArgs a, int transposed) {
  typedef typename TypeOps<T>::V8 V8;
  constexpr bool SIDE = EPI != EPI_ACT;
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int KC = 8;
  const int nkc = (a.I + 16 * KC - 1) / (16 * KC), rowb = nkc * KC * 32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
  unsigned char* const weight = smem + NT / 64 * TURN;
  fill_weight<T, NT, 256>(weight, a, transposed, 32 * YB, rowb);
  const float* bias = (const float*)(weight + 32 * YB * rowb);
  __syncthreads();
  const Turn turn(smem + wave * TURN, lane);
  const MemOrder xm(a.x_ld, a.I, lane), sm(a.side_ld, a.O, lane), om(a.out_ld, a.O, lane);
  const int64_t groups = (a.M + 31) / 32, step = (int64_t)gridDim.x * (NT / 64);
  auto load_part = [&](u32x4_t (&x)[KC / 2][2], int64_t grp, int kc) {
    const auto r = rows_rsrc<T>(a.x, grp * 32, a.M, a.x_ld, a.I);
#pragma unroll
    for (int p = 0; p < KC / 2; ++p) xm.load(x[p], r, 16 * KC * kc + 32 * p);
  };
  const unsigned char* wrow[KC];
#pragma unroll
  for (int kk = 0; kk < KC; ++kk) wrow[kk] = weight + l32 * rowb + (((2 * kk + g) ^ chunk_swizzle<256>(l32)) << 4);
  int64_t grp = (int64_t)blockIdx.x * (NT / 64) + wave;
  u32x4_t next[KC / 2][2];
  load_part(next, grp, 0);
  for (; grp < groups; grp += step) {
    const auto srs = rows_rsrc<T>(a.side, grp * 32, a.M, a.side_ld, a.O);
    const auto ors = rows_rsrc<T>(a.out, grp * 32, a.M, a.out_ld, a.O);
    u32x4_t side[YB][2];
    if (SIDE)
#pragma unroll
      for (int y = 0; y < YB; ++y) sm.load(side[y], srs, 32 * y);
    f32x16 acc[YB];
#pragma unroll
    for (int y = 0; y < YB; ++y) acc[y] = bias_tile(bias + 32 * y, g);
    for (int kc = 0; kc < nkc; ++kc) {
      u32x4_t x[KC / 2][2];
#pragma unroll
      for (int p = 0; p < KC / 2; ++p) {
        Turn::put(turn.to_mem, next[p]);
        Turn::get(turn.to_rows, x[p]);
      }
      const bool last = kc + 1 == nkc;
      load_part(next, last ? grp + step : grp, last ? 0 : kc + 1);
#pragma unroll
      for (int kk = 0; kk < KC; ++kk)
#pragma unroll
        for (int y = 0; y < YB; ++y)
          Mma<T, PREC_NATIVE>::step(acc[y], *reinterpret_cast<const V8*>(wrow[kk] + y * 32 * rowb + kc * KC * 32),
                                    __builtin_bit_cast(V8, x[kk / 2][kk % 2]));
    }
    with_activation(a.act, [&](auto act) {
#pragma unroll
      for (int y = 0; y < YB; ++y) {
        u32x4_t s[2], o[2];
        if (SIDE) {
          Turn::put(turn.to_mem, side[y]);
          Turn::get(turn.to_rows, s);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) o[t] = finish16<T, EPI, decltype(act)::value>(outputs8(acc[y], t), s[t]);
        Turn::put(turn.to_rows, o);
        Turn::get(turn.to_mem, o);
        om.store(o, ors, 32 * y);
      }
    });
  }
}

// What a form needs of LDS, 0 where it is none
struct Form {
  int ks, yb;  // rows: steps; outputs: tiles
  size_t lds;
};
Form form_for(int64_t I, int64_t O) {
  const int64_t o32 = (O + 31) / 32 * 32, o64 = (O + 63) / 64 * 64;
  if (I <= 256) {
    const int ks = I <= 64 ? 4 : I <= 128 ? 8 : 16;
    const int64_t lds = o64 * (32 * ks + 4);
    if (lds <= RS_LDS) return {ks, 0, (size_t)lds};
  }
  if (O <= 128) {
    const int yb = (int)(o32 / 32);
    const int64_t lds = o32 * ((I + 127) / 128 * 256 + 4);
    if (lds <= RS_LDS) return {0, yb, (size_t)lds};
  }
  return {0, 0, 0};
}

typedef void (*Kernel)(LinArgs, int);

template <typename T, int KS, int EPI, int NT>
Kernel rows_kernel(int act) {
  switch (act) {
    case GNN_ACT_RELU: return linear_rows_kernel<T, KS, EPI, GNN_ACT_RELU, NT>;
    case GNN_ACT_GELU: return linear_rows_kernel<T, KS, EPI, GNN_ACT_GELU, NT>;
    case GNN_ACT_SILU: return linear_rows_kernel<T, KS, EPI, GNN_ACT_SILU, NT>;
    case GNN_ACT_SIGMOID: return linear_rows_kernel<T, KS, EPI, GNN_ACT_SIGMOID, NT>;
    default: return linear_rows_kernel<T, KS, EPI, GNN_ACT_NONE, NT>;
  }
}

int launch_fn(Kernel fn, int nt, const LinArgs& a, const Form& f, int transposed, hipStream_t st) {
  const size_t lds = f.lds + nt / 64 * TURN;
  if (lds > 64 * 1024) (void)hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  const int64_t groups = (a.M + 31) / 32;
  const int64_t grid = std::min<int64_t>((groups + nt / 64 - 1) / (nt / 64), persistent_grid((const void*)fn, nt, lds));
  hipLaunchKernelGGL(fn, dim3((uint32_t)grid), dim3(nt), lds, st, a, transposed);
  return (int)hipGetLastError();
}

template <typename T, int EPI>
int launch(const LinArgs& a, const Form& f, int transposed, hipStream_t st) {
  Kernel fn = nullptr;
  switch (f.ks * 10 + f.yb) {
    case 40: fn = rows_kernel<T, 4, EPI, 512>(a.act); break;
    case 80: fn = rows_kernel<T, 8, EPI, 512>(a.act); break;
    case 160: fn = rows_kernel<T, 16, EPI, 512>(a.act); break;
    case 1: fn = linear_outputs_kernel<T, 1, EPI, 512>; break;
    case 2: fn = linear_outputs_kernel<T, 2, EPI, 512>; break;
    case 3: fn = linear_outputs_kernel<T, 3, EPI, 512>; break;
    default: fn = linear_outputs_kernel<T, 4, EPI, 512>; break;
  }
  return launch_fn(fn, 512, a, f, transposed, st);
}

template <typename T, int KS, int NT>
Kernel rows_bwd_kernel(int act) {
  switch (act) {
    case GNN_ACT_RELU: return linear_rows_bwd_kernel<T, KS, GNN_ACT_RELU, NT>;
    case GNN_ACT_GELU: return linear_rows_bwd_kernel<T, KS, GNN_ACT_GELU, NT>;
    case GNN_ACT_SILU: return linear_rows_bwd_kernel<T, KS, GNN_ACT_SILU, NT>;
    default: return linear_rows_bwd_kernel<T, KS, GNN_ACT_SIGMOID, NT>;
  }
}

template <typename T>
int launch(const LinArgs& a, int transposed, hipStream_t st) {
  const Form f = form_for(a.I, a.O);
  if (a.dx)
    return launch_fn(f.ks == 4 ? rows_bwd_kernel<T, 4, 512>(a.act) : rows_bwd_kernel<T, 8, 512>(a.act), 512, a, f, 0, st);
  if (a.dz) return launch<T, EPI_DZ>(a, f, transposed, st);
  return a.side ? launch<T, EPI_ADD>(a, f, transposed, st) : launch<T, EPI_ACT>(a, f, transposed, st);
}

}  // namespace

bool linear_resident_applicable(const gnn_linear_args& a) {
  auto rows16 = [](const void* p, int64_t ld) { return ((uintptr_t)p % 16) == 0 && ld % 8 == 0 && ld < (1 << 24); };
  return a.dtype != GNN_F32 && a.M >= RS_MIN_ROWS && a.O % 8 == 0 && a.out_cols == a.O && a.x_ld < (1 << 24) &&
         rows16(a.out, a.out_ld) && (!a.side || rows16(a.side, a.side_ld)) && form_for(a.I, a.O).lds != 0;
}

bool linear_resident_takes_dx(const gnn_linear_args& a) {
  auto rows16 = [](const void* p, int64_t ld) { return ((uintptr_t)p % 16) == 0 && ld % 8 == 0 && ld < (1 << 24); };
  const Form f = form_for(a.I, a.O);
  return linear_resident_applicable(a) && (f.ks == 4 || f.ks == 8) && a.dz && a.activation != GNN_ACT_NONE &&
         !a.w_transposed && rows16(a.dx, a.dx_ld);
}

int linear_resident(const gnn_linear_args& g, hipStream_t st) {
  LinArgs a{};
  a.dx = g.dx, a.dx_ld = g.dx_ld;
  a.x = g.x, a.w = g.w, a.bias = g.bias, a.side = g.side, a.out = g.out;
  a.M = g.M, a.x_ld = g.x_ld, a.w_ld = g.w_ld, a.side_ld = g.side_ld, a.out_ld = g.out_ld;
  a.I = (int)g.I, a.O = (int)g.O, a.out_cols = (int)g.out_cols, a.act = g.activation, a.dz = g.dz != 0;
  return g.dtype == GNN_BF16 ? launch<bf16>(a, g.w_transposed, st) : launch<f16>(a, g.w_transposed, st);
}

}  // namespace gnn
