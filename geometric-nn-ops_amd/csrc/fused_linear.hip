// A linear layer with its epilogue in one pass, y = act(x W^T + b) + r for rows x [M, I] and W [O, I], and
// the products of its backward:
//   z = x W^T + b, dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum over the rows of dz, dr = dy.
//
// The backward forms z again from x and W instead of keeping it: in 16 bits, z would put a second rounding
// under every gradient, and in fp32 it would cost 4 M O bytes written and read.
//
// linear_kernel. BM x BN output tiles, the contraction in stages of 64 or 128 bytes a row, both operands moved by
// global_load_lds into LDS (STAGES - 1 of them in flight, one barrier a stage) in 16-byte chunks whose order
// within a row the source addresses permute (chunk_swizzle). The products are formed transposed (W's rows as the
// rows of the 32x32 MFMA tile, in an order that leaves a lane 8 consecutive outputs of one row of x): these
// take bias, activation and residual in fp32, round once and leave as one 16-byte store (two in fp32).
// 8192 x 4096 -> 4096, bf16: 252 us without an activation (1090 TFLOP/s), 262 with gelu; the vendor's product alone
// 190. It is bound by how the DMA and the matrix unit overlap: with the DMA left out the products take 176, with
// the products left out the DMA 76 of the 142 us of 4096^3, and neither more stages of half the size (149), shares
// between the products (150 to 158), half of the waves a step behind (146 to 153) nor 4 waves of 128 x 128 (153)
// brought them closer together.
#include <algorithm>

#include "linear_common.hpp"

namespace gnn {

namespace {

using namespace lin;

// s_waitcnt vmcnt(VM) expcnt(7) lgkmcnt(0)
template <int VM>
__device__ __forceinline__ void wait_vm_lgkm0() {
  static_assert(VM >= 0 && VM < 64, "vmcnt immediate");
  __builtin_amdgcn_s_waitcnt(0x070 | (VM & 15) | ((VM >> 4) << 14));
}

// GM x GN waves of 32 X rows x 32 Y outputs; stages of ROWB bytes of a row
template <typename T, int GM_, int GN_, int X_, int Y_, int ROWB_, int STAGES_>
struct Tile {
  static constexpr int GM = GM_, GN = GN_, X = X_, Y = Y_, ROWB = ROWB_, STAGES = STAGES_;
  static constexpr int BM = 32 * GM * X, BN = 32 * GN * Y;
  static constexpr int NW = GM * GN, NT = 64 * NW;
  static constexpr int BK = ROWB / (int)sizeof(T);  // elements of a row a stage
  static constexpr int EPC = 16 / (int)sizeof(T);   // elements a chunk
  static constexpr int CPR = ROWB / 16, RPI = 1024 / ROWB;        // chunks a row, rows a DMA instruction
  static constexpr int QA = BM / RPI / NW, QB = BN / RPI / NW;    // DMA instructions a wave and stage
  static constexpr int QPS = QA + QB;
  static constexpr int STAGE = (BM + BN) * ROWB;
  static constexpr int LDS = STAGES * STAGE;
  static constexpr int WGS = (160 << 10) / LDS;  // workgroups a CU
  static_assert(ROWB == 64 || ROWB == 128, "swizzle");
  static_assert(QA * RPI * NW == BM && QB * RPI * NW == BN, "DMA split");
  static_assert(STAGES >= 2 && STAGES <= 4 && NW * 4096 <= LDS, "waits and the epilogue's tiles");
  static __device__ __forceinline__ int swz(int row, int chunk) { return chunk ^ chunk_swizzle<ROWB>(row); }
};

constexpr int GROUP = 4;

template <typename T, int PREC, typename Cfg>
__global__ __launch_bounds__(Cfg::NT, Cfg::WGS * Cfg::NW / 4) void linear_kernel(const LinArgs a) {
  typedef typename TypeOps<T>::V8 V8;
  __shared__ __align__(16) unsigned char smem[Cfg::LDS];
  // Consecutive workgroups of an XCD take a block of GROUP tiles of rows before the next tiles of outputs: the
  // operands that its L2 fetches at a time are those of about a square of tiles.
  const uint32_t ntn = (uint32_t)(a.out_cols + Cfg::BN - 1) / Cfg::BN;
  const uint32_t w = xcd_remap(blockIdx.x, gridDim.x), group = w / (GROUP * ntn), rest = w % (GROUP * ntn);
  const uint32_t high = min((uint32_t)GROUP, gridDim.x / ntn - group * GROUP);
  const int n0 = (int)(rest / high) * Cfg::BN;
  const int64_t m0 = (int64_t)(group * GROUP + rest % high) * Cfg::BM;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
  const int wm = wave / Cfg::GN, wn = wave % Cfg::GN;

  // DMA: an instruction moves RPI rows; lane -> row lane / CPR, stored chunk lane % CPR, which holds the row's
  // chunk swz(row, lane % CPR). Rows past the end repeat the last one (never stored), chunks past the
  // contraction's end are zeros in both operands. Tiles of 32 of W's rows are in tile_output's order.
  const int drow = lane / Cfg::CPR, dpos = lane % Cfg::CPR;
  const T* xsrc[Cfg::QA];
  const T* wsrc[Cfg::QB];
#pragma unroll
  for (int q = 0; q < Cfg::QA; ++q) {
    const int r = Cfg::RPI * (Cfg::QA * wave + q) + drow;
    xsrc[q] = (const T*)a.x + min(m0 + r, a.M - 1) * a.x_ld;
  }
#pragma unroll
  for (int q = 0; q < Cfg::QB; ++q) {
    const int r = Cfg::RPI * (Cfg::QB * wave + q) + drow, n = n0 + (r & ~31) + tile_output(r & 31);
    wsrc[q] = (const T*)a.w + (int64_t)min(n, a.O - 1) * a.w_ld;
  }
  const int nkt = (a.I + Cfg::BK - 1) / Cfg::BK;
  // instructions [q0, q1) of a stage's QPS, x's first
  auto issue = [&](int kt, int q0, int q1) {
    unsigned char* st = smem + (kt % Cfg::STAGES) * Cfg::STAGE;
    const int k0 = kt * Cfg::BK;
#pragma unroll
    for (int q = q0; q < q1; ++q) {
      const bool is_x = q < Cfg::QA;
      const int at = is_x ? Cfg::QA * wave + q : Cfg::QB * wave + q - Cfg::QA;
      const T* src = is_x ? xsrc[is_x ? q : 0] : wsrc[is_x ? 0 : q - Cfg::QA];
      const int k = k0 + Cfg::swz(Cfg::RPI * at + drow, dpos) * Cfg::EPC;
      __builtin_amdgcn_global_load_lds(k < a.I ? (const void*)(src + k) : (const void*)zero_chunk,
                                       (lds_void_t*)(st + (is_x ? 0 : Cfg::BM * Cfg::ROWB) + at * 1024), 16, 0, 0);
    }
  };
  // 8 elements kk * 16 + 8 g of a row
  auto frag = [&](const unsigned char* base, int r, int kk) -> V8 {
    const unsigned char* row = base + r * Cfg::ROWB;
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const V8*>(row + (Cfg::swz(r, 2 * kk + g) << 4));
    } else {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(row + (Cfg::swz(r, 4 * kk + 2 * g) << 4));
      const f32x4 hi = *reinterpret_cast<const f32x4*>(row + (Cfg::swz(r, 4 * kk + 2 * g + 1) << 4));
      return V8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  };

  f32x16 acc[Cfg::X][Cfg::Y];
#pragma unroll
  for (int x = 0; x < Cfg::X; ++x)
#pragma unroll
    for (int y = 0; y < Cfg::Y; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;

  // A stage's products go in steps of 16 elements; a step begins with the reads of the next step's fragments, over
  // the stage's end too. With three stages in flight the DMA of the stage after them goes in equal shares beside
  // the steps' products (4096 x 4096 -> 1024, bf16: 44 us; all at the stage's start 52). With two buffers it has
  // only until the stage's end to land and goes in the first two steps (4096^3: 142 us; in shares 149). Stages
  // past the end are zeros.
  constexpr int KS = Cfg::BK / 16, SHARE = Cfg::QPS / KS, FIRST = KS > 2 ? 2 : 1;
  constexpr bool SPREAD = Cfg::STAGES > 2;
  static_assert(KS % 2 == 0 && (!SPREAD || SHARE * KS == Cfg::QPS), "steps");
  V8 xf[2][Cfg::X], wf[2][Cfg::Y];
  auto load_frags = [&](int slot, int kt, int kk) {
    const unsigned char* sx = smem + (kt % Cfg::STAGES) * Cfg::STAGE;
    const unsigned char* sw = sx + Cfg::BM * Cfg::ROWB;
#pragma unroll
    for (int y = 0; y < Cfg::Y; ++y) wf[slot][y] = frag(sw, 32 * (Cfg::Y * wn + y) + l32, kk);
#pragma unroll
    for (int x = 0; x < Cfg::X; ++x) xf[slot][x] = frag(sx, 32 * (Cfg::X * wm + x) + l32, kk);
  };
  // This wave's DMA of a stage has landed (the later stages' may be in flight) and its reads so far have
  // returned; after the barrier every wave's have, and the buffer of the stage before is free.
  auto arrive = [&]() {
    wait_vm_lgkm0<(Cfg::STAGES - 2) * Cfg::QPS>();
    asm volatile("s_barrier" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < Cfg::STAGES - 1; ++s) issue(s, 0, Cfg::QPS);
  arrive();
  load_frags(0, 0, 0);
  if (SPREAD) issue(Cfg::STAGES - 1, 0, SHARE);
  for (int kt = 0; kt < nkt; ++kt) {
    const int next = kt + Cfg::STAGES - 1;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const bool last = kk + 1 == KS;
      if (last) arrive();
      load_frags((kk + 1) & 1, last ? kt + 1 : kt, last ? 0 : kk + 1);
      if (SPREAD)
        issue(last ? next + 1 : next, last ? 0 : (kk + 1) * SHARE, last ? SHARE : (kk + 2) * SHARE);
      else if (kk < FIRST)  // before the stage's last step, which waits for it
        issue(next, kk * Cfg::QPS / FIRST, (kk + 1) * Cfg::QPS / FIRST);
#pragma unroll
      for (int x = 0; x < Cfg::X; ++x)
#pragma unroll
        for (int y = 0; y < Cfg::Y; ++y) Mma<T, PREC>::step(acc[x][y], wf[kk & 1][y], xf[kk & 1][x]);
    }
  }

  // A lane's sums are one row's: stored like that, neighbouring lanes would write 16 bytes each to different
  // rows. Every 32 x 32 tile turns through 4 KB of LDS of the wave's own (fp32, 16-byte chunks XOR-swizzled by
  // (row / 2) % 8), and is finished with 4 lanes a row; as many tiles at a time as fit.
  wait_vm_lgkm0<0>();
  asm volatile("s_barrier" ::: "memory");
  constexpr int TILES = Cfg::X * Cfg::Y, FIT = Cfg::LDS / Cfg::NW / 4096, PASS = FIT < TILES ? FIT : TILES;
  static_assert(TILES % PASS == 0, "passes");
  unsigned char* tiles = smem + wave * PASS * 4096;
  auto at = [&](int tile, int row, int chunk) {
    return reinterpret_cast<f32x4*>(tiles + tile * 4096 + row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4));
  };
#pragma unroll
  for (int p = 0; p < TILES; p += PASS) {
#pragma unroll
    for (int t = 0; t < PASS; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16& v = acc[(p + t) % Cfg::X][(p + t) / Cfg::X];
        *at(t, l32, 4 * (q / 2) + 2 * g + q % 2) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
      }
#pragma unroll 2
    for (int h = 0; h < 2 * PASS; ++h) {
      const int t = h >> 1, x = (p + t) % Cfg::X, y = (p + t) / Cfg::X;
      const int row = 16 * (h & 1) + (lane >> 2), n = n0 + 32 * (Cfg::Y * wn + y) + 8 * (lane & 3);
      const int64_t m = m0 + 32 * (Cfg::X * wm + x) + row;
      const f32x4 lo = *at(t, row, 2 * (lane & 3)), hi = *at(t, row, 2 * (lane & 3) + 1);
      f32x8 b = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (a.bias && n < a.O) b = load8_any((const T*)a.bias + n, a.O - n);
      if (m < a.M && n < a.out_cols) finish8<T>(a, f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, b, m, n);
    }
  }
}

template <typename Cfg>
int64_t tiles_of(const LinArgs& a) {
  return (a.M + Cfg::BM - 1) / Cfg::BM * ((a.out_cols + Cfg::BN - 1) / Cfg::BN);
}

template <typename T, int PREC, typename Cfg>
int launch(const LinArgs& a, hipStream_t st) {
  const int64_t tiles = tiles_of<Cfg>(a);
  if (tiles >= ((int64_t)1 << 31)) return set_error(GNN_ERR_UNSUPPORTED, "fused_linear: grid too large");
  hipLaunchKernelGGL((linear_kernel<T, PREC, Cfg>), dim3((uint32_t)tiles), dim3(Cfg::NT), 0, st, a);
  return (int)hipGetLastError();
}

// ---- few tiles ------------------------------------------------------------------------------
// Single tokens and short sequences, whose 128 x 128 tiles would leave most CUs idle and whose time is the
// latency of one pass over the weight: a workgroup takes 32 rows x 32 outputs and its FW_NW waves split the
// contraction, each reading its fragments straight into registers, FW_AHEAD steps at a time; the partial sums
// meet in LDS and are added in wave order. (1 x 384 -> 1536, bf16: 5 us; the 128 x 128 tiles took 13.)
constexpr int FW_NW = 8, FW_NT = 64 * FW_NW, FW_AHEAD = 4;
constexpr int FW_LD = 20;  // floats a lane's 16 sums take in LDS: 4 more keep the lanes on different banks

template <typename T, int PREC>
__global__ __launch_bounds__(FW_NT, 2) void linear_few_kernel(const LinArgs a) {
  typedef typename TypeOps<T>::V8 V8;
  __shared__ __align__(16) float part[FW_NW][64][FW_LD];
  const uint32_t ntn = (uint32_t)(a.out_cols + 31) / 32;
  const int n0 = (int)(blockIdx.x % ntn) * 32, m0 = (int)(blockIdx.x / ntn) * 32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l32 = lane & 31, g = lane >> 5;
  // rows past the end repeat the last one
  const T* x = (const T*)a.x + min((int64_t)(m0 + l32), a.M - 1) * a.x_ld + 8 * g;
  const T* w = (const T*)a.w + (int64_t)min(n0 + tile_output(l32), a.O - 1) * a.w_ld + 8 * g;
  const int steps = (a.I + 15) / 16, whole = a.I / 16, each = (steps + FW_NW - 1) / FW_NW;
  const int k0 = wave * each, k1 = min(whole, k0 + each);
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  // No load in a branch: a batch's last steps may be read again, and are not multiplied
  for (int k = k0; k < k1; k += FW_AHEAD) {
    V8 xf[FW_AHEAD], wf[FW_AHEAD];
#pragma unroll
    for (int u = 0; u < FW_AHEAD; ++u) {
      const int at = 16 * min(k + u, k1 - 1);
      xf[u] = load8_global(x + at);
      wf[u] = load8_global(w + at);
    }
#pragma unroll
    for (int u = 0; u < FW_AHEAD; ++u)
      if (k + u < k1) Mma<T, PREC>::step(acc, wf[u], xf[u]);
  }
  if (whole < steps && whole >= k0 && whole < k0 + each) {  // part of a step: what lies past the row's end is zero
    V8 xf = zero8<T>(), wf = zero8<T>();
    const int left = a.I - 16 * whole - 8 * g;  // of this lane's 8 elements
    if (left >= 8) {
      xf = load8_global(x + 16 * whole), wf = load8_global(w + 16 * whole);
    } else if (sizeof(T) == 4 && left > 0) {  // fp32 rows of 16-byte chunks may end after 4
      const auto xh = load4(x + 16 * whole), wh = load4(w + 16 * whole);
#pragma unroll
      for (int e = 0; e < 4; ++e) xf[e] = xh[e], wf[e] = wh[e];
    }
    Mma<T, PREC>::step(acc, wf, xf);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<f32x4*>(&part[wave][lane][4 * q]) = f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  if (threadIdx.x >= 128) return;
  // 8 outputs 16 t + 8 g of a row a thread
  const int t = threadIdx.x >> 6, n = n0 + 16 * t + 8 * g;
  const int64_t m = m0 + l32;
  if (m >= a.M || n >= a.out_cols) return;
  f32x8 z = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < FW_NW; ++k) z += *reinterpret_cast<const f32x8*>(&part[k][lane][8 * t]);
  f32x8 b = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (a.bias && n < a.O) b = load8_any((const T*)a.bias + n, a.O - n);
  finish8<T>(a, z, b, m, n);
}

template <typename T, int PREC>
int run(const LinArgs& a, hipStream_t st) {
  // The larger the tile the less LDS is read a product, but a CU should have one at least, and the more of them it
  // holds at once the better one's epilogue hides behind another's products. 16-bit types, us (4096 x 4096 -> 1024
  // has 256 tiles of 128 x 128, one a CU; 16384 x 4096 -> 512 has two, 6977 x 384 -> 1024 440):
  //   256 x 256 (4096^3: 136; 185 in 128 x 128) where its rounds of the card, four times as long as those of 128 x 128
  //     and 1.2 times as fast, end before those of two 128 x 128 tiles a CU (45475 x 512 -> 512: 55 and 50);
  //   128 x 128, two a CU, where there are more than CUs (6977 x 384 -> 1024: 18, one a CU and four stages 23;
  //     16384 x 4096 -> 512: 76 and 92), or about one a CU with four stages (4096 x 4096 -> 1024: 44 and 60);
  //   64 x 64, two or, where there are more, five a CU (2048 x 1024 -> 1024: 11, 17 in 128 x 128; 2048 x 384 -> 1536,
  //     three a CU: 9.5, two at once 11.4);
  //   few tiles: below (384 x 384 -> 1536, 144 tiles of 64 x 64: 5.5, in that kernel 8.0).
  // fp32 products are bound by the matrix rate, and smaller tiles do (40401 x 136 -> 257: 65 us in 128 x 64, in one
  // workgroup of 128 x 128 a CU 90; 2048 x 1024 -> 1024, one tile of 128 x 64 a CU: 45 in 64 x 64, 52 in 128 x 64).
  const int64_t cus = compute_units();
  if constexpr (sizeof(T) == 4) {
    typedef Tile<T, 2, 2, 1, 1, 128, 3> Small;
    typedef Tile<T, 2, 2, 2, 1, 128, 2> Medium;
    if (tiles_of<Medium>(a) >= 2 * cus) return launch<T, PREC, Medium>(a, st);
    if (tiles_of<Small>(a) >= cus / 2) return launch<T, PREC, Small>(a, st);
  } else {
    typedef Tile<T, 2, 4, 4, 2, 128, 2> Large;
    typedef Tile<T, 2, 2, 2, 2, 128, 2> Medium;
    typedef Tile<T, 2, 2, 2, 2, 128, 4> MediumAlone;
    typedef Tile<T, 2, 2, 1, 1, 128, 2> Small;
    typedef Tile<T, 2, 2, 1, 1, 128, 4> SmallAlone;
    const int64_t large = tiles_of<Large>(a), medium = tiles_of<Medium>(a), small = tiles_of<Small>(a);
    const int64_t large_rounds = (large + cus - 1) / cus, medium_rounds = (medium + 2 * cus - 1) / (2 * cus);
    if (large >= cus && 10 * 4 * large_rounds <= 12 * 2 * medium_rounds) return launch<T, PREC, Large>(a, st);
    if (medium > cus) return launch<T, PREC, Medium>(a, st);
    if (8 * medium >= 7 * cus) return launch<T, PREC, MediumAlone>(a, st);
    if (small > 2 * cus) return launch<T, PREC, Small>(a, st);
    if (small >= cus / 2) return launch<T, PREC, SmallAlone>(a, st);
  }
  const int64_t few = (a.M + 31) / 32 * ((a.out_cols + 31) / 32);
  hipLaunchKernelGGL((linear_few_kernel<T, PREC>), dim3((uint32_t)few), dim3(FW_NT), 0, st, a);
  return (int)hipGetLastError();
}

// ---- padded rows ------------------------------------------------------------------------------
// dst[r][c] = src[r row_stride + c col_stride] for c < cols, 0 up to ld: a thread writes 16 bytes. Sources whose
// rows are not contiguous but whose columns are (a transposed weight) go through LDS in tiles of 64 x 64, read
// along the columns. (40401 x 131 fp32: 8.6 us, a fill and a strided copy 13.9; 1024 x 4096 bf16 turned: 5.7, a
// strided copy 28.4.)
template <typename E>
__global__ __launch_bounds__(256) void pad_rows_kernel(const gnn_pad_rows_args a) {
  constexpr int N = 16 / (int)sizeof(E);
  typedef E V __attribute__((ext_vector_type(N)));
  const uint32_t chunks = (uint32_t)(a.ld / N);
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = (int64_t)(i / chunks);
  if (r >= a.rows) return;
  const int64_t c = (int64_t)(i % chunks) * N;
  const E* src = (const E*)a.src + r * a.row_stride + c * a.col_stride;
  V v;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = c + e < a.cols ? src[e * a.col_stride] : (E)0;
  reinterpret_cast<V*>(a.dst)[i] = v;
}

template <typename E>
__global__ __launch_bounds__(256) void pad_rows_turned_kernel(const gnn_pad_rows_args a) {
  constexpr int N = 16 / (int)sizeof(E), B = 64;
  typedef E V __attribute__((ext_vector_type(N)));
  __shared__ E tile[B][B + 1];  // [column][row]
  const uint32_t across = (uint32_t)((a.ld + B - 1) / B);
  const int64_t r0 = (int64_t)(blockIdx.x / across) * B, c0 = (int64_t)(blockIdx.x % across) * B;
  for (int k = threadIdx.x; k < B * B; k += 256) {
    const int64_t r = r0 + k % B, c = c0 + k / B;
    tile[k / B][k % B] = r < a.rows && c < a.cols ? ((const E*)a.src)[r * a.row_stride + c * a.col_stride] : (E)0;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < B * B / N; k += 256) {
    const int r = k / (B / N), c = k % (B / N) * N;
    V v;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = tile[c + e][r];
    if (r0 + r < a.rows && c0 + c < a.ld) *reinterpret_cast<V*>((E*)a.dst + (r0 + r) * a.ld + c0 + c) = v;
  }
}

template <typename E>
int pad_rows_typed(const gnn_pad_rows_args& a, hipStream_t st) {
  const bool turned = a.col_stride != 1 && a.row_stride == 1;
  const int64_t blocks = turned ? (a.rows + 63) / 64 * ((a.ld + 63) / 64)
                                : (a.rows * (a.ld * (int64_t)sizeof(E) / 16) + 255) / 256;
  if (blocks >= ((int64_t)1 << 31)) return set_error(GNN_ERR_UNSUPPORTED, "pad_rows: grid too large");
  if (turned)
    hipLaunchKernelGGL(pad_rows_turned_kernel<E>, dim3((uint32_t)blocks), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(pad_rows_kernel<E>, dim3((uint32_t)blocks), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

// ---- column sums ---------------------------------------------------------------------------
// partial[part][n] = sum of d[m][n] over the rows m of a part: 32 lanes of 8 columns, 8 rows a turn
template <typename T>
__global__ __launch_bounds__(256) void column_sums_kernel(const T* d, int64_t ld, int64_t M, int O, int64_t rows,
                                                          float* partial) {
  __shared__ float sum[8][32 * 8 + 8];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
  const int n = (blockIdx.y * 32 + c) * 8;
  f32x8 s = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int64_t m1 = min(M, (int64_t)(blockIdx.x + 1) * rows);
  if (n < O)
    for (int64_t m = (int64_t)blockIdx.x * rows + r; m < m1; m += 8) s += load8_any(d + m * ld + n, O - n);
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[r][c * 8 + e] = s[e];
  __syncthreads();
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (col >= O) return;
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) t += sum[k][threadIdx.x];
  partial[(int64_t)blockIdx.x * O + col] = t;
}

}  // namespace

bool linear_takes_dx(const gnn_linear_args& g) { return linear_resident_takes_dx(g); }

bool linear_takes_transposed(const gnn_linear_args& g) { return linear_resident_applicable(g); }

int linear(const gnn_linear_args& g, hipStream_t st) {
  if (linear_resident_applicable(g)) return linear_resident(g, st);
  LinArgs a{};
  a.x = g.x, a.w = g.w, a.bias = g.bias, a.side = g.side, a.out = g.out;
  a.M = g.M, a.x_ld = g.x_ld, a.w_ld = g.w_ld, a.side_ld = g.side_ld, a.out_ld = g.out_ld;
  a.I = (int)g.I, a.O = (int)g.O, a.out_cols = (int)g.out_cols, a.act = g.activation, a.dz = g.dz != 0;
  switch (g.dtype) {
    case GNN_BF16: return run<bf16, PREC_NATIVE>(a, st);
    case GNN_F16: return run<f16, PREC_NATIVE>(a, st);
    default: return g.precision == GNN_PREC_BF16X3 ? run<float, PREC_BF16X3>(a, st) : run<float, PREC_IEEE>(a, st);
  }
}

int pad_rows(const gnn_pad_rows_args& a, hipStream_t st) {
  return a.dtype == GNN_F32 ? pad_rows_typed<uint32_t>(a, st) : pad_rows_typed<uint16_t>(a, st);
}

int64_t column_sums_parts(int64_t M, int64_t O) {
  const int64_t tiles = (O + 255) / 256;
  return std::max<int64_t>(1, std::min<int64_t>((M + 63) / 64, 4 * (int64_t)compute_units() / tiles));
}

int column_sums(const gnn_column_sums_args& a, hipStream_t st) {
  const int64_t rows = (a.M + a.parts - 1) / a.parts;
  const dim3 grid((uint32_t)a.parts, (uint32_t)((a.O + 255) / 256)), blk(256);
  switch (a.dtype) {
    case GNN_BF16:
      hipLaunchKernelGGL(column_sums_kernel<bf16>, grid, blk, 0, st, (const bf16*)a.d, a.ld, a.M, (int)a.O, rows, a.partial);
      break;
    case GNN_F16:
      hipLaunchKernelGGL(column_sums_kernel<f16>, grid, blk, 0, st, (const f16*)a.d, a.ld, a.M, (int)a.O, rows, a.partial);
      break;
    default:
      hipLaunchKernelGGL(column_sums_kernel<float>, grid, blk, 0, st, (const float*)a.d, a.ld, a.M, (int)a.O, rows,
                         a.partial);
      break;
  }
  return (int)hipGetLastError();
}

}  // namespace gnn
