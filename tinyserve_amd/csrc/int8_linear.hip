// The product of 8-bit rows on gfx950, out = x . W^T with one scale for each row of x (a token)
// and one for each row of W (an output channel):
//
//   out[m, n] = (T)((float)(sum_k x[m, k] w[n, k]) * xs[m] * ws[n])
//
// The sum is an int32 and exact (K <= 131071: 128 * 128 * K < 2^31), so neither the order of its
// parts nor the split of K over waves changes a bit of the output; it is rounded to float32,
// times the token's scale, times the channel's, then to T.
//
// No kernel of the reference corresponds: it stands for F.linear of the decoder layer
// (src/tinyserve/model.py:137-179) where the weights are kept in 8 bits.
#include <type_traits>

#include "common.h"

namespace ts {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4), may_alias));
typedef u32x4 u32x4_alias __attribute__((may_alias));
typedef int i32x16 __attribute__((ext_vector_type(16)));

struct LinearArgs {
  const int8_t* x;
  const int8_t* w;
  const float* xscale;
  const float* wscale;
  void* out;
  int M, N, K;
  int64_t xs, ws, os;
  int groups;  // workgroups of the launch (gridDim would be an implicit argument: 0.4 us of host time)
  int per;     // tile columns per part of K, where K is split over workgroups
};

// 16 codes at any address (gfx950 takes unaligned vector loads).
__device__ __forceinline__ i32x4 load_codes(const int8_t* p) {
  return __builtin_bit_cast(i32x4, static_cast<u32x4>(*reinterpret_cast<const u32x4_loose*>(p)));
}

// Codes k .. k + 15 of a row of K, zeros past its end.
__device__ __forceinline__ i32x4 load_codes_tail(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return load_codes(row + k);
  union {
    i32x4 v;
    int8_t b[16];
  } r;
  r.v = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (k + e < K) r.b[e] = row[k + e];
  return r.v;
}

// Four outputs: at any address, and in LDS beside other types.
template <typename T>
struct Vec4 {
  typedef T V __attribute__((ext_vector_type(4), may_alias));
  typedef V Loose __attribute__((aligned(1)));
};

// Four outputs n .. n + 3 of row m.
template <typename T>
__device__ __forceinline__ void store_outputs(const LinearArgs& a, int m, int n, i32x4 sum) {
  const float s = a.xscale[m];
  T* o = static_cast<T*>(a.out) + m * a.os + n;
  if (n + 4 <= a.N) {
    typename Vec4<T>::V y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = round_f32<T>(static_cast<float>(sum[i]) * s * a.wscale[n + i]);
    *reinterpret_cast<typename Vec4<T>::Loose*>(o) = y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) o[i] = round_f32<T>(static_cast<float>(sum[i]) * s * a.wscale[n + i]);
  }
}

// ---- few rows: the waves of a workgroup along K ------------------------------------------------
// A workgroup takes 16 NTW rows of W and 16 MT rows of x; its KP waves take 128-column units of K
// in turn, and their sums meet in LDS at the end. Each wave brings its own units into its own part
// of LDS (direct-to-LDS loads, eight lanes per row, so that whole lines of W and x are asked for
// once) and reads them back as operands of v_mfma_i32_16x16x64_i8, W the A operand: lane l holds
// row l % 16, columns 16 (l / 16) .. + 15 of each 64. No wave waits for another before the end; as
// soon as a unit is in registers, the loads of the next take its place. (Two or four units in
// flight per wave leave room for fewer workgroups: 64 x 1024 x 2048 3.9 us, 32 x 8192 x 8192 21.4
// against 18.4.)
//
// Loaded straight into operand registers, 16 rows at a time, each load takes about four times as
// long (16 rows of 64 bytes, a row's lanes apart, instead of 8 of 128): M x N x K of 64 x 1024 x
// 2048 7.3 us against 3.7, 64 x 4096 x 1024 5.9 against 4.6, 1 x 4096 x 1024 4.0 against 3.8.
//
// kAligned false: rows that are not 16-byte aligned, or are far apart, pass through registers on
// their way (unaligned vector loads).
template <int kUnits>
__device__ __forceinline__ int swizzle(int r) {
  return (kUnits == 4 ? (r >> 1) & 3 : r & 7) ^ ((r >> 3) & 1);
}

// Wait for this wave's vector-memory loads.
__device__ __forceinline__ void wait_loads() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0f70);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Wait for this wave's LDS operations.
__device__ __forceinline__ void wait_lds() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// The bytes lo .. hi - 1 of a 16-byte unit.
__device__ __forceinline__ i32x4 byte_mask(int lo, int hi) {
  auto below = [](int n) { return n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1; };
  i32x4 m;
#pragma unroll
  for (int d = 0; d < 4; ++d) m[d] = below(hi - 4 * d) & ~below(lo - 4 * d);
  return m;
}

// Division of 0 .. 2^22 by a number of the launch, 1 .. 2^22: a product with ceil(2^s / by) for s = 22 +
// ceil(log2(by)), in the scalar unit. (The compiler's division takes 0.1 us of 64 x 1024 x 2048's 3.7.)
struct Divisor {
  int by, shift;
  uint32_t factor;
  explicit Divisor(int d) : by(d), shift(0), factor(1u << 23) {
    int log = 0;
    while ((1 << log) < d) ++log;
    if (d > 1) {
      shift = log - 1;
      factor = static_cast<uint32_t>(((1ull << (22 + log)) + d - 1) / d);
    }
  }
  __device__ __forceinline__ int quotient(int n) const {
    return static_cast<int>(__umulhi(static_cast<uint32_t>(n) << 9, factor) >> shift);
  }
};

template <typename T, int NTW, int MT, bool kAligned>
__global__ __launch_bounds__(8 * kWave) void int8_rows_kernel(const LinearArgs a, const Divisor tiles_m) {
  constexpr int KP = 8, BN = 16 * NTW, BM = 16 * MT, L = (BM + BN) / 8;  // L: loads per unit
  constexpr int RED = BN + 4;  // padded row of the part sums, 16-byte aligned
  constexpr int kUnit = (BM + BN) * 128, kRing = KP * kUnit, kSums = KP * BM * RED * 4;
  __shared__ __attribute__((aligned(16))) int8_t lds[kRing > kSums ? kRing : kSums];
  const int tid = threadIdx.x, lane = tid % kWave;
  const int kp = __builtin_amdgcn_readfirstlane(tid / kWave);
  // Workgroups go round-robin over the 8 XCDs: those of the same rows of W run on one of them, which
  // reads W once (22 x 3968 x 6656 11.0 us by a grid of two dimensions, 7.9 so; 54 x 1856 x 25664 in
  // one part 32.2 and 20.6).
  const int xcd = blockIdx.x % 8, per = a.groups / 8, more = a.groups % 8;
  const int tile = xcd * per + min(xcd, more) + blockIdx.x / 8;
  const int tn = tiles_m.quotient(tile), n0 = tn * BN, m0 = (tile - tn * tiles_m.by) * BM;
  int8_t* const slot = lds + kp * kUnit;

  // Load j fills rows 8 j .. of a unit, of W and then of x; rows past the ends repeat the last one
  // (their sums are not stored). Unit row r's 16 columns c sit in slot c ^ swizzle(r).
  const int units = a.K / 128, total = (a.K + 127) / 128;
  const int padded = (a.K + 15) & ~15;
  const int last = kAligned ? max(padded - 128, 0) : max(a.K - 128, 0);  // the last unit's first column
  auto row_at = [&](int j) {
    const int r = 8 * j + lane / 8;
    return r < BN ? static_cast<int64_t>(min(r, a.N - 1 - n0)) * a.ws : static_cast<int64_t>(min(r - BN, a.M - 1 - m0)) * a.xs;
  };
  auto column = [&](int j) { return ((lane % 8) ^ swizzle<8>(8 * j + lane / 8)) * 16; };
  const int8_t* wg = a.w + static_cast<int64_t>(n0) * a.ws;
  const int8_t* xg = a.x + static_cast<int64_t>(m0) * a.xs;
  uint32_t off[kAligned ? L : 1];
  const int8_t* from[kAligned ? 1 : L];
#pragma unroll
  for (int j = 0; j < L; ++j) {
    if constexpr (kAligned) off[j] = static_cast<uint32_t>(row_at(j)) + min(column(j), padded - 16);
    else from[j] = (8 * j < BN ? wg : xg) + row_at(j);
  }
  i32x4 held[kAligned ? 1 : L];
  auto fetch = [&](int u) {
    const int k0 = min(u * 128, last);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      if constexpr (kAligned) lds_load16_s((8 * j < BN ? wg : xg) + k0, off[j], (TS_LDS void*)(slot + j * 1024));
      else if (a.K >= 128) held[j] = load_codes(from[j] + k0 + column(j));
      else held[j] = load_codes_tail(from[j], column(j), a.K);
    }
  };

  i32x4 acc[NTW][MT];
#pragma unroll
  for (int t = 0; t < NTW; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[t][u] = i32x4{0, 0, 0, 0};

  if (kp < total) fetch(kp);
  for (int u = kp; u < total; u += KP) {
    if constexpr (kAligned) {
      wait_loads();
    } else {
#pragma unroll
      for (int j = 0; j < L; ++j) *reinterpret_cast<i32x4*>(slot + j * 1024 + lane * 16) = held[j];
      if (u + KP < total) fetch(u + KP);
      wait_lds();
    }
    i32x4 wv[2][NTW], xv[2][MT];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int8_t* p = slot + (lane % 16) * 128 + (((4 * s + lane / 16) ^ swizzle<8>(lane % 16)) * 16);
#pragma unroll
      for (int t = 0; t < NTW; ++t) wv[s][t] = *reinterpret_cast<const i32x4*>(p + t * 2048);
#pragma unroll
      for (int t = 0; t < MT; ++t) xv[s][t] = *reinterpret_cast<const i32x4*>(p + (NTW + t) * 2048);
    }
    wait_lds();  // the unit is in registers: its slot is free
    if constexpr (kAligned)
      if (u + KP < total) fetch(u + KP);
    if (u == units) {  // the last, partial unit: W's columns of the unit before and past K
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int col = last + (4 * s + lane / 16) * 16;
        const i32x4 m = byte_mask(units * 128 - col, a.K - col);
#pragma unroll
        for (int t = 0; t < NTW; ++t) wv[s][t] &= m;
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < NTW; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[t][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[s][t], xv[s][m], acc[t][m], 0, 0, 0);
  }
  __syncthreads();  // every wave's units are in registers: the sums take their place

  // Lane l holds column l % 16 (a row of x) and rows 4 (l / 16) .. + 3 (of W) of each result.
  int* red = reinterpret_cast<int*>(lds);
#pragma unroll
  for (int t = 0; t < NTW; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u)
      *reinterpret_cast<i32x4*>(&red[(kp * BM + u * 16 + lane % 16) * RED + t * 16 + lane / 16 * 4]) = acc[t][u];
  __syncthreads();
  for (int i = tid; i < BM * (BN / 4); i += KP * kWave) {
    const int m = i / (BN / 4), j = i % (BN / 4) * 4;
    if (m0 + m >= a.M || n0 + j >= a.N) continue;
    i32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int p = 0; p < KP; ++p) v += *reinterpret_cast<const i32x4*>(&red[(p * BM + m) * RED + j]);
    store_outputs<T>(a, m0 + m, n0 + j, v);
  }
}

template <typename T, int NTW, int MT>
static int launch_rows8(LinearArgs a, bool aligned, hipStream_t st) {
  const int64_t tn = (a.N + 16 * NTW - 1) / (16 * NTW), tm = (a.M + 16 * MT - 1) / (16 * MT);
  if (tm * tn > 1 << 22) return TS_EUNSUPPORTED;  // 2^31 threads
  a.groups = static_cast<int>(tm * tn);
  const dim3 grid(a.groups), block(8 * kWave);
  if (aligned) hipLaunchKernelGGL((int8_rows_kernel<T, NTW, MT, true>), grid, block, 0, st, a, Divisor(static_cast<int>(tm)));
  else hipLaunchKernelGGL((int8_rows_kernel<T, NTW, MT, false>), grid, block, 0, st, a, Divisor(static_cast<int>(tm)));
  return launch_status();
}

// ---- many rows: tiles through LDS -------------------------------------------------------------
// Each of the workgroup's GM x GN waves takes 32 MW rows of x and 32 NW rows of W: MW * NW
// accumulators of v_mfma_i32_32x32x32_i8, W the A operand and x the B operand.
//
// Both operands go through a ring of kStages LDS tiles of kCols columns, filled by direct-to-LDS
// loads (kCols / 16 lanes per row) while older tiles are multiplied. Row r's 16-byte unit c sits
// in slot c ^ swizzle(r), which spreads any 8 or 16 rows' units c over all banks; the lanes of a
// load fetch the units that their slots hold. A step's operands are read from LDS while the step
// before is multiplied; the barrier that hands over the next tile stands before a tile's last
// step, so that its product covers the first reads of the next.
//
// Columns past the last whole tile: one more tile that ends where the rows (rounded up to 16
// columns) end; the columns of it that the tile before held, or that lie past K, are masked out
// of W's operand in registers.
//
// T int32_t: a part of K per workgroup, `per` tiles of it, the sums of part p as they are at row
// p * M + m of `out`.
template <typename T, int MW, int NW, int GM, int GN, int kCols, int kStages>
__global__ __launch_bounds__(GM * GN * kWave, 2) void int8_tile_kernel(LinearArgs a, int tiles_m, int tiles_n) {
  constexpr bool kPart = std::is_same_v<T, int32_t>;
  constexpr int kWaves = GM * GN, kThreads = kWaves * kWave;
  constexpr int BM = 32 * MW * GM, BN = 32 * NW * GN;
  constexpr int kUnits = kCols / 16, kSteps = kCols / 32, RPL = kWave / kUnits;  // RPL: rows per load
  constexpr int kXTile = BM * kCols, kWTile = BN * kCols;  // bytes
  constexpr int XL = BM / RPL / kWaves, WL = BN / RPL / kWaves;  // loads per wave and tile
  constexpr int kRow = 32 * NW * sizeof(T) + 16;  // bytes of a row of the output staging
  constexpr int kRing = kStages * (kXTile + kWTile), kStaged = kWaves * 32 * kRow + (BM + BN) * 4;
  constexpr int kLds = kRing > kStaged ? kRing : kStaged;
  static_assert(BM % (RPL * kWaves) == 0 && BN % (RPL * kWaves) == 0 && kLds <= 160 * 1024, "tile shape");
  __shared__ __attribute__((aligned(16))) int8_t lds[kLds];
  int8_t* const x_ring = lds;
  int8_t* const w_ring = lds + kStages * kXTile;

  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / GN, wn = wave % GN;

  // Workgroups go round-robin over the 8 XCDs: each XCD takes a contiguous run of tiles, in
  // bands of 4 tiles of x, so that the tiles running on it share rows of x and W in its L2.
  int tm, tn;
  {
    const int xcd = blockIdx.x % 8, per = a.groups / 8, more = a.groups % 8;
    int t = xcd * per + min(xcd, more) + blockIdx.x / 8;
    if constexpr (kPart) {
      const int part = t / (tiles_m * tiles_n), k0 = part * a.per * kCols;
      t -= part * tiles_m * tiles_n;
      a.x += k0;
      a.w += k0;
      a.K = min(a.K - k0, a.per * kCols);
      a.out = static_cast<T*>(a.out) + part * a.M * a.os;
    }
    const int band = t / (4 * tiles_n), first = band * 4, high = min(4, tiles_m - first);
    const int in = t - band * 4 * tiles_n;
    tm = first + in % high;
    tn = in / high;
  }
  const int m0 = tm * BM, n0 = tn * BN;
  // Each thread keeps a few of the tile's scales until the end.
  constexpr int kScales = kPart ? 0 : (BM + BN + kThreads - 1) / kThreads;
  float scale[kScales + 1];
#pragma unroll
  for (int i = 0; i < kScales; ++i) {
    const int c = threadIdx.x + i * kThreads;
    scale[i] = c < BN ? a.wscale[min(n0 + c, a.N - 1)] : a.xscale[min(m0 + c - BN, a.M - 1)];
  }
  const int8_t* wg = a.w + static_cast<int64_t>(n0) * a.ws;
  const int8_t* xg = a.x + static_cast<int64_t>(m0) * a.xs;

  // Load j of this wave fills rows RPL (wave * XL + j) .. of an x tile (WL: of a W tile), kUnits
  // lanes each; rows past the ends repeat the last one (their sums are not stored).
  const int padded = (a.K + 15) & ~15;
  auto x_row = [&](int j) { return RPL * (wave * XL + j) + lane / kUnits; };
  auto w_row = [&](int j) { return RPL * (wave * WL + j) + lane / kUnits; };
  auto column = [&](int r) { return min(((lane % kUnits) ^ swizzle<kUnits>(r)) * 16, padded - 16); };
  uint32_t x_off[XL], w_off[WL];
#pragma unroll
  for (int j = 0; j < XL; ++j)
    x_off[j] = static_cast<uint32_t>(min(x_row(j), a.M - 1 - m0) * a.xs) + column(x_row(j));
#pragma unroll
  for (int j = 0; j < WL; ++j)
    w_off[j] = static_cast<uint32_t>(min(w_row(j), a.N - 1 - n0) * a.ws) + column(w_row(j));
  // LDS bytes of unit 2 s + lane / 32 of row lane % 32 of a 32-row operand tile.
  int unit[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
    unit[s] = (lane % 32) * kCols + (((2 * s + lane / 32) ^ swizzle<kUnits>(lane % 32)) * 16);

  i32x16 acc[NW][MW];
#pragma unroll
  for (int t = 0; t < NW; ++t)
#pragma unroll
    for (int u = 0; u < MW; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][u][i] = 0;

  i32x4 wf[2][NW], xf[2][MW];  // operands of two steps, taken in turn
  auto read_all = [&](int s, const int8_t* xt, const int8_t* wt) {
#pragma unroll
    for (int t = 0; t < NW; ++t) wf[s & 1][t] = *reinterpret_cast<const i32x4*>(wt + (wn * NW + t) * 32 * kCols + unit[s]);
#pragma unroll
    for (int u = 0; u < MW; ++u) xf[s & 1][u] = *reinterpret_cast<const i32x4*>(xt + (wm * MW + u) * 32 * kCols + unit[s]);
  };
  auto multiply = [&](int s, int p) {  // product p of step s
    acc[p / MW][p % MW] =
        __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[s & 1][p / MW], xf[s & 1][p % MW], acc[p / MW][p % MW], 0, 0, 0);
  };
  auto multiply_all = [&](int s) {
#pragma unroll
    for (int p = 0; p < NW * MW; ++p) multiply(s, p);
  };

  const int whole = a.K / kCols, tiles = (a.K + kCols - 1) / kCols;
  const int last = max(padded - kCols, 0);  // the last tile's first column
  auto load_x = [&](int j, int kt, int8_t* tile) {
    lds_load16_s(xg + min(kt * kCols, last), x_off[j], (TS_LDS void*)(tile + RPL * (wave * XL + j) * kCols));
  };
  auto load_w = [&](int j, int kt, int8_t* tile) {
    lds_load16_s(wg + min(kt * kCols, last), w_off[j], (TS_LDS void*)(tile + RPL * (wave * WL + j) * kCols));
  };
  int slot = 0;
  if (tiles > 0) {
    for (int kt = 0; kt < min(kStages, tiles); ++kt) {
#pragma unroll
      for (int j = 0; j < XL; ++j) load_x(j, kt, x_ring + kt * kXTile);
#pragma unroll
      for (int j = 0; j < WL; ++j) load_w(j, kt, w_ring + kt * kWTile);
    }
    if (tiles >= kStages) ring_barrier<(kStages - 1) * (XL + WL)>();
    else ring_barrier<0>();
    read_all(0, x_ring, w_ring);
    // Step s's products with loads of tile kt spread among them: issued together, they would hold
    // up the wave's products for as long as the load path takes them in.
    int8_t *x_free = x_ring, *w_free = w_ring;  // the slots that the last barrier freed
    auto step = [&](int s, int xn, int wn, int kt) {
      constexpr int P = NW * MW;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        __builtin_amdgcn_sched_barrier(0);
        multiply(s, p);
        __builtin_amdgcn_sched_barrier(0);
        if (kt >= tiles) continue;
#pragma unroll
        for (int j = 0; j < xn; ++j)
          if (j * P / xn == p) load_x(j, kt, x_free);
#pragma unroll
        for (int j = 0; j < wn; ++j)
          if (j * P / wn == p) load_w(j, kt, w_free);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int kt = 0; kt < whole; ++kt) {
      int8_t *xt = x_ring + slot * kXTile, *wt = w_ring + slot * kWTile;
      slot = slot + 1 == kStages ? 0 : slot + 1;
#pragma unroll
      for (int s = 0; s + 1 < kSteps; ++s) {
        read_all(s + 1, xt, wt);
        step(s, 0, s == 0 ? WL : 0, kt > 0 ? kt - 1 + kStages : tiles);
      }
      // Every read of this tile is done and the next one has landed, in every wave.
      if (kt + kStages - 1 < tiles) ring_barrier<(kStages - 2) * (XL + WL)>();
      else ring_barrier<0>();
      x_free = xt;
      w_free = wt;
      if (kt + 1 < tiles) read_all(0, x_ring + slot * kXTile, w_ring + slot * kWTile);
      step(kSteps - 1, XL, 0, kt + kStages);
    }
    if (whole < tiles) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int col = last + (2 * s + lane / 32) * 16;
        const i32x4 mask = byte_mask(whole * kCols - col, a.K - col);
#pragma unroll
        for (int t = 0; t < NW; ++t) wf[s & 1][t] &= mask;
        if (s + 1 < kSteps) read_all(s + 1, x_ring + slot * kXTile, w_ring + slot * kWTile);
        multiply_all(s);
      }
    }
  }
  __syncthreads();  // the ring's last reads, before the outputs take its place

  // Lane l holds column l % 32 (a row of x) and rows 8 j + 4 (l / 32) .. + 3 (of W) of each result.
  // 32 rows of outputs at a time go through the wave's own part of LDS and out in whole vectors.
  int8_t* mine = lds + wave * 32 * kRow;
  float* scales = reinterpret_cast<float*>(lds + kWaves * 32 * kRow);  // of BN rows of W, then BM of x
#pragma unroll
  for (int i = 0; i < kScales; ++i)
    if (threadIdx.x + i * kThreads < BM + BN) scales[threadIdx.x + i * kThreads] = scale[i];
  __syncthreads();
  constexpr int E = Pack16<T>::N, VPR = 32 * NW / E;  // vectors per row
#pragma unroll
  for (int u = 0; u < MW; ++u) {
    float s = 1.f;
    if constexpr (!kPart) s = scales[BN + (wm * MW + u) * 32 + lane % 32];
#pragma unroll
    for (int t = 0; t < NW; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = t * 32 + j * 8 + lane / 32 * 4;
        typename Vec4<T>::V y;
        if constexpr (kPart) {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = acc[t][u][j * 4 + i];
        } else {
          const f32x4 sw = *reinterpret_cast<const f32x4*>(scales + wn * 32 * NW + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = round_f32<T>(static_cast<float>(acc[t][u][j * 4 + i]) * s * sw[i]);
        }
        *reinterpret_cast<typename Vec4<T>::V*>(mine + (lane % 32) * kRow + c * sizeof(T)) = y;
      }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int v = 0; v < 32 * VPR / kWave; ++v) {
      const int r = (v * kWave + lane) / VPR, c = (v * kWave + lane) % VPR * E;
      const int m = m0 + (wm * MW + u) * 32 + r, n = n0 + wn * 32 * NW + c;
      Pack16<T> y;
      y.raw = *reinterpret_cast<const u32x4_alias*>(mine + r * kRow + c * sizeof(T));
      if (m >= a.M) continue;
      T* o = static_cast<T*>(a.out) + m * a.os + n;
      if (n + E <= a.N) {
        store16_loose(o, y);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (n + e < a.N) o[e] = y.v[e];
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The sums of the parts of K, and the outputs of them: four to a thread.
template <typename T>
__global__ __launch_bounds__(256) void int8_parts_kernel(const LinearArgs a, const int32_t* sums, int parts, int quads) {
  const int i = blockIdx.x * 256 + threadIdx.x, m = i / quads, n = (i - m * quads) * 4;
  if (m >= a.M) return;
  const int64_t each = static_cast<int64_t>(a.M) * quads * 4;
  const int32_t* p = sums + static_cast<int64_t>(i) * 4;
  i32x4 v = *reinterpret_cast<const i32x4*>(p);
#pragma unroll 4
  for (int k = 1; k < parts; ++k) v += *reinterpret_cast<const i32x4*>(p + k * each);
  store_outputs<T>(a, m, n, v);
}

template <typename T, int MW, int NW, int GM, int GN, int kCols, int kStages>
static int launch_tiles(LinearArgs a, hipStream_t st) {
  constexpr int BM = 32 * MW * GM, BN = 32 * NW * GN;
  const int64_t tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
  if (tm * tn > 1 << 22) return TS_EUNSUPPORTED;  // 2^31 threads
  a.groups = static_cast<int>(tm * tn);
  hipLaunchKernelGGL((int8_tile_kernel<T, MW, NW, GM, GN, kCols, kStages>), dim3(a.groups),
                     dim3(GM * GN * kWave), 0, st, a, static_cast<int>(tm), static_cast<int>(tn));
  return launch_status();
}

template <typename T, int MW, int NW, int GM, int GN, int kCols, int kStages>
static int launch_parts(LinearArgs a, int parts, int32_t* sums, hipStream_t st) {
  constexpr int BM = 32 * MW * GM, BN = 32 * NW * GN;
  const int tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN, quads = (a.N + 3) / 4;
  LinearArgs part = a;
  part.out = sums;
  part.os = quads * 4;
  part.groups = tm * tn * parts;
  part.per = ((a.K + kCols - 1) / kCols + parts - 1) / parts;
  hipLaunchKernelGGL((int8_tile_kernel<int32_t, MW, NW, GM, GN, kCols, kStages>), dim3(part.groups),
                     dim3(GM * GN * kWave), 0, st, part, tm, tn);
  if (const int rc = launch_status()) return rc;
  hipLaunchKernelGGL(int8_parts_kernel<T>, dim3((a.M * quads + 255) / 256), dim3(256), 0, st, a, sums, parts, quads);
  return launch_status();
}

// Tile shapes, and what a tile of each takes on a compute unit: a fixed part (launch, the ring's
// first fill, outputs) and a part per 1024 columns, in us as fitted to captured launches. The
// chip takes ceil(tiles / CUs) of them one after another, so large tiles (fewer LDS reads per
// product) pay where there are many of them and small ones where there are few. Measured (us, in
// the order of the table): 8192 x 8192 x 8192 452, 502, 620, 694, 851; 2751 x 6144 x 1024 35.2,
// 28.8, 35.2, 34.1, 41.2; 1024 x 4096 x 4096 41.9, 29.9, 22.9, 25.2, 30.5; 512 x 4096 x 1024
// 16.0, 11.4, 8.5, 7.2, 7.7; 256 x 1024 x 2048 23.9, 16.3, 10.6, 8.9, 7.0.
struct TileShape {
  int bm, bn;
  float fixed, per_k;
};
constexpr TileShape kShapes[] = {
    {256, 256, 6.4f, 10.0f},  // 8 waves of 128 x 64
    {192, 128, 3.2f, 4.4f},   // 4 waves of 96 x 64, two workgroups per CU
    {128, 128, 2.4f, 4.4f},   // 8 waves of 64 x 32, three stages
    {64, 128, 1.9f, 2.55f},   // 4 waves of 32 x 64, three stages, two workgroups per CU
    {64, 64, 0.8f, 1.6f},     // 4 waves of 32 x 32, four stages, two workgroups per CU
};

// Row kernels, as 16-row tiles of W and of x per workgroup, with what a workgroup takes beside its
// loads (sums, outputs), in us.
struct RowShape {
  int ntw, mt;
  float fixed;
};
constexpr RowShape kRowShapes[] = {{1, 1, 0.2f}, {2, 1, 0.25f}, {2, 2, 0.5f}, {4, 1, 0.7f}, {4, 2, 1.2f}, {4, 4, 2.2f}};

// What runs: a tile shape (0 ..) or a row shape (-1 - index), and the parts of K that workgroups of
// their own take.
struct Pick {
  int kernel, parts;
};

// Both kinds are priced in us, by constants fitted to 357 products of 1 .. 8192 rows and 64 .. 28672
// columns and outputs, each timed with every kernel: the pick takes 0.9% longer than the best of
// them on average, 24% at most. A row kernel takes, beside its start, what its workgroups bring
// into one compute unit, at about 55 KB a us. Tiles that do not fill the chip wait for W: half as
// much again per column. Past 4096 columns loads come slower (`deep`): fewer of them find their
// lines in L2. Measured, row kernel against tiles: 128 x 2048 x 4096 6.5 and 10.6, 64 x 8192 x 8192
// 20.9 and 26.7, 64 x 16384 x 2048 11.8 and 9.6, 64 x 151936 x 1024 62 and 35.
//
// K split over workgroups: few tiles over many columns leave compute units without one, or with one
// where others have two. It costs a second launch and the sums' way through memory (5.5 us, 3.2
// TB/s). Measured, us without and with: 384 x 4096 x 11008 46.6 and 36.8 (128 x 128, two parts),
// 297 x 4288 x 15680 68 and 47 (the same), 1257 x 3392 x 27328 247 and 144 (256 x 256, three), 137 x
// 6464 x 18112 74 and 50 (256 x 256, eight); but 256 x 4096 x 4096 12.3 and 16.4, 1024 x 8192 x 8192
// 83.7 and 85.1. Parts of the other shapes would add 0.2% over all the products.
constexpr int kUnsplit = 4096;
static Pick pick_kernel(int M, int N, int K, bool may_split) {
  const unsigned cus = compute_units(), m = M, n = N;
  const float k = static_cast<float>(K) / 1024.f, deep = K > kUnsplit ? k - 4.f : 0.f;
  // 32-bit arithmetic, and constants in unrolled loops: this runs on the host at every call.
  constexpr unsigned kMost = 1 << 22;  // workgroups of 512 threads: a launch has fewer than 2^32
  auto groups = [&](unsigned bm, unsigned bn) {  // kMost + 1: more than that
    const uint64_t g = static_cast<uint64_t>((m + bm - 1) / bm) * ((n + bn - 1) / bn);
    return g > kMost ? kMost + 1 : static_cast<unsigned>(g);
  };
  auto times = [&](unsigned g) { return static_cast<float>((g + cus - 1) / cus); };  // workgroups per compute unit, one after another
  Pick best{0, 1};
  float least = 0.f;
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const TileShape& t = kShapes[i];
    const unsigned g = groups(t.bm, t.bn);
    if (i > 0 && g > kMost) continue;
    const float us = times(g) * (t.fixed + t.per_k * k);
    if (i == 0 || us < least) {
      best.kernel = i;
      least = us;
    }
  }
  const TileShape& t = kShapes[best.kernel];
  const unsigned g = groups(t.bm, t.bn);
  least += 3.0f + times(g) * t.per_k * 1.2f * deep;
  if (g < cus) least += 0.5f * t.per_k * k;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const unsigned bm = 16 * kRowShapes[i].mt, bn = 16 * kRowShapes[i].ntw, g = groups(bm, bn);
    if (g > kMost) continue;
    const float us = 3.f + times(g) * (kRowShapes[i].fixed + 0.018f * static_cast<float>(bm + bn) * (k + 0.3f * deep));
    if (us < least) {
      best.kernel = -1 - i;
      least = us;
    }
  }
  if (!may_split || K <= kUnsplit || least < 8.5f + kShapes[2].fixed) return best;
  const int columns = (K + 127) / 128;
  const float outputs = static_cast<float>(M) * static_cast<float>(N);
  for (int i : {0, 2}) {
    const TileShape& t = kShapes[i];
    for (int parts : {2, 3, 4, 6, 8}) {
      const int per = (columns + parts - 1) / parts;
      const unsigned g = groups(t.bm, t.bn) * parts;
      if ((parts - 1) * per >= columns || g > 4 * cus) continue;  // a part would be empty; nothing to fill
      if (g < cus / 4) continue;  // 16 x 16 x 131056 in 8 parts 57, as one workgroup of the row kernel 50
      const float us = 8.5f + times(g) * (t.fixed + 1.2f * t.per_k * static_cast<float>(per) / 8.f) +
                       outputs * 8.f * static_cast<float>(parts) / 3.2e6f;
      if (us < least) {
        best = {i, parts};
        least = us;
      }
    }
  }
  return best;
}

// Bytes of the sums of `parts` parts.
static int64_t parts_bytes(int M, int N, int parts) {
  return parts > 1 ? static_cast<int64_t>(parts) * M * ((static_cast<int64_t>(N) + 3) / 4 * 16) : 0;
}

// Rows for direct-to-LDS loads: 16-byte aligned, readable to a whole 16 columns, and, as rows are addressed
// by 32-bit offsets, at most 2^23 bytes apart.
static bool rows_fit(const LinearArgs& a, bool padded) {
  const int64_t at = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w)) | a.xs | a.ws;
  return at % 16 == 0 && (padded || a.K % 16 == 0) && a.xs <= 1 << 23 && a.ws <= 1 << 23;
}

template <typename T>
static int launch_linear(const LinearArgs& a, bool padded, int32_t* sums, int64_t bytes, hipStream_t st) {
  const bool aligned = rows_fit(a, padded);
  Pick pick = pick_kernel(a.M, a.N, a.K, sums != nullptr);
  if (parts_bytes(a.M, a.N, pick.parts) > bytes) pick = pick_kernel(a.M, a.N, a.K, false);
  if (pick.kernel >= 0 && !aligned) return TS_EUNSUPPORTED;
  if (pick.parts > 1) {
    switch (pick.kernel) {
      case 0: return launch_parts<T, 4, 2, 2, 4, 128, 2>(a, pick.parts, sums, st);
      default: return launch_parts<T, 2, 1, 2, 4, 128, 3>(a, pick.parts, sums, st);
    }
  }
  switch (pick.kernel) {
    case -1: return launch_rows8<T, 1, 1>(a, aligned, st);
    case -2: return launch_rows8<T, 2, 1>(a, aligned, st);
    case -3: return launch_rows8<T, 2, 2>(a, aligned, st);
    case -4: return launch_rows8<T, 4, 1>(a, aligned, st);
    case -5: return launch_rows8<T, 4, 2>(a, aligned, st);
    case -6: return launch_rows8<T, 4, 4>(a, aligned, st);
    case 0: return launch_tiles<T, 4, 2, 2, 4, 128, 2>(a, st);
    case 1: return launch_tiles<T, 3, 2, 2, 2, 128, 2>(a, st);
    case 2: return launch_tiles<T, 2, 1, 2, 4, 128, 3>(a, st);
    case 3: return launch_tiles<T, 1, 2, 2, 2, 128, 3>(a, st);
    default: return launch_tiles<T, 1, 1, 2, 2, 128, 4>(a, st);
  }
}

}  // namespace ts

using namespace ts;

extern "C" int64_t ts_int8_linear_workspace(int M, int N, int K) {
  if (M <= 0 || M > TS_INT8_MAX_DIM || N <= 0 || N > TS_INT8_MAX_DIM || K <= kUnsplit || K > TS_INT8_MAX_K) return 0;
  return parts_bytes(M, N, pick_kernel(M, N, K, true).parts);
}

extern "C" int ts_int8_linear(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride,
                              const float* w_scale, void* out, int64_t o_stride, int M, int N, int K, int padded,
                              int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (M < 0 || M > TS_INT8_MAX_DIM || N < 0 || N > TS_INT8_MAX_DIM || K < 0 || K > TS_INT8_MAX_K || x_stride < 0 || w_stride < 0) return TS_EINVAL;
  if (M > 1 && o_stride < N) return TS_EINVAL;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < 0) return TS_EINVAL;
  if (dtype < TS_F32 || dtype > TS_BF16) return TS_EUNSUPPORTED;
  if (M == 0 || N == 0) return 0;
  if (!out || !x_scale || !w_scale || (K > 0 && (!x || !w))) return TS_EINVAL;
  const LinearArgs a{x, w, x_scale, w_scale, out, M, N, K, x_stride, w_stride, o_stride, 0, 0};
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto* sums = static_cast<int32_t*>(workspace);
  switch (dtype) {
    case TS_F32: return launch_linear<float>(a, padded != 0, sums, workspace_bytes, st);
    case TS_F16: return launch_linear<f16>(a, padded != 0, sums, workspace_bytes, st);
    default: return launch_linear<bf16>(a, padded != 0, sums, workspace_bytes, st);
  }
}
