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
#include "common.h"

namespace ts {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

struct LinearArgs {
  const int8_t* x;
  const int8_t* w;
  const float* xscale;
  const float* wscale;
  void* out;
  int M, N, K;
  int64_t xs, ws, os;
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

template <typename T, int N>
struct Loose {
  typedef T Vec __attribute__((ext_vector_type(N)));
  typedef Vec V __attribute__((aligned(1), may_alias));
};

// Four outputs n .. n + 3 of row m.
template <typename T>
__device__ __forceinline__ void store_outputs(const LinearArgs& a, int m, int n, i32x4 sum) {
  const float s = a.xscale[m];
  T* o = static_cast<T*>(a.out) + m * a.os + n;
  if (n + 4 <= a.N) {
    typename Loose<T, 4>::Vec y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = from_f32<T>(static_cast<float>(sum[i]) * s * a.wscale[n + i]);
    *reinterpret_cast<typename Loose<T, 4>::V*>(o) = y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) o[i] = from_f32<T>(static_cast<float>(sum[i]) * s * a.wscale[n + i]);
  }
}

// ---- few rows: W streamed through registers ---------------------------------------------------
// A workgroup takes 16 * NTW rows of W and 16 * MT rows of x. Its KP waves take 128-column units
// of K in turn, so that the waves side by side read whole lines of W; W is the A operand of
// v_mfma_i32_16x16x64_i8 and x its B operand, both straight from global memory (16 codes per
// lane: row l % 16, columns 16 (l / 16) .. + 15 of each 64). The waves' sums meet in LDS.
template <typename T, int KP, int NTW, int MT>
__global__ __launch_bounds__(KP * kWave) void int8_rows_kernel(const LinearArgs a) {
  constexpr int BN = 16 * NTW, BM = 16 * MT;
  constexpr int RED = BN + 4;  // padded row of the part sums, 16-byte aligned
  __shared__ int red[KP > 1 ? KP * BM * RED : 1];
  const int tid = threadIdx.x, lane = tid % kWave, kp = tid / kWave;
  const int r16 = lane % 16, kq = lane / 16 * 16;
  const int n0 = blockIdx.x * BN, m0 = blockIdx.y * BM;

  // Rows past the ends repeat the last one: their sums are not stored.
  const int8_t* wp[NTW];
  const int8_t* xp[MT];
#pragma unroll
  for (int t = 0; t < NTW; ++t) wp[t] = a.w + static_cast<int64_t>(min(n0 + t * 16 + r16, a.N - 1)) * a.ws;
#pragma unroll
  for (int t = 0; t < MT; ++t) xp[t] = a.x + static_cast<int64_t>(min(m0 + t * 16 + r16, a.M - 1)) * a.xs;

  i32x4 acc[NTW][MT];
#pragma unroll
  for (int t = 0; t < NTW; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[t][u] = i32x4{0, 0, 0, 0};

  i32x4 wv[2][NTW], xv[2][MT];
  auto multiply = [&]() {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < NTW; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[s][t], xv[s][u], acc[t][u], 0, 0, 0);
  };
  const int units = a.K / 128;
  for (int u = kp; u < units; u += KP) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k = u * 128 + s * 64 + kq;
#pragma unroll
      for (int t = 0; t < NTW; ++t) wv[s][t] = load_codes(wp[t] + k);
#pragma unroll
      for (int t = 0; t < MT; ++t) xv[s][t] = load_codes(xp[t] + k);
    }
    __builtin_amdgcn_sched_barrier(0);  // every load is issued before the first product
    multiply();
  }
  if (a.K % 128 && units % KP == kp) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k = units * 128 + s * 64 + kq;
#pragma unroll
      for (int t = 0; t < NTW; ++t) wv[s][t] = load_codes_tail(wp[t], k, a.K);
#pragma unroll
      for (int t = 0; t < MT; ++t) xv[s][t] = load_codes_tail(xp[t], k, a.K);
    }
    multiply();
  }

  // Lane l holds column l % 16 (a row of x) and rows 4 (l / 16) .. + 3 (of W) of each result.
  if constexpr (KP == 1) {
#pragma unroll
    for (int t = 0; t < NTW; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        const int m = m0 + u * 16 + r16, n = n0 + t * 16 + lane / 16 * 4;
        if (m < a.M && n < a.N) store_outputs<T>(a, m, n, acc[t][u]);
      }
  } else {
#pragma unroll
    for (int t = 0; t < NTW; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u)
        *reinterpret_cast<i32x4*>(&red[(kp * BM + u * 16 + r16) * RED + t * 16 + lane / 16 * 4]) = acc[t][u];
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
}

template <typename T, int KP, int NTW, int MT>
static int launch_rows8(const LinearArgs& a, hipStream_t st) {
  const int64_t gx = (a.N + 16 * NTW - 1) / (16 * NTW), gy = (a.M + 16 * MT - 1) / (16 * MT);
  if (gy > 65535) return TS_EUNSUPPORTED;
  hipLaunchKernelGGL((int8_rows_kernel<T, KP, NTW, MT>), dim3(gx, gy), dim3(KP * kWave), 0, st, a);
  return launch_status();
}

// ---- many rows: tiles through LDS -------------------------------------------------------------
// Each of the workgroup's GM x GN waves takes 32 MW rows of x and 32 NW rows of W: MW * NW
// accumulators of v_mfma_i32_32x32x32_i8, W the A operand and x the B operand.
//
// Both operands go through a ring of kStages LDS tiles of 64 columns, filled by direct-to-LDS
// loads (four lanes per row of 64 bytes) while older tiles are multiplied. Row r's 16-byte unit c
// sits in slot c ^ swizzle(r), which spreads any 8 or 16 rows' units c over all banks; the lanes
// of a load fetch the units that their slots hold. A step's operands are read from LDS while the
// step before is multiplied; the barrier that hands over the next tile stands between a tile's
// two steps, so the last product of one tile covers the first reads of the next.
//
// kAligned false: rows that do not start at multiples of 16 bytes go through registers instead
// (unaligned vector loads), one tile ahead.
//
// The last K % 64 columns come first, alone, with zeros past the end of the rows.
__device__ __forceinline__ int swizzle(int r) { return ((r >> 1) & 3) ^ ((r >> 3) & 1); }

template <typename T, int MW, int NW, int GM, int GN, int kStages, bool kAligned>
__global__ __launch_bounds__(GM * GN * kWave) void int8_tile_kernel(const LinearArgs a, int tiles_m, int tiles_n) {
  constexpr int kWaves = GM * GN, kThreads = kWaves * kWave;
  constexpr int BM = 32 * MW * GM, BN = 32 * NW * GN;
  constexpr int kStage = (BM + BN) * 64;      // bytes: BN rows of W, then BM rows of x
  constexpr int LPW = (BM + BN) / 16 / kWaves;  // loads per wave and tile, 16 rows each
  constexpr int kRow = 32 * NW * sizeof(T) + 16;  // bytes of a row of the output staging
  constexpr int kLds = kStages * kStage > kWaves * 32 * kRow ? kStages * kStage : kWaves * 32 * kRow;
  static_assert((BM + BN) % (16 * kWaves) == 0 && kLds <= 160 * 1024, "tile shape");
  __shared__ __attribute__((aligned(16))) int8_t lds[kLds];

  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / GN, wn = wave % GN;

  // Workgroups go round-robin over the 8 XCDs: each XCD takes a contiguous run of tiles, in
  // bands of 4 tiles of x, so that the tiles running on it share rows of x and W in its L2.
  int tm, tn;
  {
    const int total = tiles_m * tiles_n, xcd = blockIdx.x % 8, per = total / 8, more = total % 8;
    const int t = xcd * per + min(xcd, more) + blockIdx.x / 8;
    const int band = t / (4 * tiles_n), first = band * 4, high = min(4, tiles_m - first);
    const int in = t - band * 4 * tiles_n;
    tm = first + in % high;
    tn = in / high;
  }
  const int m0 = tm * BM, n0 = tn * BN;
  const int8_t* wg = a.w + static_cast<int64_t>(n0) * a.ws;
  const int8_t* xg = a.x + static_cast<int64_t>(m0) * a.xs;

  // Load j of this wave fills LDS rows 16 (wave * LPW + j) .. + 15, four lanes each; rows past the
  // ends repeat the last one (their sums are not stored).
  auto load_row = [&](int j) { return 16 * (wave * LPW + j) + lane / 4; };
  const int load_unit = (lane % 4) ^ swizzle(lane / 4);
  uint32_t off[LPW];
#pragma unroll
  for (int j = 0; j < LPW; ++j) {
    const int r = load_row(j);
    const int64_t row = r < BN ? min(r, a.N - 1 - n0) * a.ws : min(r - BN, a.M - 1 - m0) * a.xs;
    off[j] = static_cast<uint32_t>(row) + load_unit * 16;
  }
  // LDS bytes of unit 2 s + lane / 32 of row lane % 32 of a 32-row operand tile.
  int unit[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) unit[s] = (lane % 32) * 64 + (((2 * s + lane / 32) ^ swizzle(lane % 32)) * 16);

  i32x16 acc[NW][MW];
#pragma unroll
  for (int t = 0; t < NW; ++t)
#pragma unroll
    for (int u = 0; u < MW; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][u][i] = 0;

  i32x4 wf[2][NW], xf[2][MW];  // operands of the two steps of a tile
  auto read_w = [&](int s, int t, const int8_t* tile) {
    wf[s][t] = *reinterpret_cast<const i32x4*>(tile + (wn * NW + t) * 2048 + unit[s]);
  };
  auto read_x = [&](int s, int u, const int8_t* tile) {
    xf[s][u] = *reinterpret_cast<const i32x4*>(tile + BN * 64 + (wm * MW + u) * 2048 + unit[s]);
  };
  auto read_all = [&](int s, const int8_t* tile) {
#pragma unroll
    for (int t = 0; t < NW; ++t) read_w(s, t, tile);
#pragma unroll
    for (int u = 0; u < MW; ++u) read_x(s, u, tile);
  };
  auto multiply = [&](int s, int p) {  // product p of step s
    acc[p / MW][p % MW] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[s][p / MW], xf[s][p % MW], acc[p / MW][p % MW], 0, 0, 0);
  };
  auto multiply_all = [&](int s) {
#pragma unroll
    for (int p = 0; p < NW * MW; ++p) multiply(s, p);
  };

  const int tiles = a.K / 64;
  if (a.K % 64) {
#pragma unroll
    for (int j = 0; j < LPW; ++j) {
      const int r = load_row(j);
      const int8_t* row = r < BN ? wg + min(r, a.N - 1 - n0) * a.ws : xg + min(r - BN, a.M - 1 - m0) * a.xs;
      *reinterpret_cast<i32x4*>(lds + r * 64 + (lane % 4) * 16) = load_codes_tail(row, tiles * 64 + load_unit * 16, a.K);
    }
    __syncthreads();
    read_all(0, lds);
    read_all(1, lds);
    multiply_all(0);
    multiply_all(1);
    __syncthreads();
  }

  if constexpr (kAligned) {
    auto load = [&](int j, int kt, int8_t* tile) {
      const int row0 = 16 * (wave * LPW + j);
      const int8_t* base = (row0 < BN ? wg : xg) + static_cast<int64_t>(kt) * 64;
      lds_load16_s(base, off[j], (TS_LDS void*)(tile + row0 * 64));
    };
    for (int kt = 0; kt < min(kStages, tiles); ++kt)
#pragma unroll
      for (int j = 0; j < LPW; ++j) load(j, kt, lds + kt * kStage);
    if (tiles >= kStages) ring_barrier<(kStages - 1) * LPW>();
    else ring_barrier<0>();
    if (tiles > 0) read_all(0, lds);
    int at = 0;  // LDS offset of tile kt
    for (int kt = 0; kt < tiles; ++kt) {
      int8_t* tile = lds + at;
      at = at + kStage == kStages * kStage ? 0 : at + kStage;
      int8_t* next = lds + at;
      read_all(1, tile);
      multiply_all(0);
      // Every read of this tile is done and the next one has landed, in every wave.
      if (kt + kStages - 1 < tiles) ring_barrier<(kStages - 2) * LPW>();
      else ring_barrier<0>();
      if (kt + kStages < tiles) {
#pragma unroll
        for (int j = 0; j < LPW; ++j) load(j, kt + kStages, tile);
      }
      if (kt + 1 < tiles) read_all(0, next);
      multiply_all(1);
    }
  } else if (tiles > 0) {
    i32x4 held[LPW];
    auto fetch = [&](int kt) {
#pragma unroll
      for (int j = 0; j < LPW; ++j)
        held[j] = load_codes((16 * (wave * LPW + j) < BN ? wg : xg) + static_cast<int64_t>(kt) * 64 + off[j]);
    };
    fetch(0);
    for (int kt = 0; kt < tiles; ++kt) {
      int8_t* tile = lds + (kt & 1) * kStage;
#pragma unroll
      for (int j = 0; j < LPW; ++j) *reinterpret_cast<i32x4*>(tile + load_row(j) * 64 + (lane % 4) * 16) = held[j];
      if (kt + 1 < tiles) fetch(kt + 1);
      __syncthreads();  // two tiles: the one before this is read by no wave that has passed it
      read_all(0, tile);
      read_all(1, tile);
      multiply_all(0);
      multiply_all(1);
    }
  }
  __syncthreads();  // the ring's last reads, before the outputs take its place

  // Lane l holds column l % 32 (a row of x) and rows 8 j + 4 (l / 32) .. + 3 (of W) of each result.
  // 32 rows of outputs at a time go through the wave's own part of LDS and out in whole vectors.
  int8_t* mine = lds + wave * 32 * kRow;
  constexpr int E = Pack16<T>::N, VPR = 32 * NW / E;  // vectors per row
#pragma unroll
  for (int u = 0; u < MW; ++u) {
    const int mrow = m0 + (wm * MW + u) * 32;
    const float s = a.xscale[min(mrow + lane % 32, a.M - 1)];
#pragma unroll
    for (int t = 0; t < NW; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = t * 32 + j * 8 + lane / 32 * 4;
        const int n = n0 + wn * 32 * NW + c;
        typename Loose<T, 4>::Vec y;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[i] = from_f32<T>(static_cast<float>(acc[t][u][j * 4 + i]) * s * a.wscale[min(n + i, a.N - 1)]);
        *reinterpret_cast<typename Loose<T, 4>::Vec*>(mine + (lane % 32) * kRow + c * sizeof(T)) = y;
      }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int v = 0; v < 32 * VPR / kWave; ++v) {
      const int r = (v * kWave + lane) / VPR, c = (v * kWave + lane) % VPR * E;
      const int m = mrow + r, n = n0 + wn * 32 * NW + c;
      const Pack16<T> y = load16(reinterpret_cast<const T*>(mine + r * kRow) + c);
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

template <typename T, int MW, int NW, int GM, int GN, int kStages, bool kAligned>
static int launch_tiles(const LinearArgs& a, hipStream_t st) {
  constexpr int BM = 32 * MW * GM, BN = 32 * NW * GN;
  const int64_t tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
  if (tm * tn > INT32_MAX) return TS_EUNSUPPORTED;
  hipLaunchKernelGGL((int8_tile_kernel<T, MW, NW, GM, GN, kStages, kAligned>), dim3(static_cast<unsigned>(tm * tn)),
                     dim3(GM * GN * kWave), 0, st, a, static_cast<int>(tm), static_cast<int>(tn));
  return launch_status();
}

template <typename T>
static int launch_linear(const LinearArgs& a, hipStream_t st) {
  if (a.M <= 16) return launch_rows8<T, 8, 1, 1>(a, st);
  if (a.M <= 32) return launch_rows8<T, 8, 1, 2>(a, st);
  // Tiles address their rows by 32-bit offsets: 255 rows of at most 2^23 bytes.
  if (a.M <= 128 || a.xs > 1 << 23 || a.ws > 1 << 23) return launch_rows8<T, 8, 1, 4>(a, st);
  const bool aligned = ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) | a.xs | a.ws) & 15) == 0;
  if (!aligned) return launch_tiles<T, 2, 2, 2, 2, 2, false>(a, st);
  if (a.M >= 1024 && a.N >= 1024) return launch_tiles<T, 4, 4, 2, 2, 4, true>(a, st);
  return launch_tiles<T, 2, 2, 2, 2, 4, true>(a, st);
}

}  // namespace ts

using namespace ts;

extern "C" int ts_int8_linear(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride,
                              const float* w_scale, void* out, int64_t o_stride, int M, int N, int K, int dtype,
                              void* stream) {
  if (M < 0 || M > TS_INT8_MAX_DIM || N < 0 || N > TS_INT8_MAX_DIM || K < 0 || K > TS_INT8_MAX_K || x_stride < 0 || w_stride < 0) return TS_EINVAL;
  if (M > 1 && o_stride < N) return TS_EINVAL;
  if (dtype < TS_F32 || dtype > TS_BF16) return TS_EUNSUPPORTED;
  if (M == 0 || N == 0) return 0;
  if (!out || !x_scale || !w_scale || (K > 0 && (!x || !w))) return TS_EINVAL;
  const LinearArgs a{x, w, x_scale, w_scale, out, M, N, K, x_stride, w_stride, o_stride};
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TS_F32: return launch_linear<float>(a, st);
    case TS_F16: return launch_linear<f16>(a, st);
    default: return launch_linear<bf16>(a, st);
  }
}
