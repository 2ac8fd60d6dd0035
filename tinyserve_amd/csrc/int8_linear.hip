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
typedef u32x4 u32x4_loose __attribute__((aligned(1), may_alias));

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

template <typename T>
static int launch_linear(const LinearArgs& a, hipStream_t st) {
  if (a.M <= 16) return launch_rows8<T, 8, 1, 1>(a, st);
  if (a.M <= 32) return launch_rows8<T, 8, 1, 2>(a, st);
  return launch_rows8<T, 8, 1, 4>(a, st);
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
