// Rows in 8 bits on gfx950: quantisation with one scale per row (as the rows stand, after the
// residual add and RMSNorm, after SiLU x up), and the lookup of rows of an 8-bit table.
//
// No kernel of the reference corresponds: its model runs in one 16- or 32-bit type
// (src/tinyserve/model.py:137-179). These feed the 8-bit projections of int8_linear.hip.
//
// Quantisation of a row v:
//   a = max |v|;  q = rint(v * (127 / a)) in -127 .. 127;  scale = a / 127
// so that q * scale is within half a step, a / 254, of v. Two rows have no such a: one whose a
// is below 2^-100 (127 / a could overflow) is all zeros with scale 0, and one that holds a NaN
// or an infinity gets zeros and a NaN scale, so that whatever is computed from it is NaN, as it
// would be in floating point.
//
// RMSNorm: the row is x * r * w with r = 1 / sqrt(mean x^2 + eps). r is common to the row, so it
// cancels in q: v = x * w is quantised and r goes into the scale, (a / 127) * r. Nothing is
// rounded between the norm and the 8 bits, and the codes do not wait for the sum of squares.
// A row whose sum of squares leaves float32 is a NaN row. With the residual add, x = (T)(x + y)
// is written back in place first, rounded to T as the rest of the framework holds it.
//
// SiLU x up: v = g / (1 + exp(-g)) * u in float32, not rounded to T in between.
//
// All are bound by HBM: each input is read once into registers (both maxima and sums are taken
// there), each output written once.
#include "common.h"

namespace ts {

enum Int8Form { kPlain = 0, kNorm = 1, kAddNorm = 2, kSilu = 3 };

constexpr uint32_t kInfBits = 0x7f800000u;
constexpr uint32_t kTinyBits = 0x0d800000u;  // 2^-100

// Elements i .. i + E - 1 of a row of N >= E elements, zeros past its end. The load itself is
// moved back to the row's last whole vector and its elements shifted down: no branch, so the
// loads of a row's chunks are all in flight together.
template <typename T>
__device__ __forceinline__ Pack16<T> load_chunk(const T* row, int i, int N) {
  constexpr int E = Pack16<T>::N;
  const int at = min(i, N - E);
  Pack16<T> r = load16_loose(row + at);
  if (N % E) {
    const int bits = (i - at) * static_cast<int>(sizeof(T)) * 8;
    unsigned __int128 v = static_cast<unsigned __int128>(r.raw[3]) << 96 | static_cast<unsigned __int128>(r.raw[2]) << 64 |
                          static_cast<unsigned __int128>(r.raw[1]) << 32 | r.raw[0];
    v = bits < 128 ? v >> (bits & 127) : 0;
    r.raw = u32x4{static_cast<uint32_t>(v), static_cast<uint32_t>(v >> 32), static_cast<uint32_t>(v >> 64),
                  static_cast<uint32_t>(v >> 96)};
  } else if (i >= N) {
    r.raw = u32x4{0, 0, 0, 0};
  }
  return r;
}

// g / (1 + exp(-g)), within about 2^-21: exp(-g) as 2^t of t = -g log2(e), with the rounding of t put
// right to first order (t alone would be off by |g| 2^-24), and the quotient by the reciprocal.
// The exponent is taken from g cut to where 2^t is finite: below -88.7 the result, under 1e-36 in
// magnitude, is -88.7's; the last term makes an infinity or a NaN in g a NaN.
// The hardware's exp2 and reciprocal are within one unit in the last place; expf and a correctly
// rounded quotient made the kernel wait for its arithmetic (8192 x 8192 bf16 82 us, then 68).
__device__ __forceinline__ float silu(float g) {
  constexpr float kLog2eLow = 1.92596299e-8f;  // log2(e) - (float)log2(e)
  constexpr float kLn2 = 0.693147180559945f;
  const float cut = fminf(fmaxf(g, -88.7f), 88.7f);
  const float t = -cut * kLog2e;
  const float off = fmaf(-cut, kLog2e, -t) - cut * kLog2eLow;
  const float e = fast_exp2(t);
  return fmaf(g, 0.0f, fmaxf(g, -88.7f) * __builtin_amdgcn_rcpf(1.0f + fmaf(e, off * kLn2, e)));
}

// |v| as bits: ordered as the magnitudes are, infinities above every finite value and NaN above
// those, so one unsigned maximum carries all three.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <int OFF>
__device__ __forceinline__ uint32_t xor_lane_u(uint32_t x) {
  return __float_as_uint(xor_lane<OFF>(__uint_as_float(x)));
}

// The largest x of each group of N consecutive lanes.
template <int N>
__device__ __forceinline__ uint32_t group_umax(uint32_t x) {
  x = max(x, xor_lane_u<1>(x));
  x = max(x, xor_lane_u<2>(x));
  x = max(x, xor_lane_u<4>(x));
  x = max(x, xor_lane_u<8>(x));
  if constexpr (N >= 32) x = max(x, xor_lane_u<16>(x));
  if constexpr (N >= 64) x = max(x, xor_lane_u<32>(x));
  return x;
}

// A row's factor for its codes (0: all codes are zero) and its scale, from the largest
// magnitude, and for a norm the sum of squares.
struct RowScale {
  float inv, scale;
};

template <int FORM>
__device__ __forceinline__ RowScale row_scale(uint32_t top, float ss, int N, float eps) {
  RowScale r;
  const float a = __uint_as_float(top);
  const bool zero = top < kTinyBits;
  r.inv = zero ? 0.0f : 127.0f / a;
  r.scale = zero ? 0.0f : a / 127.0f;
  if constexpr (FORM == kNorm || FORM == kAddNorm) {
    if (!zero) r.scale *= 1.0f / sqrtf(ss / static_cast<float>(N) + eps);
  }
  // top >= inf: an infinity or a NaN in the row; a scale that is not finite: a sum of squares
  // past float32, or eps 0 under one that underflows.
  if (top >= kInfBits || magnitude(r.scale) >= kInfBits || (FORM != kPlain && FORM != kSilu && magnitude(ss) >= kInfBits)) {
    r.inv = 0.0f;
    r.scale = __uint_as_float(0x7fc00000u);
  }
  return r;
}

// The codes of four values, a byte each. Adding 1.5 * 2^23 leaves rint(v * inv), at most 127, in
// the sum's low bits. A row without a scale has inv 0, whatever its values: all codes zero.
__device__ __forceinline__ uint32_t codes4(const float* v, float inv) {
  constexpr float kMagic = 12582912.0f;
  uint32_t b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(fmaf(v[e], inv, kMagic));
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);  // low bytes of b[0], b[1]
  const uint32_t hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);  // of b[2], b[3], above them
  return inv == 0.0f ? 0u : lo | hi;
}

struct QuantArgs {
  const void* x;  // [T, N] (kSilu: [T, 2N], gate | up)
  void* xo;       // kAddNorm: x again, written
  const void* y;
  const void* w;
  int8_t* q;
  float* scale;
  int rows, N;
  int64_t xs, ys, qs;
  float eps;
  int threads;  // of a workgroup (blockDim would be an implicit argument, which costs host time)
};

// CPT chunks of E elements per thread. LPR lanes of a wave on one row, a workgroup of 256 threads on
// 256 / LPR rows; or LPR 0: the whole workgroup, of any number of waves up to 16, on one row.
template <typename T, int FORM, int LPR, int CPT>
__global__ __launch_bounds__(LPR ? 256 : 1024) void quantize_rows_kernel(const QuantArgs a) {
  constexpr int E = Pack16<T>::N;
  const int wave = threadIdx.x / kWave, TPR = LPR ? LPR : a.threads;
  const int64_t row = LPR ? static_cast<int64_t>(blockIdx.x) * (256 / (LPR ? LPR : 1)) + threadIdx.x / (LPR ? LPR : 1) : blockIdx.x;
  const int t = LPR ? threadIdx.x % (LPR ? LPR : 1) : threadIdx.x;
  if (LPR && row >= a.rows) return;
  const int N = a.N;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  const T* y = static_cast<const T*>(a.y) + row * a.ys;  // kAddNorm
  const T* w = static_cast<const T*>(a.w);

  Pack16<T> xv[CPT], sv[CPT], wv[CPT];
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * TPR + t) * E;
    xv[c] = load_chunk(x, i, N);
    if constexpr (FORM == kAddNorm) sv[c] = load_chunk(y, i, N);
    if constexpr (FORM == kSilu) sv[c] = load_chunk(x + N, i, N);
    if constexpr (FORM == kNorm || FORM == kAddNorm) wv[c] = load_chunk(w, i, N);
  }

  float v[CPT][E];
  uint32_t top = 0;
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    if constexpr (FORM == kAddNorm) {
      const int i = (c * TPR + t) * E;
#pragma unroll
      for (int e = 0; e < E; ++e) xv[c].v[e] = round_f32<T>(to_f32(xv[c].v[e]) + to_f32(sv[c].v[e]));
      T* xo = static_cast<T*>(a.xo) + row * a.xs + i;
      if (i + E <= N) {
        store16_loose(xo, xv[c]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (i + e < N) xo[e] = xv[c].v[e];
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float f = to_f32(xv[c].v[e]);
      if constexpr (FORM == kSilu) f = silu(f) * to_f32(sv[c].v[e]);
      if constexpr (FORM == kNorm || FORM == kAddNorm) {
        ss = fmaf(f, f, ss);
        f *= to_f32(wv[c].v[e]);
      }
      v[c][e] = f;
      top = max(top, magnitude(f));
    }
  }

  constexpr int kLanes = LPR ? LPR : kWave;
  top = group_umax<kLanes>(top);
  if constexpr (FORM == kNorm || FORM == kAddNorm) ss = group_sum<kLanes>(ss);
  if constexpr (LPR == 0) {
    __shared__ uint32_t tops[16];
    __shared__ float sums[16];
    if (threadIdx.x % kWave == 0) {
      tops[wave] = top;
      sums[wave] = ss;
    }
    __syncthreads();
    top = 0;
    ss = 0.f;
    for (int k = 0; k < TPR / kWave; ++k) {  // in the waves' order in every thread
      top = max(top, tops[k]);
      ss += sums[k];
    }
  }
  const RowScale r = row_scale<FORM>(top, ss, N, a.eps);
  if (t == 0) a.scale[row] = r.scale;

  int8_t* q = a.q + row * a.qs;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * TPR + t) * E;
    if (i >= N) continue;
    uint32_t word[E / 4];
#pragma unroll
    for (int k = 0; k < E / 4; ++k) word[k] = codes4(&v[c][4 * k], r.inv);
    // Whole words: the row's padding, up to its stride, takes zeros.
    if constexpr (E == 8) *reinterpret_cast<uint2*>(q + i) = uint2{word[0], word[1]};
    else *reinterpret_cast<uint32_t*>(q + i) = word[0];
  }
}

// Any row length, one element at a time: rows shorter than one 16-byte vector, and rows longer
// than a workgroup's registers hold, which are read twice. A workgroup per row.
template <typename T, int FORM>
__global__ __launch_bounds__(1024) void quantize_rows_any_kernel(const QuantArgs a) {
  const int64_t row = blockIdx.x;
  const int N = a.N, wave = threadIdx.x / kWave, threads = a.threads;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  T* xo = static_cast<T*>(a.xo) + row * a.xs;
  const T* y = static_cast<const T*>(a.y) + row * a.ys;
  const T* w = static_cast<const T*>(a.w);
  // kAddNorm: the second pass reads the sums that this same thread wrote in the first.
  auto value = [&](int i, float f) {
    if constexpr (FORM == kSilu) return silu(f) * to_f32(x[N + i]);
    else if constexpr (FORM == kPlain) return f;
    else return f * to_f32(w[i]);
  };
  uint32_t top = 0;
  float ss = 0.f;
  for (int i = threadIdx.x; i < N; i += threads) {
    float f;
    if constexpr (FORM == kAddNorm) {
      const T s = round_f32<T>(to_f32(xo[i]) + to_f32(y[i]));
      xo[i] = s;
      f = to_f32(s);
    } else {
      f = to_f32(x[i]);
    }
    if constexpr (FORM == kNorm || FORM == kAddNorm) ss = fmaf(f, f, ss);
    top = max(top, magnitude(value(i, f)));
  }
  top = group_umax<kWave>(top);
  ss = group_sum<kWave>(ss);
  __shared__ uint32_t tops[16];
  __shared__ float sums[16];
  if (threadIdx.x % kWave == 0) {
    tops[wave] = top;
    sums[wave] = ss;
  }
  __syncthreads();
  top = 0;
  ss = 0.f;
  for (int k = 0; k < threads / kWave; ++k) {
    top = max(top, tops[k]);
    ss += sums[k];
  }
  const RowScale r = row_scale<FORM>(top, ss, N, a.eps);
  if (threadIdx.x == 0) a.scale[row] = r.scale;
  int8_t* q = a.q + row * a.qs;
  for (int i = threadIdx.x; i < N; i += threads) {
    float f;
    if constexpr (FORM == kAddNorm) f = to_f32(xo[i]);
    else f = to_f32(x[i]);
    const float v[4] = {value(i, f), 0.f, 0.f, 0.f};
    q[i] = static_cast<int8_t>(codes4(v, r.inv) & 0xffu);
  }
}

template <typename T, int FORM>
static int launch_quantize(QuantArgs a, hipStream_t st) {
  constexpr int E = Pack16<T>::N;
  const int chunks = (a.N + E - 1) / E;
  // Wide rows: a workgroup of as many threads as there are chunks, up to 1024, then two to four
  // chunks a thread. Where one array is read and there is much of it, a thread takes two from 256
  // chunks on: more loads in flight then pay more than more waves. Measured (us, one and two
  // chunks): quantising 8192 x 8192 bf16 37.0 and 33.3, 32768 x 2048 39.3 and 32.9, 1024 x 2048 3.67
  // and 3.72, 32 x 2048 3.18 and 3.32; norm 51.6 and 40.2, 44.5 and 40.4, 4.1 and 4.2, 3.5 and 3.8
  // (2751 x 2048 7.3 and 7.7, 1024 x 8192 9.9 and 9.4); residual + norm 83.1 and 91.5, 81.3 and 89.5,
  // 5.8 and 6.3; SiLU 62.1 and 64.0, 59.6 and 62.6, 4.7 and 4.8. From 1025 to 1536 chunks three a
  // thread: four workgroups of up to 512 threads fill a compute unit, two of 704 do not (4096 x 11008,
  // two and three: quantising 27.9 and 24.6, SiLU 48.3 and 45.6). Narrow rows: 8192 x 512 in one wave
  // each, four to a workgroup, 5.1 and 8.6 (quantising; residual + norm), a workgroup each 5.4 and
  // 8.1; 32768 x 64 in 16 lanes each 4.0 and 6.9, in a wave each 10.5 and 15.1.
#define TS_NARROW(L)                                                                                                 \
  hipLaunchKernelGGL((quantize_rows_kernel<T, FORM, L, 1>), dim3((a.rows + 256 / (L) - 1) / (256 / (L))), dim3(256), 0, st, a)
#define TS_WIDE(C)                                                                                           \
  do {                                                                                                       \
    a.threads = ((chunks + (C) - 1) / (C) + kWave - 1) / kWave * kWave;                                      \
    hipLaunchKernelGGL((quantize_rows_kernel<T, FORM, 0, C>), dim3(a.rows), dim3(a.threads), 0, st, a);      \
  } while (0)
  constexpr int kMost = 1024;  // threads of a workgroup
  const int64_t much = FORM == kPlain ? 1 << 18 : FORM == kNorm ? 1 << 20 : INT64_MAX;  // chunks in all
  const bool two = chunks > kMost || (chunks >= 256 && static_cast<int64_t>(a.rows) * chunks >= much);
  if (a.N < E || chunks > 4 * kMost) {
    a.threads = a.N < E ? kWave : kMost;
    hipLaunchKernelGGL((quantize_rows_any_kernel<T, FORM>), dim3(a.rows), dim3(a.threads), 0, st, a);
  } else if (chunks <= 16) TS_NARROW(16);
  else if (chunks <= 32) TS_NARROW(32);
  else if (chunks <= 64) TS_NARROW(64);
  else if (!two) TS_WIDE(1);
  else if (chunks <= kMost || (chunks > kMost * 3 / 2 && chunks <= 2 * kMost)) TS_WIDE(2);
  else if (chunks <= 3 * kMost) TS_WIDE(3);
  else TS_WIDE(4);
#undef TS_NARROW
#undef TS_WIDE
  return launch_status();
}

// Rows per launch: a launch has fewer than 2^32 threads, up to 1024 of them per row.
constexpr int kRowsPerLaunch = 1 << 21;

template <typename T>
static int launch_form(QuantArgs a, int form, hipStream_t st) {
  for (int left = a.rows; left > 0; left -= kRowsPerLaunch) {
    a.rows = left < kRowsPerLaunch ? left : kRowsPerLaunch;
    const int rc = form == kPlain ? launch_quantize<T, kPlain>(a, st) : form == kNorm ? launch_quantize<T, kNorm>(a, st)
                   : form == kAddNorm ? launch_quantize<T, kAddNorm>(a, st) : launch_quantize<T, kSilu>(a, st);
    if (rc) return rc;
    a.x = static_cast<const T*>(a.x) + a.rows * a.xs;
    a.xo = static_cast<T*>(a.xo) + a.rows * a.xs;
    a.y = static_cast<const T*>(a.y) + a.rows * a.ys;
    a.q += a.rows * a.qs;
    a.scale += a.rows;
  }
  return 0;
}

// ---- rows of an 8-bit table -----------------------------------------------------------------
// out[t] = (T)(q[ids[t]] * scale[ids[t]]): one thread per 16 codes. Bound by HBM (and, for few
// ids, by the chain id -> row). An id outside the table gives a row of NaN.
constexpr int kMostBlocks = 1 << 20;  // of a launch; one of fewer has a thread for every 16 bytes

struct TableArgs {
  const int8_t* q;
  const float* scale;
  const int64_t* ids;  // null: row t itself
  void* out;
  int64_t qs, os, table;  // table: its rows
  int rows, N, per_row;   // per_row: threads per row
};

template <typename T>
__global__ __launch_bounds__(256) void int8_embedding_kernel(const TableArgs a) {
  const int N = a.N;
  const int64_t total = static_cast<int64_t>(a.rows) * a.per_row;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; u < total; u += kMostBlocks * 256ll) {
    const int64_t t = u / a.per_row;
    const int i = static_cast<int>(u - t * a.per_row) * 16;
    const int64_t id = a.ids ? a.ids[t] : t;
    const bool in = id >= 0 && id < a.table;
    const float s = in ? a.scale[id] : __uint_as_float(0x7fc00000u);
    const int8_t* p = a.q + (in ? id : 0) * a.qs + i;
    T* o = static_cast<T*>(a.out) + t * a.os + i;
    if (i + 16 <= N) {
      union {
        u32x4 raw;
        int8_t b[16];
      } c;
      c.raw = load16_loose(p).raw;
      constexpr int E = Pack16<T>::N;
#pragma unroll
      for (int k = 0; k < 16 / E; ++k) {
        Pack16<T> y;
#pragma unroll
        for (int e = 0; e < E; ++e) y.v[e] = round_f32<T>(static_cast<float>(c.b[k * E + e]) * s);
        store16_loose(o + k * E, y);
      }
    } else {
      for (int e = 0; e < N - i; ++e) o[e] = round_f32<T>(static_cast<float>(p[e]) * s);
    }
  }
}

// Rows of one matrix, or of two, copied to a stride of whole 16 bytes, zeros past their ends. One
// thread per 16 bytes.
struct PadArgs {
  const int8_t *a, *b;
  int8_t *a_out, *b_out;
  int64_t as, bs, os;
  int a_rows, b_rows, N, per_row;
};

__global__ __launch_bounds__(256) void int8_pad_rows_kernel(const PadArgs p) {
  const int64_t total = (static_cast<int64_t>(p.a_rows) + p.b_rows) * p.per_row;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; u < total; u += kMostBlocks * 256ll) {
    const int64_t row = u / p.per_row;
    const int i = static_cast<int>(u - row * p.per_row) * 16;
    const bool first = row < p.a_rows;
    const int64_t t = first ? row : row - p.a_rows;
    const int8_t* q = (first ? p.a + t * p.as : p.b + t * p.bs) + i;
    union {
      u32x4 raw;
      int8_t b[16];
    } c;
    c.raw = u32x4{0, 0, 0, 0};
    if (i + 16 <= p.N) {
      c.raw = load16_loose(q).raw;
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (i + e < p.N) c.b[e] = q[e];
    }
    *reinterpret_cast<u32x4*>((first ? p.a_out : p.b_out) + t * p.os + i) = c.raw;
  }
}

template <typename T>
static int launch_embedding(TableArgs a, hipStream_t st) {
  a.per_row = (a.N + 15) / 16;
  const int64_t blocks = (static_cast<int64_t>(a.rows) * a.per_row + 255) / 256;
  hipLaunchKernelGGL(int8_embedding_kernel<T>, dim3(static_cast<unsigned>(blocks < kMostBlocks ? blocks : kMostBlocks)), dim3(256),
                     0, st, a);
  return launch_status();
}

}  // namespace ts

using namespace ts;

extern "C" int ts_int8_quantize_rows(void* x, const void* y, const void* w, int8_t* q, float* scale, int T, int N,
                                     int64_t x_stride, int64_t y_stride, int64_t q_stride, float eps, int form, int dtype,
                                     void* stream) {
  if (T < 0 || T > TS_INT8_MAX_DIM || N <= 0 || N > TS_INT8_MAX_DIM || form < kPlain || form > kSilu) return TS_EINVAL;
  const int64_t padded = (static_cast<int64_t>(N) + 15) / 16 * 16;
  if (q_stride < padded || q_stride % 16 || reinterpret_cast<uintptr_t>(q) % 16) return TS_EINVAL;
  if (dtype < TS_F32 || dtype > TS_BF16) return TS_EUNSUPPORTED;
  if (T == 0) return 0;
  if (!x || !q || !scale || x_stride < 0) return TS_EINVAL;
  if ((form == kNorm || form == kAddNorm) && !w) return TS_EINVAL;
  if (form == kAddNorm) {
    // x is written: its rows may not overlap each other, nor y's, unless y is x itself or lies
    // beside it in the same rows.
    if (!y || y_stride < 0 || (T > 1 && x_stride < N)) return TS_EINVAL;
    const int64_t es = elem_size(dtype);
    const int64_t x0 = reinterpret_cast<int64_t>(x), y0 = reinterpret_cast<int64_t>(y);
    const int64_t x1 = x0 + ((T - 1) * x_stride + N) * es, y1 = y0 + ((T - 1) * y_stride + N) * es;
    if (x0 < y1 && y0 < x1 && !(x0 == y0 && (x_stride == y_stride || T == 1))) {
      const int64_t pitch = x_stride * es, d = T > 1 && x_stride == y_stride ? ((y0 - x0) % pitch + pitch) % pitch : 0;
      if (T == 1 || x_stride != y_stride || d < N * es || d > pitch - N * es) return TS_EINVAL;
    }
  }
  const QuantArgs a{x, x, y, w, q, scale, T, N, x_stride, y_stride, q_stride, eps, 0};
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TS_F32: return launch_form<float>(a, form, st);
    case TS_F16: return launch_form<f16>(a, form, st);
    default: return launch_form<bf16>(a, form, st);
  }
}

extern "C" int ts_int8_embedding(const int8_t* table, int64_t t_stride, const float* scale, int64_t table_rows,
                                 const int64_t* ids, void* out, int64_t o_stride, int T, int N, int dtype, void* stream) {
  if (T < 0 || T > TS_INT8_MAX_DIM || N < 0 || N > TS_INT8_MAX_DIM || t_stride < 0 || table_rows < 0 || (T > 1 && o_stride < N)) return TS_EINVAL;
  if (dtype < TS_F32 || dtype > TS_BF16) return TS_EUNSUPPORTED;
  if (T == 0 || N == 0) return 0;
  // The rows of an empty table do not exist: there is nothing to read for any id.
  if (!table || !scale || !out || table_rows == 0 || (!ids && T > table_rows)) return TS_EINVAL;
  const TableArgs a{table, scale, ids, out, t_stride, o_stride, table_rows, T, N, 0};
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TS_F32: return launch_embedding<float>(a, st);
    case TS_F16: return launch_embedding<f16>(a, st);
    default: return launch_embedding<bf16>(a, st);
  }
}

extern "C" int ts_int8_pad_rows(const int8_t* a, int64_t a_stride, int8_t* a_out, int a_rows, const int8_t* b,
                                int64_t b_stride, int8_t* b_out, int b_rows, int64_t o_stride, int N, void* stream) {
  const int64_t padded = (static_cast<int64_t>(N) + 15) / 16 * 16;
  if (a_rows < 0 || a_rows > TS_INT8_MAX_DIM || b_rows < 0 || b_rows > TS_INT8_MAX_DIM || N < 0 || N > TS_INT8_MAX_DIM)
    return TS_EINVAL;
  if (a_stride < 0 || b_stride < 0 || o_stride < padded || o_stride % 16) return TS_EINVAL;
  if ((reinterpret_cast<uintptr_t>(a_out) | reinterpret_cast<uintptr_t>(b_out)) % 16) return TS_EINVAL;
  if ((a_rows == 0 && b_rows == 0) || N == 0) return 0;
  if ((a_rows > 0 && (!a || !a_out)) || (b_rows > 0 && (!b || !b_out))) return TS_EINVAL;
  const PadArgs p{a, b, a_out, b_out, a_stride, b_stride, o_stride, a_rows, b_rows, N, static_cast<int>(padded / 16)};
  const int64_t blocks = ((static_cast<int64_t>(a_rows) + b_rows) * p.per_row + 255) / 256;
  hipLaunchKernelGGL(int8_pad_rows_kernel, dim3(static_cast<unsigned>(blocks < kMostBlocks ? blocks : kMostBlocks)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), p);
  return launch_status();
}
