// Microscaled 4-bit floating point (OCP MX, format MXFP4) on gfx950: quantisation, the way back, and the product of two
// such matrices on the scaled matrix instruction.
//
// A (rows, K) matrix is cut into blocks of 32 along K.  A block holds 32 E2M1 elements (sign, 2 exponent bits, 1 mantissa
// bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one E8M0 scale 2^se: se = floor(log2(largest magnitude)) - 2, not below -127;
// elements are x / 2^se rounded half to even and held to 6.  A block with a NaN or an infinity gets the scale byte 255 (NaN):
// everything made from it is NaN.
//
// Layout: the one the matrix instruction reads, for both operands.  v_mfma_scale_f32_16x16x128_f8f6f4 takes of each
// operand 16 rows x 128 k; lane l holds row l % 16, k block l / 16: 32 consecutive elements, 16 bytes, exactly one block,
// and in one byte that block's scale.  Rows are padded to 64, K to 128 (zero elements, scale byte 0), and stored as
//   codes  [rows/64][K/128][4 fragments][64 lanes][16 bytes]     (element j of a block in nibble j, low nibble first)
//   scales [rows/64][K/128][64 lanes][4 bytes]                   (byte f: the lane's block of fragment f)
// so that a fragment is 1 KB and the scales of four are 256 bytes, read without a gap.  Row r of fragment f is row
// 32 (f / 2) + 8 (r / 4) + 4 (f % 2) + r % 4 of its 64: with the weights as the instruction's first operand, whose rows come
// out four to a lane, the accumulators of two fragments are then 8 consecutive output columns of one row.
#include "epilogue.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int frag_row(int f, int r) { return ((f >> 1) << 5) + ((r >> 2) << 3) + ((f & 1) << 2) + (r & 3); }

// 32 values -> 32 codes and the scale byte.  Everything is exact but the rounding itself (the scale is a power of two), and
// the conversion instructions do that rounding: half to even, held to 6, for every scale byte from 0 on.
__device__ __forceinline__ uint32_t scale_of(uint32_t ex) { return ex == 255u ? 255u : (ex > 2u ? ex - 2u : 0u); }

template <typename T> struct RawBlock {      // a lane's 32 elements as loaded
  static constexpr int N = 32 * sizeof(T) / 16;
  u32x4 v[N];
};

__device__ __forceinline__ uint32_t mx_block(const RawBlock<bf16>& x, u32x4& codes) {
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  us2 m = {0, 0};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, x.v[j / 4][j % 4] & 0x7fff7fffu));
  const uint32_t big = m[0] > m[1] ? m[0] : m[1];
  const uint32_t scale = scale_of(big >> 7);
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  const float s = __builtin_bit_cast(float, scale << 23);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(b2, (uint32_t)x.v[q][0]), s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(b2, (uint32_t)x.v[q][1]), s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(b2, (uint32_t)x.v[q][2]), s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(b2, (uint32_t)x.v[q][3]), s, 3);
    codes[q] = scale == 255u ? 0u : w;
  }
#endif
  return scale;
}

__device__ __forceinline__ uint32_t mx_block(const RawBlock<float>& x, u32x4& codes) {
  uint32_t big = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint32_t b = x.v[i / 4][i % 4] & 0x7fffffffu;
    big = b > big ? b : big;
  }
  const uint32_t scale = scale_of(big >> 23);
#if defined(__HIP_DEVICE_COMPILE__)
  const float s = __builtin_bit_cast(float, scale << 23);
  auto f = [&](int i) __attribute__((always_inline)) { return __builtin_bit_cast(float, (uint32_t)x.v[i / 4][i % 4]); };
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(8 * q), f(8 * q + 1), s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(8 * q + 2), f(8 * q + 3), s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(8 * q + 4), f(8 * q + 5), s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(8 * q + 6), f(8 * q + 7), s, 3);
    codes[q] = scale == 255u ? 0u : w;
  }
#endif
  return scale;
}

// 32 consecutive elements of a row, zeros past its end (and for a row that is not there)
template <typename T, bool VEC>
__device__ __forceinline__ void load_block(const T* row, int k0, int K, bool there, RawBlock<T>& x) {
  constexpr int E = Vec16<T>::N;
#pragma unroll
  for (int j = 0; j < RawBlock<T>::N; ++j) {
    Vec16<T> r = zero16<T>();
    if (VEC) {
      if (there && k0 + j * E < K) r = load16(row + k0 + j * E);
    } else if (there) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (k0 + j * E + e < K) r.v[e] = row[k0 + j * E + e];
    }
    x.v[j] = __builtin_bit_cast(u32x4, r);
  }
}

// One wave: 64 rows x 128 k, each lane whole blocks.  Bound by the read of x.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, int64_t ldx, uint32_t rows, int K,
                                                          uint32_t kt, uint64_t units, u32x4* __restrict__ codes,
                                                          uint32_t* __restrict__ scales) {
  const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int lane = threadIdx.x & 63;
  const uint32_t g = (uint32_t)(unit / kt);
  const int k0 = (int)(unit % kt) * 128 + (lane >> 4) * 32;
  uint32_t sc = 0;
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    const uint32_t row = g * 64 + frag_row(f, lane & 15);
    RawBlock<T> r;
    load_block<T, VEC>(x + (int64_t)(row < rows ? row : 0) * ldx, k0, K, row < rows, r);
    u32x4 c;
    sc |= mx_block(r, c) << (8 * f);
    codes[(unit * 4 + f) * 64 + lane] = c;
  }
  scales[unit * 64 + lane] = sc;
}

// value of a code times 2^(scale byte - 127); the bf16 result is exact, the fp32 one too
__device__ __forceinline__ float mx_value(uint32_t code, uint32_t scale) {
  const uint32_t m = code & 7u;
  // 2^(scale - 127) as two factors that are both normal numbers
  const float s0 = __builtin_bit_cast(float, ((scale >> 1) + 64u) << 23);              // 2^(floor(scale / 2) - 63)
  const float s1 = __builtin_bit_cast(float, (scale - (scale >> 1) + 63u) << 23);      // 2^(ceil(scale / 2) - 64)
  float v = m < 2u ? 0.5f * (float)m : __builtin_bit_cast(float, (m + 252u) << 22);
  v = v * s0 * s1;
  v = scale == 255u ? __builtin_nanf("") : v;
  return (code & 8u) ? -v : v;
}

template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const u32x4* __restrict__ codes, const uint32_t* __restrict__ scales,
                                                            uint32_t rows, int K, uint32_t kt, uint64_t units,
                                                            T* __restrict__ out, int64_t ldo, int vec) {
  const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  constexpr int E = Vec16<T>::N;
  const int lane = threadIdx.x & 63;
  const uint32_t g = (uint32_t)(unit / kt);
  const int k0 = (int)(unit % kt) * 128 + (lane >> 4) * 32;
  const uint32_t sc = scales[unit * 64 + lane];
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    const uint32_t row = g * 64 + frag_row(f, lane & 15);
    if (row >= rows) continue;
    const u32x4 c = codes[(unit * 4 + f) * 64 + lane];
    T* o = out + (int64_t)row * ldo + k0;
#pragma unroll
    for (int j = 0; j < 32 / E; ++j) {
      Vec16<T> v;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = j * E + e;
        v.v[e] = from_f32<T>(mx_value(c[i / 8] >> (4 * (i % 8)), (sc >> (8 * f)) & 255u));
      }
      if (vec) {
        if (k0 + j * E < K) store16(o + j * E, v);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (k0 + j * E + e < K) o[j * E + e] = v.v[e];
      }
    }
  }
}

struct MxArgs {
  const u32x4 *xc, *wc;
  const uint32_t *xs, *ws;
  const void* x;          // the activations themselves, where a kernel quantises them on the way
  void* out;
  const float* bias;
  const void* resid;
  int64_t ldx, ldo, ldr;
  uint32_t M, N, kt;      // rows, output columns, steps of 128 k
  int K, act, vec;
  uint32_t ngroups, per;  // mx_rows_kernel: groups of 64 columns, and how many of them a workgroup takes
};

// fragments FW of the weights and FX of the activations (their scales: byte FW / FX of the lane's word)
template <int FW, int FX>
__device__ __forceinline__ f32x4 mma4(const u32x4& w, const u32x4& x, f32x4 c, uint32_t sw, uint32_t sx) {
#if defined(__HIP_DEVICE_COMPILE__)
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, FW, (int)sw, FX, (int)sx);
#else
  return c;
#endif
}

// GELU for bfloat16 results: v Phi(v) = (v or 0, whichever is larger) - |v| Phi(-|v|), and log2 Phi(-a) is so smooth that
// a polynomial of degree 6 in a suffices: the result is off by less than 2.4e-7 of v, and by less than 1.6e-4 of itself
// far into the tail (least squares in the Chebyshev basis on [0, 5.5], reweighted towards the largest error against those
// two; Phi(-5.5) = 2e-8 stands for what lies beyond).  Seven multiply-adds and one exponential instead of the erf form's
// reciprocal, exponential and more.  NaN and +infinity pass through the first term.
__device__ __forceinline__ float gelu_bf16(float v) {
  const float a = __builtin_amdgcn_fmed3f(fabsf(v), 0.f, 5.5f);
  float p = 3.13768651e-05f;
  p = fmaf(p, a, -0.000742790464f);
  p = fmaf(p, a, 0.00795761682f);
  p = fmaf(p, a, -0.0531759113f);
  p = fmaf(p, a, -0.458968848f);
  p = fmaf(p, a, -1.15113544f);
  p = fmaf(p, a, -0.999999404f);
  return fmaf(-a, __builtin_amdgcn_exp2f(p), v < 0.f ? 0.f : v);
}

template <typename T, int ACT> __device__ __forceinline__ float mx_act(float v) {
  if (ACT == 1) return v < 0.f ? 0.f : v;
  if (ACT == 2) return sizeof(T) == 2 ? gelu_bf16(v) : 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f));
  return v;
}

// The columns of a lane's accumulators: pair j of fragments (2j, 2j + 1) holds columns n0 + 32 j + 8 (lane / 16) + 0...7
// of one row.  Accumulators begin as the bias.
__device__ __forceinline__ f32x4 bias4(const MxArgs& a, uint32_t n0, int f, int lane) {
  const uint32_t n = n0 + ((f >> 1) << 5) + ((lane >> 4) << 3) + ((f & 1) << 2);
  f32x4 b = {0.f, 0.f, 0.f, 0.f};
  if (a.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) b[i] = a.bias[n + i];
  }
  return b;
}

// activation, residual and store of 8 consecutive columns of row m (lo, hi: accumulators of two fragments)
template <typename T, int ACT, bool VEC>
__device__ __forceinline__ void store8(const MxArgs& a, uint32_t m, uint32_t n, const f32x4& lo, const f32x4& hi) {
  constexpr int E = Vec16<T>::N;
  if (m >= a.M) return;
  T* o = reinterpret_cast<T*>(a.out) + (int64_t)m * a.ldo + n;
#pragma unroll
  for (int j = 0; j < 8 / E; ++j) {
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = mx_act<T, ACT>(j * E + e < 4 ? lo[(j * E + e) % 4] : hi[(j * E + e) % 4]);
    if (a.resid != nullptr) {
      const T* rs = reinterpret_cast<const T*>(a.resid) + (int64_t)m * a.ldr + n + j * E;
      if (VEC) {
        if (n + j * E < a.N) {
          const Vec16<T> r = load16(rs);
#pragma unroll
          for (int e = 0; e < E; ++e) y[e] += to_f32(r.v[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (n + j * E + e < a.N) y[e] += to_f32(rs[e]);
      }
    }
    if (VEC) {
      Vec16<T> v;
#pragma unroll
      for (int e = 0; e < E; ++e) v.v[e] = from_f32<T>(y[e]);
      if (n + j * E < a.N) store16(o + j * E, v);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (n + j * E + e < a.N) o[j * E + e] = from_f32<T>(y[e]);
    }
  }
}

// f(activation, whole 16-byte stores or not) as constants: the branch is taken once a tile, not once an element
template <typename F> __device__ __forceinline__ void with_epilogue(const MxArgs& a, F&& f) {
  using std::integral_constant;
  if (a.vec) {
    if (a.act == 0) f(integral_constant<int, 0>{}, integral_constant<bool, true>{});
    else if (a.act == 1) f(integral_constant<int, 1>{}, integral_constant<bool, true>{});
    else f(integral_constant<int, 2>{}, integral_constant<bool, true>{});
  } else {
    if (a.act == 0) f(integral_constant<int, 0>{}, integral_constant<bool, false>{});
    else if (a.act == 1) f(integral_constant<int, 1>{}, integral_constant<bool, false>{});
    else f(integral_constant<int, 2>{}, integral_constant<bool, false>{});
  }
}

// ---- few tiles: the W waves of a workgroup share the steps of K of one tile of 16 F x 16 F outputs and add their sums
// through LDS in a fixed tree.  SRC: the activations' own type, quantised by each wave for its steps, or void: packed.
// A step's fragments are fetched one step ahead.
template <typename T, typename SRC, int F>
__global__ __launch_bounds__(F == 4 ? 512 : 1024) void mx_split_kernel(MxArgs a) {
  constexpr bool RAW = !std::is_void<SRC>::value;
  typedef typename std::conditional<RAW, SRC, bf16>::type S;
  extern __shared__ f32x4 xch[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
  const uint32_t ng = blockIdx.x / (4 / F), f0 = blockIdx.x % (4 / F) * F;      // weights: group of 64, first fragment in it
  const uint32_t m0 = blockIdx.y * 16 * F;
  const u32x4* wc = a.wc + (uint64_t)ng * a.kt * 256 + f0 * 64 + lane;
  const uint32_t* ws = a.ws + (uint64_t)ng * a.kt * 64 + lane;
  // row of this lane in fragment fx of the tile; the packed order where the tile is a whole group
  auto row_of = [&](int fx) __attribute__((always_inline)) { return m0 + (F == 4 ? frag_row(fx, lane & 15) : fx * 16 + (lane & 15)); };
  f32x4 acc[F][F];
#pragma unroll
  for (int w = 0; w < F; ++w) {
    const f32x4 b = wave == 0 ? bias4(a, ng * 64, f0 + w, lane) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < F; ++x) acc[w][x] = b;
  }
  struct Step {
    u32x4 w[F], x[F];
    RawBlock<S> raw[RAW ? F : 1];
    uint32_t sw, sx;
  };
  auto fetch = [&](Step& s, uint32_t k) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < F; ++f) s.w[f] = wc[(uint64_t)k * 256 + f * 64];
    s.sw = ws[(uint64_t)k * 64] >> (8 * f0);
    s.sx = 0;
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const uint32_t row = row_of(f);
      if constexpr (RAW) {
        const bool there = row < a.M;
        load_block<S, true>(reinterpret_cast<const S*>(a.x) + (int64_t)(there ? row : 0) * a.ldx, (int)k * 128 + (lane >> 4) * 32, a.K,
                           there, s.raw[f]);
      } else if (F == 4) {
        s.x[f] = a.xc[((uint64_t)blockIdx.y * a.kt + k) * 256 + f * 64 + lane];
        if (f == 0) s.sx = a.xs[((uint64_t)blockIdx.y * a.kt + k) * 64 + lane];
      } else {
        // where the packed order has this row: fragment and lane
        const uint32_t g = row >> 6, r = row & 63, pf = (r >> 5 << 1) + (r >> 2 & 1), pl = (lane & 48) + (r >> 3 & 3) * 4 + (r & 3);
        s.x[f] = a.xc[((uint64_t)g * a.kt + k) * 256 + pf * 64 + pl];
        s.sx |= (a.xs[((uint64_t)g * a.kt + k) * 64 + pl] >> (8 * pf) & 255u) << (8 * f);
      }
    }
  };
  Step nx;
  uint32_t k = wave;
  if (k < a.kt) fetch(nx, k);
  while (k < a.kt) {
    Step s = nx;
    k += W;
    if (k < a.kt) fetch(nx, k);
    if constexpr (RAW) {
#pragma unroll
      for (int f = 0; f < F; ++f) s.sx |= mx_block(s.raw[f], s.x[f]) << (8 * f);
    }
    static_for<F>([&](auto fw) __attribute__((always_inline)) {
      static_for<F>([&](auto fx) __attribute__((always_inline)) {
        constexpr int w = decltype(fw)::value, x = decltype(fx)::value;
        acc[w][x] = mma4<w, x>(s.w[w], s.x[x], acc[w][x], s.sw, s.sx);
      });
    });
  }
  for (int half = W >> 1; half >= 1; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int i = 0; i < F * F; ++i) xch[((wave - half) * F * F + i) * 64 + lane] = acc[i / F][i % F];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int i = 0; i < F * F; ++i) acc[i / F][i % F] += xch[(wave * F * F + i) * 64 + lane];
    }
    __syncthreads();
  }
  if (wave != 0) return;
  const int q = lane >> 4;
  with_epilogue(a, [&](auto act, auto vec) __attribute__((always_inline)) {
    constexpr int ACT = decltype(act)::value;
    constexpr bool V = decltype(vec)::value;
#pragma unroll
    for (int x = 0; x < F; ++x) {
      const uint32_t m = row_of(x);
      if constexpr (F == 1) {
        // one fragment: four columns out of eight
        const uint32_t n = ng * 64 + ((f0 >> 1) << 5) + (q << 3) + ((f0 & 1) << 2);
        if (m < a.M) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n + i < a.N) {
              float y = mx_act<T, ACT>(acc[0][0][i]);
              if (a.resid != nullptr) y += to_f32(reinterpret_cast<const T*>(a.resid)[(int64_t)m * a.ldr + n + i]);
              reinterpret_cast<T*>(a.out)[(int64_t)m * a.ldo + n + i] = from_f32<T>(y);
            }
        }
      } else {
#pragma unroll
        for (int j = 0; j < F / 2; ++j)
          store8<T, ACT, V>(a, m, ng * 64 + (f0 >> 1) * 32 + j * 32 + q * 8, acc[2 * j][x], acc[2 * j + 1][x]);
      }
    }
  });
}

// ---- many rows, short K (KS steps of 128): a wave quantises its 64 rows once and keeps them in registers; the workgroup
// runs over its groups of 64 columns, whose weights the next group's LDS-DMA brings while this one is multiplied and
// written.  Bound by the write of the output and the arithmetic on it.
template <typename T, typename SRC, int KS>
__global__ __launch_bounds__(256, KS <= 2 ? 3 : 2) void mx_rows_kernel(MxArgs a) {
  constexpr bool RAW = !std::is_void<SRC>::value;
  typedef typename std::conditional<RAW, SRC, bf16>::type S;
  constexpr int STAGE = KS * (4096 + 256);      // codes of KS steps, their scales
  constexpr int PIECES = KS * 4 + (KS + 3) / 4, PER = (PIECES + 3) / 4;      // of 1 KB (the last may be part empty), a wave
  __shared__ __attribute__((aligned(1024))) char st0[PIECES * 1024];
  __shared__ __attribute__((aligned(1024))) char st1[PIECES * 1024];
  static_assert(STAGE <= PIECES * 1024, "stage");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups are dealt round-robin to the 8 XCDs: XCD x takes the x-th eighth of the list (rows, columns), columns
  // fastest, so that the workgroups that read the same rows do so through the same L2
  const uint32_t pos = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const uint32_t splits = (a.ngroups + a.per - 1) / a.per;
  const uint32_t mb = pos / splits, g0 = pos % splits * a.per;
  if ((uint64_t)mb * 256 >= a.M) return;      // (the whole workgroup)
  const uint32_t g1 = g0 + a.per < a.ngroups ? g0 + a.per : a.ngroups;
  const uint32_t mg = mb * 4 + wave;
  // pieces wave, wave + 4, ... of a group's weights; the surplus ones repeat the last, lanes past the scales' end read
  // their first bytes again
  auto request = [&](uint32_t g, char* st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int p = wave + 4 * i < PIECES ? wave + 4 * i : PIECES - 1;
      if (p < KS * 4) {
        glds16e(a.wc + ((uint64_t)g * KS * 4 + p) * 64 + lane, st + p * 1024);
      } else {
        const int o = (p - KS * 4) * 64 + lane;
        glds16e(reinterpret_cast<const u32x4*>(a.ws) + (uint64_t)g * KS * 16 + (o < KS * 16 ? o : 0), st + p * 1024);
      }
    }
  };
  request(g0, st0);
  u32x4 xf[KS][4];
  uint32_t sx[KS];
  const bool work = (uint64_t)mg * 64 < a.M;      // (a wave without rows only helps to fetch)
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    if constexpr (RAW) {
      // (a step, or in fp32 half a step, at a time: more in flight costs more registers than the multiplication has)
      constexpr int FB = sizeof(S) == 2 ? 4 : 2;
      sx[k] = 0;
#pragma unroll
      for (int f0 = 0; f0 < 4; f0 += FB) {
        RawBlock<S> r[FB];
#pragma unroll
        for (int f = 0; f < FB; ++f) {
          const uint32_t row = mg * 64 + frag_row(f0 + f, lane & 15);
          load_block<S, true>(reinterpret_cast<const S*>(a.x) + (int64_t)(row < a.M ? row : 0) * a.ldx, k * 128 + (lane >> 4) * 32,
                              a.K, row < a.M, r[f]);
        }
#pragma unroll
        for (int f = 0; f < FB; ++f) {
          sx[k] |= mx_block(r[f], xf[k][f0 + f]) << (8 * (f0 + f));
          asm volatile("" : "+v"(xf[k][f0 + f]) : : "memory");
        }
      }
    } else {
      const uint32_t g = work ? mg : 0;
#pragma unroll
      for (int f = 0; f < 4; ++f) xf[k][f] = a.xc[((uint64_t)g * KS + k) * 256 + f * 64 + lane];
      sx[k] = a.xs[((uint64_t)g * KS + k) * 64 + lane];
    }
  }
  auto group = [&](uint32_t g, const char* st, char* other) __attribute__((always_inline)) {
    // this group's weights have landed for every wave, and everyone is done with the other stage
    wait_vm_then_barrier<0, true>();
    if (g + 1 < g1) request(g + 1, other);
    if (!work) return;
    f32x4 acc[4][4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f32x4 b = bias4(a, g * 64, w, lane);
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[w][x] = b;
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      u32x4 wf[4];
#pragma unroll
      for (int f = 0; f < 4; ++f) wf[f] = *reinterpret_cast<const u32x4*>(st + (k * 4 + f) * 1024 + lane * 16);
      const uint32_t sw = *reinterpret_cast<const uint32_t*>(st + KS * 4096 + k * 256 + lane * 4);
      static_for<4>([&](auto fw) __attribute__((always_inline)) {
        static_for<4>([&](auto fx) __attribute__((always_inline)) {
          constexpr int w = decltype(fw)::value, x = decltype(fx)::value;
          acc[w][x] = mma4<w, x>(wf[w], xf[k][x], acc[w][x], sw, sx[k]);
        });
      });
    }
    // (opaque: the compiler would otherwise move the multiplications in front of each row's store and keep every weight
    // fragment of the group for them)
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(acc[i / 4][i % 4]));
    with_epilogue(a, [&](auto act, auto vec) __attribute__((always_inline)) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t m = mg * 64 + frag_row(x, lane & 15), n = g * 64 + (lane >> 4) * 8;
        store8<T, decltype(act)::value, decltype(vec)::value>(a, m, n, acc[0][x], acc[1][x]);
        store8<T, decltype(act)::value, decltype(vec)::value>(a, m, n + 32, acc[2][x], acc[3][x]);
      }
    });
  };
#pragma unroll 1
  for (uint32_t g = g0; g < g1; g += 2) {
    group(g, st0, st1);
    if (g + 1 < g1) group(g + 1, st1, st0);
  }
}

// ---- large products: 256 x 256 outputs a workgroup, 128 x 128 a wave, so that a byte read from LDS meets 128 others.
// Four LDS stages of a step (128 k) each, filled by LDS-DMA: while step s multiplies from registers, the fragments of step
// s + 1 are read from their stage between the multiplications, stage s + 2 is landing and s + 3 is requested.
constexpr int LG_STAGE = 2 * (16 * 1024 + 1024);      // codes of 256 rows and 256 columns, their scales

template <typename T>
__global__ __launch_bounds__(256, 1) void mx_large_kernel(MxArgs a) {
  __shared__ __attribute__((aligned(1024))) char st0[LG_STAGE];
  __shared__ __attribute__((aligned(1024))) char st1[LG_STAGE];
  __shared__ __attribute__((aligned(1024))) char st2[LG_STAGE];
  __shared__ __attribute__((aligned(1024))) char st3[LG_STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const uint32_t tm = (a.M + 255) / 256, tn = (a.N + 255) / 256, total = tm * tn;
  // XCD x takes the x-th eighth of the tiles, in bands of eight row tiles: the 32 tiles an XCD has in work form a patch
  // of 8 x 4, which share rows and columns in its L2
  const uint32_t pos = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (pos >= total) return;
  const uint32_t band = pos / (8 * tn), rest = pos - band * 8 * tn, high = tm - band * 8 < 8 ? tm - band * 8 : 8;
  const uint32_t mt = band * 8 + rest % high, nt = rest / high;
  const uint32_t mgs = (a.M + 63) / 64, ngs = (a.N + 63) / 64;
  // what this wave requests of a stage: eight of the 32 fragments (waves 0, 1 the activations', 2, 3 the weights') and,
  // twice over, one of the two scale pieces (so every wave has nine requests a stage)
  const u32x4* src[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t g = (wave & 1) * 2 + i;
    if (wave < 2) {
      const uint32_t mg = mt * 4 + g < mgs ? mt * 4 + g : mgs - 1;      // past the last group: any that is there
      src[i] = a.xc + (uint64_t)mg * a.kt * 256 + lane;
    } else {
      const uint32_t gg = nt * 4 + g < ngs ? nt * 4 + g : ngs - 1;
      src[i] = a.wc + (uint64_t)gg * a.kt * 256 + lane;
    }
  }
  const u32x4* ssrc;      // scales: lane / 16 is the group, 16 bytes a lane
  {
    const uint32_t g = lane >> 4;
    if ((wave & 1) == 0) {
      const uint32_t mg = mt * 4 + g < mgs ? mt * 4 + g : mgs - 1;
      ssrc = reinterpret_cast<const u32x4*>(a.xs) + (uint64_t)mg * a.kt * 16 + (lane & 15);
    } else {
      const uint32_t gg = nt * 4 + g < ngs ? nt * 4 + g : ngs - 1;
      ssrc = reinterpret_cast<const u32x4*>(a.ws) + (uint64_t)gg * a.kt * 16 + (lane & 15);
    }
  }
  auto request = [&](uint32_t k, char* st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int f = 0; f < 4; ++f) glds16e(src[i] + (uint64_t)k * 256 + f * 64, st + (wave * 8 + i * 4 + f) * 1024);
    glds16e(ssrc + (uint64_t)k * 16, st + 32 * 1024 + (wave & 1) * 1024);
  };
  struct Frags {
    u32x4 x[8], w[8];
    uint32_t sx[2], sw[2];
  } fr[2];
  // fragment i of both operands out of a stage (and the scales with the first)
  auto read1 = [&](Frags& f, const char* st, int i) __attribute__((always_inline)) {
    f.x[i] = *reinterpret_cast<const u32x4*>(st + (wm * 8 + i) * 1024 + lane * 16);
    f.w[i] = *reinterpret_cast<const u32x4*>(st + (16 + wn * 8 + i) * 1024 + lane * 16);
    if (i % 4 == 0) {
      f.sx[i / 4] = *reinterpret_cast<const uint32_t*>(st + 32 * 1024 + (wm * 2 + i / 4) * 256 + lane * 4);
      f.sw[i / 4] = *reinterpret_cast<const uint32_t*>(st + 33 * 1024 + (wn * 2 + i / 4) * 256 + lane * 4);
    }
  };
  f32x4 acc[8][8];      // [weights' fragment][activations' fragment]
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const f32x4 b = bias4(a, nt * 256 + wn * 128 + (w >> 2) * 64, w & 3, lane);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      acc[w][x] = b;
      asm volatile("" : "+a"(acc[w][x]));
    }
  }
  const uint32_t kt = a.kt;
  char* const stages[4] = {st0, st1, st2, st3};
  request(0, st0);
  request(1 < kt ? 1 : 0, st1);
  request(2 < kt ? 2 : 0, st2);
  wait_vm_then_barrier<18, false>();
#pragma unroll
  for (int i = 0; i < 8; ++i) read1(fr[0], st0, i);
  // step s (s % 4 == P): nine requests of step s + 2 may be out, those of s + 1 have landed.  Steps past the end repeat
  // the last one's requests, so that the count holds.
  auto step = [&](uint32_t s, auto pc) __attribute__((always_inline)) {
    constexpr int P = decltype(pc)::value;
    wait_vm_then_barrier<9, true>();
    request(s + 3 < kt ? s + 3 : kt - 1, stages[(P + 3) & 3]);
    Frags& cur = fr[P & 1];
    Frags& nxt = fr[(P & 1) ^ 1];
    static_for<8>([&](auto ic) __attribute__((always_inline)) {
      constexpr int x = decltype(ic)::value;
      read1(nxt, stages[(P + 1) & 3], x);
      static_for<8>([&](auto wc) __attribute__((always_inline)) {
        constexpr int w = decltype(wc)::value;
        acc[w][x] = mma4<w % 4, x % 4>(cur.w[w], cur.x[x], acc[w][x], cur.sw[w / 4], cur.sx[x / 4]);
      });
    });
  };
  // (one loop left from four places, the accumulators pinned where the multiplications update them in place: with the
  // last steps behind the loop the compiler shuffles and spills all 256 of them between the two)
  uint32_t s = 0;
#pragma unroll 1
  while (true) {
    step(s, std::integral_constant<int, 0>{});
    if (s + 1 >= kt) break;
    step(s + 1, std::integral_constant<int, 1>{});
    if (s + 2 >= kt) break;
    step(s + 2, std::integral_constant<int, 2>{});
    if (s + 3 >= kt) break;
    step(s + 3, std::integral_constant<int, 3>{});
    s += 4;
    if (s >= kt) break;
  }
  wait_vm_then_barrier<0, true>();      // nothing of this workgroup writes LDS after its end
#pragma unroll
  for (int i = 0; i < 64; ++i) asm volatile("" : "+a"(acc[i / 8][i % 8]));
  with_epilogue(a, [&](auto act, auto vec) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const uint32_t m = mt * 256 + wm * 128 + (x >> 2) * 64 + frag_row(x & 3, lane & 15);
      const uint32_t n = nt * 256 + wn * 128 + (lane >> 4) * 8;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        store8<T, decltype(act)::value, decltype(vec)::value>(a, m, n + j * 32, acc[2 * j][x], acc[2 * j + 1][x]);
    }
  });
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int64_t MX_MAX_ROWS = (int64_t)1 << 30;
constexpr int MX_MAX_K = 1 << 20;

int64_t units_of(int64_t rows, int K) { return ((rows + 63) / 64) * ((K + 127) / 128); }

int check_mx(const char* who, int64_t rows, int64_t K, int dtype) {
  UNETK_CHECK_ARG(dtype == UNETK_F32 || dtype == UNETK_BF16, "%s: unsupported dtype %d", who, dtype);
  UNETK_CHECK_ARG(rows >= 1 && rows <= MX_MAX_ROWS && K >= 1 && K <= MX_MAX_K, "%s: a %lld x %lld matrix", who,
                  (long long)rows, (long long)K);
  UNETK_CHECK_ARG(units_of(rows, (int)K) < (int64_t)1 << 26, "%s: a %lld x %lld matrix", who, (long long)rows, (long long)K);
  return UNETK_OK;
}

// Which kernel takes an M x N x K product: by sizes alone, so that activations quantised beforehand give the same bits.
enum Plan { SPLIT, ROWS, LARGE };
Plan plan_of(int64_t M, int64_t K, int64_t N) {
  const int64_t kt = (K + 127) / 128;
  if (kt <= 6 && M >= 1024) return ROWS;
  if (((M + 255) / 256) * ((N + 255) / 256) >= 160) return LARGE;
  return SPLIT;
}

template <typename T, typename SRC, int F> void launch_split(const MxArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)cdiv(a.N, 64) * (4 / F), (unsigned)cdiv(a.M, 16 * F));
  // waves a tile: about 4096 in all, at least a step each
  const int64_t tiles = (int64_t)grid.x * grid.y;
  int W = 1;
  while (W < (F == 4 ? 8 : 16) && tiles * W < 4096 && (uint32_t)W * 2 <= a.kt) W *= 2;
  hipLaunchKernelGGL((mx_split_kernel<T, SRC, F>), grid, dim3(64 * W), W / 2 * F * F * 1024, stream, a);
}
template <typename T, typename SRC> void launch_split_f(const MxArgs& a, hipStream_t stream) {
  if (a.M <= 16) launch_split<T, SRC, 1>(a, stream);
  else if constexpr (std::is_same<SRC, float>::value) return;      // (never asked for: unetk_mx_linear_x_supported)
  else if (a.M <= 32) launch_split<T, SRC, 2>(a, stream);
  else launch_split<T, SRC, 4>(a, stream);
}

template <typename T, typename SRC> void launch_rows(MxArgs& a, hipStream_t stream) {
  a.ngroups = (uint32_t)cdiv(a.N, 64);
  const uint32_t blocks = (uint32_t)cdiv(a.M, 256);
  // the columns are split until there are workgroups enough for the chip
  uint32_t splits = 1;
  while (blocks * splits < 512 && splits < a.ngroups) ++splits;
  a.per = (a.ngroups + splits - 1) / splits;
  splits = (a.ngroups + a.per - 1) / a.per;
  const dim3 grid((blocks * splits + 7) / 8 * 8);
  switch (a.kt) {
    case 1: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 1>), grid, dim3(256), 0, stream, a); break;
    case 2: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 2>), grid, dim3(256), 0, stream, a); break;
    case 3: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 3>), grid, dim3(256), 0, stream, a); break;
    case 4: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 4>), grid, dim3(256), 0, stream, a); break;
    case 5: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 5>), grid, dim3(256), 0, stream, a); break;
    default: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 6>), grid, dim3(256), 0, stream, a); break;
  }
}

template <typename T> void launch_mx(MxArgs& a, Plan plan, hipStream_t stream) {
  if (plan == ROWS) {
    if (a.x) launch_rows<T, T>(a, stream);
    else launch_rows<T, void>(a, stream);
  } else if (plan == LARGE) {
    const unsigned tiles = (unsigned)cdiv(a.M, 256) * (unsigned)cdiv(a.N, 256);
    hipLaunchKernelGGL(mx_large_kernel<T>, dim3((tiles + 7) / 8 * 8), dim3(256), 0, stream, a);
  } else {
    if (a.x) launch_split_f<T, T>(a, stream);
    else launch_split_f<T, void>(a, stream);
  }
}

int mx_linear_impl(const void* x, int64_t ldx, const void* xcodes, const void* xscales, const void* wcodes, const void* wscales,
                   void* out, int64_t ldo, int64_t M, int64_t K, int64_t N, const float* bias, int act, const void* resid,
                   int64_t ldr, int dtype, hipStream_t stream) {
  int rc = check_mx("mx_linear", M, K, dtype);
  if (rc == UNETK_OK) rc = check_mx("mx_linear", N, K, dtype);
  if (rc != UNETK_OK) return rc;
  UNETK_CHECK_ARG(wcodes && wscales && out && ldo >= N && (resid == nullptr || ldr >= N),
                  "mx_linear: null operand or overlapping rows");
  UNETK_CHECK_ARG(aligned16(wcodes) && aligned16(wscales), "mx_linear: misaligned packed operand");
  UNETK_CHECK_ARG(act >= 0 && act <= 2, "mx_linear: activation %d", act);
  // (grids: one block axis per 16 columns, one per 16...64 rows)
  UNETK_CHECK_ARG(N <= (int64_t)1 << 24 && (M <= (int64_t)1 << 21 || plan_of(M, K, N) != SPLIT), "mx_linear: %lld x %lld outputs",
                  (long long)M, (long long)N);
  MxArgs a = {};
  a.x = x; a.ldx = ldx;
  a.xc = (const u32x4*)xcodes; a.xs = (const uint32_t*)xscales; a.wc = (const u32x4*)wcodes; a.ws = (const uint32_t*)wscales;
  a.out = out; a.bias = bias; a.resid = resid; a.ldo = ldo; a.ldr = ldr; a.M = (uint32_t)M; a.N = (uint32_t)N;
  a.kt = (uint32_t)((K + 127) / 128); a.K = (int)K; a.act = act;
  const int E = dtype == UNETK_BF16 ? 8 : 4;
  a.vec = N % E == 0 && ldo % E == 0 && aligned16(out) && (!resid || (ldr % E == 0 && aligned16(resid)));
  const Plan plan = plan_of(M, K, N);
  if (dtype == UNETK_BF16) launch_mx<bf16>(a, plan, stream);
  else launch_mx<float>(a, plan, stream);
  UNETK_CHECK_LAUNCH();
  return UNETK_OK;
}

}  // namespace

extern "C" {

int64_t unetk_mx_codes_bytes(int64_t rows, int64_t K) {
  return rows < 1 || rows > MX_MAX_ROWS || K < 1 || K > MX_MAX_K ? 0 : units_of(rows, (int)K) * 4096;
}

int64_t unetk_mx_scales_bytes(int64_t rows, int64_t K) { return unetk_mx_codes_bytes(rows, K) / 16; }

int unetk_mx_quantize(const void* x, int64_t ldx, int64_t rows, int64_t K, int dtype, void* codes, void* scales,
                      hipStream_t stream) {
  const int rc = check_mx("mx_quantize", rows, K, dtype);
  if (rc != UNETK_OK) return rc;
  UNETK_CHECK_ARG(x && codes && scales && ldx >= K && aligned16(codes) && aligned16(scales),
                  "mx_quantize: null or misaligned operand, or overlapping rows");
  const uint32_t kt = (uint32_t)((K + 127) / 128);
  const uint64_t units = (uint64_t)units_of(rows, (int)K);
  const dim3 grid((unsigned)((units + 3) / 4));
  const int E = dtype == UNETK_BF16 ? 8 : 4;
  const bool vec = K % E == 0 && ldx % E == 0 && aligned16(x);
#define MX_QUANT(T, V)                                                                                                \
  hipLaunchKernelGGL((mx_quantize_kernel<T, V>), grid, dim3(256), 0, stream, (const T*)x, ldx, (uint32_t)rows, (int)K, kt, \
                     units, (u32x4*)codes, (uint32_t*)scales)
  if (dtype == UNETK_BF16) {
    if (vec) MX_QUANT(bf16, true);
    else MX_QUANT(bf16, false);
  } else {
    if (vec) MX_QUANT(float, true);
    else MX_QUANT(float, false);
  }
#undef MX_QUANT
  UNETK_CHECK_LAUNCH();
  return UNETK_OK;
}

int unetk_mx_dequantize(const void* codes, const void* scales, int64_t rows, int64_t K, void* out, int64_t ldo, int dtype,
                        hipStream_t stream) {
  const int rc = check_mx("mx_dequantize", rows, K, dtype);
  if (rc != UNETK_OK) return rc;
  UNETK_CHECK_ARG(out && codes && scales && ldo >= K && aligned16(codes) && aligned16(scales),
                  "mx_dequantize: null or misaligned operand, or overlapping rows");
  const uint32_t kt = (uint32_t)((K + 127) / 128);
  const uint64_t units = (uint64_t)units_of(rows, (int)K);
  const dim3 grid((unsigned)((units + 3) / 4));
  const int E = dtype == UNETK_BF16 ? 8 : 4;
  const int vec = K % E == 0 && ldo % E == 0 && aligned16(out);
  if (dtype == UNETK_BF16)
    hipLaunchKernelGGL(mx_dequantize_kernel<bf16>, grid, dim3(256), 0, stream, (const u32x4*)codes, (const uint32_t*)scales,
                       (uint32_t)rows, (int)K, kt, units, (bf16*)out, ldo, vec);
  else
    hipLaunchKernelGGL(mx_dequantize_kernel<float>, grid, dim3(256), 0, stream, (const u32x4*)codes, (const uint32_t*)scales,
                       (uint32_t)rows, (int)K, kt, units, (float*)out, ldo, vec);
  UNETK_CHECK_LAUNCH();
  return UNETK_OK;
}

/* Whether mx_linear quantises activations on the way (unetk_mx_linear_x) for this problem: a few rows, where the launch
 * counts, and short K, where the rows are kept in registers. */
int unetk_mx_linear_x_supported(int64_t M, int64_t K, int64_t N, int dtype) {
  if (M < 1 || K < 1 || N < 1 || M > MX_MAX_ROWS || N > MX_MAX_ROWS || K > MX_MAX_K) return 0;
  if (K % (dtype == UNETK_BF16 ? 8 : 4) != 0) return 0;
  return M <= (dtype == UNETK_BF16 ? 64 : 16) || plan_of(M, K, N) == ROWS;
}

int unetk_mx_linear_x(const void* x, int64_t ldx, const void* wcodes, const void* wscales, void* out, int64_t ldo, int64_t M,
                      int64_t K, int64_t N, const float* bias, int act, const void* resid, int64_t ldr, int dtype,
                      hipStream_t stream) {
  const int E = dtype == UNETK_BF16 ? 8 : 4;
  UNETK_CHECK_ARG(x && ldx >= K && ldx % E == 0 && aligned16(x), "mx_linear_x: null or unaligned activations");
  UNETK_CHECK_ARG(unetk_mx_linear_x_supported(M, K, N, dtype), "mx_linear_x: %lld x %lld x %lld is quantised first", (long long)M,
                  (long long)K, (long long)N);
  return mx_linear_impl(x, ldx, nullptr, nullptr, wcodes, wscales, out, ldo, M, K, N, bias, act, resid, ldr, dtype, stream);
}

int unetk_mx_linear(const void* xcodes, const void* xscales, const void* wcodes, const void* wscales, void* out, int64_t ldo,
                    int64_t M, int64_t K, int64_t N, const float* bias, int act, const void* resid, int64_t ldr, int dtype,
                    hipStream_t stream) {
  UNETK_CHECK_ARG(xcodes && xscales && aligned16(xcodes) && aligned16(xscales), "mx_linear: null or misaligned activations");
  return mx_linear_impl(nullptr, 0, xcodes, xscales, wcodes, wscales, out, ldo, M, K, N, bias, act, resid, ldr, dtype, stream);
}

}  // extern "C"
