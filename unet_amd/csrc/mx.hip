// Microscaled 4-bit floating point (OCP MX, format MXFP4) on gfx950: quantisation, the way back, and the product of two
// such matrices on the scaled matrix instruction.
//
// A (rows, K) matrix is cut into blocks of 32 along K.  A block holds 32 E2M1 elements (sign, 2 exponent bits, 1 mantissa
// bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one E8M0 scale 2^se: se = floor(log2(largest magnitude)) - 2, not below -127;
// elements are x / 2^se rounded half to even and held to 6.  A block with a NaN or an infinity gets the scale byte 255 (NaN):
// everything made from it is NaN.
//
// Layout: the one the matrix instruction reads, for both operands.  v_mfma_scale_f32_32x32x64_f8f6f4 takes of each operand
// 32 rows x 64 k; lane l holds row l % 32, k block l / 32: 32 consecutive elements, 16 bytes, exactly one block, and in one
// byte that block's scale.  (The 16x16x128 shape multiplies at 5.0...6.4 PFLOP/s here, this one at 9.3.)  Rows are padded to
// 64, K to 128 (zero elements, scale byte 0), and stored in units of 64 rows x 128 k:
//   codes  [rows/64][K/128][4 fragments][64 lanes][16 bytes]     (element j of a block in nibble j, low nibble first)
//   scales [rows/64][K/128][64 lanes][4 bytes]                   (byte f: the lane's block of fragment f)
// fragment f: rows 32 (f % 2) + ..., k 64 (f / 2) + ..., so that a fragment is 1 KB and the scales of four are 256 bytes, read
// without a gap.  Row r of a fragment is row 16 (r / 16) + 8 (r / 4 % 2) + 4 (r / 8 % 2) + r % 4 of its 32: with the weights as the
// instruction's first operand, whose rows come out in fours eight apart, a lane's accumulators are then two runs of 8
// consecutive output columns of one row.
#include "epilogue.h"
#include "unaligned.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// row of a fragment's 32 (or the other way round: the map is its own inverse)
__device__ __forceinline__ int frag_row(int r) { return (r & 16) + ((r & 4) << 1) + ((r & 8) >> 1) + (r & 3); }

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
template <typename T, bool WHOLE>
__device__ __forceinline__ void load_block(const T* row, int k0, int K, bool there, RawBlock<T>& x) {
  constexpr int E = Vec16<T>::N;
#pragma unroll
  for (int j = 0; j < RawBlock<T>::N; ++j)
    x.v[j] = __builtin_bit_cast(u32x4, load_part<WHOLE>(row + k0 + j * E, there ? K - (k0 + j * E) : 0));
}

// One wave: a fragment (32 rows x 64 k), each lane one block.  Bound by the read of x: 65536 x 768 bf16 28.5 us (127 MB,
// 4.5 TB/s), 8192 x 8192 40.1 us (170 MB, 4.2 TB/s), operands out of the caches.  (One workgroup of four waves a unit: with a
// wave a unit, four fragments in turn, a small matrix has too few waves to hide its loads.)
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, int64_t ldx, uint32_t rows, int K,
                                                          uint32_t kt, u32x4* __restrict__ codes, uint8_t* __restrict__ scales) {
  const uint64_t unit = blockIdx.x;
  const int lane = threadIdx.x & 63, f = threadIdx.x >> 6;
  const uint32_t row = (uint32_t)(unit / kt) * 64 + (f & 1) * 32 + frag_row(lane & 31);
  const int k0 = (int)(unit % kt) * 128 + (f >> 1) * 64 + (lane >> 5) * 32;
  RawBlock<T> r;
  load_block<T, WHOLE>(x + (int64_t)(row < rows ? row : 0) * ldx, k0, K, row < rows, r);
  u32x4 c;
  scales[(unit * 64 + lane) * 4 + f] = (uint8_t)mx_block(r, c);
  codes[(unit * 4 + f) * 64 + lane] = c;
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

// One workgroup a unit; a lane makes 8 consecutive values, 16 lanes the 128 of a row: runs of 256 bytes (bf16) a row.  Bound
// by the write of the values: 65536 x 768 to bf16 22.5 us (127 MB, 5.6 TB/s: much of the codes still lies in the last cache).
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            uint32_t rows, int K, uint32_t kt, T* __restrict__ out, int64_t ldo) {
  constexpr int E = Vec16<T>::N;
  const uint64_t unit = blockIdx.x;
  const int k8 = threadIdx.x & 15, kb = k8 >> 2;      // which 8 values of the row, in which block
  const int k0 = (int)(unit % kt) * 128 + k8 * 8;
  if (k0 >= K) return;
  uint32_t c[4], sc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 16 + (threadIdx.x >> 4);      // row of the unit
    const int f = (kb >> 1) * 2 + (r >> 5), slot = (kb & 1) * 32 + frag_row(r & 31);
    c[i] = codes[((unit * 4 + f) * 64 + slot) * 4 + (k8 & 3)];
    sc[i] = scales[(unit * 64 + slot) * 4 + f];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t row = (uint32_t)(unit / kt) * 64 + i * 16 + (threadIdx.x >> 4);
    if (row >= rows) return;
    T* o = out + (int64_t)row * ldo + k0;
#pragma unroll
    for (int j = 0; j < 8 / E; ++j) {
      Vec16<T> v;
#pragma unroll
      for (int e = 0; e < E; ++e) v.v[e] = from_f32<T>(mx_value(c[i] >> (4 * (j * E + e)), sc[i]));
      store_part<WHOLE>(o + j * E, v, K - (k0 + j * E));
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
  int K, act, whole;
  uint32_t ngroups, per;  // mx_rows_kernel: groups of 64 columns, and how many of them a workgroup takes
};

// a fragment of the weights and one of the activations (their scales: bytes FW / FX of the lane's words)
template <int FW, int FX>
__device__ __forceinline__ f32x16 mma32(const u32x4& w, const u32x4& x, f32x16 c, uint32_t sw, uint32_t sx) {
#if defined(__HIP_DEVICE_COMPILE__)
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 4, FW, (int)sw, FX, (int)sx);
#else
  return c;
#endif
}
__device__ __forceinline__ f32x4 mma16(const u32x4& w, const u32x4& x, f32x4 c, uint32_t sw, uint32_t sx) {
#if defined(__HIP_DEVICE_COMPILE__)
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, 0, (int)sw, 0, (int)sx);
#else
  return c;
#endif
}

// GELU for bfloat16 results: v Phi(v) = (v or 0, whichever is larger) - |v| Phi(-|v|), and log2 Phi(-a) is so smooth that
// a polynomial of degree 6 in a suffices: the result is off by less than 2.4e-7 of v, and by less than 1.6e-4 of itself
// far into the tail (least squares in the Chebyshev basis on [0, 5.5], reweighted towards the largest error against those
// two; Phi(-5.5) = 2e-8 stands for what lies beyond).  Seven multiply-adds and one exponential instead of the erf form's
// reciprocal, exponential and more.  The first term is v / 2 + |v| / 2, exact for normal numbers: NaN and +infinity pass
// through it, and -infinity makes it NaN, as the erf form does (infinity times zero).
__device__ __forceinline__ float gelu_bf16(float v) {
  const float a = __builtin_amdgcn_fmed3f(fabsf(v), 0.f, 5.5f);
  float p = 3.13768651e-05f;
  p = fmaf(p, a, -0.000742790464f);
  p = fmaf(p, a, 0.00795761682f);
  p = fmaf(p, a, -0.0531759113f);
  p = fmaf(p, a, -0.458968848f);
  p = fmaf(p, a, -1.15113544f);
  p = fmaf(p, a, -0.999999404f);
  return fmaf(-a, __builtin_amdgcn_exp2f(p), fmaf(0.5f, fabsf(v), 0.5f * v));
}

template <typename T, bool GELU> __device__ __forceinline__ float mx_act(float v) {
  if (!GELU) return v;
  return sizeof(T) == 2 ? gelu_bf16(v) : 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f));
}

// Accumulators begin as the bias: run j (of two) of a 32-column fragment at n0 is columns n0 + 16 j + 8 (lane / 32) + 0...7.
__device__ __forceinline__ f32x16 bias16(const MxArgs& a, uint32_t n0, int lane) {
  f32x16 b;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t n = n0 + ((i >> 3) << 4) + ((lane >> 5) << 3) + (i & 7);
    b[i] = (a.bias != nullptr && n < a.N) ? a.bias[n] : 0.f;
  }
  return b;
}

// activation, residual and store of run J of a fragment: 8 consecutive columns, from n on, of row m
template <typename T, bool ACT, bool WHOLE, int J>
__device__ __forceinline__ void store8(const MxArgs& a, uint32_t m, uint32_t n, const f32x16& acc) {
  constexpr int E = Vec16<T>::N;
  if (m >= a.M) return;
  T* o = reinterpret_cast<T*>(a.out) + (int64_t)m * a.ldo + n;
#pragma unroll
  for (int j = 0; j < 8 / E; ++j) {
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = mx_act<T, ACT>(acc[J * 8 + j * E + e]);
    const int left = (int)(a.N - n) - j * E;      // (n may lie past the last column: below zero)
    if (a.resid != nullptr) {
      const Vec16<T> r = load_part<WHOLE>(reinterpret_cast<const T*>(a.resid) + (int64_t)m * a.ldr + n + j * E, left);
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] += to_f32(r.v[e]);
    }
    Vec16<T> v;
#pragma unroll
    for (int e = 0; e < E; ++e) v.v[e] = from_f32<T>(y[e]);
    store_part<WHOLE>(o + j * E, v, left);
  }
}

// a 32 x 32 tile: row m (this lane's), columns n0 + ...
template <typename T, bool ACT, bool WHOLE>
__device__ __forceinline__ void store_tile(const MxArgs& a, uint32_t m, uint32_t n0, int lane, const f32x16& acc) {
  const uint32_t n = n0 + ((lane >> 5) << 3);
  store8<T, ACT, WHOLE, 0>(a, m, n, acc);
  store8<T, ACT, WHOLE, 1>(a, m, n + 16, acc);
}

// Four vectors of each of a quad's lanes the other way round: v[k] of lane i <- v[i] of lane k
template <int CTRL> __device__ __forceinline__ uint32_t quad_swap(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ void transpose_quad(u32x4 (&v)[4], int lane) {
  const bool b0 = lane & 1, b1 = lane & 2;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {      // lanes 1 apart
      const uint32_t lo = v[k][e], hi = v[k + 1][e], from_lo = quad_swap<0xB1>(lo), from_hi = quad_swap<0xB1>(hi);
      v[k][e] = b0 ? from_hi : lo;
      v[k + 1][e] = b0 ? hi : from_lo;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {      // 2 apart
      const uint32_t lo = v[k][e], hi = v[k + 2][e], from_lo = quad_swap<0x4E>(lo), from_hi = quad_swap<0x4E>(hi);
      v[k][e] = b1 ? from_hi : lo;
      v[k + 2][e] = b1 ? hi : from_lo;
    }
  }
}

// 32 rows x 64 columns (c0, c1: the columns' halves), activation and no residual, in stores whose quads of lanes write 64
// consecutive bytes of a row: a quad holds four rows' 16-byte pieces, and turned round each of its vectors is one row's.
// All lanes come here.
template <typename T, bool ACT, bool WHOLE>
__device__ __forceinline__ void store_rows(const MxArgs& a, uint32_t m0, uint32_t n0, int lane, const f32x16& c0, const f32x16& c1) {
  constexpr int E = Vec16<T>::N;
  const uint32_t m = m0 + frag_row(lane & 28), i = lane & 3, h = (lane >> 5) << 3;
#pragma unroll
  for (int part = 0; part < 8 / E; ++part) {      // (float: 128 bytes are 32 columns)
    u32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x16& c = (E == 8 ? j >> 1 : part) ? c1 : c0;
      const int at = E == 8 ? 8 * (j & 1) : 8 * (j >> 1) + 4 * (j & 1);
      Vec16<T> o;
#pragma unroll
      for (int e = 0; e < E; ++e) o.v[e] = from_f32<T>(mx_act<T, ACT>(c[at + e]));
      v[j] = __builtin_bit_cast(u32x4, o);
      asm volatile("" : "+v"(v[j]));      // (one vector at a time: the registers are needed)
    }
    if (E == 8) {      // the lower half of the wave takes the left 32 columns, the upper half the right ones
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const auto t = __builtin_amdgcn_permlane32_swap(v[j][e], v[j + 2][e], false, false);
          v[j][e] = t[0];
          v[j + 2][e] = t[1];
        }
      const u32x4 t = v[1];
      v[1] = v[2];
      v[2] = t;
    }
    transpose_quad(v, lane);
    const uint32_t n = n0 + (E == 8 ? 8 * i + 4 * h : 32 * part + 16 * (i >> 1) + 4 * (i & 1) + h);
    const int left = (int)(a.N - n);              // (n may lie past the last column: below zero)
    T* o = reinterpret_cast<T*>(a.out) + (int64_t)m * a.ldo + n;
#pragma unroll
    for (int k = 0; k < 4; ++k, o += a.ldo)
      if (m + k < a.M) store_part<WHOLE>(o, __builtin_bit_cast(Vec16<T>, v[k]), left);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// A wave's 64 x 64 tile in bfloat16 through LDS (TILE_LDS bytes of its own): stores of eight rows x 128 bytes instead of 32
// rows x 32 bytes (8192^3: 295 us for the whole call, 313 without; in mx_rows_kernel the LDS it takes costs waves, and
// 262144 x 96 -> 384 went from 66 to 87 us when the results stayed in the last cache).  cWX: half W of the columns, half X of the rows.
constexpr int TILE_LDS = 64 * 144;
template <bool ACT, bool WHOLE>
__device__ __forceinline__ void store_through_lds(const MxArgs& a, uint32_t m0, uint32_t n0, int lane, const f32x16& c00,
                                                  const f32x16& c01, const f32x16& c10, const f32x16& c11, char* lds) {
  auto put = [&](const f32x16& c, int wf, int xf) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      Vec16<bf16> v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v.v[e] = from_f32<bf16>(mx_act<bf16, ACT>(c[j * 8 + e]));
      store16(reinterpret_cast<bf16*>(lds + (xf * 32 + frag_row(lane & 31)) * 144 + (wf * 32 + j * 16 + ((lane >> 5) << 3)) * 2), v);
    }
  };
  put(c00, 0, 0);
  put(c01, 0, 1);
  put(c10, 1, 0);
  put(c11, 1, 1);
  // (the wave's own LDS operations are carried out in order; the compiler must not turn them round)
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const uint32_t n = n0 + (lane & 7) * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t r = i * 8 + (lane >> 3), m = m0 + r;
    const Vec16<bf16> v = load16(reinterpret_cast<const bf16*>(lds + r * 144 + (lane & 7) * 16));
    if (m < a.M) store_part<WHOLE>(reinterpret_cast<bf16*>(a.out) + (int64_t)m * a.ldo + n, v, (int)(a.N - n));
  }
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// f(GELU or not, rows of whole 16-byte pieces or not) as constants: the branch is taken once a tile, not once an element
template <typename F> __device__ __forceinline__ void with_epilogue(const MxArgs& a, F&& f) {
  std::integral_constant<bool, false> no;
  std::integral_constant<bool, true> yes;
  if (a.whole) {
    if (a.act == 0) f(no, yes);
    else f(yes, yes);
  } else {
    if (a.act == 0) f(no, no);
    else f(yes, no);
  }
}

// ---- few tiles: the W waves of a workgroup share the steps of K of one tile of SIDE x SIDE outputs and add their sums
// through LDS in a fixed tree.  SRC: the activations' own type, quantised by each wave for its steps, or void: packed.
// A step's fragments are fetched one step ahead.  Bound by latency: 1 x 4096 -> 4096, quantising on the way, 7.6 us with the
// weights out of the caches (8.9 MB, 1.8 us at 5 TB/s), 6.1 with them in; 1037 x 2072 -> 1511 fp32, quantised before, 13.8 and
// 11.6.  (A launch among others replayed from a graph takes about 1 us less than alone: 5.2 and 10.8, cached.)

// one 16 x 16 tile (16x16x128: lane l holds row l % 16, k block l / 16), its fragments gathered from the units by blocks
struct Tile16 {
  static constexpr int SIDE = 16, NF = 1, NA = 1;      // fragments a step, accumulators (of four floats)
  f32x4 acc[1];
  static __device__ __forceinline__ int unit_slot(int lane, int r) {      // 16-byte slot of (row r of 64, this lane's block)
    const int kb = lane >> 4;
    return ((kb >> 1) * 2 + (r >> 5)) * 64 + (kb & 1) * 32 + frag_row(r & 31);
  }
  __device__ __forceinline__ void mma(const u32x4 (&w)[1], const u32x4 (&x)[1], uint32_t sw, uint32_t sx) {
    acc[0] = mma16(w[0], x[0], acc[0], sw, sx);
  }
};
// one 32 x 32 tile: two fragments a step
struct Tile32 {
  static constexpr int SIDE = 32, NF = 2, NA = 4;
  f32x16 acc[1];
  __device__ __forceinline__ void mma(const u32x4 (&w)[2], const u32x4 (&x)[2], uint32_t sw, uint32_t sx) {
    acc[0] = mma32<0, 0>(w[0], x[0], acc[0], sw, sx);
    acc[0] = mma32<1, 1>(w[1], x[1], acc[0], sw, sx);
  }
};
template <typename T, typename SRC, typename TILE>
__global__ __launch_bounds__(1024) void mx_split_kernel(MxArgs a) {
  constexpr bool RAW = !std::is_void<SRC>::value;
  typedef typename std::conditional<RAW, SRC, bf16>::type S;
  constexpr int SIDE = TILE::SIDE, NF = TILE::NF, NA = TILE::NA;
  extern __shared__ f32x4 xch[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
  const uint32_t across = (a.N + SIDE - 1) / SIDE, mt = blockIdx.x / across, nt = blockIdx.x - mt * across;
  const uint32_t n0 = nt * SIDE, m0 = mt * SIDE, ng = n0 >> 6, xg = m0 >> 6;
  // where this lane's blocks of fragment f lie in a unit (16-byte slots), for the rows from r0 (in the unit) on
  auto slot = [&](uint32_t r0, int f) __attribute__((always_inline)) -> int {
    if constexpr (SIDE == 16) return Tile16::unit_slot(lane, r0 + (lane & 15));
    else return (f * 2 + (r0 >> 5)) * 64 + lane;
  };
  // row and first k (in the step) of this lane's block of fragment f, for activations quantised here: in a unit's order,
  // so that both sources give the same tile
  auto raw_row = [&](int f) __attribute__((always_inline)) -> uint32_t {
    if constexpr (SIDE == 16) return m0 + (lane & 15);
    else return m0 + frag_row(lane & 31);
  };
  auto raw_k = [&](int f) __attribute__((always_inline)) -> int {
    if constexpr (SIDE == 16) return (lane >> 4) * 32;
    else return f * 64 + (lane >> 5) * 32;
  };
  // the scale bytes of this lane's blocks out of a unit's word(s), byte f: fragment f
  auto scales = [&](const uint32_t* unit, uint32_t r0) __attribute__((always_inline)) -> uint32_t {
    if constexpr (SIDE == 32) {
      const uint32_t v = unit[lane] >> (8 * (r0 >> 5));      // fragments r0 / 32 and 2 + r0 / 32
      return (v & 255u) | (v >> 8 & 0xff00u);
    } else {
      const int sl = slot(r0, 0);
      return unit[sl & 63] >> (8 * (sl >> 6)) & 255u;
    }
  };
  TILE t;
  if constexpr (SIDE == 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t n = n0 + (lane >> 4) * 4 + i;
      t.acc[0][i] = (wave == 0 && a.bias != nullptr && n < a.N) ? a.bias[n] : 0.f;
    }
  } else {
    t.acc[0] = bias16(a, n0, lane);
    if (wave != 0)
#pragma unroll
      for (int j = 0; j < 16; ++j) t.acc[0][j] = 0.f;
  }
  struct Step {
    u32x4 w[NF], x[NF];
    RawBlock<S> raw[RAW ? NF : 1];
    uint32_t sw, sx;
  };
  auto fetch = [&](Step& s, uint32_t k) __attribute__((always_inline)) {
    const uint64_t wu = (uint64_t)ng * a.kt + k, xu = (uint64_t)xg * a.kt + k;
#pragma unroll
    for (int f = 0; f < NF; ++f) s.w[f] = a.wc[wu * 256 + slot(n0 & 63, f)];
    s.sw = scales(a.ws + wu * 64, n0 & 63);
    s.sx = 0;
    if constexpr (RAW) {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const uint32_t row = raw_row(f);
        const bool there = row < a.M;
        load_block<S, true>(reinterpret_cast<const S*>(a.x) + (int64_t)(there ? row : 0) * a.ldx, (int)k * 128 + raw_k(f), a.K, there,
                            s.raw[f]);
      }
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f) s.x[f] = a.xc[xu * 256 + slot(m0 & 63, f)];
      s.sx = scales(a.xs + xu * 64, m0 & 63);
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
      for (int f = 0; f < NF; ++f) s.sx |= mx_block(s.raw[f], s.x[f]) << (8 * f);
    }
    t.mma(s.w, s.x, s.sw, s.sx);
  }
  auto part = [&](int i) __attribute__((always_inline)) -> f32x4 {
    if constexpr (SIDE == 16) return t.acc[0];
    else return f32x4{t.acc[0][i * 4], t.acc[0][i * 4 + 1], t.acc[0][i * 4 + 2], t.acc[0][i * 4 + 3]};
  };
  // down to two waves (one for 16 x 16) by halves, then each of those sums and finishes its share of the tile
  constexpr int FIN = SIDE == 32 ? 2 : 1;
  const int left = W < FIN ? W : FIN, each = NA / left;
  auto add = [&](int i, const f32x4& v) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (SIDE == 16) t.acc[0][j] += v[j];
      else t.acc[0][i * 4 + j] += v[j];
    }
  };
  for (int half = W >> 1; half >= FIN; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int i = 0; i < NA; ++i) xch[((wave - half) * NA + i) * 64 + lane] = part(i);
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int i = 0; i < NA; ++i) add(i, xch[(wave * NA + i) * 64 + lane]);
    }
    __syncthreads();
  }
  if (left > 1) {
    if (wave < left) {
#pragma unroll
      for (int i = 0; i < NA; ++i) xch[(wave * NA + i) * 64 + lane] = part(i);
    }
    __syncthreads();
    if (wave < left) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
        if (i / each == wave) {
          f32x4 v = xch[i * 64 + lane];
          for (int w = 1; w < left; ++w) v += xch[(w * NA + i) * 64 + lane];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (SIDE == 16) t.acc[0][j] = v[j];
            else t.acc[0][i * 4 + j] = v[j];
          }
        }
    }
  }
  if constexpr (SIDE == 16) {
    if (wave != 0) return;
    const uint32_t m = m0 + (lane & 15), n = n0 + (lane >> 4) * 4;
    if (m >= a.M) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) {
        float y = a.act ? mx_act<T, true>(t.acc[0][i]) : t.acc[0][i];
        if (a.resid != nullptr) y += to_f32(reinterpret_cast<const T*>(a.resid)[(int64_t)m * a.ldr + n + i]);
        reinterpret_cast<T*>(a.out)[(int64_t)m * a.ldo + n + i] = from_f32<T>(y);
      }
  } else {
    // parts i, i + 1 (i even): 8 consecutive columns of this lane's row
    with_epilogue(a, [&](auto act, auto whole) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NA; i += 2) {
        if (wave >= left || i / each != wave) continue;
        f32x16 r;
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = t.acc[0][i * 4 + (j & 7)];
        store8<T, decltype(act)::value, decltype(whole)::value, 0>(a, m0 + frag_row(lane & 31), n0 + i * 8 + ((lane >> 5) << 3), r);
      }
    });
  }
}

// ---- many rows, short K (KS steps of 128): a workgroup of W (four or eight) waves quantises 64 rows once into LDS and its
// waves take every W-th group of 64 columns.  The weights' fragments come straight from the caches into
// a ring of registers, a group ahead; the rows' are read from LDS a step at a time.  Bound by the write of the output (a
// store instruction whose lanes lie in many rows holds the CU's address path for some 100 cycles) and the arithmetic on it.
// 262144 x 96 -> 384 with GELU 70.3 us (252 MB, 3.6 TB/s, a floor of 50), 62.9 with the operands cached; 16384 x 384 -> 1152 16.9
// us (50 MB, 3.0 TB/s), 15.8 cached.  (Stores of 32 bytes in each of 32 rows took 18 us more on the first, 17 of them behind
// the kernel's end, and nothing more where the output stayed in the last cache; stores past the caches 130 more.  With a residual
// they are still taken: 262144 x 96 -> 96 31.1 us, 262144 x 384 -> 96 80.4, replayed from a graph; floors of 30 and 60.)
template <typename T, typename SRC, int KS>
__global__ __launch_bounds__(512, KS <= 2 ? 4 : KS <= 4 ? 3 : 2) void mx_rows_kernel(MxArgs a) {
  constexpr bool RAW = !std::is_void<SRC>::value;
  typedef typename std::conditional<RAW, SRC, bf16>::type S;
  __shared__ u32x4 xl[KS][4][64];
  __shared__ uint8_t sl[KS][64][4];
  // The bias of this workgroup's columns.  (Loaded from memory at the head of a group it would be waited for behind the
  // stores of the group before: loads and stores share one counter.)
  extern __shared__ float bias[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups are dealt round-robin to the 8 XCDs: XCD x takes the x-th eighth of the list (rows, columns), columns
  // fastest, so that the workgroups that read the same rows do so through the same L2
  const uint32_t pos = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const uint32_t splits = (a.ngroups + a.per - 1) / a.per;
  const uint32_t mg = pos / splits, g0 = pos % splits * a.per;
  if ((uint64_t)mg * 64 >= a.M) return;      // (the whole workgroup)
  const uint32_t g1 = g0 + a.per < a.ngroups ? g0 + a.per : a.ngroups;
  // the ring: fragments and scales of the KS steps of this wave's next group
  u32x4 wr[KS][4];
  uint32_t ws[KS];
  auto refill = [&](uint32_t g, int k) __attribute__((always_inline)) {
    const uint64_t u = (uint64_t)(g < a.ngroups ? g : a.ngroups - 1) * KS + k;
#pragma unroll
    for (int f = 0; f < 4; ++f) wr[k][f] = a.wc[u * 256 + f * 64 + lane];
    ws[k] = a.ws[u * 64 + lane];
  };
#pragma unroll
  for (int k = 0; k < KS; ++k) refill(g0 + wave, k);
  const int W = blockDim.x >> 6;
  for (uint32_t i = threadIdx.x; i < (g1 - g0) * 64; i += blockDim.x)
    bias[i] = (a.bias != nullptr && g0 * 64 + i < a.N) ? a.bias[g0 * 64 + i] : 0.f;
#pragma unroll 1
  for (int f = wave; f < 4; f += W) {
    const uint32_t row = mg * 64 + (f & 1) * 32 + frag_row(lane & 31);
    if constexpr (RAW) {
      constexpr int KB = sizeof(S) == 2 ? 3 : 2;      // blocks in flight at a time
#pragma unroll
      for (int k0 = 0; k0 < KS; k0 += KB) {
        RawBlock<S> r[KB];
#pragma unroll
        for (int k = 0; k < KB; ++k)
          if (k0 + k < KS)
            load_block<S, true>(reinterpret_cast<const S*>(a.x) + (int64_t)(row < a.M ? row : 0) * a.ldx,
                                (k0 + k) * 128 + (f >> 1) * 64 + (lane >> 5) * 32, a.K, row < a.M, r[k]);
#pragma unroll
        for (int k = 0; k < KB; ++k)
          if (k0 + k < KS) {
            u32x4 c;
            sl[k0 + k][lane][f] = (uint8_t)mx_block(r[k], c);
            xl[k0 + k][f][lane] = c;
          }
      }
    } else {
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint64_t u = (uint64_t)mg * KS + k;
        xl[k][f][lane] = a.xc[u * 256 + f * 64 + lane];
        if (f == 0) *reinterpret_cast<uint32_t*>(&sl[k][lane][0]) = a.xs[u * 64 + lane];
      }
    }
  }
  __syncthreads();
#pragma unroll 1
  for (uint32_t g = g0 + wave; g < g1; g += W) {
    // (opaque: the addresses of all forms of the epilogue would otherwise be kept in registers across the loop)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    // 32 rows at a time, so that half the accumulators are alive
    static_for<2>([&](auto xc) __attribute__((always_inline)) {
      constexpr int x = decltype(xc)::value;
      f32x16 acc[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const float* b = bias + (g - g0) * 64 + w * 32 + ((lane >> 5) << 3);
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[w][i] = b[((i >> 3) << 4) + (i & 7)];
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4 x0 = xl[k][x][lane], x1 = xl[k][2 + x][lane];
        const uint32_t sx = *reinterpret_cast<const uint32_t*>(&sl[k][lane][0]);
        acc[0] = mma32<0, x>(wr[k][0], x0, acc[0], ws[k], sx);
        acc[1] = mma32<1, x>(wr[k][1], x0, acc[1], ws[k], sx);
        acc[0] = mma32<2, 2 + x>(wr[k][2], x1, acc[0], ws[k], sx);
        acc[1] = mma32<3, 2 + x>(wr[k][3], x1, acc[1], ws[k], sx);
        if constexpr (x == 1) refill(g + W, k);
      }
      // (opaque: the compiler would otherwise move the multiplications in front of each row's store)
      asm volatile("" : "+v"(acc[0]), "+v"(acc[1]));
      const uint32_t m = mg * 64 + x * 32;
      with_epilogue(a, [&](auto act, auto whole) __attribute__((always_inline)) {
        if (a.resid == nullptr) {
          store_rows<T, decltype(act)::value, decltype(whole)::value>(a, m, g * 64, ln, acc[0], acc[1]);
        } else {
          store_tile<T, decltype(act)::value, decltype(whole)::value>(a, m + frag_row(ln & 31), g * 64, ln, acc[0]);
          store_tile<T, decltype(act)::value, decltype(whole)::value>(a, m + frag_row(ln & 31), g * 64 + 32, ln, acc[1]);
        }
      });
    });
  }
}

// ---- large products: 256 x 256 outputs a workgroup, 128 x 128 a wave, so that a byte read from LDS meets 128 others.
// Four LDS stages of a step (128 k) each, filled by LDS-DMA: while step s multiplies from registers, the fragments of step
// s + 1 are read from their stage between the multiplications, stage s + 2 is landing and s + 3 is requested.
// 8192^3: 263...275 us with pauses between the launches, 260...320 one behind the other (3.4...4.2 PFLOP/s; 10 are nominal, 8.4 what
// the instruction reaches from registers alone with such data).  Replayed from a graph: 248, with a residual 303, fp32 results
// 409 (both stored straight from the registers, the latter with 48 of them spilled in the epilogue).
// The chip lowers its clock to 1.87 GHz during it and the matrix pipe is busy half of the cycles.
// LDS-DMA of 16 bytes a lane as an instruction of its own.  Through the builtin the compiler follows which transfers may
// still be filling which array, loses track at the loop's end and waits for all of them there, the newest included; here
// it knows of none, and the kernel's own counted waits are the only ones.  (No register is written; the address registers
// are read when the instruction issues.)
__device__ __forceinline__ void dma16(const void* src, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds) : "memory", "m0");
#endif
}
__device__ __forceinline__ uint32_t lds_address(const char* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

constexpr int LG_STAGE = 2 * (16 * 1024 + 1024);      // codes of 256 rows and 256 columns, their scales
static_assert(3 * TILE_LDS <= LG_STAGE, "three waves' output tiles in a stage");

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
  // request p (of nine) of step k's data into a stage
  auto request1 = [&](uint32_t k, uint32_t base, int p) __attribute__((always_inline)) {
    if (p < 8) dma16(src[p / 4] + (uint64_t)k * 256 + (p % 4) * 64, base + (wave * 8 + p) * 1024);
    else dma16(ssrc + (uint64_t)k * 16, base + 32 * 1024 + (wave & 1) * 1024);
  };
  auto request = [&](uint32_t k, char* st) __attribute__((always_inline)) {
    const uint32_t base = __builtin_amdgcn_readfirstlane(lds_address(st));
#pragma unroll
    for (int p = 0; p < 9; ++p) request1(k, base, p);
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
  f32x16 acc[4][4];      // [32 columns][32 rows]
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const f32x16 b = bias16(a, nt * 256 + wn * 128 + w * 32, lane);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      acc[w][x] = b;
      asm volatile("" : "+a"(acc[w][x]));
    }
  }
  const uint32_t kt = a.kt;
  char* const stages[4] = {st0, st1, st2, st3};
  // (in this order: the waits count requests)
  request(0, st0);
  request(1 < kt ? 1 : 0, st1);
  request(2 < kt ? 2 : 0, st2);
  wait_vm_then_barrier<18, false>();
#pragma unroll
  for (int i = 0; i < 8; ++i) read1(fr[0], st0, i);
  wait_vm_then_barrier<9, true>();
  // step s (s % 4 == P): when it begins, those of step s + 1 have landed for every wave and the nine of s + 2 may be out.  Steps past the end repeat
  // the last one's requests, so that the count holds.
  auto step = [&](uint32_t s, auto pc) __attribute__((always_inline)) {
    constexpr int P = decltype(pc)::value;
    const uint32_t later = s + 3 < kt ? s + 3 : kt - 1, base = __builtin_amdgcn_readfirstlane(lds_address(stages[(P + 3) & 3]));
    Frags& cur = fr[P & 1];
    Frags& nxt = fr[(P & 1) ^ 1];
    // fragment i of an operand: rows 64 (i / 4) + 32 (i % 2) + ... of the wave's 128, half i / 2 % 2 of the step's k
    static_for<8>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value, kh = i >> 2, xr = i & 3, xi = (xr >> 1) * 4 + kh * 2 + (xr & 1);
      // (a request occupies the CU's address path for some 33 cycles and holds up what its wave issues behind it: one at
      // a time between the multiplications, not nine in front of them)
      request1(later, base, i);
      if (i == 7) request1(later, base, 8);
      read1(nxt, stages[(P + 1) & 3], i);
      static_for<4>([&](auto wc) __attribute__((always_inline)) {
        constexpr int wr = decltype(wc)::value, wi = (wr >> 1) * 4 + kh * 2 + (wr & 1);
        acc[wr][xr] = mma32<wi % 4, xi % 4>(cur.w[wi], cur.x[xi], acc[wr][xr], cur.sw[wi / 4], cur.sx[xi / 4]);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    // (the reads belong to this step: the compiler would otherwise move each in front of its use, one step later, and
    // wait there)
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(nxt.x[i]), "+v"(nxt.w[i]));
    asm volatile("" : "+v"(nxt.sx[0]), "+v"(nxt.sx[1]), "+v"(nxt.sw[0]), "+v"(nxt.sw[1]));
    wait_vm_then_barrier<9, true>();
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
  for (int i = 0; i < 16; ++i) asm volatile("" : "+a"(acc[i / 4][i % 4]));
  with_epilogue(a, [&](auto act, auto whole) __attribute__((always_inline)) {
    constexpr bool ACT = decltype(act)::value, WH = decltype(whole)::value;
    if constexpr (sizeof(T) == 2) {
      if (a.resid == nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          store_through_lds<ACT, WH>(a, mt * 256 + wm * 128 + (i & 1) * 64, nt * 256 + wn * 128 + (i >> 1) * 64, lane,
                                     acc[(i >> 1) * 2][(i & 1) * 2], acc[(i >> 1) * 2][(i & 1) * 2 + 1],
                                     acc[(i >> 1) * 2 + 1][(i & 1) * 2], acc[(i >> 1) * 2 + 1][(i & 1) * 2 + 1],
                                     wave < 3 ? st0 + wave * TILE_LDS : st1);
        return;
      }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int w = 0; w < 4; ++w)
        store_tile<T, ACT, WH>(a, mt * 256 + wm * 128 + x * 32 + frag_row(lane & 31), nt * 256 + wn * 128 + w * 32, lane, acc[w][x]);
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
  UNETK_CHECK_ARG(units_of(rows, (int)K) < (int64_t)1 << 24, "%s: a %lld x %lld matrix", who, (long long)rows, (long long)K);
  return UNETK_OK;
}

// Which kernel takes an M x N x K product: by sizes alone, so that activations quantised beforehand give the same bits.
// Times in us, bf16, replayed from a graph on the same operands (as all figures of the rules below).
//   rows against quantisation and split (short K): 1024 x 192 -> 768 5.8 and 5.8, 2048 rows 6.0 and 6.6; x 384 -> 1152: 1024 rows
//   7.2 and 6.8, 2048 7.6 and 8.1; x 768 -> 2304: 2048 rows 14.5 and 13.3, 4096 19.0 and 21.7: from 512 rows a step of K on;
//   large against split: 64 tiles (2048 x 2048) 28.2 and 24.3 with K = 4096, 14.5 and 9.6 with 1024; 96 tiles (2048 x 3000) 28.9
//   and 41.3, 15.1 and 14.2.  A side of 64 fills a quarter of its tiles: 64 x 4096 -> 65536 45.2 and 28.9, 65536 x 2048 -> 64 27.7
//   and 24.8; of 128: 128 x 2048 -> 65536 29.6 and 38.0, 65536 x 1024 -> 128 21.8 and 25.8.
enum Plan { SPLIT, ROWS, LARGE };
Plan plan_of(int64_t M, int64_t K, int64_t N) {
  const int64_t kt = (K + 127) / 128;
  if (kt <= 6 && M >= 512 * kt) return ROWS;
  if (M > 64 && N > 64 && ((M + 255) / 256) * ((N + 255) / 256) >= 96) return LARGE;
  return SPLIT;
}
// the split kernel's tile, 16 or 32 a side: 32 x 4096 -> 4096 4.4 and 4.9 us, 64 x 4096 -> 4096 5.6 and 5.2, 256 x 1024 -> 1024 3.7
// both, 512 x 4096 -> 512 5.6 and 5.2.  (64 a side: 1024 x 1024 -> 1024 7.5 against 4.7 with 32, 2048 x 4096 -> 2048 22.6 against 24.3.)
bool small_tiles(int64_t M, int64_t N) { return M * N < 1 << 18; }
// Activations quantised inside the product, by every tile of columns again, or by a launch of their own: bf16 1 x 4096 -> 4096
// 5.4 and 6.5 us, 4 x 4096 -> 4096 5.6 and 6.7, 8 x 4096 -> 4096 6.1 and 6.7, 16 x 2048 -> 2048 5.4 and 5.9, 16 x 4096 -> 4096 7.8 and 6.8;
// fp32 1 x 4096 -> 4096 6.3 and 6.6, 4 x 4096 -> 4096 7.0 and 6.7.  The rule does not see N: with many columns the launch of its own
// would win (4 x 4096 -> 16384 15.8 and 12.5, 8 x 4096 -> 65536 45.6 and 25.7).
bool quantised_inside(int64_t M, int64_t K, int64_t N, int dtype) {
  if (K % (dtype == UNETK_BF16 ? 8 : 4) != 0) return false;
  const Plan p = plan_of(M, K, N);
  if (p != SPLIT) return p == ROWS;
  return dtype == UNETK_BF16 ? M * K <= 32768 : M * K <= 16384 && small_tiles(M, N);
}

template <typename T, typename SRC, typename TILE> void launch_split(const MxArgs& a, hipStream_t stream) {
  // waves a tile: about 2048 in all, at least a step each (256 x 4096 -> 4096: 9.5 us with 1024, 7.7 with 2048, 8.7 with 4096; 1 x
  // 4096 -> 4096 4.1, 3.7, 4.0)
  const int64_t tiles = ((a.M + TILE::SIDE - 1) / TILE::SIDE) * (int64_t)((a.N + TILE::SIDE - 1) / TILE::SIDE);
  int W = 1;
  while (W < 16 && tiles * W < 2048 && (uint32_t)W * 2 <= a.kt) W *= 2;
  const int fin = TILE::SIDE == 32 ? 2 : 1, parts = W / 2 > fin ? W / 2 : W < fin ? W : fin;
  hipLaunchKernelGGL((mx_split_kernel<T, SRC, TILE>), dim3((unsigned)tiles), dim3(64 * W), W > 1 ? parts * TILE::NA * 1024 : 0, stream, a);
}
template <typename T, typename SRC> void launch_split_f(const MxArgs& a, hipStream_t stream) {
  if (small_tiles(a.M, a.N)) launch_split<T, SRC, Tile16>(a, stream);
  else if constexpr (!std::is_same<SRC, float>::value) launch_split<T, SRC, Tile32>(a, stream);      // (floats: never asked for)
}

template <typename T, typename SRC> void launch_rows(MxArgs& a, hipStream_t stream) {
  a.ngroups = (uint32_t)cdiv(a.N, 64);
  const uint32_t blocks = (uint32_t)cdiv(a.M, 64);
  // Whether four or eight waves share 64 rows (whole SIMDs: 65536 x 192 -> 576 26.9 us with four, 30.0 with five), and over how
  // many workgroups their columns are split, from what bounds the kernel, in cycles of a CU: its address path (about 100 for
  // a load or store whose lanes lie in many rows: 16 of a step's rows, 8 of a group's results; 33 for 1 KB of weights), and
  // the rounds of resident workgroups times a wave's own way through its share.  (262144 x 96 -> 384 75.5 with four waves, 81.7 with
  // eight; 16384 x 384 -> 1152 16.6 and 15.1; 4096 x 768 -> 2304 23.8 with eight, 16.6 split in two.)
  const double ks = a.kt, resident = 256.0 * (a.kt <= 2 ? 16 : a.kt <= 4 ? 12 : 8);
  uint32_t W = 4, splits = 1;
  double best = 1e30;
  const uint32_t s0 = (a.ngroups + 127) / 128;      // (at most 128 groups a workgroup: 32 KB of bias)
  for (uint32_t s = s0; s < s0 + 16 && s <= a.ngroups; ++s)
    for (uint32_t w = 4; w <= 8; w += 4) {
      const uint32_t per = (a.ngroups + s - 1) / s, used = (a.ngroups + per - 1) / per;
      const double path = blocks * (used * ks * 1600.0 + a.ngroups * (800.0 + ks * 140.0)) / 256.0;
      const double rounds = (double)blocks * used * w / resident;
      const double way = ((4 + w - 1) / w) * (1500.0 + ks * 500.0) + ((per + w - 1) / w) * (1800.0 + ks * 400.0);
      const double waves = (rounds > 1.0 ? rounds : 1.0) * way, cost = (path > waves ? path : waves) + 0.2 * (path + waves);
      if (cost < best) best = cost, W = w, splits = s;
    }
  a.per = (a.ngroups + splits - 1) / splits;
  splits = (a.ngroups + a.per - 1) / a.per;
  const dim3 grid((blocks * splits + 7) / 8 * 8), threads(64 * W);
  const unsigned lds = a.per * 256;      // the bias
  switch (a.kt) {
    case 1: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 1>), grid, threads, lds, stream, a); break;
    case 2: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 2>), grid, threads, lds, stream, a); break;
    case 3: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 3>), grid, threads, lds, stream, a); break;
    case 4: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 4>), grid, threads, lds, stream, a); break;
    case 5: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 5>), grid, threads, lds, stream, a); break;
    default: hipLaunchKernelGGL((mx_rows_kernel<T, SRC, 6>), grid, threads, lds, stream, a); break;
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
  UNETK_CHECK_ARG(act == 0 || act == 2, "mx_linear: activation %d", act);
  // (a launch has fewer than 2^32 lanes)
  UNETK_CHECK_ARG(N <= (int64_t)1 << 24 && M <= (int64_t)1 << 28 && M * N <= (int64_t)1 << 39, "mx_linear: %lld x %lld outputs",
                  (long long)M, (long long)N);
  MxArgs a = {};
  a.x = x; a.ldx = ldx;
  a.xc = (const u32x4*)xcodes; a.xs = (const uint32_t*)xscales; a.wc = (const u32x4*)wcodes; a.ws = (const uint32_t*)wscales;
  a.out = out; a.bias = bias; a.resid = resid; a.ldo = ldo; a.ldr = ldr; a.M = (uint32_t)M; a.N = (uint32_t)N;
  a.kt = (uint32_t)((K + 127) / 128); a.K = (int)K; a.act = act;
  a.whole = N % (dtype == UNETK_BF16 ? 8 : 4) == 0;
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
  const dim3 grid((unsigned)units_of(rows, (int)K));
  const bool whole = K % (dtype == UNETK_BF16 ? 8 : 4) == 0;
#define MX_QUANT(T, V)                                                                                                \
  hipLaunchKernelGGL((mx_quantize_kernel<T, V>), grid, dim3(256), 0, stream, (const T*)x, ldx, (uint32_t)rows, (int)K, kt, \
                     (u32x4*)codes, (uint8_t*)scales)
  if (dtype == UNETK_BF16) {
    if (whole) MX_QUANT(bf16, true);
    else MX_QUANT(bf16, false);
  } else {
    if (whole) MX_QUANT(float, true);
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
  const dim3 grid((unsigned)units_of(rows, (int)K));
  const bool whole = K % (dtype == UNETK_BF16 ? 8 : 4) == 0;
#define MX_DEQUANT(T, V)                                                                                              \
  hipLaunchKernelGGL((mx_dequantize_kernel<T, V>), grid, dim3(256), 0, stream, (const uint32_t*)codes, (const uint8_t*)scales, \
                     (uint32_t)rows, (int)K, kt, (T*)out, ldo)
  if (dtype == UNETK_BF16) {
    if (whole) MX_DEQUANT(bf16, true);
    else MX_DEQUANT(bf16, false);
  } else {
    if (whole) MX_DEQUANT(float, true);
    else MX_DEQUANT(float, false);
  }
#undef MX_DEQUANT
  UNETK_CHECK_LAUNCH();
  return UNETK_OK;
}

int64_t unetk_mx_linear_x_workspace_bytes(int64_t M, int64_t K, int64_t N, int dtype) {
  const int64_t codes = unetk_mx_codes_bytes(M, K);
  if (codes == 0 || N < 1 || N > MX_MAX_ROWS) return 0;
  return quantised_inside(M, K, N, dtype) ? 0 : codes + codes / 16;
}

int unetk_mx_linear_x(const void* x, int64_t ldx, const void* wcodes, const void* wscales, void* out, int64_t ldo, int64_t M,
                      int64_t K, int64_t N, const float* bias, int act, const void* resid, int64_t ldr, int dtype,
                      void* workspace, hipStream_t stream) {
  UNETK_CHECK_ARG(x && ldx >= K, "mx_linear_x: null activations or overlapping rows");
  const int64_t ws = unetk_mx_linear_x_workspace_bytes(M, K, N, dtype);
  if (ws == 0)
    return mx_linear_impl(x, ldx, nullptr, nullptr, wcodes, wscales, out, ldo, M, K, N, bias, act, resid, ldr, dtype, stream);
  UNETK_CHECK_ARG(workspace != nullptr, "mx_linear_x: this problem takes a workspace");
  const char* scales = (const char*)workspace + unetk_mx_codes_bytes(M, K);
  const int rc = unetk_mx_quantize(x, ldx, M, K, dtype, workspace, (void*)scales, stream);
  if (rc != UNETK_OK) return rc;
  return mx_linear_impl(nullptr, 0, workspace, scales, wcodes, wscales, out, ldo, M, K, N, bias, act, resid, ldr, dtype, stream);
}

int unetk_mx_linear(const void* xcodes, const void* xscales, const void* wcodes, const void* wscales, void* out, int64_t ldo,
                    int64_t M, int64_t K, int64_t N, const float* bias, int act, const void* resid, int64_t ldr, int dtype,
                    hipStream_t stream) {
  UNETK_CHECK_ARG(xcodes && xscales && aligned16(xcodes) && aligned16(xscales), "mx_linear: null or misaligned activations");
  return mx_linear_impl(nullptr, 0, xcodes, xscales, wcodes, wscales, out, ldo, M, K, N, bias, act, resid, ldr, dtype, stream);
}

}  // extern "C"
