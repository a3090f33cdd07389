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
// 16 (r / 4) + 4 f + r % 4 of its 64: with the weights as the instruction's first operand a lane's four accumulators over the four
// fragments are then 16 consecutive output columns.
#include "epilogue.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int frag_row(int f, int r) { return ((r >> 2) << 4) + (f << 2) + (r & 3); }

// 32 values -> 32 codes and the scale byte.  Everything is exact but the rounding itself: the scale is a power of two.
__device__ __forceinline__ uint32_t mx_block(const float (&v)[32], u32x4& codes) {
  uint32_t big = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu;
    big = b > big ? b : big;
  }
  const uint32_t ex = big >> 23;                           // biased exponent of the largest magnitude
  const uint32_t scale = ex == 255 ? 255u : (ex > 2 ? ex - 2 : 0u);
  const float inv = __builtin_bit_cast(float, (scale == 255 ? 127u : 254u - scale) << 23);      // 2^-(scale - 127)
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = v[q * 8 + j] * inv;
      const uint32_t u = __builtin_bit_cast(uint32_t, y), m = u & 0x7fffffffu;
      // from 1 on: the float's exponent and first mantissa bit, rounded half to even, are the code up to an offset;
      // below 1 the steps are halves
      uint32_t c = ((m + 0x1fffffu + ((m >> 22) & 1u)) >> 22) - 252u;
      if (m < 0x3f800000u) c = (uint32_t)__float2int_rn(2.0f * fabsf(y));
      c = c > 7u ? 7u : c;
      w |= (c | ((u >> 28) & 8u)) << (4 * j);
    }
    codes[q] = scale == 255 ? 0u : w;
  }
  return scale;
}

// 32 consecutive elements of a row, zeros past its end
template <typename T, bool VEC>
__device__ __forceinline__ void load_block(const T* row, int k0, int K, float (&v)[32]) {
  constexpr int E = Vec16<T>::N;
  if (VEC) {
#pragma unroll
    for (int j = 0; j < 32 / E; ++j) {
      const Vec16<T> r = k0 + j * E < K ? load16(row + k0 + j * E) : zero16<T>();
#pragma unroll
      for (int e = 0; e < E; ++e) v[j * E + e] = to_f32(r.v[e]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = k0 + j < K ? to_f32(row[k0 + j]) : 0.f;
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
    u32x4 c = {0u, 0u, 0u, 0u};
    if (row < rows && k0 < K) {
      float v[32];
      load_block<T, VEC>(x + (int64_t)row * ldx, k0, K, v);
      sc |= mx_block(v, c) << (8 * f);
    }
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
  void* out;
  const float* bias;
  const void* resid;
  int64_t ldo, ldr;
  uint32_t M, N, kt;      // rows, output columns, steps of 128 k
  int act, vec;
};


template <int FW, int FX> __device__ __forceinline__ f32x4 mma4(const u32x4& w, const u32x4& x, f32x4 c, uint32_t sw, uint32_t sx) {
#if defined(__HIP_DEVICE_COMPILE__)
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, FW, (int)sw, FX, (int)sx);
#else
  return c;
#endif
}

template <typename T> __device__ __forceinline__ float mx_act(float v, int act) {
  if (act == 1) return v > 0.f ? v : 0.f;
  if (act == 2) return sizeof(T) == 2 ? gelu_erf_g(v) : 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f));
  return v;
}

// bias, activation, residual and the store of a wave's 64 x 64 tile: row frag_row(fx, lane % 16) of its rows, columns
// 16 (lane / 16) + 4 fw + i of its columns
template <typename T>
__device__ __forceinline__ void mx_store(const MxArgs& a, uint32_t m0, uint32_t n0, const f32x4 (&acc)[4][4], int lane) {
  constexpr int E = Vec16<T>::N;
  const uint32_t n = n0 + (lane >> 4) * 16;
  float b[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) b[j] = (a.bias != nullptr && n + j < a.N) ? a.bias[n + j] : 0.f;
#pragma unroll
  for (int fx = 0; fx < 4; ++fx) {
    const uint32_t m = m0 + frag_row(fx, lane & 15);
    if (m >= a.M) continue;
    T* o = reinterpret_cast<T*>(a.out) + (int64_t)m * a.ldo + n;
    const T* rs = a.resid != nullptr ? reinterpret_cast<const T*>(a.resid) + (int64_t)m * a.ldr + n : nullptr;
#pragma unroll
    for (int j = 0; j < 16 / E; ++j) {
      Vec16<T> v, r = zero16<T>();
      if (rs != nullptr) {
        if (a.vec) {
          if (n + j * E < a.N) r = load16(rs + j * E);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (n + j * E + e < a.N) r.v[e] = rs[j * E + e];
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = j * E + e;
        v.v[e] = from_f32<T>(mx_act<T>(acc[i / 4][fx][i % 4] + b[i], a.act) + to_f32(r.v[e]));
      }
      if (a.vec) {
        if (n + j * E < a.N) store16(o + j * E, v);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (n + j * E + e < a.N) o[j * E + e] = v.v[e];
      }
    }
  }
}

// 128 x 128 of the output a workgroup, 64 x 64 a wave, fragments straight from memory
template <typename T>
__global__ __launch_bounds__(256) void mx_linear_kernel(MxArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t mg = blockIdx.x * 2 + (wave & 1), ng = blockIdx.y * 2 + (wave >> 1);
  if (mg * 64 >= a.M || ng * 64 >= a.N) return;
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const u32x4* xc = a.xc + (uint64_t)mg * a.kt * 256 + lane;
  const u32x4* wc = a.wc + (uint64_t)ng * a.kt * 256 + lane;
  const uint32_t* xs = a.xs + (uint64_t)mg * a.kt * 64 + lane;
  const uint32_t* ws = a.ws + (uint64_t)ng * a.kt * 64 + lane;
  for (uint32_t k = 0; k < a.kt; ++k) {
    u32x4 xf[4], wf[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      xf[f] = xc[(uint64_t)k * 256 + f * 64];
      wf[f] = wc[(uint64_t)k * 256 + f * 64];
    }
    const uint32_t sx = xs[(uint64_t)k * 64], sw = ws[(uint64_t)k * 64];
    static_for<4>([&](auto fw) __attribute__((always_inline)) {
      static_for<4>([&](auto fx) __attribute__((always_inline)) {
        constexpr int W = decltype(fw)::value, X = decltype(fx)::value;
        acc[W][X] = mma4<W, X>(wf[W], xf[X], acc[W][X], sw, sx);
      });
    });
  }
  mx_store<T>(a, mg * 64, ng * 64, acc, lane);
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

int unetk_mx_linear(const void* xcodes, const void* xscales, const void* wcodes, const void* wscales, void* out, int64_t ldo,
                    int64_t M, int64_t K, int64_t N, const float* bias, int act, const void* resid, int64_t ldr, int dtype,
                    hipStream_t stream) {
  int rc = check_mx("mx_linear", M, K, dtype);
  if (rc == UNETK_OK) rc = check_mx("mx_linear", N, K, dtype);
  if (rc != UNETK_OK) return rc;
  UNETK_CHECK_ARG(xcodes && xscales && wcodes && wscales && out && ldo >= N && (resid == nullptr || ldr >= N),
                  "mx_linear: null operand or overlapping rows");
  UNETK_CHECK_ARG(aligned16(xcodes) && aligned16(xscales) && aligned16(wcodes) && aligned16(wscales),
                  "mx_linear: misaligned packed operand");
  UNETK_CHECK_ARG(act >= 0 && act <= 2, "mx_linear: activation %d", act);
  MxArgs a = {};
  a.xc = (const u32x4*)xcodes; a.xs = (const uint32_t*)xscales; a.wc = (const u32x4*)wcodes; a.ws = (const uint32_t*)wscales;
  a.out = out; a.bias = bias; a.resid = resid; a.ldo = ldo; a.ldr = ldr; a.M = (uint32_t)M; a.N = (uint32_t)N;
  a.kt = (uint32_t)((K + 127) / 128); a.act = act;
  const int E = dtype == UNETK_BF16 ? 8 : 4;
  a.vec = N % E == 0 && ldo % E == 0 && aligned16(out) && (!resid || (ldr % E == 0 && aligned16(resid)));
  UNETK_CHECK_ARG(cdiv(N, 128) <= 65535, "mx_linear: %lld output columns", (long long)N);
  const dim3 grid((unsigned)cdiv(M, 128), (unsigned)cdiv(N, 128));
  if (dtype == UNETK_BF16) hipLaunchKernelGGL(mx_linear_kernel<bf16>, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(mx_linear_kernel<float>, grid, dim3(256), 0, stream, a);
  UNETK_CHECK_LAUNCH();
  return UNETK_OK;
}

}  // extern "C"
