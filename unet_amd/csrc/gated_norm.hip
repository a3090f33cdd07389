// Norm behind a branch, gate, residual and norm in front of the next branch, in one pass each way (gfx950).
//
//   h = post(f) (or f)      r = res_scale * x + keep[sample] * gate * h      n = pre(r)
//
// post and pre are LayerNorm ((v - mean) * rstd * w + b) or RMSNorm (v * rms * w + b) over the C channels of a row;
// f is the branch's output, x the residual stream, keep the DropPath factor of the row's sample, gate one factor a
// channel.  Backward, from dr (the residual stream's gradient) and dn:
//   rhat = (r - mean) rstd, q = dn w_pre:   g = dr + rstd (q - mean(q) - rhat mean(q rhat)),  dx = res_scale g
//   u = keep g:  dgate = sum u h, dh = u gate;   fhat = (f - mean) rstd, p = dh w_post:
//   df = rstd (p - mean(p) - fhat mean(p fhat));  dw_pre = sum dn rhat, db_pre = sum dn, dw_post = sum dh fhat, db_post = sum dh
// (RMSNorm: no means of v, q and p.)  HBM-bound: the forward pass moves 4 tensors, the backward pass 6, a few dozen
// operations an element.  All arithmetic is fp32; r, n, dx, df are rounded once, when they are stored.  n comes from the
// unrounded r (which is in registers), and the backward pass forms r again from x and f for the same reason: it reads
// as many bytes as with a stored r.
//
// Measured (MI355X; a large copy reaches 5.0 TB/s here; the kernel alone, operands out of the caches), bf16 unless noted:
// forward 262144 x 96 43.7 us (4.6 TB/s), 65536 x 192 27.5 us (3.7), 8192 x 4096 RMS 52.0 us (5.2); backward 65536 x 192 30.7 us
// (4.9 TB/s), 8192 x 4096 72.8 us (5.5), each followed by 5...8 us of column sums; 5003 x 1001 fp32 19.0, 26.4 and 6.6 us (4.2
// and 4.6 TB/s); 64 x 768 forward 7.3 us (5.4 with its operands in the caches), which is a launch and one pass through the loads.
//
// Infinities and NaN stay in their row, and in the column sums of their channels.  (With a bias behind the branch dgate is two
// sums' combination: where both are infinite it may be NaN for an infinity of the definition.)
#include "unaligned.h"

namespace {

struct NormArgs {
  const void* x;
  const void* f;
  const void* dr;
  const void* dn;
  int64_t ldx, ldf, lddr, lddn;
  const float *gate, *keep, *post_w, *post_b, *pre_w, *pre_b;
  const float* stats_in;
  float* stats_out;      // [M][4]: mean and rstd of f, mean and rstd of r
  void* o0;              // r / dx
  void* o1;              // n / df
  float* partials;       // [workgroups][4][C]
  uint32_t M, rps;       // rows; rows per sample
  int C, rms;
  float res_scale, post_eps, pre_eps;
};

// The elements of a row that one of its G lanes holds: N = NV 16-byte vectors, at whatever address the row begins.
// WHOLE: C is a multiple of the vector's elements; else the lanes take single elements side by side (20000 x 1001 bf16
// forward: 44.4 us so, 59.2 with vectors off their alignment; 5003 x 1001 fp32: 17.2 and 22.0; operands cached).
template <typename T, int G, int NV, bool WHOLE> struct Lane {
  static constexpr int E = Vec16<T>::N, N = NV * E;
  static constexpr bool SINGLE = !WHOLE;
  int gl, C;
  __device__ __forceinline__ int chan(int i) const { return SINGLE ? i * G + gl : ((i / E) * G + gl) * E + i % E; }
  __device__ __forceinline__ bool has(int i) const { return WHOLE ? ((i / E) * G + gl) * E < C : chan(i) < C; }
  struct Raw {
    Vec16<T> v[NV];
  };
  __device__ __forceinline__ void load(Raw& r, const T* row) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (SINGLE) {
        r.v[k] = zero16<T>();
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (has(k * E + e)) r.v[k].v[e] = row[chan(k * E + e)];
      } else {
        r.v[k] = load_part<true>(row + chan(k * E), C - chan(k * E));
      }
    }
  }
  static __device__ __forceinline__ float at(const Raw& r, int i) { return to_f32(r.v[i / E].v[i % E]); }
  __device__ __forceinline__ void store(T* row, const float (&d)[N]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (SINGLE) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (has(k * E + e)) row[chan(k * E + e)] = from_f32<T>(d[k * E + e]);
      } else {
        Vec16<T> o;
#pragma unroll
        for (int e = 0; e < E; ++e) o.v[e] = from_f32<T>(d[k * E + e]);
        store_part<true>(row + chan(k * E), o, C - chan(k * E));
      }
    }
  }
  __device__ __forceinline__ void param(float (&d)[N], const float* p, float none) const {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = (p != nullptr && has(i)) ? p[chan(i)] : none;
  }
};

constexpr int threads_of(int G) { return G > 256 ? G : 256; }

// v plus its partner's: lanes 1, 2, 4 and 8 apart inside a row of 16 through DPP (the last two as mirrors: by then all
// lanes of a half hold the same sum), 16 through the swizzle, 32 by reading the two halves' sums as scalars.
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  const int i = __builtin_bit_cast(int, v);
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, true));
}
template <int W> __device__ __forceinline__ float lane_sum(float v) {
  if (W >= 2) v = dpp_add<0xB1>(v);
  if (W >= 4) v = dpp_add<0x4E>(v);
  if (W >= 8) v = dpp_add<0x141>(v);
  if (W >= 16) v = dpp_add<0x140>(v);
  if (W >= 32)
    v += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F));      // lane ^ 16
  if (W >= 64) {
    const int i = __builtin_bit_cast(int, v);
    v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 0)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 32));
  }
  return v;
}

// Sums over the G lanes of a row.  Rows of more than a wave go through LDS (two areas in turn: the barrier of the next
// call is what frees this one's).
template <int G> struct RowSum {
  float (*red)[2][threads_of(G) / 64];
  int phase = 0;
  __device__ __forceinline__ void sum2(float& a, float& b) {
    constexpr int W = G < 64 ? G : 64;
    a = lane_sum<W>(a);
    b = lane_sum<W>(b);
    if (G > 64) {
      constexpr int WPR = G / 64;
      const int wave = threadIdx.x >> 6, w0 = wave / WPR * WPR;
      if ((threadIdx.x & 63) == 0) {
        red[phase][0][wave] = a;
        red[phase][1][wave] = b;
      }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) {
        a += red[phase][0][w0 + w];
        b += red[phase][1][w0 + w];
      }
      phase ^= 1;
    }
  }
  __device__ __forceinline__ float sum(float a) {
    if (G <= 64) return lane_sum<(G < 64 ? G : 64)>(a);
    float b = 0.f;
    sum2(a, b);
    return a;
  }
};

// mean (0 for RMSNorm) and 1 / sqrt(mean square distance from it + eps) of the row whose elements the lanes hold: from
// registers, in two passes, so that rows far from zero keep their digits
template <typename L, int G>
__device__ __forceinline__ void moments(const L& ln, const float (&v)[L::N], RowSum<G>& rs, const NormArgs& a, float eps,
                                        float inv_c, float& mean, float& rstd) {
  mean = 0.f;
  if (!a.rms) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < L::N; ++i) s += v[i];
    mean = rs.sum(s) / (float)a.C;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < L::N; ++i) {
    const float d = ln.has(i) ? v[i] - mean : 0.f;
    q += d * d;
  }
  rstd = 1.0f / sqrtf(rs.sum(q) * inv_c + eps);
}

// One element of r, in the operations that both directions use (explicit fused multiply-adds: whatever the compiler
// would contract in each, the backward pass finds the bits of the forward pass, and rows whose deviation is nothing but
// rounding keep it).  gw = gate w_post, gb = gate b_post.
__device__ __forceinline__ float norm_hat(float v, float mean, float rstd) { return (v - mean) * rstd; }
__device__ __forceinline__ float residual(float x, float fhat, float gw, float gb, float keep, float scale) {
  return fmaf(keep, fmaf(fhat, gw, gb), x * scale);
}

template <typename T, int G, int NV, bool WHOLE>
__global__ __launch_bounds__(threads_of(G)) void gated_norm_fwd_kernel(NormArgs a) {
  using L = Lane<T, G, NV, WHOLE>;
  constexpr int N = L::N, RPB = threads_of(G) / G;
  __shared__ float red[2][2][threads_of(G) / 64];
  RowSum<G> rs{red};
  const L ln{(int)(threadIdx.x % G), a.C};
  const uint32_t rg = threadIdx.x / G;
  const float inv_c = 1.0f / (float)a.C;
  const bool post = a.post_w != nullptr, pre = a.pre_w != nullptr;
  // gate * (fhat * w_post + b_post) = fhat * (gate w_post) + gate b_post, the second term 0 without a bias (a gate may be
  // infinite, and infinity times zero is NaN)
  float qw[N], qb[N], pw[N], pb[N];
  {
    float gate[N];
    ln.param(gate, a.gate, 1.f);
    ln.param(qw, a.post_w, 1.f);
    ln.param(qb, a.post_b, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) qw[i] *= gate[i], qb[i] = a.post_b != nullptr ? qb[i] * gate[i] : 0.f;
  }
  ln.param(pw, a.pre_w, 1.f);
  ln.param(pb, a.pre_b, 0.f);
  // the next row is on its way while this one is reduced
  typename L::Raw xn, fn;
  auto fetch = [&](uint32_t row0) __attribute__((always_inline)) {
    const uint32_t row = row0 + rg < a.M ? row0 + rg : a.M - 1;
    ln.load(xn, reinterpret_cast<const T*>(a.x) + (int64_t)row * a.ldx);
    ln.load(fn, reinterpret_cast<const T*>(a.f) + (int64_t)row * a.ldf);
  };
  const uint32_t step = gridDim.x * RPB;
  if (blockIdx.x * RPB < a.M) fetch(blockIdx.x * RPB);
  for (uint32_t row0 = blockIdx.x * RPB; row0 < a.M; row0 += step) {      // (the same trips for every wave)
    const bool live = row0 + rg < a.M;
    const uint32_t row = live ? row0 + rg : row0;
    const typename L::Raw xr = xn, fr = fn;
    if (row0 + step < a.M) fetch(row0 + step);
    const float keep = a.keep != nullptr ? a.keep[row / a.rps] : 1.f;
    float h[N], r[N];
    float fm = 0.f, fs = 0.f, rm = 0.f, rsd = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = L::at(fr, i);
    if (post) moments(ln, h, rs, a, a.post_eps, inv_c, fm, fs);
    const float hs = post ? fs : 1.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      r[i] = ln.has(i) ? residual(L::at(xr, i), norm_hat(h[i], fm, hs), qw[i], qb[i], keep, a.res_scale) : 0.f;
    if (live) ln.store(reinterpret_cast<T*>(a.o0) + (int64_t)row * a.C, r);
    if (pre) {
      moments(ln, r, rs, a, a.pre_eps, inv_c, rm, rsd);
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = norm_hat(r[i], rm, rsd) * pw[i] + pb[i];
      if (live) ln.store(reinterpret_cast<T*>(a.o1) + (int64_t)row * a.C, r);
    }
    if (a.stats_out != nullptr && live && ln.gl == 0)
      *reinterpret_cast<f32x4*>(a.stats_out + 4 * (int64_t)row) = f32x4{fm, fs, rm, rsd};
  }
}

// Each workgroup walks rows blockIdx.x * RPB, + gridDim.x * RPB, ... and keeps its share of four sums a channel in
// registers: dn rhat, dn, u fhat and u (u = keep g; without a norm behind the branch fhat is f).  The gradients of gate,
// w_post and b_post are these times constants of the channel: dgate = w_post sum(u fhat) + b_post sum(u), dw_post = gate
// sum(u fhat), db_post = gate sum(u).  The sums leave as one [4][C] row of partials a workgroup, added in a fixed order by
// column_sums_kernel: no atomics, the same bits every time.
template <typename T, int G, int NV, bool WHOLE>
__global__ __launch_bounds__(threads_of(G)) void gated_norm_bwd_kernel(NormArgs a) {
  using L = Lane<T, G, NV, WHOLE>;
  constexpr int N = L::N, RPB = threads_of(G) / G;
  __shared__ float red[2][2][threads_of(G) / 64];
  __shared__ float xch[RPB > 1 ? threads_of(G) * N : 1];
  RowSum<G> rs{red};
  const L ln{(int)(threadIdx.x % G), a.C};
  const uint32_t rg = threadIdx.x / G;
  const float inv_c = 1.0f / (float)a.C;
  const bool post = a.post_w != nullptr, pre = a.pre_w != nullptr;
  // gate w_post, gate b_post, w_pre of this lane's channels: in registers, or, where a lane holds 16 channels and the
  // registers do not suffice, in LDS (each lane reads back only what it wrote itself)
  constexpr bool PL = N > 8;
  float preg[PL ? 1 : 3][N];
  __shared__ float plds[PL ? 3 : 1][PL ? N * G : 1];
  auto put = [&](int s, const float (&d)[N]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (PL) plds[s][i * G + ln.gl] = d[i];
      else preg[PL ? 0 : s][i] = d[i];
    }
  };
  auto prm = [&](int s, int i) __attribute__((always_inline)) { return PL ? plds[s][i * G + ln.gl] : preg[PL ? 0 : s][i]; };
  {
    float gate[N], w[N];
    ln.param(gate, a.gate, 1.f);
    ln.param(w, a.post_w, 1.f);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] *= gate[i];
    put(0, w);
    ln.param(w, a.post_b, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = a.post_b != nullptr ? w[i] * gate[i] : 0.f;
    put(1, w);
    ln.param(w, a.pre_w, 0.f);
    put(2, w);
  }
  float acc[4][N];
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < N; ++i) acc[s][i] = 0.f;
  // the next row is on its way while this one is reduced
  struct Next {
    typename L::Raw x, f, dr, dn;
    f32x4 st;
    float keep;
  } nx;
  auto fetch = [&](uint32_t row0) __attribute__((always_inline)) {
    const uint32_t row = row0 + rg < a.M ? row0 + rg : a.M - 1;
    nx.st = *reinterpret_cast<const f32x4*>(a.stats_in + 4 * (int64_t)row);
    nx.keep = a.keep != nullptr ? a.keep[row / a.rps] : 1.f;
    ln.load(nx.f, reinterpret_cast<const T*>(a.f) + (int64_t)row * a.ldf);
    if (pre) {
      ln.load(nx.x, reinterpret_cast<const T*>(a.x) + (int64_t)row * a.ldx);
      ln.load(nx.dn, reinterpret_cast<const T*>(a.dn) + (int64_t)row * a.lddn);
    }
    if (a.dr != nullptr) {
      ln.load(nx.dr, reinterpret_cast<const T*>(a.dr) + (int64_t)row * a.lddr);
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k) nx.dr.v[k] = zero16<T>();
    }
  };
  const uint32_t step = gridDim.x * RPB;
  if (blockIdx.x * RPB < a.M) fetch(blockIdx.x * RPB);
  for (uint32_t row0 = blockIdx.x * RPB; row0 < a.M; row0 += step) {
    const bool live = row0 + rg < a.M;
    const uint32_t row = live ? row0 + rg : row0;
    const typename L::Raw xr = nx.x, dr = nx.dr, dn = nx.dn;
    typename L::Raw fr = nx.f;
    if (RPB > 1) {      // (lanes past the last row hold its values again: zero times an infinite one would be NaN)
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        u32x4 v = __builtin_bit_cast(u32x4, fr.v[k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = live ? v[e] : 0u;
        fr.v[k] = __builtin_bit_cast(Vec16<T>, v);
      }
    }
    const f32x4 st = nx.st;
    const float keep = nx.keep;
    if (row0 + step < a.M) fetch(row0 + step);
    const float fm = post ? st[0] : 0.f, fs = post ? st[1] : 1.f;
    float g[N];
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = L::at(dr, i);
    if (pre) {
      float s1 = 0.f, s2 = 0.f, rhat[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float r = residual(L::at(xr, i), norm_hat(L::at(fr, i), fm, fs), prm(0, i), prm(1, i), keep, a.res_scale);
        rhat[i] = ln.has(i) ? norm_hat(r, st[2], st[3]) : 0.f;
        const float d = live ? L::at(dn, i) : 0.f, q = d * prm(2, i);
        acc[0][i] += d * rhat[i];
        acc[1][i] += d;
        s1 += q;
        s2 += q * rhat[i];
      }
      rs.sum2(s1, s2);
      s1 = a.rms ? 0.f : s1 * inv_c;
      s2 *= inv_c;
#pragma unroll
      for (int i = 0; i < N; ++i) g[i] += st[3] * (L::at(dn, i) * prm(2, i) - s1 - rhat[i] * s2);
    }
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = a.res_scale * g[i];
    if (live) ln.store(reinterpret_cast<T*>(a.o0) + (int64_t)row * a.C, o);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float u = (live && ln.has(i)) ? keep * g[i] : 0.f, fh = norm_hat(L::at(fr, i), fm, fs);
      acc[2][i] += u * fh;
      acc[3][i] += u;
      o[i] = u * prm(0, i);
      s1 += o[i];
      s2 += o[i] * fh;
    }
    if (post) {
      rs.sum2(s1, s2);
      s1 = a.rms ? 0.f : s1 * inv_c;
      s2 *= inv_c;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = fs * (o[i] - s1 - norm_hat(L::at(fr, i), fm, fs) * s2);
    }
    if (live) ln.store(reinterpret_cast<T*>(a.o1) + (int64_t)row * a.C, o);
  }
  float* out = a.partials + (int64_t)blockIdx.x * 4 * a.C;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    if (s < 2 && !pre) continue;      // (uniform)
    if (RPB == 1) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (ln.has(i)) out[s * a.C + ln.chan(i)] = acc[s][i];
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) xch[(rg * N + i) * G + ln.gl] = acc[s][i];
      __syncthreads();
      for (int j = threadIdx.x; j < N * G; j += threads_of(G)) {
        const L lj{j % G, a.C};
        const int i = j / G;
        float t = 0.f;
        for (int w = 0; w < RPB; ++w) t += xch[w * N * G + j];
        if (lj.has(i)) out[s * a.C + lj.chan(i)] = t;
      }
    }
  }
}

// Sums of partials [rows][4][C] down the rows, in double, and the gradients made of them: blockIdx.y 0: the norm in front
// (d0: weight, d1: bias), 1: gate, weight and bias of the norm behind (d2, d3, d4).  16 columns a workgroup, 32 row lanes a
// sum with eight loads in flight each (a few MB that were just written: latency, not bytes; rows past the end load the last
// one, since a condition would turn the eight into branches: the whole backward call at 65536 x 192 41.8 us with it, 37...40
// without; 8 columns a workgroup take 8192 x 4096 from 87 to 93).
struct SumArgs {
  float *d0, *d1, *d2, *d3, *d4;
  const float *gate, *post_w, *post_b;
};
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* __restrict__ partials, int rows, int C, SumArgs o) {
  __shared__ double red[2][32][17];
  const bool behind = blockIdx.y != 0;
  if (behind ? !(o.d2 || o.d3 || o.d4) : !(o.d0 || o.d1)) return;
  const int cl = threadIdx.x & 15, which = (threadIdx.x >> 4) & 1, rl = threadIdx.x >> 5, col = blockIdx.x * 16 + cl;
  double t = 0.0;
  if (col < C) {
    const float* p = partials + (int64_t)(2 * blockIdx.y + which) * C + col;
    for (int r0 = rl; r0 < rows; r0 += 32 * 8) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = p[(int64_t)min(r0 + 32 * j, rows - 1) * 4 * C];
#pragma unroll
      for (int j = 0; j < 8; ++j) t += r0 + 32 * j < rows ? (double)v[j] : 0.0;
    }
  }
  red[which][rl][cl] = t;
  __syncthreads();
  if (threadIdx.x >= 64) return;      // one wave adds: lane = (half of the row lanes, sum, column)
  {
    const int half = threadIdx.x >> 5;
    t = 0.0;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += red[which][half * 16 + w][cl];
    t += __shfl_xor(t, 32, 64);
    const double other = __shfl_xor(t, 16, 64);
    if (threadIdx.x >= 16 || col >= C) return;
    if (!behind) {
      if (o.d0) o.d0[col] = (float)t;
      if (o.d1) o.d1[col] = (float)other;
    } else {
      const double gate = o.gate ? (double)o.gate[col] : 1.0;
      if (o.d2) {      // (an absent bias adds no term: a sum may be infinite, and infinity times zero is NaN)
        double d = t * (o.post_w ? (double)o.post_w[col] : 1.0);
        if (o.post_b) d += other * (double)o.post_b[col];
        o.d2[col] = (float)d;
      }
      if (o.d3) o.d3[col] = (float)(gate * t);
      if (o.d4) o.d4[col] = (float)(gate * other);
    }
  }
}

constexpr int NORM_MAX_C = 8192;

// lanes a row and 8-element groups a lane: the fewest lanes that hold the row in eight elements each, from four lanes
// up to eight waves
struct Shape {
  int G, K;
};
Shape norm_shape(int C) {
  const int need = (C + 7) / 8;
  int G = 4;
  while (G < need && G < 512) G *= 2;
  return {G, (need + G - 1) / G > 1 ? 2 : 1};
}

unsigned norm_grid(int64_t M, int C, int cap) {
  const int rpb = threads_of(norm_shape(C).G) / norm_shape(C).G;
  const int64_t b = (M + rpb - 1) / rpb;
  return (unsigned)(b < cap ? b : cap);
}

#define NORM_LAUNCH(KERNEL, T, G_, K_, WHOLE_)                                                                  \
  hipLaunchKernelGGL((KERNEL<T, G_, K_ * (8 / Vec16<T>::N), WHOLE_>), dim3(grid), dim3(threads_of(G_)), 0, stream, a)
#define NORM_TAIL(KERNEL, T, G_, K_)              \
  do {                                           \
    if (whole) NORM_LAUNCH(KERNEL, T, G_, K_, true); \
    else NORM_LAUNCH(KERNEL, T, G_, K_, false);  \
  } while (0)
#define NORM_DISPATCH(KERNEL, T)                                   \
  do {                                                             \
    const Shape sh = norm_shape(a.C);                              \
    switch (sh.G) {                                                \
      case 4: NORM_TAIL(KERNEL, T, 4, 1); break;                    \
      case 8: NORM_TAIL(KERNEL, T, 8, 1); break;                    \
      case 16: NORM_TAIL(KERNEL, T, 16, 1); break;                  \
      case 32: NORM_TAIL(KERNEL, T, 32, 1); break;                  \
      case 64: NORM_TAIL(KERNEL, T, 64, 1); break;                  \
      case 128: NORM_TAIL(KERNEL, T, 128, 1); break;                \
      case 256: NORM_TAIL(KERNEL, T, 256, 1); break;                \
      default:                                                     \
        if (sh.K == 1) NORM_TAIL(KERNEL, T, 512, 1);                \
        else NORM_TAIL(KERNEL, T, 512, 2);                          \
    }                                                              \
  } while (0)

int check_norm(const char* who, int64_t M, int C, int dtype, const float* keep, int64_t rps) {
  UNETK_CHECK_ARG(dtype == UNETK_F32 || dtype == UNETK_BF16, "%s: unsupported dtype %d", who, dtype);
  UNETK_CHECK_ARG(C >= 1 && C <= NORM_MAX_C, "%s: C=%d (1...%d)", who, C, NORM_MAX_C);
  UNETK_CHECK_ARG(M >= 1 && M < ((int64_t)1 << 31) - (1 << 20), "%s: %lld rows", who, (long long)M);
  UNETK_CHECK_ARG(keep == nullptr || (rps >= 1 && M % rps == 0), "%s: %lld rows are not whole samples of %lld", who,
                  (long long)M, (long long)rps);
  return UNETK_OK;
}

}  // namespace

extern "C" {

int unetk_gated_norm_max_channels(void) { return NORM_MAX_C; }

int unetk_gated_norm_fwd_eps(const void* x, int64_t ldx, const void* f, int64_t ldf, const float* gate, const float* keep,
                             int64_t rows_per_sample, float res_scale, const float* post_w, const float* post_b,
                             const float* pre_w, const float* pre_b, int rms, float post_eps, float pre_eps, void* r, void* n,
                             float* stats, int64_t M, int C, int dtype, hipStream_t stream) {
  const int rc = check_norm("gated_norm_fwd", M, C, dtype, keep, rows_per_sample);
  if (rc != UNETK_OK) return rc;
  UNETK_CHECK_ARG(x && f && r && ldx >= C && ldf >= C, "gated_norm_fwd: null operand or overlapping rows");
  UNETK_CHECK_ARG((pre_w != nullptr) == (n != nullptr), "gated_norm_fwd: n goes with the norm in front");
  UNETK_CHECK_ARG((post_w || !post_b) && (pre_w || !pre_b), "gated_norm_fwd: a norm's bias without its weight");
  NormArgs a = {};
  a.x = x; a.f = f; a.ldx = ldx; a.ldf = ldf; a.gate = gate; a.keep = keep; a.post_w = post_w; a.post_b = post_b;
  a.pre_w = pre_w; a.pre_b = pre_b; a.stats_out = stats; a.o0 = r; a.o1 = n; a.M = (uint32_t)M;
  a.rps = keep ? (uint32_t)rows_per_sample : 1; a.C = C; a.rms = rms; a.res_scale = res_scale;
  a.post_eps = post_eps; a.pre_eps = pre_eps;
  const bool whole = C % (dtype == UNETK_BF16 ? 8 : 4) == 0;
  // about what the chip holds at once, so that a workgroup has many rows to fetch ahead over (262144 x 96: 43.2 us with
  // 1536, 50.1 with 4096; 8192 x 4096: 47.9 with 1024, 49.1 with 1536, 53.4 with 4096)
  const unsigned grid = norm_grid(M, C, norm_shape(C).G > 64 ? 1024 : 1536);
  if (dtype == UNETK_BF16) NORM_DISPATCH(gated_norm_fwd_kernel, bf16);
  else NORM_DISPATCH(gated_norm_fwd_kernel, float);
  UNETK_CHECK_LAUNCH();
  return UNETK_OK;
}

int unetk_gated_norm_fwd(const void* x, int64_t ldx, const void* f, int64_t ldf, const float* gate, const float* keep,
                         int64_t rows_per_sample, float res_scale, const float* post_w, const float* post_b,
                         const float* pre_w, const float* pre_b, int rms, float eps, void* r, void* n, float* stats,
                         int64_t M, int C, int dtype, hipStream_t stream) {
  return unetk_gated_norm_fwd_eps(x, ldx, f, ldf, gate, keep, rows_per_sample, res_scale, post_w, post_b, pre_w, pre_b, rms, eps,
                                  eps, r, n, stats, M, C, dtype, stream);
}

int unetk_gated_norm_bwd_rows(int64_t M, int C) {
  // As many workgroups as the chip holds at once (three a CU; two where a row takes several waves and another 10
  // registers, one where it takes eight): each leaves a row of partials.  65536 x 192: 40.6 us with 768, 55.1 with 256;
  // 5003 x 1001 fp32: 34.8 with 512, 42.6 with 768; 8192 x 4096: 83.7 with 256, 94.5 with 768.
  if (M < 1 || C < 1 || C > NORM_MAX_C) return 0;
  const int G = norm_shape(C).G;
  return (int)norm_grid(M, C, G > 256 ? 256 : G > 64 ? 512 : 768);
}

int unetk_gated_norm_bwd(const void* dr, int64_t lddr, const void* dn, int64_t lddn, const void* x, int64_t ldx,
                         const void* f, int64_t ldf, const float* stats, const float* gate, const float* keep,
                         int64_t rows_per_sample, float res_scale, const float* post_w, const float* post_b,
                         const float* pre_w, int rms, void* dx, void* df, float* dgate, float* dpost_w, float* dpost_b,
                         float* dpre_w, float* dpre_b, float* partials, int64_t M, int C, int dtype, hipStream_t stream) {
  const int rc = check_norm("gated_norm_bwd", M, C, dtype, keep, rows_per_sample);
  if (rc != UNETK_OK) return rc;
  UNETK_CHECK_ARG(x && f && stats && dx && df && partials && ldx >= C && ldf >= C && (dr || dn),
                  "gated_norm_bwd: null operand or overlapping rows");
  UNETK_CHECK_ARG((dr == nullptr || lddr >= C) && (dn == nullptr || lddn >= C), "gated_norm_bwd: overlapping rows");
  UNETK_CHECK_ARG((pre_w != nullptr) == (dn != nullptr), "gated_norm_bwd: dn goes with the norm in front");
  UNETK_CHECK_ARG((gate || !dgate) && (post_w || !(post_b || dpost_w || dpost_b)) && (pre_w || !(dpre_w || dpre_b)),
                  "gated_norm_bwd: a gradient of a parameter that is not there");
  NormArgs a = {};
  a.x = x; a.f = f; a.dr = dr; a.dn = dn; a.ldx = ldx; a.ldf = ldf; a.lddr = lddr; a.lddn = lddn; a.gate = gate;
  a.keep = keep; a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.stats_in = stats; a.o0 = dx; a.o1 = df;
  a.partials = partials; a.M = (uint32_t)M; a.rps = keep ? (uint32_t)rows_per_sample : 1; a.C = C; a.rms = rms;
  a.res_scale = res_scale;
  const bool whole = C % (dtype == UNETK_BF16 ? 8 : 4) == 0;
  const unsigned grid = (unsigned)unetk_gated_norm_bwd_rows(M, C);
  if (dtype == UNETK_BF16) NORM_DISPATCH(gated_norm_bwd_kernel, bf16);
  else NORM_DISPATCH(gated_norm_bwd_kernel, float);
  UNETK_CHECK_LAUNCH();
  if (dgate || dpost_w || dpost_b || dpre_w || dpre_b) {
    const SumArgs o = {dpre_w, dpre_b, dgate, dpost_w, dpost_b, gate, post_w, post_b};
    hipLaunchKernelGGL(column_sums_kernel, dim3(cdiv(C, 16), 2), dim3(1024), 0, stream, partials, (int)grid, C, o);
    UNETK_CHECK_LAUNCH();
  }
  return UNETK_OK;
}

}  // extern "C"
