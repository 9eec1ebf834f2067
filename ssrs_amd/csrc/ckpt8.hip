// 8-bit activation checkpoints and their use in the backward pass (format: ckpt8.h):
//
//   pack / unpack        a tensor into its checkpoint and back
//   gelu                 act = x Phi(x), checkpoint of x;      dx = dy (Phi(x8) + x8 phi(x8)), optionally act again
//   layernorm            y = (x - mean) rstd gamma + beta, checkpoint of x, mean and rstd of the exact x;
//                        xh = (x8 - mean) rstd, t = dy gamma: dx = rstd (t - mean(t) - xh mean(t xh)) (+ dres),
//                        dgamma = sum_rows dy xh, dbeta = sum_rows dy, optionally y again from xh
//
// All are bound by memory: every operand is streamed once, 16 bytes per lane and request, and the codes cost 33/32 byte per element
// instead of the 2 (bf16) or 4 (fp32, LayerNorm's input) that the backward would read otherwise.
#include "ckpt8.h"

// ------------------------------------------------------------------------------------------------ GELU
// Phi(x) = erfc(-x / sqrt 2) / 2. erfc(z) = exp(-z^2) t P(t), t = 1 / (1 + 0.4 z), z = |x| / sqrt 2, P of degree 8: least squares on
// Chebyshev nodes over z in [0, 10], reweighted until the relative error is level (6.2e-8; 3.8e-7 with every step rounded to fp32).
// The error is RELATIVE also in the left tail, where an absolute 1.5e-7 (common.h) would be all of the value.
__device__ __forceinline__ float ck_half_erfc_exp(float x, float* e_out) {      // erfc(|x| / sqrt 2) / 2; *e_out = exp(-x^2 / 2)
  const float z = fabsf(x) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.4f, z, 1.0f));
  float p = fmaf(t, 0.041253041476011276f, -0.14031924307346344f);
  p = fmaf(p, t, 0.083987295627594f);
  p = fmaf(p, t, 0.08796432614326477f);
  p = fmaf(p, t, 0.07975649833679199f);
  p = fmaf(p, t, 0.19339320063591003f);
  p = fmaf(p, t, 0.2018875926733017f);
  p = fmaf(p, t, 0.2264431118965149f);
  p = fmaf(p, t, 0.22563423216342926f);
  const float e = __expf(-0.5f * x * x);
  *e_out = e;
  return 0.5f * p * t * e;
}
__device__ __forceinline__ float ck_gelu(float x) {
  float e;
  const float q = ck_half_erfc_exp(x, &e);
  return x * (x < 0.f ? q : 1.0f - q);
}
// act and slope share everything but the last steps
__device__ __forceinline__ float ck_gelu_slope(float x, float* act) {
  float e;
  const float q = ck_half_erfc_exp(x, &e);
  const float cdf = x < 0.f ? q : 1.0f - q;
  *act = x * cdf;
  return fmaf(x, 0.3989422804014327f * e, cdf);
}

// ------------------------------------------------------------------------------------------------ 8 elements of a row per lane
struct Vec8 { float v[8]; };
__device__ __forceinline__ Vec8 load8(const float* p) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ Vec8 load8(const bf16_t* p) {
  const u32x4_t w = *reinterpret_cast<const u32x4_t*>(p);
  return {{bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y), bf16_lo(w.z), bf16_hi(w.z), bf16_lo(w.w), bf16_hi(w.w)}};
}
__device__ __forceinline__ void store8(float* p, const Vec8& x) {
  *reinterpret_cast<float4*>(p) = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
}
__device__ __forceinline__ void store8(bf16_t* p, const Vec8& x) {
  u32x4_t w;
  w.x = pack_bf16x2(x.v[0], x.v[1]); w.y = pack_bf16x2(x.v[2], x.v[3]); w.z = pack_bf16x2(x.v[4], x.v[5]); w.w = pack_bf16x2(x.v[6], x.v[7]);
  *reinterpret_cast<u32x4_t*>(p) = w;
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const bf16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(bf16_t* p, float v) { *p = f32_to_bf16(v); }

__device__ __forceinline__ unsigned int umax3(unsigned int a, unsigned int b, unsigned int c) {
  const unsigned int m = a > b ? a : b;
  return m > c ? m : c;
}
// largest value among the 4 lanes of a quad (quad_perm 1,0,3,2 then 2,3,0,1)
__device__ __forceinline__ unsigned int quad_umax(unsigned int v) {
  unsigned int o = (unsigned int)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);
  v = v > o ? v : o;
  o = (unsigned int)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);
  return v > o ? v : o;
}

// Geometry of the elementwise kernels. A block of 256 threads is (tx, ty): tx lanes along a row, ty rows; grid.y strides over the rows.
// A tensor whose rows follow each other without a gap and hold whole blocks is passed as ONE row.
struct CkGeom { int64_t rows, C, nb, ldx, ld2; int tx_shift; };      // nb: blocks per row; ldx: row stride of x / dy; ld2: of act / dx

// C % 8 == 0 and 16-byte aligned rows: 8 elements per lane, a block is a quad of lanes (lanes past the row's end hold zeros)
template <typename T, bool GELU>
__global__ __launch_bounds__(256) void ckpt8_fwd_vec_kernel(const T* __restrict__ x, T* __restrict__ act, signed char* __restrict__ codes,
                                                            unsigned char* __restrict__ exps, const CkGeom g) {
  const int tx = threadIdx.x & ((1 << g.tx_shift) - 1), ty = threadIdx.x >> g.tx_shift;
  const int64_t v = ((int64_t)blockIdx.x << g.tx_shift) + tx;
  const int64_t c = v * 8;
  const int rpb = 256 >> g.tx_shift;
  for (int64_t row = (int64_t)blockIdx.y * rpb + ty; row < g.rows; row += (int64_t)gridDim.y * rpb) {
    Vec8 e = {{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
    const bool on = c < g.C;
    if (on) e = load8(x + row * g.ldx + c);
    unsigned int m = 0u;
#pragma unroll
    for (int i = 0; i < 8; i += 2) m = umax3(m, ckpt8_abs_bits(e.v[i]), ckpt8_abs_bits(e.v[i + 1]));
    const unsigned int byte = ckpt8_exp_byte(quad_umax(m));
    const float inv = ckpt8_inv_step(byte);
    if (on) {
      u32x2_t w;
      w.x = ckpt8_code4(e.v[0], e.v[1], e.v[2], e.v[3], inv);
      w.y = ckpt8_code4(e.v[4], e.v[5], e.v[6], e.v[7], inv);
      if (byte == 255u) w.x = w.y = 0u;                       // (NaN * 0: keep the codes of a marked block zero)
      *reinterpret_cast<u32x2_t*>(codes + row * g.C + c) = w;
      if ((v & 3) == 0) exps[row * g.nb + (v >> 2)] = (unsigned char)byte;
      if (GELU) {
        Vec8 a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a.v[i] = ck_gelu(e.v[i]);
        store8(act + row * g.ld2 + c, a);
      }
    }
  }
}

// the same from the checkpoint: MODE 0 unpack (dx = value), 1 GELU backward (dx = dy * slope; act too if it is given)
template <typename T, int MODE>
__global__ __launch_bounds__(256) void ckpt8_bwd_vec_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                            const T* __restrict__ dy, T* __restrict__ dx, T* __restrict__ act, const CkGeom g) {
  const int tx = threadIdx.x & ((1 << g.tx_shift) - 1), ty = threadIdx.x >> g.tx_shift;
  const int64_t v = ((int64_t)blockIdx.x << g.tx_shift) + tx;
  const int64_t c = v * 8;
  if (c >= g.C) return;
  const int rpb = 256 >> g.tx_shift;
  for (int64_t row = (int64_t)blockIdx.y * rpb + ty; row < g.rows; row += (int64_t)gridDim.y * rpb) {
    const u32x2_t w = *reinterpret_cast<const u32x2_t*>(codes + row * g.C + c);
    const float step = ckpt8_step(exps[row * g.nb + (v >> 2)]);
    Vec8 o;
    if (MODE == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[i] = ckpt8_value(i < 4 ? w.x : w.y, i & 3, step);
      store8(dx + row * g.ld2 + c, o);
    } else {
      const Vec8 d = load8(dy + row * g.ldx + c);
      Vec8 a;
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[i] = d.v[i] * ck_gelu_slope(ckpt8_value(i < 4 ? w.x : w.y, i & 3, step), &a.v[i]);
      store8(dx + row * g.ld2 + c, o);
      if (act) store8(act + row * g.ld2 + c, a);
    }
  }
}

// any C, any alignment: one element per lane, a block is half a wave (odd widths: rows of codes start at any byte)
template <typename T, bool GELU>
__global__ __launch_bounds__(256) void ckpt8_fwd_any_kernel(const T* __restrict__ x, T* __restrict__ act, signed char* __restrict__ codes,
                                                            unsigned char* __restrict__ exps, const CkGeom g) {
  const int tx = threadIdx.x & ((1 << g.tx_shift) - 1), ty = threadIdx.x >> g.tx_shift;
  const int64_t c = ((int64_t)blockIdx.x << g.tx_shift) + tx;
  const int rpb = 256 >> g.tx_shift;
  for (int64_t row = (int64_t)blockIdx.y * rpb + ty; row < g.rows; row += (int64_t)gridDim.y * rpb) {
    const bool on = c < g.C;
    const float e = on ? load1(x + row * g.ldx + c) : 0.f;
    unsigned int m = ckpt8_abs_bits(e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned int q = (unsigned int)__shfl_xor((int)m, o, 64);
      m = m > q ? m : q;
    }
    const unsigned int byte = ckpt8_exp_byte(m);
    if (on) {
      codes[row * g.C + c] = byte == 255u ? (signed char)0 : (signed char)ckpt8_code(e, ckpt8_inv_step(byte));
      if ((c & 31) == 0) exps[row * g.nb + (c >> 5)] = (unsigned char)byte;
      if (GELU) store1(act + row * g.ld2 + c, ck_gelu(e));
    }
  }
}
template <typename T, int MODE>
__global__ __launch_bounds__(256) void ckpt8_bwd_any_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                            const T* __restrict__ dy, T* __restrict__ dx, T* __restrict__ act, const CkGeom g) {
  const int tx = threadIdx.x & ((1 << g.tx_shift) - 1), ty = threadIdx.x >> g.tx_shift;
  const int64_t c = ((int64_t)blockIdx.x << g.tx_shift) + tx;
  if (c >= g.C) return;
  const int rpb = 256 >> g.tx_shift;
  for (int64_t row = (int64_t)blockIdx.y * rpb + ty; row < g.rows; row += (int64_t)gridDim.y * rpb) {
    const float x8 = (float)codes[row * g.C + c] * ckpt8_step(exps[row * g.nb + (c >> 5)]);
    if (MODE == 0) store1(dx + row * g.ld2 + c, x8);
    else {
      float a;
      const float s = ck_gelu_slope(x8, &a);
      store1(dx + row * g.ld2 + c, load1(dy + row * g.ldx + c) * s);
      if (act) store1(act + row * g.ld2 + c, a);
    }
  }
}

// ------------------------------------------------------------------------------------------------ LayerNorm
// One wave per row, the row in registers: lane holds elements 4 (lane + 64 j) .. + 3, j < NV = ceil(C / 256), a block is 8 lanes.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <> __device__ __forceinline__ float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <> __device__ __forceinline__ float4 load4<bf16_t>(const bf16_t* p) {
  const u32x2_t w = *reinterpret_cast<const u32x2_t*>(p);
  return make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
}

// four elements as they lie in memory
template <typename T> struct Raw4;
template <> struct Raw4<float> {
  float4 v;
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void zero() { v = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ float4 value() const { return v; }
};
template <> struct Raw4<bf16_t> {
  u32x2_t v;
  __device__ __forceinline__ void load(const bf16_t* p) { v = *reinterpret_cast<const u32x2_t*>(p); }
  __device__ __forceinline__ void zero() { v = (u32x2_t){0u, 0u}; }
  __device__ __forceinline__ float4 value() const { return make_float4(bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y)); }
};

template <typename T, int NV>
__global__ __launch_bounds__(256) void ln_fwd_ckpt8_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ gamma,
                                                           const float* __restrict__ beta, bf16_t* __restrict__ y, float* __restrict__ mean_out,
                                                           float* __restrict__ rstd_out, signed char* __restrict__ codes,
                                                           unsigned char* __restrict__ exps, int64_t rows, int C, float eps) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  float4 e[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = 4 * (lane + 64 * j);
    e[j] = c < C ? load4(x + row * ldx + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) s += (e[j].x + e[j].y) + (e[j].z + e[j].w);
  const float mean = wave_sum(s) / (float)C;
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (4 * (lane + 64 * j) < C) {
      const float a = e[j].x - mean, b = e[j].y - mean, c = e[j].z - mean, d = e[j].w - mean;
      q += (a * a + b * b) + (c * c + d * d);
    }
  }
  const float rstd = 1.0f / sqrtf(wave_sum(q) / (float)C + eps);
  if (lane == 0) { mean_out[row] = mean; rstd_out[row] = rstd; }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = 4 * (lane + 64 * j);
    const unsigned int a0 = ckpt8_abs_bits(e[j].x), a1 = ckpt8_abs_bits(e[j].y), a2 = ckpt8_abs_bits(e[j].z), a3 = ckpt8_abs_bits(e[j].w);
    unsigned int m = quad_umax(umax3(umax3(a0, a1, a2), a3, 0u));
    const unsigned int o = (unsigned int)__shfl_xor((int)m, 4, 64);
    m = m > o ? m : o;
    const unsigned int byte = ckpt8_exp_byte(m);
    if (c < C) {
      unsigned int w = ckpt8_code4(e[j].x, e[j].y, e[j].z, e[j].w, ckpt8_inv_step(byte));
      if (byte == 255u) w = 0u;
      *reinterpret_cast<unsigned int*>(codes + row * C + c) = w;
      if ((lane & 7) == 0) exps[row * (C >> 5) + (c >> 5)] = (unsigned char)byte;
      const float4 ga = *reinterpret_cast<const float4*>(gamma + c), be = *reinterpret_cast<const float4*>(beta + c);
      u32x2_t o2;
      o2.x = pack_bf16x2(fmaf((e[j].x - mean) * rstd, ga.x, be.x), fmaf((e[j].y - mean) * rstd, ga.y, be.y));
      o2.y = pack_bf16x2(fmaf((e[j].z - mean) * rstd, ga.z, be.z), fmaf((e[j].w - mean) * rstd, ga.w, be.w));
      *reinterpret_cast<u32x2_t*>(y + row * C + c) = o2;
    }
  }
}

// Backward: 8 waves per workgroup, a wave strides over the rows; dgamma / dbeta stay in its registers, the waves' sums are added in
// order through LDS and leave one slab [2][C] per workgroup, which the second kernel adds in order: no atomics, the same bits each run.
#define LNB_WAVES 8
#define LNB_MAX_WG 512
#define LNB_FEW 2048
// Few rows: dgamma and dbeta of 32 columns (a block of the checkpoint) by one workgroup more per block in the same launch, which reads
// dy and the codes of all rows again: 64 groups of rows, added in order. [512, 768]: 8.9 us with slabs and a second launch, 4.4 so (18.3
// and 13.7 issued one by one); [2048, 1280] 14.0 and 12.3; [4096, 768] 17.4 and 20.4, where re-reading costs more than the launch.
template <typename T>
__device__ __forceinline__ void ln_bwd_ckpt8_columns(const T* __restrict__ dy, int64_t lddy, const signed char* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                     const float* __restrict__ mean_in, const float* __restrict__ rstd_in, float* __restrict__ dgamma,
                                                     float* __restrict__ dbeta, int rows, int C, int block) {
  __shared__ float part[2][64][33];
  const int l = threadIdx.x & 7, k = threadIdx.x >> 3, c = 32 * block + 4 * l;
  float dg[4] = {0.f, 0.f, 0.f, 0.f}, db[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int row = k; row < rows; row += 64) {
    Raw4<T> q;
    q.load(dy + (int64_t)row * lddy + c);
    const float4 d = q.value();
    const unsigned int w = *reinterpret_cast<const unsigned int*>(codes + (int64_t)row * C + c);
    const float step = ckpt8_step(exps[(int64_t)row * (C >> 5) + block]), mean = mean_in[row], rstd = rstd_in[row];
    const float dv[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      dg[i] = fmaf(dv[i], (ckpt8_value(w, i, step) - mean) * rstd, dg[i]);
      db[i] += dv[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) { part[0][k][4 * l + i] = dg[i]; part[1][k][4 * l + i] = db[i]; }
  __syncthreads();
  const int j = threadIdx.x & 31, z = (threadIdx.x >> 5) & 1;
  if (threadIdx.x >= 64) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 64; ++i) t += part[z][i][j];
  (z ? dbeta : dgamma)[32 * block + j] = t;
}
template <typename T, int NV, bool WG>
__global__ __launch_bounds__(64 * LNB_WAVES) void ln_bwd_ckpt8_kernel(const T* __restrict__ dy, int64_t lddy, const signed char* __restrict__ codes,
                                                                      const unsigned char* __restrict__ exps, const float* __restrict__ mean_in,
                                                                      const float* __restrict__ rstd_in, const float* __restrict__ gamma,
                                                                      const float* __restrict__ beta, const float* __restrict__ dres,
                                                                      float* __restrict__ dx, bf16_t* __restrict__ dx_bf, bf16_t* __restrict__ y,
                                                                      float* __restrict__ slabs, int64_t rows, int C, int col_wgs, float* __restrict__ dgamma,
                                                                      float* __restrict__ dbeta) {
  extern __shared__ float lds_w[];      // WG: [2][C]
  if (!WG && (int)blockIdx.x < col_wgs) {
    ln_bwd_ckpt8_columns<T>(dy, lddy, codes, exps, mean_in, rstd_in, dgamma, dbeta, (int)rows, C, blockIdx.x);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float4 ga[NV], dg[NV], db[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = 4 * (lane + 64 * j);
    ga[j] = c < C ? *reinterpret_cast<const float4*>(gamma + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    dg[j] = db[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float invC = 1.0f / (float)C;
  const int64_t stride = (int64_t)(gridDim.x - col_wgs) * LNB_WAVES;
  // Operands of a row as they lie in memory. Up to NV = 5 the next row's are requested before this row's arithmetic (registers end it
  // there): with one row in flight per wave the loop reached 4.1 TB/s.
  struct Raw { Raw4<T> d[NV]; unsigned int w[NV], by[NV]; float4 r[NV]; float mean, rstd; };
  auto request = [&](int64_t row, Raw& q) __attribute__((always_inline)) {
    q.mean = mean_in[row];
    q.rstd = rstd_in[row];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = 4 * (lane + 64 * j);
      const bool on = c < C;
      if (on && dy) q.d[j].load(dy + row * lddy + c); else q.d[j].zero();
      q.w[j] = on ? *reinterpret_cast<const unsigned int*>(codes + row * C + c) : 0u;
      q.by[j] = on ? exps[row * (C >> 5) + (c >> 5)] : 0u;
      q.r[j] = on && dres ? *reinterpret_cast<const float4*>(dres + row * C + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  constexpr bool AHEAD = NV <= 5;
  Raw cur, nxt;
  int64_t row = (int64_t)(blockIdx.x - col_wgs) * LNB_WAVES + wave;
  if (AHEAD && row < rows) request(row, nxt);
  for (; row < rows; row += stride) {
    if (AHEAD) {
      cur = nxt;
      if (row + stride < rows) request(row + stride, nxt);
    } else request(row, cur);
    float4 d[NV], xh[NV];
    const float mean = cur.mean, rstd = cur.rstd;
#pragma unroll
    for (int j = 0; j < NV; ++j) d[j] = cur.d[j].value();
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float step = ckpt8_step(cur.by[j]);
      xh[j].x = (ckpt8_value(cur.w[j], 0, step) - mean) * rstd; xh[j].y = (ckpt8_value(cur.w[j], 1, step) - mean) * rstd;
      xh[j].z = (ckpt8_value(cur.w[j], 2, step) - mean) * rstd; xh[j].w = (ckpt8_value(cur.w[j], 3, step) - mean) * rstd;
      const float tx = d[j].x * ga[j].x, ty = d[j].y * ga[j].y, tz = d[j].z * ga[j].z, tw = d[j].w * ga[j].w;
      s1 += (tx + ty) + (tz + tw);
      if (4 * (lane + 64 * j) < C) s2 += fmaf(tx, xh[j].x, ty * xh[j].y) + fmaf(tz, xh[j].z, tw * xh[j].w);
      if (WG) {
        dg[j].x = fmaf(d[j].x, xh[j].x, dg[j].x); dg[j].y = fmaf(d[j].y, xh[j].y, dg[j].y);
        dg[j].z = fmaf(d[j].z, xh[j].z, dg[j].z); dg[j].w = fmaf(d[j].w, xh[j].w, dg[j].w);
        db[j].x += d[j].x; db[j].y += d[j].y; db[j].z += d[j].z; db[j].w += d[j].w;
      }
    }
    const float m1 = wave_sum(s1) * invC, m2 = wave_sum(s2) * invC;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = 4 * (lane + 64 * j);
      if (c >= C) continue;
      float4 o;
      o.x = rstd * (fmaf(d[j].x, ga[j].x, -m1) - xh[j].x * m2); o.y = rstd * (fmaf(d[j].y, ga[j].y, -m1) - xh[j].y * m2);
      o.z = rstd * (fmaf(d[j].z, ga[j].z, -m1) - xh[j].z * m2); o.w = rstd * (fmaf(d[j].w, ga[j].w, -m1) - xh[j].w * m2);
      if (dres) { o.x += cur.r[j].x; o.y += cur.r[j].y; o.z += cur.r[j].z; o.w += cur.r[j].w; }
      if (dx) *reinterpret_cast<float4*>(dx + row * C + c) = o;
      if (dx_bf) {
        u32x2_t p; p.x = pack_bf16x2(o.x, o.y); p.y = pack_bf16x2(o.z, o.w);
        *reinterpret_cast<u32x2_t*>(dx_bf + row * C + c) = p;
      }
      if (y) {
        const float4 be = *reinterpret_cast<const float4*>(beta + c);
        u32x2_t p;
        p.x = pack_bf16x2(fmaf(xh[j].x, ga[j].x, be.x), fmaf(xh[j].y, ga[j].y, be.y));
        p.y = pack_bf16x2(fmaf(xh[j].z, ga[j].z, be.z), fmaf(xh[j].w, ga[j].w, be.w));
        *reinterpret_cast<u32x2_t*>(y + row * C + c) = p;
      }
    }
  }
  if (WG) {
    for (int k = 0; k < LNB_WAVES; ++k) {
      if (wave == k) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int c = 4 * (lane + 64 * j);
          if (c >= C) continue;
          float4* pg = reinterpret_cast<float4*>(lds_w + c);
          float4* pb = reinterpret_cast<float4*>(lds_w + C + c);
          if (k) {
            const float4 og = *pg, ob = *pb;
            dg[j].x += og.x; dg[j].y += og.y; dg[j].z += og.z; dg[j].w += og.w;
            db[j].x += ob.x; db[j].y += ob.y; db[j].z += ob.z; db[j].w += ob.w;
          }
          *pg = dg[j]; *pb = db[j];
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * C; i += 64 * LNB_WAVES) slabs[(int64_t)blockIdx.x * 2 * C + i] = lds_w[i];
  }
}

// out[j] = sum over the n slabs of slab[j], j < 2 C: 32 columns x 32 slab groups per workgroup (64 x 4 with the loads of a thread one
// after the other took 32 us for 512 slabs of 2560 columns)
__global__ __launch_bounds__(1024) void ln_bwd_ckpt8_sum_kernel(const float* __restrict__ slabs, int n, int C, float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float part[32][33];
  const int l = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + l;                      // (2 C is a multiple of 64)
  const float* s = slabs + j;
  float t = 0.f;
#pragma unroll 4
  for (int i = k; i < n; i += 32) t += s[(int64_t)i * 2 * C];
  part[k][l] = t;
  __syncthreads();
  if (k < 4) {
    float u = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) u += part[8 * k + i][l];
    part[8 * k][l] = u;
  }
  __syncthreads();
  if (k == 0) {
    const float v = (part[0][l] + part[8][l]) + (part[16][l] + part[24][l]);
    if (j < C) dgamma[j] = v; else dbeta[j - C] = v;
  }
}

// ------------------------------------------------------------------------------------------------ host
static bool ck_dtype(int d) { return d == MFNET_F32 || d == MFNET_BF16; }

// geometry and grid of an elementwise call; vec: 8 elements per lane
static bool ck_geometry(CkGeom* g, dim3* grid, int64_t rows, int64_t C, int64_t ldx, int64_t ld2, bool vec) {
  if (vec && C % CKPT8_BLOCK == 0 && ldx == C && ld2 == C) { C *= rows; rows = 1; ldx = ld2 = C; }
  g->rows = rows; g->C = C; g->nb = ceil_div64(C, CKPT8_BLOCK); g->ldx = ldx; g->ld2 = ld2;
  const int64_t lanes = vec ? g->nb * 4 : g->nb * 32;
  int sh = vec ? 2 : 5;
  while (sh < 8 && (1ll << sh) < lanes) ++sh;
  g->tx_shift = sh;
  const int64_t gx = ceil_div64(lanes, 1ll << sh);
  int64_t gy = ceil_div64(rows, 256 >> sh);
  if (gy > 65535) gy = 65535;
  *grid = dim3((unsigned)gx, (unsigned)gy);
  return gx < (1ll << 24);                                // (a grid dimension holds less than 2^32 threads)
}

#define CK_CHECK_SHAPE(name)                                                                                                         \
  MF_CHECK_ARG(rows >= 0 && C >= 1 && C < (1ll << 40) && rows < (1ll << 40) && (rows == 0 || C <= (1ll << 42) / rows), name ": bad shape [%lld, %lld]", (long long)rows, (long long)C)

static int ck_fwd(const char* name, bool gelu, const void* x, int dt, int64_t ldx, void* act, int64_t ldact, void* codes, void* exps,
                  int64_t rows, int64_t C, hipStream_t stream) {
  CK_CHECK_SHAPE("ckpt8");
  MF_CHECK_ARG(ck_dtype(dt), "%s: dtype must be MFNET_F32 or MFNET_BF16", name);
  if (rows == 0) return MFNET_OK;
  MF_CHECK_ARG(x && codes && exps && (!gelu || act), "%s: null pointer", name);
  const int64_t es = dt == MFNET_F32 ? 4 : 2;
  MF_CHECK_ARG(ldx >= C && (!gelu || ldact >= C), "%s: row stride below C", name);
  MF_CHECK_ARG((uintptr_t)x % es == 0 && (uintptr_t)act % es == 0, "%s: misaligned tensor", name);
  const bool vec = C % 8 == 0 && ldx % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)codes % 8 == 0 && (!gelu || (ldact % 8 == 0 && (uintptr_t)act % 16 == 0));
  CkGeom g; dim3 grid;
  MF_CHECK_ARG(ck_geometry(&g, &grid, rows, C, ldx, gelu ? ldact : ldx, vec), "%s: tensor too large", name);
#define CK_FWD(T_, G_) do { if (vec) hipLaunchKernelGGL((ckpt8_fwd_vec_kernel<T_, G_>), grid, dim3(256), 0, stream, (const T_*)x, (T_*)act, (signed char*)codes, (unsigned char*)exps, g); \
                            else hipLaunchKernelGGL((ckpt8_fwd_any_kernel<T_, G_>), grid, dim3(256), 0, stream, (const T_*)x, (T_*)act, (signed char*)codes, (unsigned char*)exps, g); } while (0)
  if (dt == MFNET_F32) { if (gelu) CK_FWD(float, true); else CK_FWD(float, false); }
  else { if (gelu) CK_FWD(bf16_t, true); else CK_FWD(bf16_t, false); }
#undef CK_FWD
  MF_LAUNCH_CHECK(name);
  return MFNET_OK;
}

static int ck_bwd(const char* name, int mode, const void* codes, const void* exps, const void* dy, int64_t lddy, void* dx, int dt,
                  int64_t lddx, void* act, int64_t rows, int64_t C, hipStream_t stream) {
  CK_CHECK_SHAPE("ckpt8");
  MF_CHECK_ARG(ck_dtype(dt), "%s: dtype must be MFNET_F32 or MFNET_BF16", name);
  if (rows == 0) return MFNET_OK;
  MF_CHECK_ARG(codes && exps && dx && (mode == 0 || dy), "%s: null pointer", name);
  const int64_t es = dt == MFNET_F32 ? 4 : 2;
  if (mode == 0) lddy = lddx;
  MF_CHECK_ARG(lddx >= C && lddy >= C, "%s: row stride below C", name);
  MF_CHECK_ARG((uintptr_t)dx % es == 0 && (uintptr_t)dy % es == 0 && (uintptr_t)act % es == 0, "%s: misaligned tensor", name);
  const bool vec = C % 8 == 0 && lddx % 8 == 0 && lddy % 8 == 0 && (uintptr_t)dx % 16 == 0 && (uintptr_t)dy % 16 == 0 && (uintptr_t)act % 16 == 0 && (uintptr_t)codes % 8 == 0;
  CkGeom g; dim3 grid;
  MF_CHECK_ARG(ck_geometry(&g, &grid, rows, C, lddy, lddx, vec), "%s: tensor too large", name);
#define CK_BWD(T_, M_) do { if (vec) hipLaunchKernelGGL((ckpt8_bwd_vec_kernel<T_, M_>), grid, dim3(256), 0, stream, (const signed char*)codes, (const unsigned char*)exps, (const T_*)dy, (T_*)dx, (T_*)act, g); \
                            else hipLaunchKernelGGL((ckpt8_bwd_any_kernel<T_, M_>), grid, dim3(256), 0, stream, (const signed char*)codes, (const unsigned char*)exps, (const T_*)dy, (T_*)dx, (T_*)act, g); } while (0)
  if (dt == MFNET_F32) { if (mode) CK_BWD(float, 1); else CK_BWD(float, 0); }
  else { if (mode) CK_BWD(bf16_t, 1); else CK_BWD(bf16_t, 0); }
#undef CK_BWD
  MF_LAUNCH_CHECK(name);
  return MFNET_OK;
}

extern "C" int mfnet_ckpt8_pack(const void* x, int x_dtype, int64_t ldx, void* codes, void* exps, int64_t rows, int64_t C, hipStream_t stream) {
  return ck_fwd("ckpt8_pack", false, x, x_dtype, ldx, nullptr, 0, codes, exps, rows, C, stream);
}
extern "C" int mfnet_ckpt8_unpack(const void* codes, const void* exps, void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t C, hipStream_t stream) {
  return ck_bwd("ckpt8_unpack", 0, codes, exps, nullptr, 0, x, x_dtype, ldx, nullptr, rows, C, stream);
}
extern "C" int mfnet_gelu_fwd_ckpt8(const void* x, int dtype, int64_t ldx, void* act, int64_t ldact, void* codes, void* exps, int64_t rows, int64_t C, hipStream_t stream) {
  return ck_fwd("gelu_fwd_ckpt8", true, x, dtype, ldx, act, ldact, codes, exps, rows, C, stream);
}
extern "C" int mfnet_gelu_bwd_ckpt8(const void* codes, const void* exps, const void* dy, int dtype, int64_t lddy, void* dx, void* act, int64_t lddx, int64_t rows, int64_t C, hipStream_t stream) {
  return ck_bwd("gelu_bwd_ckpt8", 1, codes, exps, dy, lddy, dx, dtype, lddx, act, rows, C, stream);
}

static bool ln_ck_shape(int64_t rows, int64_t C) { return rows >= 0 && C >= 32 && C % CKPT8_BLOCK == 0 && C <= 2048 && rows <= (1ll << 40); }

extern "C" int mfnet_layernorm_fwd_ckpt8(const void* x, int x_dtype, int64_t ldx, const float* gamma, const float* beta, void* y, float* mean,
                                         float* rstd, void* codes, void* exps, int64_t rows, int64_t C, float eps, hipStream_t stream) {
  MF_CHECK_ARG(ln_ck_shape(rows, C), "layernorm_fwd_ckpt8: C=%lld must be a multiple of 32, at most 2048", (long long)C);
  MF_CHECK_ARG(ck_dtype(x_dtype), "layernorm_fwd_ckpt8: bad dtype");
  if (rows == 0) return MFNET_OK;
  MF_CHECK_ARG(x && gamma && beta && y && mean && rstd && codes && exps, "layernorm_fwd_ckpt8: null pointer");
  MF_CHECK_ARG(ldx >= C && ldx % 4 == 0, "layernorm_fwd_ckpt8: ldx must be >= C and a multiple of 4");
  MF_CHECK_ARG(((uintptr_t)gamma | (uintptr_t)beta) % 16 == 0 && (uintptr_t)x % (x_dtype == MFNET_F32 ? 16 : 8) == 0 && (uintptr_t)y % 8 == 0 && (uintptr_t)codes % 4 == 0,
               "layernorm_fwd_ckpt8: misaligned tensor");
  const int64_t gx = ceil_div64(rows, 4);
  MF_CHECK_ARG(gx < (1ll << 24), "layernorm_fwd_ckpt8: too many rows");
#define LNF(T_, NV_) hipLaunchKernelGGL((ln_fwd_ckpt8_kernel<T_, NV_>), dim3((unsigned)gx), dim3(256), 0, stream, (const T_*)x, ldx, gamma, beta, (bf16_t*)y, mean, rstd, (signed char*)codes, (unsigned char*)exps, rows, (int)C, eps)
#define LNF_CASE(NV_) case NV_: if (x_dtype == MFNET_F32) LNF(float, NV_); else LNF(bf16_t, NV_); break;
  switch ((int)ceil_div64(C, 256)) { LNF_CASE(1) LNF_CASE(2) LNF_CASE(3) LNF_CASE(4) LNF_CASE(5) LNF_CASE(6) LNF_CASE(7) LNF_CASE(8) }
#undef LNF_CASE
#undef LNF
  MF_LAUNCH_CHECK("layernorm_fwd_ckpt8");
  return MFNET_OK;
}

// few rows (see ln_bwd_ckpt8_columns)
static bool ln_ck_few(int64_t rows) { return rows <= LNB_FEW; }
static int64_t ln_ck_wgs(int64_t rows) {
  const int64_t n = ceil_div64(rows, LNB_WAVES);
  return n < LNB_MAX_WG ? n : LNB_MAX_WG;
}
// floats of workspace of mfnet_layernorm_bwd_ckpt8 with weight gradients
extern "C" int64_t mfnet_layernorm_ckpt8_workspace_floats(int64_t rows, int64_t C) {
  return rows <= 0 || C <= 0 || ln_ck_few(rows) ? 0 : ln_ck_wgs(rows) * 2 * C;
}

extern "C" int mfnet_layernorm_bwd_ckpt8(const void* dy, int dy_dtype, int64_t lddy, const void* codes, const void* exps, const float* mean,
                                         const float* rstd, const float* gamma, const float* beta, const float* dres, float* dx, void* dx_bf16,
                                         void* y, float* dgamma, float* dbeta, float* ws, int64_t ws_floats, int64_t rows, int64_t C, hipStream_t stream) {
  MF_CHECK_ARG(ln_ck_shape(rows, C), "layernorm_bwd_ckpt8: C=%lld must be a multiple of 32, at most 2048", (long long)C);
  MF_CHECK_ARG(ck_dtype(dy_dtype), "layernorm_bwd_ckpt8: bad dtype");
  MF_CHECK_ARG((dgamma == nullptr) == (dbeta == nullptr), "layernorm_bwd_ckpt8: dgamma and dbeta go together");
  const bool wg = dgamma != nullptr;
  MF_CHECK_ARG(rows == 0 || (codes && exps && mean && rstd && gamma && (dy ? dx || dx_bf16 : y && !dx && !dx_bf16 && !wg)),
               "layernorm_bwd_ckpt8: null pointer (dy with dx, or y alone)");
  MF_CHECK_ARG(!y || beta, "layernorm_bwd_ckpt8: y needs beta");
  const int64_t n = rows ? ln_ck_wgs(rows) : 0;
  const bool few = rows && ln_ck_few(rows), slabs = wg && !few;
  const int col_wgs = wg && few ? (int)(C / 32) : 0;
  MF_CHECK_ARG(!slabs || n == 0 || (ws && ws_floats >= n * 2 * C), "layernorm_bwd_ckpt8: workspace too small");
  if (rows) {
    MF_CHECK_ARG(!dy || (lddy >= C && lddy % 4 == 0), "layernorm_bwd_ckpt8: lddy must be >= C and a multiple of 4");
    MF_CHECK_ARG(((uintptr_t)gamma | (uintptr_t)beta | (uintptr_t)dres | (uintptr_t)dx) % 16 == 0 && (uintptr_t)dy % (dy_dtype == MFNET_F32 ? 16 : 8) == 0 &&
                 ((uintptr_t)dx_bf16 | (uintptr_t)y) % 8 == 0 && (uintptr_t)codes % 4 == 0, "layernorm_bwd_ckpt8: misaligned tensor");
#define LNB(T_, NV_, W_) hipLaunchKernelGGL((ln_bwd_ckpt8_kernel<T_, NV_, W_>), dim3((unsigned)(n + col_wgs)), dim3(64 * LNB_WAVES), W_ ? 2 * (size_t)C * 4 : 0, stream, (const T_*)dy, lddy, \
    (const signed char*)codes, (const unsigned char*)exps, mean, rstd, gamma, beta, dres, dx, (bf16_t*)dx_bf16, (bf16_t*)y, ws, rows, (int)C, col_wgs, dgamma, dbeta)
#define LNB_CASE(NV_) case NV_: if (dy_dtype == MFNET_F32) { if (slabs) LNB(float, NV_, true); else LNB(float, NV_, false); } else { if (slabs) LNB(bf16_t, NV_, true); else LNB(bf16_t, NV_, false); } break;
    switch ((int)ceil_div64(C, 256)) { LNB_CASE(1) LNB_CASE(2) LNB_CASE(3) LNB_CASE(4) LNB_CASE(5) LNB_CASE(6) LNB_CASE(7) LNB_CASE(8) }
#undef LNB_CASE
#undef LNB
    MF_LAUNCH_CHECK("layernorm_bwd_ckpt8");
  }
  if (slabs) {      // (no rows: the sums of nothing, zeros)
    hipLaunchKernelGGL(ln_bwd_ckpt8_sum_kernel, dim3((unsigned)(C / 16)), dim3(1024), 0, stream, ws, (int)n, (int)C, dgamma, dbeta);
    MF_LAUNCH_CHECK("layernorm_bwd_ckpt8 (sums)");
  }
  return MFNET_OK;
}
