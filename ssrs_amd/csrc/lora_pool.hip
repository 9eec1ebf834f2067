// A pool of low-rank adapters beside one shared projection, forward and backward. Every row m names its adapter i = ids[m] (none if the
// index lies outside [0, n)): rows of many requests, tiles or jobs, in any order, in one call.
//
//   down[m]  = s_i A_i x_m                                  (fp32 [M, RP], kept for the backward pass)
//   out[m]   = W x_m + bias + B_i down[m]
//   p[m]     = s_i B_i^T dy_m
//   dx[m]    = W^T dy_m + A_i^T p[m]
//   dA_i     = sum over the rows of adapter i of p[m] x_m^T,     dB_i = sum of dy_m down[m]^T
//
// The factors are held as bf16 images padded to RP = 16, 32 or 64 ranks (mfnet_lora_pool_pack): "down" images [n][RP][C] for products
// that contract over the long axis, "up" images [n][C][RP] for products that contract over the ranks, so that both are read as MFMA
// operands in 16-byte pieces. fp32 factors of a product (down, p) are split into bf16 parts hi + lo (+ lo'), never rounded once.
//
// A workgroup that meets rows of several adapters multiplies all its rows with each adapter in turn and SELECTS the rows it belongs to:
// a sum of zeros would let one adapter's infinities and NaN into another request's rows.
#include "ckpt8.h"

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef const __attribute__((address_space(1))) void* gbl_ptr_t;

// source of the k-chunks behind the last column (zero-initialised device memory, never written)
__device__ __attribute__((aligned(128))) unsigned char g_pool_zero[128];

union Frag { bf16x8_t v; s16x4_t h[2]; unsigned int w[4]; u32x4_t q; };

// part 0 / 1 / 2 of the split x = hi + lo + lo' (bf16 each, 8 + 8 + 8 significant bits) of eight values
__device__ __forceinline__ bf16x8_t split_part(const float (&x)[8], int part) {
  Frag f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
    unsigned int h = pack_bf16x2(a, b);
    if (part >= 1) {
      a -= bf16_lo(h); b -= bf16_hi(h);
      h = pack_bf16x2(a, b);
      if (part >= 2) h = pack_bf16x2(a - bf16_lo(h), b - bf16_hi(h));
    }
    f.w[i] = h;
  }
  return f.v;
}

// smallest index above `last` among the lanes' candidates (lane quarters hold copies of the same 16 rows); INT_MAX: none left
__device__ __forceinline__ int next_id(int cand) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const int q = __shfl_xor(cand, o, 64);
    cand = cand < q ? cand : q;
  }
  return __builtin_amdgcn_readfirstlane(cand);
}
#define NO_ID 0x7fffffff

// ------------------------------------------------------------------------------------------------ images
// long_first: src [n][C][r] (B), else src [n][r][C] (A). One thread per (adapter, position on the long axis).
template <typename T, bool LONG_FIRST>
__global__ __launch_bounds__(256) void pool_pack_kernel(const T* __restrict__ src, int C, int r, int RP, bf16_t* __restrict__ down, bf16_t* __restrict__ up) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  const int64_t i = blockIdx.y;
  if (c >= C) return;
  const T* s = src + i * (int64_t)C * r;
  for (int j0 = 0; j0 < RP; j0 += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = j0 + j;
      if (k < r) {
        const T t = LONG_FIRST ? s[(int64_t)c * r + k] : s[(int64_t)k * C + c];
        if constexpr (sizeof(T) == 4) v[j] = t; else v[j] = bf16_to_f32(t);
      } else v[j] = 0.f;
    }
    Frag f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.w[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
    if (up) *reinterpret_cast<u32x4_t*>(up + (i * C + c) * RP + j0) = f.q;
    if (down) {
#pragma unroll
      for (int j = 0; j < 8; ++j) down[(i * RP + j0 + j) * C + c] = (bf16_t)(f.w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// ------------------------------------------------------------------------------------------------ rows grouped by adapter
// Workgroup i: how many rows belong to adapters below i (their places come first), then the rows of adapter i in ascending order.
// Deterministic without a sort; the indices are read from L2 twice per adapter.
__global__ __launch_bounds__(256) void pool_plan_kernel(const int* __restrict__ ids, int M, int n, int* __restrict__ offs, int* __restrict__ perm) {
  const int i = blockIdx.x;                               // 0 .. n; workgroup n only writes offs[n]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ int part[4];
  int below = 0;
  for (int m = threadIdx.x; m < M; m += 256) {
    const int v = ids[m];
    below += (v >= 0 && v < i) ? 1 : 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o, 64);
  if (lane == 0) part[wave] = below;
  __syncthreads();
  int pos = part[0] + part[1] + part[2] + part[3];
  if (threadIdx.x == 0) offs[i] = pos;
  if (i == n) return;
  for (int m0 = 0; m0 < M; m0 += 256) {
    const int m = m0 + threadIdx.x;
    const bool mine = m < M && ids[m] == i;
    const unsigned long long b = __ballot(mine);
    __syncthreads();
    if (lane == 0) part[wave] = __popcll(b);
    __syncthreads();
    int at = pos;
    for (int w = 0; w < wave; ++w) at += part[w];
    if (mine) perm[at + __popcll(b & ((1ull << lane) - 1))] = m;
    pos += part[0] + part[1] + part[2] + part[3];
  }
}
// chunks of at most ch rows of one adapter: table[k] = {adapter, first, last + 1 place in perm, 0}, base[i] = first chunk of adapter i.
// Entries behind the last chunk keep adapter -1.
__global__ __launch_bounds__(256) void pool_chunks_kernel(const int* __restrict__ offs, int n, int ch, int max_chunks, int* __restrict__ base, int4* __restrict__ table) {
  const int i = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ int part[4];
  int b = 0;
  for (int j = threadIdx.x; j < i; j += 256) b += (offs[j + 1] - offs[j] + ch - 1) / ch;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) b += __shfl_xor(b, o, 64);
  if (lane == 0) part[wave] = b;
  __syncthreads();
  b = part[0] + part[1] + part[2] + part[3];
  if (threadIdx.x == 0) base[i] = b;
  if (i == n) {
    for (int k = b + threadIdx.x; k < max_chunks; k += 256) table[k] = make_int4(-1, 0, 0, 0);
    return;
  }
  const int lo = offs[i], hi = offs[i + 1];
  for (int k = threadIdx.x; k < (hi - lo + ch - 1) / ch; k += 256) {
    const int s = lo + k * ch;
    table[b + k] = make_int4(i, s, s + ch < hi ? s + ch : hi, 0);
  }
}

// ------------------------------------------------------------------------------------------------ down: s_i F_i y_m
// 16 rows per workgroup, the four waves take every fourth 32-wide k-step. The factor is the MFMA's "A" operand, the rows its "B"
// operand, so a lane ends with four consecutive ranks of row fr. Bound by reading the rows once (the factors come from L2).
template <int NR>      // RP / 16
__global__ __launch_bounds__(256) void pool_down_kernel(const bf16_t* __restrict__ X, int64_t ldx, const bf16_t* __restrict__ F, const float* __restrict__ scale,
                                                        const int* __restrict__ ids, int n, float* __restrict__ out, int64_t M, int K) {
  __shared__ f32x4_t red[3][NR][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const int64_t m = (int64_t)blockIdx.x * 16 + fr;
  int id = m < M ? ids[m] : -1;
  if ((unsigned)id >= (unsigned)n) id = -1;
  const bf16_t* xp = X + (m < M ? m : M - 1) * ldx + 8 * fq;
  f32x4_t sel[NR];
#pragma unroll
  for (int f = 0; f < NR; ++f) sel[f] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  const int nks = (K + 31) / 32;
  for (int last = -1;;) {
    const int cur = next_id(id > last ? id : NO_ID);
    if (cur == NO_ID) break;
    last = cur;
    const bf16_t* fp = F + ((int64_t)cur * 16 * NR + fr) * K + 8 * fq;
    f32x4_t acc[NR];
#pragma unroll
    for (int f = 0; f < NR; ++f) acc[f] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int ks = wave; ks < nks; ks += 4) {
      Frag x, a[NR];
      const bool on = 32 * ks + 8 * fq < K;               // chunks behind the last column are zeros on both sides
      x.q = on ? *reinterpret_cast<const u32x4_t*>(xp + 32 * ks) : (u32x4_t){0u, 0u, 0u, 0u};
#pragma unroll
      for (int f = 0; f < NR; ++f) a[f].q = on ? *reinterpret_cast<const u32x4_t*>(fp + (int64_t)16 * f * K + 32 * ks) : (u32x4_t){0u, 0u, 0u, 0u};
#pragma unroll
      for (int f = 0; f < NR; ++f) acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[f].v, x.v, acc[f], 0, 0, 0);
    }
#pragma unroll
    for (int f = 0; f < NR; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r) sel[f][r] = id == cur ? acc[f][r] : sel[f][r];
  }
  if (wave) {
#pragma unroll
    for (int f = 0; f < NR; ++f) red[wave - 1][f][lane] = sel[f];
  }
  __syncthreads();
  if (wave == 0 && m < M) {
    const float s = id >= 0 ? scale[id] : 0.f;
#pragma unroll
    for (int f = 0; f < NR; ++f) {
      const f32x4_t t = (sel[f] + red[0][f][lane]) + (red[1][f][lane] + red[2][f][lane]);
      // (no adapter: zeros, whatever the sums hold)
      const float4 o = id >= 0 ? make_float4(s * t[0], s * t[1], s * t[2], s * t[3]) : make_float4(0.f, 0.f, 0.f, 0.f);
      *reinterpret_cast<float4*>(out + m * (16 * NR) + 16 * f + 4 * fq) = o;
    }
  }
}

// ------------------------------------------------------------------------------------------------ out = X W^T + bias + Up_i down
struct PoolGemm {
  const bf16_t* X; int64_t ldx; const bf16_t* W; int64_t ldw; const float* bias;
  const float* D; const bf16_t* Up; const int* ids; int n, RP;
  void* out; int64_t ldo; int out_f32;
  int64_t M; int N, K, tiles_m, tiles_n;
};

// chunk XOR of W row o of a wave's columns: conflict-free ds_read_b128 for the permuted row sets (G fragments per group)
template <int G> __device__ __forceinline__ int pool_swz_w(int o) {
  return G == 4 ? ((((o >> 4) & 3) << 1) | ((o >> 1) & 1)) : ((((o >> 3) & 3) << 1) | ((o >> 1) & 1));
}

// WM x WN waves, each 16 XF rows x 16 G columns; k-tiles of 64 in two LDS buffers filled by global_load_lds. The W rows are the MFMA's
// "A" operand, read in a permuted order so that a lane ends with 4 G consecutive columns of row fr of each row fragment.
template <int WM, int WN, int XF, int G>
__global__ __launch_bounds__(64 * WM * WN, (WM * WN) / 4) void pool_gemm_kernel(const PoolGemm p) {
  constexpr int NW = WM * WN, BM = 16 * XF * WM, BN = 16 * G * WN, ROWS = BM + BN, STAGE = ROWS * 128, PPW = ROWS / 8 / NW;
  static_assert(ROWS % (8 * NW) == 0, "whole 1-KB pieces per wave");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane & 15, fq = lane >> 4;
  // XCD-aware: workgroup ids go round-robin over the 8 XCDs; each XCD walks a contiguous run of tiles
  const int nwg = p.tiles_m * p.tiles_n;
  int wg;
  {
    const int orig = blockIdx.x, xcd = orig & 7, q = nwg >> 3, r = nwg & 7;
    wg = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (orig >> 3);
  }
  const int tm = wg / p.tiles_n, tn = wg - tm * p.tiles_n;
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN;

  // staging: piece j holds stage rows 8j .. 8j+7; lane -> row 8j + (lane >> 3), destination chunk lane & 7
  const bf16_t* src[PPW];
  int kch[PPW];
#pragma unroll
  for (int i = 0; i < PPW; ++i) {
    const int row = 8 * (wave + NW * i) + (lane >> 3);
    if (row < BM) {
      const int64_t m = m0 + row < p.M ? m0 + row : p.M - 1;           // rows and columns past the end repeat the last one: never stored
      kch[i] = ((lane & 7) ^ (row & 7)) << 3;
      src[i] = p.X + m * p.ldx + kch[i];
    } else {
      const int jw = row - BM, nn = n0 + jw < p.N ? n0 + jw : p.N - 1;
      kch[i] = ((lane & 7) ^ pool_swz_w<G>(jw % (16 * G))) << 3;
      src[i] = p.W + (int64_t)nn * p.ldw + kch[i];
    }
  }
  const int nt = (p.K + 63) / 64;
  auto stage = [&](int kt, int buf) {
    unsigned char* base = lds + buf * STAGE;
#pragma unroll
    for (int i = 0; i < PPW; ++i) {
      const bf16_t* s = src[i] + kt * 64;
      if (kt * 64 + 64 > p.K) s = kt * 64 + kch[i] < p.K ? s : reinterpret_cast<const bf16_t*>(g_pool_zero);     // (uniform branch: the last k-tile of a ragged K)
      __builtin_amdgcn_global_load_lds((gbl_ptr_t)s, (lds_ptr_t)(base + (wave + NW * i) * 1024), 16, 0, 0);
    }
  };

  int x_off[XF], x_sw, w_off[G], w_sw[G];
#pragma unroll
  for (int i = 0; i < XF; ++i) x_off[i] = (wm * 16 * XF + i * 16 + fr) * 128;
  x_sw = fr & 7;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int o = 4 * G * (fr >> 2) + 4 * i + (fr & 3);
    w_off[i] = (BM + wn * 16 * G + o) * 128;
    w_sw[i] = pool_swz_w<G>(o);
  }
  f32x4_t acc[G][XF];
#pragma unroll
  for (int a = 0; a < G; ++a)
#pragma unroll
    for (int b = 0; b < XF; ++b) acc[a][b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

  stage(0, 0);
  for (int t = 0; t < nt; ++t) {
    if (t + 1 < nt) {
      stage(t + 1, (t + 1) & 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PPW) : "memory");      // tile t landed, tile t + 1 in flight
    } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const unsigned char* base = lds + (t & 1) * STAGE;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      bf16x8_t xf[XF], wf[G];
      const int ch = fq + 4 * ks;
#pragma unroll
      for (int i = 0; i < XF; ++i) xf[i] = *reinterpret_cast<const bf16x8_t*>(base + x_off[i] + ((ch ^ x_sw) << 4));
#pragma unroll
      for (int i = 0; i < G; ++i) wf[i] = *reinterpret_cast<const bf16x8_t*>(base + w_off[i] + ((ch ^ w_sw[i]) << 4));
#pragma unroll
      for (int a = 0; a < G; ++a)
#pragma unroll
        for (int b = 0; b < XF; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[a], xf[b], acc[a][b], 0, 0, 0);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                // this wave's reads of tile t are done: its buffer may be refilled
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // ---- epilogue: lane owns rows m0 + wm*16*XF + 16 b + fr and columns cb .. cb + 4G - 1
  const int64_t mw = m0 + wm * 16 * XF + fr;
  const int ncol = n0 + wn * 16 * G;
  if (p.D) {
    int id[XF];
#pragma unroll
    for (int b = 0; b < XF; ++b) {
      const int64_t m = mw + 16 * b;
      id[b] = m < p.M ? p.ids[m] : -1;
      if ((unsigned)id[b] >= (unsigned)p.n) id[b] = -1;
    }
    const int RP = p.RP, wide = RP > 16;
    // k-slots of one MFMA: RP = 16: ranks 0..15 of part hi, then of part lo; wider: 32 ranks of one part
    const int parts = p.out_f32 ? 3 : 2;                   // a bf16 result needs 16 bits of the product's fp32 factor, an fp32 one all
    for (int last = -1;;) {
      int cand = NO_ID;
#pragma unroll
      for (int b = 0; b < XF; ++b) cand = id[b] > last && id[b] < cand ? id[b] : cand;
      const int cur = next_id(cand);
      if (cur == NO_ID) break;
      last = cur;
      bool same = true;
#pragma unroll
      for (int b = 0; b < XF; ++b) same = same && (id[b] == cur || mw + 16 * b >= p.M);
      const bool uniform = __all(same);
      for (int s = 0; s < (wide ? parts * (RP / 32) : parts - 1); ++s) {
        const int rk = wide ? 32 * (s / parts) + 8 * fq : 8 * (fq & 1);
        const int part = wide ? s % parts : 2 * s + (fq >> 1);      // (RP = 16, s = 1: parts 2 and 3; the fourth is left out)
        Frag up[G];
#pragma unroll
        for (int a = 0; a < G; ++a) {
          int c = ncol + 4 * G * (fr >> 2) + 4 * a + (fr & 3);
          c = c < p.N ? c : p.N - 1;
          up[a].q = *reinterpret_cast<const u32x4_t*>(p.Up + ((int64_t)cur * p.N + c) * RP + rk);
        }
#pragma unroll
        for (int b = 0; b < XF; ++b) {
          const int64_t m = mw + 16 * b < p.M ? mw + 16 * b : p.M - 1;
          const float4 u0 = *reinterpret_cast<const float4*>(p.D + m * RP + rk), u1 = *reinterpret_cast<const float4*>(p.D + m * RP + rk + 4);
          const float x[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
          Frag u;
          if (part == 0) u.v = split_part(x, 0);
          else if (part == 1) u.v = split_part(x, 1);
          else if (part == 2) u.v = split_part(x, 2);
          else u.q = (u32x4_t){0u, 0u, 0u, 0u};
          if (uniform) {
#pragma unroll
            for (int a = 0; a < G; ++a) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(up[a].v, u.v, acc[a][b], 0, 0, 0);
          } else {
#pragma unroll
            for (int a = 0; a < G; ++a) {
              const f32x4_t t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(up[a].v, u.v, acc[a][b], 0, 0, 0);
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[a][b][r] = id[b] == cur ? t[r] : acc[a][b][r];
            }
          }
        }
      }
    }
  }
  const int cb = ncol + 4 * G * fq;
  float bv[4 * G];
#pragma unroll
  for (int a = 0; a < G; ++a) {
    const float4 b4 = p.bias && cb + 4 * a < p.N ? *reinterpret_cast<const float4*>(p.bias + cb + 4 * a) : make_float4(0.f, 0.f, 0.f, 0.f);
    bv[4 * a] = b4.x; bv[4 * a + 1] = b4.y; bv[4 * a + 2] = b4.z; bv[4 * a + 3] = b4.w;
  }
#pragma unroll
  for (int b = 0; b < XF; ++b) {
    const int64_t m = mw + 16 * b;
    if (m >= p.M) continue;
    if (p.out_f32) {
      float* o = (float*)p.out + m * p.ldo + cb;
#pragma unroll
      for (int a = 0; a < G; ++a)
        if (cb + 4 * a < p.N)
          *reinterpret_cast<float4*>(o + 4 * a) = make_float4(acc[a][b][0] + bv[4 * a], acc[a][b][1] + bv[4 * a + 1], acc[a][b][2] + bv[4 * a + 2], acc[a][b][3] + bv[4 * a + 3]);
    } else {
      bf16_t* o = (bf16_t*)p.out + m * p.ldo + cb;
#pragma unroll
      for (int h = 0; h < G / 2; ++h)
        if (cb + 8 * h < p.N) {
          u32x4_t w;
          w.x = pack_bf16x2(acc[2 * h][b][0] + bv[8 * h], acc[2 * h][b][1] + bv[8 * h + 1]);
          w.y = pack_bf16x2(acc[2 * h][b][2] + bv[8 * h + 2], acc[2 * h][b][3] + bv[8 * h + 3]);
          w.z = pack_bf16x2(acc[2 * h + 1][b][0] + bv[8 * h + 4], acc[2 * h + 1][b][1] + bv[8 * h + 5]);
          w.w = pack_bf16x2(acc[2 * h + 1][b][2] + bv[8 * h + 6], acc[2 * h + 1][b][3] + bv[8 * h + 7]);
          *reinterpret_cast<u32x4_t*>(o + 8 * h) = w;
        }
    }
  }
}

// ------------------------------------------------------------------------------------------------ dA / dB: sums over an adapter's rows
// part[chunk] = sum over the chunk's rows of y_m u_m^T. 256 columns of y per workgroup, the four waves take every fourth step of 32 rows:
// a step is copied into wave-private [32][64] LDS slabs (row-major, swizzled) and read transposed (ds_read_b64_tr_b16) as one MFMA
// operand; the other is u (fp32), split into three bf16 parts. Rows behind the chunk are zeros on BOTH sides, rows of other adapters are
// never read. y is bf16 or an 8-bit checkpoint, whose values are exact in bf16. RANK_MAJOR: part [RP][C] (dA), else [C][RP] (dB).
struct PoolTn {
  const bf16_t* Y; int64_t ldy; const signed char* codes; const unsigned char* exps;
  const float* U; int RP; const int* perm; const int4* table; float* part; int C;
};
#define TN_MAX_CH 512
template <int NR, bool CKPT, bool RANK_MAJOR>
__global__ __launch_bounds__(256, 2) void pool_tn_kernel(const PoolTn p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[4][4][32 * 128];
  __shared__ int rows[TN_MAX_CH];
  const int4 ck = p.table[blockIdx.y];
  if (ck.x < 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const int cw = blockIdx.x * 256, C = p.C, len = ck.z - ck.y;
  const int j0 = 16 * NR * blockIdx.z;                               // first rank of this workgroup
  for (int i = threadIdx.x; i < len; i += 256) rows[i] = p.perm[ck.y + i];
  __syncthreads();
  f32x4_t acc[4][4][NR];
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int f = 0; f < NR; ++f) acc[s][t][f] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  const int srow = lane >> 3, sch = lane & 7;
  const int nb = (C + 31) >> 5;
  u32x4_t yv[4][4];
  unsigned int eb[4][4];
  float uv[NR][8];
  auto issue = [&](int i0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = i0 + srow + 8 * i;
      const int64_t m = k < len ? rows[k] : -1;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int c = cw + 64 * s + 8 * sch;
        const bool on = m >= 0 && c < C;
        if (CKPT) {
          const u32x2_t w = on ? *reinterpret_cast<const u32x2_t*>(p.codes + m * C + c) : (u32x2_t){0u, 0u};
          yv[s][i].x = w.x; yv[s][i].y = w.y;
          eb[s][i] = on ? p.exps[m * nb + (c >> 5)] : 0u;
        } else yv[s][i] = on ? *reinterpret_cast<const u32x4_t*>(p.Y + m * p.ldy + c) : (u32x4_t){0u, 0u, 0u, 0u};
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = i0 + 16 * (j >> 2) + 4 * fq + (j & 3);             // k-slot j of lane quarter fq <-> this row of the step
      const int64_t m = k < len ? rows[k] : -1;
#pragma unroll
      for (int f = 0; f < NR; ++f) uv[f][j] = m >= 0 ? p.U[m * p.RP + j0 + 16 * f + fr] : 0.f;
    }
  };
  int i0 = 32 * wave;
  if (i0 < len) issue(i0);
  for (; i0 < len; i0 += 128) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = srow + 8 * i;
        u32x4_t v = yv[s][i];
        if (CKPT) {
          const float step = ckpt8_step(eb[s][i]);
          u32x4_t o;
          o.x = pack_bf16x2(ckpt8_value(v.x, 0, step), ckpt8_value(v.x, 1, step)); o.y = pack_bf16x2(ckpt8_value(v.x, 2, step), ckpt8_value(v.x, 3, step));
          o.z = pack_bf16x2(ckpt8_value(v.y, 0, step), ckpt8_value(v.y, 1, step)); o.w = pack_bf16x2(ckpt8_value(v.y, 2, step), ckpt8_value(v.y, 3, step));
          v = o;
        }
        *reinterpret_cast<u32x4_t*>(lds[wave][s] + row * 128 + ((sch ^ (row & 7)) << 4)) = v;
      }
    bf16x8_t up[NR][3];
#pragma unroll
    for (int f = 0; f < NR; ++f)
#pragma unroll
      for (int q = 0; q < 3; ++q) up[f][q] = split_part(uv[f], q);
    if (i0 + 128 < len) issue(i0 + 128);
    const int trow = 4 * fq + (fr >> 2);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const unsigned char* img = lds[wave][s];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const unsigned char* a = img + trow * 128 + (((2 * t + ((fr >> 1) & 1)) ^ (trow & 7)) << 4) + ((fr & 1) << 3);
        Frag y;
        y.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr_t)a);
        y.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr_t)(a + 16 * 128));
#pragma unroll
        for (int f = 0; f < NR; ++f)
#pragma unroll
          for (int q = 2; q >= 0; --q)
            acc[s][t][f] = RANK_MAJOR ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(up[f][q], y.v, acc[s][t][f], 0, 0, 0)
                                      : __builtin_amdgcn_mfma_f32_16x16x32_bf16(y.v, up[f][q], acc[s][t][f], 0, 0, 0);
      }
    }
  }
  // sum of the four waves, one slab of 64 columns after the other (16 KB per wave and fragment column); wave w writes tile t = w
  float* out = p.part + (int64_t)blockIdx.y * p.RP * C;
#pragma unroll
  for (int f = 0; f < NR; ++f) {
    __syncthreads();
    float* mine = reinterpret_cast<float*>(lds[wave][0]);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) mine[((s * 4 + t) * 4 + r) * 64 + lane] = acc[s][t][f][r];
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int idx = ((wave * 4 + t) * 4 + r) * 64 + lane;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) v += reinterpret_cast<const float*>(lds[w][0])[idx];
        const int a = 4 * fq + r;
        const int c = cw + 64 * wave + 16 * t + (RANK_MAJOR ? fr : a), j = j0 + 16 * f + (RANK_MAJOR ? a : fr);
        if (c < C) out[RANK_MAJOR ? (int64_t)j * C + c : (int64_t)c * p.RP + j] = v;
      }
  }
}

// out[i] = sum over the chunks of adapter i, in order; part entries [d0][ld] -> out [d0][d1] (the padded ranks are dropped). No rows: zeros.
__global__ __launch_bounds__(256) void pool_sum_kernel(const float* __restrict__ part, const int* __restrict__ base, int64_t per, int ld, int d0, int d1, float* __restrict__ out) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= (int64_t)d0 * d1) return;
  const int i = blockIdx.y;
  const int64_t src = (e / d1) * ld + e % d1;
  float s = 0.f;
  for (int k = base[i]; k < base[i + 1]; ++k) s += part[k * per + src];
  out[(int64_t)i * d0 * d1 + e] = s;
}

// ------------------------------------------------------------------------------------------------ host
static bool pool_rp(int RP) { return RP == 16 || RP == 32 || RP == 64; }

extern "C" int mfnet_lora_pool_pack(const void* src, int dtype, int long_first, int64_t n, int64_t C, int r, int RP, void* down, void* up, hipStream_t stream) {
  MF_CHECK_ARG(src && (down || up), "lora_pool_pack: null pointer");
  MF_CHECK_ARG(dtype == MFNET_F32 || dtype == MFNET_BF16, "lora_pool_pack: bad dtype");
  MF_CHECK_ARG(n >= 1 && n <= 65535 && C >= 8 && C % 8 == 0 && C < (1 << 24) && r >= 1 && r <= RP && pool_rp(RP), "lora_pool_pack: bad sizes (n=%lld C=%lld r=%d RP=%d)",
               (long long)n, (long long)C, r, RP);
  MF_CHECK_ARG((uintptr_t)src % (dtype == MFNET_F32 ? 4 : 2) == 0 && (uintptr_t)up % 16 == 0 && (uintptr_t)down % 16 == 0, "lora_pool_pack: misaligned tensor");
  const dim3 grid((unsigned)ceil_div64(C, 256), (unsigned)n);
#define PP(T_, L_) hipLaunchKernelGGL((pool_pack_kernel<T_, L_>), grid, dim3(256), 0, stream, (const T_*)src, (int)C, r, RP, (bf16_t*)down, (bf16_t*)up)
  if (dtype == MFNET_F32) { if (long_first) PP(float, true); else PP(float, false); }
  else { if (long_first) PP(bf16_t, true); else PP(bf16_t, false); }
#undef PP
  MF_LAUNCH_CHECK("lora_pool_pack");
  return MFNET_OK;
}

// rows of a chunk of the backward sums
static int pool_chunk_rows(int64_t M) { return M <= 16384 ? 128 : TN_MAX_CH; }
extern "C" int64_t mfnet_lora_pool_chunks(int64_t M, int64_t n) {
  return M <= 0 || n <= 0 ? 0 : M / pool_chunk_rows(M) + (n < M ? n : M);
}

extern "C" int mfnet_lora_pool_plan(const int* ids, int64_t M, int64_t n, int* offs, int* perm, int* base, int* table, hipStream_t stream) {
  MF_CHECK_ARG(M >= 0 && M < (1ll << 31) - 256 && n >= 1 && n <= 65535, "lora_pool_plan: bad sizes (M=%lld n=%lld)", (long long)M, (long long)n);
  MF_CHECK_ARG(offs && base && (M == 0 || (ids && perm && table)), "lora_pool_plan: null pointer");
  MF_CHECK_ARG((uintptr_t)table % 16 == 0, "lora_pool_plan: table must be 16-byte aligned");
  hipLaunchKernelGGL(pool_plan_kernel, dim3((unsigned)n + 1), dim3(256), 0, stream, ids, (int)M, (int)n, offs, perm);
  MF_LAUNCH_CHECK("lora_pool_plan");
  hipLaunchKernelGGL(pool_chunks_kernel, dim3((unsigned)n + 1), dim3(256), 0, stream, offs, (int)n, pool_chunk_rows(M), (int)mfnet_lora_pool_chunks(M, n), base, (int4*)table);
  MF_LAUNCH_CHECK("lora_pool_plan (chunks)");
  return MFNET_OK;
}

#define POOL_CHECK_ROWS(name, T_, ld_, C_)                                                                                          \
  MF_CHECK_ARG((C_) >= 8 && (C_) % 8 == 0 && (C_) < (1 << 24) && (ld_) >= (C_) && (ld_) % 8 == 0 && (uintptr_t)(T_) % 16 == 0,      \
               name ": rows must hold a multiple of 8 elements, 16-byte aligned, row stride a multiple of 8 (C=%lld ld=%lld)", (long long)(C_), (long long)(ld_))

extern "C" int mfnet_lora_pool_down(const void* X, int64_t ldx, const void* down, const float* scale, const int* ids, int64_t n, int RP,
                                    float* out, int64_t M, int64_t K, hipStream_t stream) {
  MF_CHECK_ARG(M >= 0 && M < (1ll << 31) - 256 && n >= 1 && n <= 65535 && pool_rp(RP), "lora_pool_down: bad sizes (M=%lld n=%lld RP=%d)", (long long)M, (long long)n, RP);
  if (M == 0) return MFNET_OK;
  MF_CHECK_ARG(X && down && scale && ids && out, "lora_pool_down: null pointer");
  POOL_CHECK_ROWS("lora_pool_down", X, ldx, K);
  MF_CHECK_ARG(((uintptr_t)down | (uintptr_t)out) % 16 == 0, "lora_pool_down: misaligned tensor");
  const dim3 grid((unsigned)ceil_div64(M, 16));
#define PD(NR_) hipLaunchKernelGGL((pool_down_kernel<NR_>), grid, dim3(256), 0, stream, (const bf16_t*)X, ldx, (const bf16_t*)down, scale, ids, (int)n, out, M, (int)K)
  if (RP == 16) PD(1); else if (RP == 32) PD(2); else PD(4);
#undef PD
  MF_LAUNCH_CHECK("lora_pool_down");
  return MFNET_OK;
}

extern "C" int mfnet_lora_pool_gemm(const void* X, int64_t ldx, const void* W, int64_t ldw, const float* bias, const float* D, const void* up,
                                    const int* ids, int64_t n, int RP, void* out, int out_dtype, int64_t ldo, int64_t M, int64_t N, int64_t K,
                                    hipStream_t stream) {
  MF_CHECK_ARG(M >= 0 && M < (1ll << 31) - 256, "lora_pool_gemm: bad row count");
  MF_CHECK_ARG(out_dtype == MFNET_BF16 || out_dtype == MFNET_F32, "lora_pool_gemm: bad out dtype");
  if (M == 0) return MFNET_OK;
  MF_CHECK_ARG(X && W && out && (!D || (up && ids)), "lora_pool_gemm: null pointer");
  MF_CHECK_ARG(!D || (n >= 1 && n <= 65535 && pool_rp(RP)), "lora_pool_gemm: bad pool (n=%lld RP=%d)", (long long)n, RP);
  POOL_CHECK_ROWS("lora_pool_gemm", X, ldx, K);
  POOL_CHECK_ROWS("lora_pool_gemm (weight)", W, ldw, K);
  POOL_CHECK_ROWS("lora_pool_gemm (out)", out, ldo, N);
  MF_CHECK_ARG(((uintptr_t)bias | (uintptr_t)D | (uintptr_t)up) % 16 == 0, "lora_pool_gemm: misaligned tensor");
  PoolGemm p;
  p.X = (const bf16_t*)X; p.ldx = ldx; p.W = (const bf16_t*)W; p.ldw = ldw; p.bias = bias;
  p.D = D; p.Up = (const bf16_t*)up; p.ids = ids; p.n = (int)n; p.RP = RP;
  p.out = out; p.ldo = ldo; p.out_f32 = out_dtype == MFNET_F32;
  p.M = M; p.N = (int)N; p.K = (int)K;
#define PG(WM_, WN_, XF_, G_) do { p.tiles_m = (int)ceil_div64(M, 16 * XF_ * WM_); p.tiles_n = (int)ceil_div64(N, 16 * G_ * WN_); \
    MF_CHECK_ARG((int64_t)p.tiles_m * p.tiles_n < (1ll << 31), "lora_pool_gemm: too many tiles"); \
    hipLaunchKernelGGL((pool_gemm_kernel<WM_, WN_, XF_, G_>), dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(64 * WM_ * WN_), 0, stream, p); } while (0)
  if (ceil_div64(M, 256) * ceil_div64(N, 256) >= 200) PG(2, 4, 8, 4);
  else if (ceil_div64(M, 128) * ceil_div64(N, 128) >= 200) PG(2, 2, 4, 4);
  else PG(2, 2, 2, 2);
#undef PG
  MF_LAUNCH_CHECK("lora_pool_gemm");
  return MFNET_OK;
}

// floats of workspace of mfnet_lora_pool_tn
extern "C" int64_t mfnet_lora_pool_tn_workspace_floats(int64_t M, int64_t n, int64_t C, int RP) { return mfnet_lora_pool_chunks(M, n) * C * RP; }

extern "C" int mfnet_lora_pool_tn(const void* Y, int64_t ldy, const void* codes, const void* exps, const float* U, int RP, const int* perm, const int* base,
                                  const int* table, int64_t M, int64_t n, int64_t C, int r, int rank_major, float* out, float* ws, int64_t ws_floats, hipStream_t stream) {
  MF_CHECK_ARG(M >= 0 && M < (1ll << 31) - 256 && n >= 1 && n <= 65535 && pool_rp(RP) && r >= 1 && r <= RP, "lora_pool_tn: bad sizes");
  MF_CHECK_ARG(out && base, "lora_pool_tn: null pointer");
  MF_CHECK_ARG(C >= 8 && C % 8 == 0 && C < (1 << 24), "lora_pool_tn: C=%lld must be a multiple of 8", (long long)C);
  const int64_t chunks = mfnet_lora_pool_chunks(M, n);
  if (M > 0) {
    MF_CHECK_ARG(U && perm && table && ((Y != nullptr) != (codes != nullptr)) && (!codes || exps), "lora_pool_tn: null pointer (rows as bf16 or as a checkpoint)");
    if (Y) POOL_CHECK_ROWS("lora_pool_tn", Y, ldy, C);
    MF_CHECK_ARG((uintptr_t)codes % 8 == 0 && (uintptr_t)table % 16 == 0 && (uintptr_t)U % 4 == 0, "lora_pool_tn: misaligned tensor");
    MF_CHECK_ARG(ws && ws_floats >= chunks * C * RP, "lora_pool_tn: workspace too small");
    MF_CHECK_ARG(chunks <= 65535, "lora_pool_tn: too many chunks of rows (%lld)", (long long)chunks);
    PoolTn p;
    p.Y = (const bf16_t*)Y; p.ldy = ldy; p.codes = (const signed char*)codes; p.exps = (const unsigned char*)exps;
    p.U = U; p.RP = RP; p.perm = perm; p.table = (const int4*)table; p.part = ws; p.C = (int)C;
    const dim3 grid((unsigned)ceil_div64(C, 256), (unsigned)chunks, RP == 64 ? 2 : 1);
#define PT(NR_, CK_, RM_) hipLaunchKernelGGL((pool_tn_kernel<NR_, CK_, RM_>), grid, dim3(256), 0, stream, p)
#define PT2(NR_, CK_) do { if (rank_major) PT(NR_, CK_, true); else PT(NR_, CK_, false); } while (0)
    if (RP == 16) { if (codes) PT2(1, true); else PT2(1, false); }
    else { if (codes) PT2(2, true); else PT2(2, false); }
#undef PT2
#undef PT
    MF_LAUNCH_CHECK("lora_pool_tn");
  }
  const int d0 = rank_major ? r : (int)C, d1 = rank_major ? (int)C : r;
  hipLaunchKernelGGL(pool_sum_kernel, dim3((unsigned)ceil_div64((int64_t)d0 * d1, 256), (unsigned)n), dim3(256), 0, stream, ws, base, C * RP,
                     rank_major ? (int)C : RP, d0, d1, out);
  MF_LAUNCH_CHECK("lora_pool_tn (sums)");
  return MFNET_OK;
}
