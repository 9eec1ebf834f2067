// A pool of low-rank adapters beside one shared projection, forward and backward. Every row m names its adapter i = ids[m] (none if the
// index lies outside [0, n)): rows of many requests, tiles or jobs, in any order, in one call.
//
//   down[m]  = s_i A_i x_m                                  (fp32 [M, RP], kept for the backward pass)
//   out[m]   = W x_m + bias + B_i down[m]
//   p[m]     = s_i B_i^T dy_m
//   dx[m]    = W^T dy_m + A_i^T p[m]
//   dA_i     = sum over the rows of adapter i of p[m] x_m^T,     dB_i = sum of dy_m down[m]^T
//
// The factors are held as bf16 images padded to RP = 16, 32 or 64 ranks (mfnet_lora_pool_pack): "down" images for products that contract
// over the long axis, "up" images for products that contract over the ranks, so that both are read as MFMA
// operands in 16-byte pieces. Adapters given in fp32 are rounded to bf16 there, once. The fp32 factors that a call makes itself (down, p)
// are split into bf16 parts hi + lo (+ lo').
//
// A workgroup that meets rows of several adapters multiplies all its rows with each adapter in turn and SELECTS the rows it belongs to:
// a sum of zeros would let one adapter's infinities and NaN into another request's rows. In its own rows an infinity may end as NaN: padded
// ranks hold 0 * inf, the split inf - inf.
#include "ckpt8.h"
#include <math.h>
#include <type_traits>

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

// smallest index above `last` among the lanes' candidates (lane quarters hold copies of the same 16 rows); INT_MAX: none left. Rotations
// inside 16 lanes are single instructions: with shuffles through LDS [1500, 768] -> 768 took 14.2 us instead of 13.3 for 2 adapters in
// runs, 38.6 instead of 35.3 for 100 in random order.
__device__ __forceinline__ int next_id(int cand) {
  int q = __builtin_amdgcn_mov_dpp(cand, 0x128, 0xf, 0xf, true);      // by 8, 4, 2 and 1
  cand = cand < q ? cand : q;
  q = __builtin_amdgcn_mov_dpp(cand, 0x124, 0xf, 0xf, true);
  cand = cand < q ? cand : q;
  q = __builtin_amdgcn_mov_dpp(cand, 0x122, 0xf, 0xf, true);
  cand = cand < q ? cand : q;
  q = __builtin_amdgcn_mov_dpp(cand, 0x121, 0xf, 0xf, true);
  cand = cand < q ? cand : q;
  return __builtin_amdgcn_readfirstlane(cand);
}
#define NO_ID 0x7fffffff

// ------------------------------------------------------------------------------------------------ images
// The "down" image is kept in MFMA operand order: [n][k-step of 32][RP / 16][lane][8], lane = (rank % 16) + 16 (k % 32 / 8), zeros behind
// the last column up to a multiple of 64: a fragment is one dense KB. The "up" image is [n][C][RP].
__device__ __host__ __forceinline__ int64_t pool_image(int64_t C, int RP) { return (C + 63) / 64 * 64 * RP; }      // elements of a down image per adapter
struct PoolPack { const void* src[2]; bf16_t* down[2]; bf16_t* up[2]; int C[2], r, RP; const float* scale; float* scale_out; };
template <typename T>
__global__ __launch_bounds__(256) void pool_pack_kernel(const PoolPack p) {
  const int z = blockIdx.z, C = p.C[z], r = p.r, RP = p.RP;                    // z = 0: A [n][r][K], 1: B [n][N][r]
  const int64_t i = blockIdx.y;
  const T* s = (const T*)p.src[z] + i * (int64_t)C * r;
  auto at = [&](int c, int k) {
    if (c >= C || k >= r) return 0.f;
    const T t = z ? s[(int64_t)c * r + k] : s[(int64_t)k * C + c];
    if constexpr (sizeof(T) == 4) return t; else return bf16_to_f32(t);
  };
  if (z == 0 && blockIdx.x == 0 && threadIdx.x == 0) p.scale_out[i] = p.scale ? p.scale[i] : 1.f;
  const int chunks = (C + 63) / 64 * 8 * RP;                                   // 16-byte pieces of the down image, then of the up image
  const int t = blockIdx.x * 256 + threadIdx.x;
  float v[8];
  bf16_t* dst;
  if (t < chunks) {
    const int lane = t & 63, f = t >> 6, ks = f / (RP / 16), k = 16 * (f % (RP / 16)) + (lane & 15), c = 32 * ks + 8 * (lane >> 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at(c + j, k);
    dst = p.down[z] + i * pool_image(C, RP) + (int64_t)t * 8;
  } else {
    const int u = t - chunks, c = u / (RP / 8), k = 8 * (u % (RP / 8));
    if (c >= C) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at(c, k + j);
    dst = p.up[z] + (i * C + c) * RP + k;
  }
  Frag f;
#pragma unroll
  for (int j = 0; j < 4; ++j) f.w[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<u32x4_t*>(dst) = f.q;
}

// ------------------------------------------------------------------------------------------------ rows grouped by adapter
// Workgroup i: how many rows belong to adapters below i (their places come first), then the rows of adapter i in ascending order.
// Deterministic without a sort; the indices are read from L2 twice per adapter, four per thread and step (32768 rows, 8 adapters: 17 us;
// one per thread of 256: 96).
__global__ __launch_bounds__(1024) void pool_plan_kernel(const int* __restrict__ ids, int M, int n, int* __restrict__ offs, int* __restrict__ perm) {
  const int i = blockIdx.x;                               // 0 .. n; workgroup n only writes offs[n]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ int part[2][16];
  int below = 0;
  for (int m = threadIdx.x; m < M; m += 4096)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = m + 1024 * j, v = k < M ? ids[k] : -1;
      below += (v >= 0 && v < i) ? 1 : 0;
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o, 64);
  if (lane == 0) part[0][wave] = below;
  __syncthreads();
  int pos = 0;
  for (int w = 0; w < 16; ++w) pos += part[0][w];
  if (threadIdx.x == 0) offs[i] = pos;
  if (i == n) return;
  __syncthreads();
  for (int m0 = 0, step = 0; m0 < M; m0 += 4096, ++step) {
    int mine[4], cnt = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {                         // four rows in a row: the order inside a thread is the rows' order
      const int m = m0 + 4 * threadIdx.x + j;
      mine[j] = m < M && ids[m] == i;
      cnt += mine[j];
    }
    int scan = cnt;                                       // inclusive over the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int q = __shfl_up(scan, o, 64);
      if (lane >= o) scan += q;
    }
    int* pt = part[step & 1];
    if (lane == 63) pt[wave] = scan;
    __syncthreads();
    int at = pos + scan - cnt, all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      const int c = pt[w];
      at += w < wave ? c : 0;
      all += c;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (mine[j]) perm[at++] = m0 + 4 * threadIdx.x + j;
    pos += all;
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
// One row by one wave: the MFMA's 16 columns all hold the row - a sixteenth of the products, but one instruction where 8 multiply-adds
// and their conversions would stand. Four sums over every fourth k-step, as pool_down_row_kernel's waves have them: the same bits.
// Lanes with fr = 0 hold the result: ranks 16 f + 4 fq + r.
template <int NR>
__device__ __forceinline__ void pool_row_sums(const bf16_t* __restrict__ x, const bf16_t* __restrict__ fp, int K, int lane, f32x4_t (&t)[NR]) {
  const int fq = lane >> 4;
  const u32x4_t zero = (u32x4_t){0u, 0u, 0u, 0u};
  f32x4_t s[4][NR];
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int f = 0; f < NR; ++f) s[q][f] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  constexpr int IN = NR == 1 ? 8 : 4;                        // k-steps in flight
  for (int ks0 = 0; 32 * ks0 < K; ks0 += IN) {
    Frag xv[IN], a[IN][NR];
#pragma unroll
    for (int j = 0; j < IN; ++j) {
      const int ks = ks0 + j;
      const bool in = 32 * ks + 8 * fq < K;
      xv[j].q = in ? *reinterpret_cast<const u32x4_t*>(x + 32 * ks + 8 * fq) : zero;
#pragma unroll
      for (int f = 0; f < NR; ++f) a[j][f].q = in ? *reinterpret_cast<const u32x4_t*>(fp + ((int64_t)ks * NR + f) * 512 + 8 * lane) : zero;
    }
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
      for (int f = 0; f < NR; ++f) s[j & 3][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j][f].v, xv[j].v, s[j & 3][f], 0, 0, 0);
  }
#pragma unroll
  for (int f = 0; f < NR; ++f) t[f] = (s[0][f] + s[1][f]) + (s[2][f] + s[3][f]);
}
// The result: fp32 [M, RP], and (P > 0) the same in P bf16 parts [M][P][RP], hi + lo (+ lo'), as the up product's MFMA reads them: split
// once here, not by every wave that meets the row ([32768, 1280] x [1280, 5120]: 422 -> 397 us, [8192, 768] x [768, 2304]: 39 -> 36).
struct PoolDown { float* out; bf16_t* parts; int P; };
__device__ __forceinline__ void pool_store_down(const PoolDown& o, int64_t m, int RP, int j, float4 v) {      // ranks j .. j + 3 of row m
  *reinterpret_cast<float4*>(o.out + m * RP + j) = v;
  for (int q = 0; q < o.P; ++q) {
    u32x2_t w;
    w.x = pack_bf16x2(v.x, v.y); w.y = pack_bf16x2(v.z, v.w);
    *reinterpret_cast<u32x2_t*>(o.parts + (m * o.P + q) * RP + j) = w;
    v.x -= bf16_lo(w.x); v.y -= bf16_hi(w.x); v.z -= bf16_lo(w.y); v.w -= bf16_hi(w.y);
  }
}
template <int NR>
__device__ __forceinline__ void pool_down_row(const bf16_t* __restrict__ X, int64_t ldx, const bf16_t* __restrict__ F, const float* __restrict__ scale,
                                              const int* __restrict__ ids, int n, const PoolDown& out, int64_t m, int K, int lane) {
  const int id = ids[m];
  const bool on = (unsigned)id < (unsigned)n;
  f32x4_t t[NR];
#pragma unroll
  for (int f = 0; f < NR; ++f) t[f] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  if (on) {
    pool_row_sums<NR>(X + m * ldx, F + id * pool_image(K, 16 * NR), K, lane, t);
    const float s = scale[id];
#pragma unroll
    for (int f = 0; f < NR; ++f) t[f] *= s;
  }
  if ((lane & 15) == 0) {
#pragma unroll
    for (int f = 0; f < NR; ++f) pool_store_down(out, m, 16 * NR, 16 * f + 4 * (lane >> 4), make_float4(t[f][0], t[f][1], t[f][2], t[f][3]));
  }
}

// 16 XR rows per workgroup, the four waves take every fourth piece of 64 columns. The factor is the MFMA's "A" operand, the rows its "B"
// operand, so a lane ends with four consecutive ranks of row fr. Bound by reading the rows once. Both operands come through a ring of
// three pieces in LDS of the wave's own (global_load_lds, counted vmcnt, no barrier): rows in whole 128-byte lines, swizzled, the factor
// as dense KBs of its image. Read straight into registers the rows go 64 bytes at a time and the factor's rows again as often as the
// rows themselves: 77 us for [32768, 3840] instead of 45 (5.5 TB/s).
// perm: the k-th row of the call is perm[k], and only the *count rows that have an adapter are taken (the backward pass, whose plan has
// them grouped). A workgroup that meets more adapters than pay takes its rows one by one: each of the rows' own factor once, where the
// other way reads all its rows again for every adapter (20000 rows in random order over 48 adapters, K = 1280: 147 us to 76).
template <int NR, int XR>      // NR = RP / 16
__global__ __launch_bounds__(256) void pool_down_kernel(const bf16_t* __restrict__ X, int64_t ldx, const bf16_t* __restrict__ F, const float* __restrict__ scale,
                                                        const int* __restrict__ ids, int n, const int* __restrict__ perm, const int* __restrict__ count,
                                                        const PoolDown out, int64_t M, int K) {
  constexpr int RING = 3, XL = 2 * XR, FL = 2 * NR, PIECE = (XL + FL) * 1024;      // requests of 1 KB per piece: rows, factor
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4][RING][PIECE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int64_t mw = (int64_t)blockIdx.x * (16 * XR);
  if (count) M = *count;
  if (mw >= M) return;
  auto row_of = [&](int64_t k) { k = k < M ? k : M - 1; return perm ? (int64_t)perm[k] : k; };
  int id[XR];
  int64_t mrow[XR];
  f32x4_t sel[XR][NR];
#pragma unroll
  for (int b = 0; b < XR; ++b) {
    mrow[b] = row_of(mw + 16 * b + fr);
    id[b] = mw + 16 * b + fr < M ? ids[mrow[b]] : -1;
    if ((unsigned)id[b] >= (unsigned)n) id[b] = -1;
#pragma unroll
    for (int f = 0; f < NR; ++f) sel[b][f] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }
  {
    constexpr int FEW = XR == 1 ? 8 : 10;                    // reads of all rows and a factor against reads of a factor per row
    int met = 0;
    for (int last = -1; met <= FEW; ++met) {
      int cand = NO_ID;
#pragma unroll
      for (int b = 0; b < XR; ++b) cand = id[b] > last && id[b] < cand ? id[b] : cand;
      last = next_id(cand);
      if (last == NO_ID) break;
    }
    if (met > FEW) {
      for (int j = wave; j < 16 * XR && mw + j < M; j += 4) pool_down_row<NR>(X, ldx, F, scale, ids, n, out, row_of(mw + j), K, lane);
      return;
    }
  }
  const bf16_t* src[XL];                                     // request i: rows 8 i + (lane >> 3), chunk (lane & 7) of its 128 bytes
  const int swz = (lane & 7) ^ (lane >> 3);
#pragma unroll
  for (int i = 0; i < XL; ++i) src[i] = X + row_of(mw + 8 * i + (lane >> 3)) * ldx + 8 * swz;
  const int np = ((K + 63) / 64 - wave + 3) / 4;             // pieces of this wave (0 if it has none)
  unsigned char* ring = lds[wave][0];
  for (int last = -1;;) {
    int cand = NO_ID;
#pragma unroll
    for (int b = 0; b < XR; ++b) cand = id[b] > last && id[b] < cand ? id[b] : cand;
    const int cur = next_id(cand);
    if (cur == NO_ID) break;
    last = cur;
    const bf16_t* fp = F + cur * pool_image(K, 16 * NR) + 8 * lane;
    auto request = [&](int j) __attribute__((always_inline)) {
      const int piece = wave + 4 * j;
      unsigned char* l = ring + (j % RING) * PIECE;
#pragma unroll
      for (int i = 0; i < XL; ++i) {
        const bf16_t* s = 64 * piece + 8 * swz < K ? src[i] + 64 * piece : reinterpret_cast<const bf16_t*>(g_pool_zero);      // behind the last column: zeros
        __builtin_amdgcn_global_load_lds((gbl_ptr_t)s, (lds_ptr_t)(l + i * 1024), 16, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < FL; ++i) __builtin_amdgcn_global_load_lds((gbl_ptr_t)(fp + ((int64_t)piece * FL + i) * 512), (lds_ptr_t)(l + (XL + i) * 1024), 16, 0, 0);
    };
    f32x4_t acc[XR][NR];
#pragma unroll
    for (int b = 0; b < XR; ++b)
#pragma unroll
      for (int f = 0; f < NR; ++f) acc[b][f] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < RING - 1 && j < np; ++j) request(j);
    for (int j = 0; j < np; ++j) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the place of piece j - 1 has been read
      if (j + RING - 1 < np) {
        request(j + RING - 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * (XL + FL)) : "memory");
      } else if (j + 1 < np) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(XL + FL) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      const unsigned char* l = ring + (j % RING) * PIECE;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        bf16x8_t a[NR];
#pragma unroll
        for (int f = 0; f < NR; ++f) a[f] = *reinterpret_cast<const bf16x8_t*>(l + (XL + ks * NR + f) * 1024 + lane * 16);
#pragma unroll
        for (int b = 0; b < XR; ++b) {
          const bf16x8_t x = *reinterpret_cast<const bf16x8_t*>(l + (16 * b + fr) * 128 + (((fq + 4 * ks) ^ (fr & 7)) << 4));
#pragma unroll
          for (int f = 0; f < NR; ++f) acc[b][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[f], x, acc[b][f], 0, 0, 0);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int b = 0; b < XR; ++b)
#pragma unroll
      for (int f = 0; f < NR; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) sel[b][f][r] = id[b] == cur ? acc[b][f][r] : sel[b][f][r];
  }
  __syncthreads();
  f32x4_t (*red)[NR * XR][64] = reinterpret_cast<f32x4_t (*)[NR * XR][64]>(lds);
  if (wave) {
#pragma unroll
    for (int b = 0; b < XR; ++b)
#pragma unroll
      for (int f = 0; f < NR; ++f) red[wave - 1][b * NR + f][lane] = sel[b][f];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int b = 0; b < XR; ++b) {
    if (mw + 16 * b + fr >= M) continue;
    const float s = id[b] >= 0 ? scale[id[b]] : 0.f;
#pragma unroll
    for (int f = 0; f < NR; ++f) {
      const int i = b * NR + f;
      const f32x4_t t = (sel[b][f] + red[0][i][lane]) + (red[1][i][lane] + red[2][i][lane]);
      // (no adapter: zeros, whatever the sums hold)
      const float4 o = id[b] >= 0 ? make_float4(s * t[0], s * t[1], s * t[2], s * t[3]) : make_float4(0.f, 0.f, 0.f, 0.f);
      pool_store_down(out, mrow[b], 16 * NR, 16 * f + 4 * fq, o);
    }
  }
}

// One row per workgroup, the four waves take every fourth k-step.
template <int NR>
__global__ __launch_bounds__(256) void pool_down_row_kernel(const bf16_t* __restrict__ X, int64_t ldx, const bf16_t* __restrict__ F, const float* __restrict__ scale,
                                                            const int* __restrict__ ids, int n, const PoolDown out, int K) {
  __shared__ float red[4][16 * NR];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const int64_t m = blockIdx.x;
  const int id = ids[m];
  f32x4_t s[NR];
#pragma unroll
  for (int f = 0; f < NR; ++f) s[f] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  const bool on = (unsigned)id < (unsigned)n;
  if (on) {
    const bf16_t* fp = F + id * pool_image(K, 16 * NR) + 8 * lane;
    const bf16_t* x = X + m * ldx + 8 * fq;
    for (int k0 = wave; 32 * k0 < K; k0 += 16) {             // four k-steps in flight
      Frag xv[4], a[4][NR];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int ks = k0 + 4 * j;
        const bool in = 32 * ks + 8 * fq < K;
        xv[j].q = in ? *reinterpret_cast<const u32x4_t*>(x + 32 * ks) : (u32x4_t){0u, 0u, 0u, 0u};
#pragma unroll
        for (int f = 0; f < NR; ++f) a[j][f].q = in ? *reinterpret_cast<const u32x4_t*>(fp + ((int64_t)ks * NR + f) * 512) : (u32x4_t){0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int f = 0; f < NR; ++f) s[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j][f].v, xv[j].v, s[f], 0, 0, 0);
    }
  }
  if (fr == 0) {
#pragma unroll
    for (int f = 0; f < NR; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[wave][16 * f + 4 * fq + r] = s[f][r];
  }
  __syncthreads();
  const int t = threadIdx.x;
  if (t >= 4 * NR) return;
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = on ? scale[id] * ((red[0][4 * t + r] + red[1][4 * t + r]) + (red[2][4 * t + r] + red[3][4 * t + r])) : 0.f;
  pool_store_down(out, m, 16 * NR, 4 * t, make_float4(v[0], v[1], v[2], v[3]));
}

// ------------------------------------------------------------------------------------------------ out = X W^T + bias + Up_i down
struct PoolGemm {
  const bf16_t* X; int64_t ldx; const bf16_t* W; int64_t ldw; const float* bias;
  const float* D; const bf16_t* U; int P;                   // the down products: fp32 (few rows), in P parts
  const bf16_t* Up; const int* ids; int n, RP;
  void* out; int64_t ldo; int out_f32;
  int64_t M; int N, K, tiles_m, tiles_n;
};

// Column order inside a wave's 16 G columns: a pair of fragments covers 32 columns, operand row fr of its fragment i <-> column
// 8 (fr >> 2) + 4 i + (fr & 3), a last single fragment (G = 3) its 16 columns in order. A lane ends with 8 consecutive columns per pair,
// so that one 16-byte store instruction of a wave fills 64 consecutive bytes of each of its 16 rows (16 consecutive columns per lane, in
// two instructions of every second 16 bytes, took 6.7 us per 256 x 256 tile instead of 3). Chunk XOR of column o's LDS row: the 16
// rows of a fragment fall on 16 different 16-byte slots; it depends on fr alone.
template <int G> __device__ __forceinline__ constexpr bool pool_single(int i) { return (G & 1) && i == G - 1; }
template <int G> __device__ __forceinline__ int pool_col(int fr, int i) {
  return pool_single<G>(i) ? 16 * i + fr : 32 * (i >> 1) + 8 * (fr >> 2) + 4 * (i & 1) + (fr & 3);
}
template <int G> __device__ __forceinline__ int pool_swz_w(int o) {
  return (((G & 1) && o >= 16 * (G - 1) ? o >> 2 : o >> 3) & 3) << 1 | ((o >> 1) & 1);
}
// first of the four columns a lane holds of fragment i
template <int G> __device__ __forceinline__ int pool_out_col(int fq, int i) { return pool_single<G>(i) ? 16 * i + 4 * fq : 32 * (i >> 1) + 8 * fq + 4 * (i & 1); }

// Low-rank update, bias and store of a wave's tile: the lane owns rows m0 + r0 + 16 b and four columns per fragment (pool_out_col; rows past
// the end repeat the last one and are not stored). The update is MFMA k-steps of 32 slots: RP = 16: ranks 0..15 of the down product's part
// hi, then of its part lo; wider: 32 ranks of one part. A bf16 result needs 16 bits of the fp32 factor (hi + lo), an fp32 one a third part.
// `pre`: indices and the first step's parts, requested before the main loop (PRE).
template <int XF> struct PoolPre { int id[XF]; Frag u[XF]; };
__device__ __forceinline__ int pool_part(const PoolGemm& p, int s, int fq) { return p.RP > 16 ? s % p.P : 2 * s + (fq >> 1); }      // of step s; >= P: none
__device__ __forceinline__ int pool_rank(const PoolGemm& p, int s, int fq) { return p.RP > 16 ? 32 * (s / p.P) + 8 * fq : 8 * (fq & 1); }
__device__ __forceinline__ u32x4_t pool_parts(const PoolGemm& p, int64_t m, int s, int fq) {
  const int q = pool_part(p, s, fq);
  return q < p.P ? *reinterpret_cast<const u32x4_t*>(p.U + (m * p.P + q) * p.RP + pool_rank(p, s, fq)) : (u32x4_t){0u, 0u, 0u, 0u};
}
template <int XF>
__device__ __forceinline__ void pool_prefetch(const PoolGemm& p, PoolPre<XF>& pre, int64_t m0, int r0, int fq) {
  const int mlim = p.M - m0 - 1 < r0 + 16 * XF ? (int)(p.M - m0) - 1 : r0 + 16 * XF;
#pragma unroll
  for (int b = 0; b < XF; ++b) {
    const int r = r0 + 16 * b < mlim ? r0 + 16 * b : mlim;
    pre.id[b] = p.ids[m0 + r];
    pre.u[b].q = pool_parts(p, m0 + r, 0, fq);
  }
}
template <int XF, int G, bool PRE>
__device__ __forceinline__ void pool_epilogue(const PoolGemm& p, f32x4_t (&acc)[G][XF], int64_t m0, int r0, int ncol, int fr, int fq, unsigned char* bounce, const PoolPre<XF>& pre) {
  const int mlim = p.M - m0 - 1 < r0 + 16 * XF ? (int)(p.M - m0) - 1 : r0 + 16 * XF;       // last row of the matrix, from m0
  {
    const int* ids = p.ids + m0;
    const int RP = p.RP;
    int id[XF];
#pragma unroll
    for (int b = 0; b < XF; ++b) {
      const int r = r0 + 16 * b;
      id[b] = PRE ? pre.id[b] : ids[r < mlim ? r : mlim];
      if ((unsigned)id[b] >= (unsigned)p.n) id[b] = -1;
    }
    const int steps = RP > 16 ? p.P * (RP / 32) : p.P - 1;
    for (int s = 0; s < steps; ++s) {
      const int rk = pool_rank(p, s, fq);
      Frag u[XF];
#pragma unroll
      for (int b = 0; b < XF; ++b) {
        const int r = r0 + 16 * b;
        if (PRE && s == 0) u[b] = pre.u[b];
        else u[b].q = pool_parts(p, m0 + (r < mlim ? r : mlim), s, fq);
      }
      auto above = [&](int last) __attribute__((always_inline)) {
        int cand = NO_ID;
#pragma unroll
        for (int b = 0; b < XF; ++b) cand = id[b] > last && id[b] < cand ? id[b] : cand;
        return next_id(cand);
      };
      auto factors = [&](int i, Frag (&f)[G]) __attribute__((always_inline)) {
        const bf16_t* up = p.Up + (int64_t)i * p.N * RP;
#pragma unroll
        for (int a = 0; a < G; ++a) {
          const int c = ncol + pool_col<G>(fr, a);
          f[a].q = *reinterpret_cast<const u32x4_t*>(up + ((int64_t)(c < p.N ? c : p.N - 1) * RP + rk));
        }
      };
      Frag f[G];
      int cur = above(-1);
      if (cur != NO_ID) factors(cur, f);
      while (cur != NO_ID) {                                               // the next adapter's factors are on their way meanwhile
        const int nxt = above(cur);
        Frag g[G];
        if (nxt != NO_ID) factors(nxt, g);
#pragma unroll
        for (int b = 0; b < XF; ++b) {
          if (!__any(id[b] == cur)) continue;                              // (none of these 16 rows)
#pragma unroll
          for (int a = 0; a < G; ++a) {
            const f32x4_t t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[a].v, u[b].v, acc[a][b], 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[a][b][r] = id[b] == cur ? t[r] : acc[a][b][r];
          }
        }
#pragma unroll
        for (int a = 0; a < G; ++a) f[a] = g[a];
        cur = nxt;
      }
    }
  }
  float4 bv[G];
  int cb[G];
#pragma unroll
  for (int a = 0; a < G; ++a) {
    cb[a] = ncol + pool_out_col<G>(fq, a);
    bv[a] = p.bias && cb[a] < p.N ? *reinterpret_cast<const float4*>(p.bias + cb[a]) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (G == 4 && bounce && !p.out_f32) {                      // through 8 KB of LDS of this wave's own: stores of whole 128-byte lines
    const int lane = threadIdx.x & 63, rr = lane >> 3, ch = lane & 7;
#pragma unroll
    for (int b = 0; b < XF; ++b) {
      u32x2_t w[G];
#pragma unroll
      for (int a = 0; a < G; ++a) {
        w[a].x = pack_bf16x2(acc[a][b][0] + bv[a].x, acc[a][b][1] + bv[a].y);
        w[a].y = pack_bf16x2(acc[a][b][2] + bv[a].z, acc[a][b][3] + bv[a].w);
      }
      unsigned char* l = bounce + (b & 3) * 2048;
      *reinterpret_cast<u32x4_t*>(l + fr * 128 + ((fq ^ (fr & 7)) << 4)) = (u32x4_t){w[0].x, w[0].y, w[1].x, w[1].y};
      *reinterpret_cast<u32x4_t*>(l + fr * 128 + (((4 + fq) ^ (fr & 7)) << 4)) = (u32x4_t){w[2].x, w[2].y, w[3].x, w[3].y};
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int row = 8 * q + rr, m = r0 - fr + 16 * b + row;
        const u32x4_t v = *reinterpret_cast<const u32x4_t*>(l + row * 128 + ((ch ^ (row & 7)) << 4));
        if (m <= mlim && ncol + 8 * ch < p.N) *reinterpret_cast<u32x4_t*>((bf16_t*)p.out + (m0 + m) * p.ldo + ncol + 8 * ch) = v;
      }
    }
    return;
  }
#pragma unroll
  for (int b = 0; b < XF; ++b) {
    if (r0 + 16 * b > mlim) continue;
    if (p.out_f32) {
      float* o = (float*)p.out + (m0 + r0 + 16 * b) * p.ldo;
#pragma unroll
      for (int a = 0; a < G; ++a)
        if (cb[a] < p.N) *reinterpret_cast<float4*>(o + cb[a]) = make_float4(acc[a][b][0] + bv[a].x, acc[a][b][1] + bv[a].y, acc[a][b][2] + bv[a].z, acc[a][b][3] + bv[a].w);
    } else {
      bf16_t* o = (bf16_t*)p.out + (m0 + r0 + 16 * b) * p.ldo;
      u32x2_t w[G];
#pragma unroll
      for (int a = 0; a < G; ++a) {
        w[a].x = pack_bf16x2(acc[a][b][0] + bv[a].x, acc[a][b][1] + bv[a].y);
        w[a].y = pack_bf16x2(acc[a][b][2] + bv[a].z, acc[a][b][3] + bv[a].w);
      }
#pragma unroll
      for (int a = 0; a < G; ++a) {
        if (cb[a] >= p.N) continue;                          // (N is a multiple of 8: a pair is in or out as a whole)
        if (pool_single<G>(a)) *reinterpret_cast<u32x2_t*>(o + cb[a]) = w[a];
        else if (!(a & 1)) *reinterpret_cast<u32x4_t*>(o + cb[a]) = (u32x4_t){w[a].x, w[a].y, w[a + 1 < G ? a + 1 : a].x, w[a + 1 < G ? a + 1 : a].y};
      }
    }
  }
}

// Few rows: 16 XF of them and 16 columns per workgroup, the four waves take every fourth 64-wide piece of K and add up through LDS: the
// weight is streamed once and every request of a wave is independent. Bound by latency. The low-rank update needs no matrix
// instruction here: a lane owns one row and four columns, whose RP factors lie in one piece; they are requested before the products.
template <int XF>
__global__ __launch_bounds__(256) void pool_gemm_rows_kernel(const PoolGemm p) {
  __shared__ f32x4_t red[4][XF][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int m0 = blockIdx.y * 16 * XF, n0 = blockIdx.x * 16, K = p.K, M = (int)p.M;
  const int mf = m0 + 16 * wave + fr, cb = n0 + 4 * fq;           // the row and columns this lane finishes (waves below XF)
  const bool fin = wave < XF && mf < M && cb < p.N;
  float add[4] = {0.f, 0.f, 0.f, 0.f};
  if (fin && p.bias) {
    const float4 b = *reinterpret_cast<const float4*>(p.bias + cb);
    add[0] = b.x; add[1] = b.y; add[2] = b.z; add[3] = b.w;
  }
  if (fin) {
    const int id = p.ids[mf];
    if ((unsigned)id < (unsigned)p.n) {
      const int RP = p.RP;
      const bf16_t* up = p.Up + ((int64_t)id * p.N + cb) * RP;
      const float* d = p.D + (int64_t)mf * RP;
      float lr[4] = {0.f, 0.f, 0.f, 0.f};
      for (int j = 0; j < RP; j += 8) {
        const float4 d0 = *reinterpret_cast<const float4*>(d + j), d1 = *reinterpret_cast<const float4*>(d + j + 4);
        const float x[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const u32x4_t u = *reinterpret_cast<const u32x4_t*>(up + (int64_t)c * RP + j);
#pragma unroll
          for (int q = 0; q < 4; ++q) lr[c] = fmaf(x[2 * q], bf16_lo(u[q]), fmaf(x[2 * q + 1], bf16_hi(u[q]), lr[c]));
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) add[c] += lr[c];
    }
  }
  const bf16_t* w = p.W + (int64_t)(n0 + fr < p.N ? n0 + fr : p.N - 1) * p.ldw + 8 * fq;
  const bf16_t* x[XF];
#pragma unroll
  for (int b = 0; b < XF; ++b) x[b] = p.X + (int64_t)(m0 + 16 * b + fr < M ? m0 + 16 * b + fr : M - 1) * p.ldx + 8 * fq;
  f32x4_t acc[XF];
#pragma unroll
  for (int b = 0; b < XF; ++b) acc[b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  const u32x4_t zero = (u32x4_t){0u, 0u, 0u, 0u};
  for (int k0 = 64 * wave; k0 < K; k0 += 256 * 2) {          // two pieces of 64 in flight
    Frag wf[4], xf[4][XF];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + 256 * (j >> 1) + 32 * (j & 1);
      const bool on = k + 8 * fq < K;                        // chunks behind column K: zeros on both sides
      wf[j].q = on ? *reinterpret_cast<const u32x4_t*>(w + k) : zero;
#pragma unroll
      for (int b = 0; b < XF; ++b) xf[j][b].q = on ? *reinterpret_cast<const u32x4_t*>(x[b] + k) : zero;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int b = 0; b < XF; ++b) acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[j].v, xf[j][b].v, acc[b], 0, 0, 0);
  }
#pragma unroll
  for (int b = 0; b < XF; ++b) red[wave][b][lane] = acc[b];
  __syncthreads();
  if (!fin) return;
  const f32x4_t t = (red[0][wave][lane] + red[1][wave][lane]) + (red[2][wave][lane] + red[3][wave][lane]);
  const int64_t at = (int64_t)mf * p.ldo + cb;
  if (p.out_f32) *reinterpret_cast<float4*>((float*)p.out + at) = make_float4(t[0] + add[0], t[1] + add[1], t[2] + add[2], t[3] + add[3]);
  else {
    u32x2_t o;
    o.x = pack_bf16x2(t[0] + add[0], t[1] + add[1]);
    o.y = pack_bf16x2(t[2] + add[2], t[3] + add[3]);
    *reinterpret_cast<u32x2_t*>((bf16_t*)p.out + at) = o;
  }
}

// At most 16 rows, short ones: both products in one launch. 16 waves per workgroup and 32 columns: wave w computes down of row w (every workgroup
// again: M 16 NR K products beside the 32 M K of its own, the factors come from L2) while the weight is on its way, then the waves
// split K for the 32 columns, add up through LDS and add the update.
template <int NR>
__global__ __launch_bounds__(1024) void pool_rows_fused_kernel(const PoolGemm p, const bf16_t* __restrict__ F, const float* __restrict__ scale, float* __restrict__ down) {
  constexpr int RP = 16 * NR;
  __shared__ f32x4_t red[16][2][64];
  __shared__ float dn[16][RP + 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int n0 = blockIdx.x * 32, K = p.K, M = (int)p.M;
  const u32x4_t zero = (u32x4_t){0u, 0u, 0u, 0u};
  // this wave's 64-wide pieces of K: the first one is requested before the down product
  const bf16_t* x = p.X + (int64_t)(fr < M ? fr : M - 1) * p.ldx + 8 * fq;
  const bf16_t* w[2];
#pragma unroll
  for (int a = 0; a < 2; ++a) w[a] = p.W + (int64_t)(n0 + 16 * a + fr < p.N ? n0 + 16 * a + fr : p.N - 1) * p.ldw + 8 * fq;
  const int my = wave < M ? p.ids[wave] : -1;                // the adapter of the row whose down product this wave makes
  const int cb = n0 + 16 * wave + 4 * fq;                    // waves 0 and 1 finish 16 columns each: row fr, columns cb .. cb + 3
  const bool fin = wave < 2 && fr < M && cb < p.N;
  const int fid = fin ? p.ids[fr] : -1;
  const bool flr = (unsigned)fid < (unsigned)p.n;
  Frag wf[2][2], xf[2];
  auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int k = k0 + 32 * j;
      const bool on = k + 8 * fq < K;                        // chunks behind column K: zeros on both sides
      xf[j].q = on ? *reinterpret_cast<const u32x4_t*>(x + k) : zero;
#pragma unroll
      for (int a = 0; a < 2; ++a) wf[j][a].q = on ? *reinterpret_cast<const u32x4_t*>(w[a] + k) : zero;
    }
  };
  if (64 * wave < K) load(64 * wave);
  if (wave < M) {
    const int id = my;
    const bool on = (unsigned)id < (unsigned)p.n;
    f32x4_t s[NR];
#pragma unroll
    for (int f = 0; f < NR; ++f) s[f] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    float sc = 0.f;
    if (on) {
      sc = scale[id];
      pool_row_sums<NR>(p.X + (int64_t)wave * p.ldx, F + id * pool_image(K, RP), K, lane, s);
    }
    if (fr == 0) {
#pragma unroll
      for (int f = 0; f < NR; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 16 * f + 4 * fq + r;
          const float v = on ? sc * s[f][r] : 0.f;
          dn[wave][j] = v;
          if (blockIdx.x == 0) down[wave * RP + j] = v;
        }
    }
  }
  // what the finishing waves need beside the sums (RP = 16: in registers before the barrier)
  const bf16_t* up = p.Up + ((int64_t)(flr ? fid : 0) * p.N + (fin ? cb : 0)) * RP;
  u32x4_t uv[NR == 1 ? 8 : 1];
  if (NR == 1 && flr) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int j = 0; j < 2; ++j) uv[2 * c + j] = *reinterpret_cast<const u32x4_t*>(up + c * RP + 8 * j);
  }
  float4 bias = make_float4(0.f, 0.f, 0.f, 0.f);
  if (fin && p.bias) bias = *reinterpret_cast<const float4*>(p.bias + cb);
  f32x4_t acc[2];
#pragma unroll
  for (int a = 0; a < 2; ++a) acc[a] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  for (int k0 = 64 * wave; k0 < K; k0 += 1024) {
    if (k0 != 64 * wave) load(k0);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int a = 0; a < 2; ++a) acc[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[j][a].v, xf[j].v, acc[a], 0, 0, 0);
  }
#pragma unroll
  for (int a = 0; a < 2; ++a) red[wave][a][lane] = acc[a];
  __syncthreads();
  if (!fin) return;
  f32x4_t t = red[0][wave][lane];
#pragma unroll
  for (int q = 1; q < 16; ++q) t += red[q][wave][lane];
  t[0] += bias.x; t[1] += bias.y; t[2] += bias.z; t[3] += bias.w;
  if (flr) {
    f32x4_t lr = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int j = 0; j < RP; j += 8)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const u32x4_t u = NR == 1 ? uv[(2 * c + j / 8) % (NR == 1 ? 8 : 1)] : *reinterpret_cast<const u32x4_t*>(up + (int64_t)c * RP + j);
#pragma unroll
        for (int q = 0; q < 4; ++q) lr[c] = fmaf(dn[fr][j + 2 * q], bf16_lo(u[q]), fmaf(dn[fr][j + 2 * q + 1], bf16_hi(u[q]), lr[c]));
      }
    t += lr;
  }
  const int64_t at = (int64_t)fr * p.ldo + cb;
  if (p.out_f32) *reinterpret_cast<float4*>((float*)p.out + at) = make_float4(t[0], t[1], t[2], t[3]);
  else {
    u32x2_t o;
    o.x = pack_bf16x2(t[0], t[1]);
    o.y = pack_bf16x2(t[2], t[3]);
    *reinterpret_cast<u32x2_t*>((bf16_t*)p.out + at) = o;
  }
}

// Workgroup -> tile. Workgroup ids go round-robin over the 8 XCDs: each XCD takes a contiguous run of tiles, and a run walks down 4
// tile rows before it moves to the next column, so that the 32 tiles an XCD holds at a time share 4 + 8 panels in its L2 (32 tiles of
// one tile row: 1 + 32).
__device__ __forceinline__ void pool_tile(const PoolGemm& p, int* tm, int* tn) {
  const int nwg = p.tiles_m * p.tiles_n, orig = blockIdx.x, xcd = orig & 7, q = nwg >> 3, r = nwg & 7;
  const int wg = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (orig >> 3);
  const int per = 4 * p.tiles_n, g = wg / per, rem = wg - g * per;
  const int rows = p.tiles_m - 4 * g < 4 ? p.tiles_m - 4 * g : 4;
  *tm = 4 * g + rem % rows;
  *tn = rem / rows;
}

// Few tiles: 64 x 64 columns per workgroup, waves of 32 x 32, k-tiles of 64 in a ring of three LDS buffers filled by global_load_lds two
// tiles ahead; KS groups of four waves take every KS-th k-tile, each with a ring of its own, and add up through LDS at the end (a chip
// that is not full is bound by the length of this loop: 0.36 us per k-tile). One barrier per k-tile: behind it every wave's requests of
// tile t have landed and every wave is done with tile t - 1, whose buffer takes tile t + 2. The W rows are the MFMA's "A" operand.
template <int KS>
__global__ __launch_bounds__(256 * KS) void pool_gemm_kernel(const PoolGemm p) {
  constexpr int WN = 2, XF = 2, G = 2, RING = 3, BM = 64, BN = 64, ROWS = BM + BN, STAGE = ROWS * 128, PPW = ROWS / 8 / 4;
  __shared__ __attribute__((aligned(1024))) unsigned char lds_all[KS * RING * STAGE];
  const int lane = threadIdx.x & 63;
  const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave_all >> 2, wave = wave_all & 3;
  unsigned char* lds = lds_all + kg * RING * STAGE;
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane & 15, fq = lane >> 4;
  int tm, tn;
  pool_tile(p, &tm, &tn);
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN;
  PoolPre<XF> pre;
  if (kg == 0) pool_prefetch<XF>(p, pre, m0, wm * 16 * XF + fr, fq);

  // staging: piece j holds stage rows 8j .. 8j+7; lane -> row 8j + (lane >> 3), destination chunk lane & 7
  const bf16_t* src[PPW];
  int kch[PPW];
#pragma unroll
  for (int i = 0; i < PPW; ++i) {
    const int row = 8 * (wave + 4 * i) + (lane >> 3);
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
  const int nt_all = (p.K + 63) / 64, rounds = (nt_all + KS - 1) / KS, nt = (nt_all - kg + KS - 1) / KS;      // k-tiles of this group: kg + KS t
  auto stage = [&](int t) {
    unsigned char* base = lds + (t % RING) * STAGE;
    const int kt = kg + KS * t;
#pragma unroll
    for (int i = 0; i < PPW; ++i) {
      const bf16_t* s = src[i] + kt * 64;
      if (kt * 64 + 64 > p.K) s = kt * 64 + kch[i] < p.K ? s : reinterpret_cast<const bf16_t*>(g_pool_zero);     // (uniform branch: the last k-tile of a ragged K)
      __builtin_amdgcn_global_load_lds((gbl_ptr_t)s, (lds_ptr_t)(base + (wave + 4 * i) * 1024), 16, 0, 0);
    }
  };

  const int x_row = (wm * 16 * XF + fr) * 128, x_sw = fr & 7;
  const int w_row = (BM + wn * 16 * G + pool_col<G>(fr, 0)) * 128, w_sw = pool_swz_w<G>(pool_col<G>(fr, 0));      // (fragment 1: 4 rows further, the same swizzle)
  f32x4_t acc[G][XF];
#pragma unroll
  for (int a = 0; a < G; ++a)
#pragma unroll
    for (int b = 0; b < XF; ++b) acc[a][b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

  for (int t = 0; t < RING - 1 && t < nt; ++t) stage(t);
  for (int t = 0; t < rounds; ++t) {
    if (t + 1 < nt) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PPW) : "memory");      // tile t landed, tile t + 1 may be in flight
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                // this wave's reads of tile t - 1
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (t >= nt) continue;                                            // (the other groups' last round)
    if (t + RING - 1 < nt) stage(t + RING - 1);
    const unsigned char* base = lds + (t % RING) * STAGE;
    bf16x8_t xf[2][XF], wf[2][G];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int ch = fq + 4 * ks;
#pragma unroll
      for (int i = 0; i < XF; ++i) xf[ks][i] = *reinterpret_cast<const bf16x8_t*>(base + x_row + i * 2048 + ((ch ^ x_sw) << 4));
#pragma unroll
      for (int i = 0; i < G; ++i) wf[ks][i] = *reinterpret_cast<const bf16x8_t*>(base + w_row + i * 512 + ((ch ^ w_sw) << 4));
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int a = 0; a < G; ++a)
#pragma unroll
        for (int b = 0; b < XF; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[ks][a], xf[ks][b], acc[a][b], 0, 0, 0);
  }
  if (KS > 1) {
    __syncthreads();
    f32x4_t* red = reinterpret_cast<f32x4_t*>(lds_all);
    if (kg) {
#pragma unroll
      for (int a = 0; a < G; ++a)
#pragma unroll
        for (int b = 0; b < XF; ++b) red[(((kg - 1) * 4 + wave) * (G * XF) + a * XF + b) * 64 + lane] = acc[a][b];
    }
    __syncthreads();
    if (kg) return;
#pragma unroll
    for (int g = 0; g < KS - 1; ++g)
#pragma unroll
      for (int a = 0; a < G; ++a)
#pragma unroll
        for (int b = 0; b < XF; ++b) acc[a][b] += red[((g * 4 + wave) * (G * XF) + a * XF + b) * 64 + lane];
  }
  pool_epilogue<XF, G, true>(p, acc, m0, wm * 16 * XF + fr, n0 + wn * 16 * G, fr, fq, nullptr, pre);
}

// The same product for many rows: 8 waves as 2 (rows) x 4 (columns), wave tile 16 XF x 16 G, two k-tiles of 64 in LDS. A k-tile is
// four phases, one quadrant of the wave's tile each (half the row fragments x half the column fragments x both k-steps):
//
//   phase 0  reads the rest of x-lo                        multiplies x-lo w-lo      requests x-hi of tile t + 1
//   phase 1  reads w-hi, a fragment of x-hi                multiplies x-lo w-hi      requests x-lo of tile t + 2
//   phase 2  reads the rest of x-hi                        multiplies x-hi w-hi      requests half of W of tile t + 2
//   phase 3  reads w-lo, a fragment of x-lo of tile t + 1  multiplies x-hi w-lo      requests the rest of W of tile t + 2
//
// Each phase is a read slot and a multiply slot with a barrier behind each; the waves of the second row half run one slot late, so
// that on every SIMD one of its two waves multiplies while the other reads. For that the slots have to be alike: 6 reads in each, where
// x-lo and w-lo in phase 0 would be 12 of the 24 (with zeros as operands, which leave the clock alone, 3 to 7 % less time; with random
// ones, where large products are held by the chip's power, 0 to 3 %: [32768, 3840] x [3840, 1280] 270 -> 265 us). The smaller tiles, two
// workgroups per CU, read everything where it is multiplied first: two workgroups fill each other's gaps, and the early reads cost them
// up to 6 %. A request overwrites only what both halves have read (waited for by lgkmcnt(0) inside the read slot, published by its
// barrier) at least one slot earlier. vmcnt counts in order: each wait leaves the requests younger than the wanted ones. Addresses: a fragment's LDS address is one of four lane addresses plus a constant, a
// request's global one a constant 32-bit offset beside a scalar that advances by 128 bytes a tile, so that the loop has next to no vector
// instructions beside the MFMAs.
template <int XF, int G>
__global__ __launch_bounds__(512, XF * G <= 12 ? 4 : 2) void pool_gemm_phased_kernel(const PoolGemm p) {
  constexpr int BM = 32 * XF, BN = 64 * G, STAGE = (BM + BN) * 128;
  constexpr int XH = XF / 2, GL = (G + 1) / 2;               // fragments of a row half; column fragments of the first half
  constexpr int XP = XF / 4, WP = G, W0 = (G + 1) / 2;       // requests per wave: a row half, all of W, its first part
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int fr = lane & 15, fq = lane >> 4;
  int tm, tn;
  pool_tile(p, &tm, &tn);
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN;

  // Requests: 1-KB pieces of 8 rows; byte offsets from the tile's first row fit 31 bits (row strides up to 2^22 elements). A row half
  // (lo / hi) holds rows wm * 16 XF + half * 8 XF ... of both wave rows: 2 XF pieces, XP per wave. W: 8 G pieces, G per wave.
  const int mlim = p.M - m0 < BM ? (int)(p.M - m0) - 1 : BM - 1, nlim = p.N - n0 < BN ? p.N - n0 - 1 : BN - 1;
  const bf16_t* xbase = p.X + m0 * p.ldx;
  const bf16_t* wbase = p.W + (int64_t)n0 * p.ldw;
#if defined(__HIP_DEVICE_COMPILE__)                          // (buffer resources are a type of the device pass only)
  const __amdgpu_buffer_rsrc_t xres = __builtin_amdgcn_make_buffer_rsrc((void*)xbase, 0, (int)(mlim * (2 * p.ldx) + 2 * p.K), 0x00020000);
  const __amdgpu_buffer_rsrc_t wres = __builtin_amdgcn_make_buffer_rsrc((void*)wbase, 0, (int)(nlim * (2 * p.ldw) + 2 * p.K), 0x00020000);
  int xo[2][XP], wo[WP];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < XP; ++i) {
      const int j = wave + 8 * i, row = (j / XF) * 16 * XF + h * 8 * XF + (j % XF) * 8 + (lane >> 3);       // piece of the half: XF of them per wave row
      xo[h][i] = (row < mlim ? row : mlim) * (int)(2 * p.ldx) + (((lane & 7) ^ (row & 7)) << 4);
    }
#pragma unroll
  for (int i = 0; i < WP; ++i) {
    const int row = (wave + 8 * i) * 8 + (lane >> 3);
    wo[i] = (row < nlim ? row : nlim) * (int)(2 * p.ldw) + (((lane & 7) ^ pool_swz_w<G>(row % (16 * G))) << 4);
  }
  const int nt = p.K / 64, ragged = p.K & 63;                // whole k-tiles; columns behind them
  auto req_x = [&](int h, int kt) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < XP; ++i) {
      const int j = wave + 8 * i, row0 = (j / XF) * 16 * XF + h * 8 * XF + (j % XF) * 8;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xres, (lds_ptr_t)(lds + (kt & 1) * STAGE + row0 * 128), 16, xo[h][i], kt * 128, 0, 0);
    }
  };
  auto req_w = [&](int i0, int i1, int kt) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < WP; ++i)
      if (i >= i0 && i < i1)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wres, (lds_ptr_t)(lds + (kt & 1) * STAGE + (BM + (wave + 8 * i) * 8) * 128), 16, wo[i], kt * 128, 0, 0);
  };

  // fragment addresses: both swizzles depend on the lane alone, so a fragment is a constant offset from one address per k-step
  unsigned int xa[2], wa[2], wa1[2];                         // wa1: a last single fragment
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    const unsigned int l0 = (unsigned int)(uintptr_t)(lds_ptr_t)lds;
    xa[ks] = l0 + (wm * 16 * XF + fr) * 128 + (((fq + 4 * ks) ^ (fr & 7)) << 4);
    wa[ks] = l0 + (BM + wn * 16 * G + pool_col<G>(fr, 0)) * 128 + (((fq + 4 * ks) ^ pool_swz_w<G>(pool_col<G>(fr, 0))) << 4);
    wa1[ks] = l0 + (BM + wn * 16 * G + pool_col<G>(fr, G - 1)) * 128 + (((fq + 4 * ks) ^ pool_swz_w<G>(pool_col<G>(fr, G - 1))) << 4);
  }
  f32x4_t acc[G][XF];
#pragma unroll
  for (int a = 0; a < G; ++a)
#pragma unroll
    for (int b = 0; b < XF; ++b) acc[a][b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  bf16x8_t xf[XH][2], wf[G][2];
  bf16x8_t xe[2], we[GL][2];                                 // read a phase early: the last fragment of x-lo or x-hi, w-lo
  constexpr bool EARLY = XF * G >= 32;
  typedef const __attribute__((address_space(3))) bf16x8_t* frag_ptr_t;
  auto read_x = [&](int h, int i1) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < XH; ++i)
        if (i < i1) xf[i][ks] = *(frag_ptr_t)(uintptr_t)(xa[ks] + (h * XH + i) * 2048);
  };
  auto read_w = [&](int i0, int i1) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < G; ++i)
        if (i >= i0 && i < i1) wf[i][ks] = *(frag_ptr_t)(uintptr_t)(pool_single<G>(i) ? wa1[ks] : wa[ks] + (i >> 1) * 4096 + (i & 1) * 512);
  };
  auto early_x = [&](int h) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) xe[ks] = *(frag_ptr_t)(uintptr_t)(xa[ks] + (h * XH + XH - 1) * 2048);
  };
  auto early_w = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < GL; ++i) we[i][ks] = *(frag_ptr_t)(uintptr_t)(wa[ks] + (i >> 1) * 4096 + (i & 1) * 512);
  };
  auto rest_x = [&](int h) __attribute__((always_inline)) {
    read_x(h, XH - 1);
    xf[XH - 1][0] = xe[0];
    xf[XH - 1][1] = xe[1];
  };
  auto mul = [&](int h, int i0, int i1) __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int a = 0; a < G; ++a)
        if (a >= i0 && a < i1) {
#pragma unroll
          for (int b = 0; b < XH; ++b) acc[a][h * XH + b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[a][ks], xf[b][ks], acc[a][h * XH + b], 0, 0, 0);
        }
    __builtin_amdgcn_s_setprio(0);
  };
  // end of a read slot: this wave's fragments are in registers; end of either slot: barrier
  auto end_read = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto end_mul = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  if (nt > 0) {
    req_x(0, 0); req_w(0, WP, 0); req_x(1, 0);
  }
  if (nt > 1) {
    req_x(0, 1); req_w(0, WP, 1);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(XP + WP) : "memory");
  } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (wm) __builtin_amdgcn_s_barrier();                      // the second row half runs one slot late
  auto flip = [&](unsigned int (&at)[2], int t) __attribute__((always_inline)) {      // to the other buffer
    const unsigned int d = t & 1 ? (unsigned int)-STAGE : (unsigned int)STAGE;
    at[0] += d;
    at[1] += d;
  };
  // MORE: two further tiles exist. What the next phase reads has to have landed at a read slot's end: x-hi of this tile (before phase 1,
  // or 2), x-lo and W of the next one (before phase 3, or 0).
  auto tile = [&](auto more, int t) __attribute__((always_inline)) {
    constexpr bool MORE = decltype(more)::value;
    const bool next = MORE || t + 1 < nt;
    if (!EARLY) { early_w(); early_x(0); }
    rest_x(0);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < GL; ++i) wf[i][ks] = we[i][ks];
    if (next) req_x(1, t + 1);
    if (EARLY && next) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * XP + WP) : "memory");
    else if (EARLY) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    end_read();
    mul(0, 0, GL);
    end_mul();
    read_w(GL, G);
    if (EARLY) early_x(1);
    if (MORE) req_x(0, t + 2);
    if (!EARLY && MORE) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * XP + WP) : "memory");
    else if (!EARLY && next) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(XP) : "memory");
    else if (!EARLY) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    end_read();
    mul(0, GL, G);
    end_mul();
    if (!EARLY) early_x(1);
    rest_x(1);
    if (MORE) req_w(0, W0, t + 2);
    if (EARLY) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MORE ? 2 * XP + W0 : XP) : "memory");
    end_read();
    mul(1, GL, G);
    end_mul();
    flip(xa, t); flip(wa, t); flip(wa1, t);
    if (EARLY && next) { early_w(); early_x(0); }
    if (MORE) req_w(W0, WP, t + 2);
    if (!EARLY) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MORE ? 2 * XP + WP : XP) : "memory");
    end_read();
    mul(1, 0, GL);
    end_mul();
  };
  if (EARLY && nt > 0) { early_w(); early_x(0); }
  int t = 0;
  for (; t + 2 < nt; ++t) tile(std::true_type{}, t);
  for (; t < nt; ++t) tile(std::false_type{}, t);
  if (!wm) __builtin_amdgcn_s_barrier();
  if (ragged) {                                              // the columns behind the last whole k-tile; zeros behind column K on both sides
    __syncthreads();
    for (int i = 0; i < (BM + BN) / 64; ++i) {
      const int row0 = (wave + 8 * i) * 8, row = row0 + (lane >> 3), o = row - BM;
      const int c = ((lane & 7) ^ (row < BM ? row & 7 : pool_swz_w<G>(o % (16 * G)))) << 3;
      const bf16_t* s = row < BM ? xbase + (int64_t)(row < mlim ? row : mlim) * p.ldx : wbase + (int64_t)(o < nlim ? o : nlim) * p.ldw;
      s = c < ragged ? s + nt * 64 + c : reinterpret_cast<const bf16_t*>(g_pool_zero);
      __builtin_amdgcn_global_load_lds((gbl_ptr_t)s, (lds_ptr_t)(lds + row0 * 128), 16, 0, 0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (nt & 1) { flip(xa, 1); flip(wa, 1); flip(wa1, 1); }  // the chunks went to buffer 0
    read_w(0, G);
    read_x(0, XH);
    mul(0, 0, G);
    read_x(1, XH);
    mul(1, 0, G);
    __syncthreads();                                         // (the epilogue writes to the same LDS)
  }
  const PoolPre<XF> none = {};
  pool_epilogue<XF, G, false>(p, acc, m0, wm * 16 * XF + fr, n0 + wn * 16 * G, fr, fq, lds + wave * 8192, none);
#endif
}

// ------------------------------------------------------------------------------------------------ dA / dB: sums over an adapter's rows
// part[chunk] = sum over the chunk's rows of y_m u_m^T. 256 columns of y per workgroup, its W waves take every W-th step of 32 rows:
// a step is copied into wave-private [32][64] LDS slabs (row-major, swizzled) and read transposed (ds_read_b64_tr_b16) as one MFMA
// operand; the other is u (fp32), split into three bf16 parts. Rows behind the chunk are zeros on BOTH sides, rows of other adapters are
// never read. y is bf16 or an 8-bit checkpoint, whose values are exact in bf16. RANK_MAJOR: part [RP][C] (dA), else [C][RP] (dB).
struct PoolTn {
  const bf16_t* Y; int64_t ldy; const signed char* codes; const unsigned char* exps;
  const float* U; int RP; const int* perm; const int4* table; float* part; int C;
  float* out; int r;                                       // != NULL (no adapter has more than one chunk): the result itself, without the padded ranks
  const int* base;
};
#define TN_MAX_CH 512
template <int NR, bool CKPT, bool RANK_MAJOR, int W>
__device__ __forceinline__ void pool_tn_body(unsigned char (*lds)[4][32 * 128], int* rows, const PoolTn& p, const int4 ck, int strip) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const int cw = strip * 256, C = p.C, len = ck.z - ck.y;
  const int j0 = 16 * NR * blockIdx.z;                               // first rank of this workgroup
  for (int i = threadIdx.x; i < len; i += 64 * W) rows[i] = p.perm[ck.y + i];
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
  for (; i0 < len; i0 += 32 * W) {
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
    if (i0 + 32 * W < len) issue(i0 + 32 * W);
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
  // sum of the waves, in order (16 KB per wave and fragment column); wave w writes slab w % 4, of eight waves each half of its tiles
  float* out = p.out ? p.out + (int64_t)blockIdx.y * p.r * C : p.part + (int64_t)blockIdx.y * p.RP * C;
  const int ld = p.out ? p.r : p.RP, jmax = p.out ? p.r : p.RP;
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
    for (int ti = 0; ti < 16 / W; ++ti)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = ti + 16 / W * (wave >> 2), idx = (((wave & 3) * 4 + t) * 4 + r) * 64 + lane;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += reinterpret_cast<const float*>(lds[w][0])[idx];
        const int a = 4 * fq + r;
        const int c = cw + 64 * (wave & 3) + 16 * t + (RANK_MAJOR ? fr : a), j = j0 + 16 * f + (RANK_MAJOR ? a : fr);
        if (c < C && j < jmax) out[RANK_MAJOR ? (int64_t)j * C + c : (int64_t)c * ld + j] = v;
      }
  }
}

// both sums of a layer in one launch: the first strips_a workgroups of a chunk row take dA, the others dB
template <int NR, bool CKPT, int W>
__global__ __launch_bounds__(64 * W, 2) void pool_tn_kernel(const PoolTn a, const PoolTn b, int strips_a) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[W][4][32 * 128];
  __shared__ int rows[TN_MAX_CH];
  int4 ck;
  if (a.out) {                                             // blockIdx.y is an adapter: its only chunk, or no rows (sums of nothing)
    const int k = a.base[blockIdx.y];
    ck = k < a.base[blockIdx.y + 1] ? a.table[k] : make_int4((int)blockIdx.y, 0, 0, 0);
  } else ck = a.table[blockIdx.y];
  if (ck.x < 0) return;
  if ((int)blockIdx.x < strips_a) pool_tn_body<NR, CKPT, true, W>(lds, rows, a, ck, blockIdx.x);
  else pool_tn_body<NR, false, false, W>(lds, rows, b, ck, blockIdx.x - strips_a);
}

// out[i] = sum over the chunks of adapter i, in order; part entries [d0][ld] -> out [d0][d1] (the padded ranks are dropped). No rows: zeros.
struct PoolSum { const float* part; float* out; int64_t per; int ld, d0, d1; };
__global__ __launch_bounds__(256) void pool_sum_kernel(const PoolSum a, const PoolSum b, const int* __restrict__ base) {
  const PoolSum p = blockIdx.z ? b : a;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= (int64_t)p.d0 * p.d1) return;
  const int i = blockIdx.y;
  const float* src = p.part + (e / p.d1) * p.ld + e % p.d1;
  float s = 0.f;
  const int k1 = base[i + 1];
#pragma unroll 8
  for (int k = base[i]; k < k1; ++k) s += src[k * p.per];
  p.out[(int64_t)i * p.d0 * p.d1 + e] = s;
}

// ------------------------------------------------------------------------------------------------ host
static bool pool_rp(int RP) { return RP == 16 || RP == 32 || RP == 64; }
// (a launch holds less than 2^32 threads: 2^27 rows keep every grid here below that)
static bool pool_counts(int64_t M, int64_t n) { return M >= 0 && M < (1ll << 27) && n >= 1 && n <= 65535; }
// a matrix whose rows are read in 16-byte pieces
static bool pool_rows(const void* t, int64_t ld, int64_t C) { return C >= 8 && C % 8 == 0 && C < (1 << 24) && ld >= C && ld % 8 == 0 && (uintptr_t)t % 16 == 0; }
#define POOL_CHECK_ROWS(name, T_, ld_, C_)                                                                                              \
  MF_CHECK_ARG(pool_rows(T_, ld_, C_), name ": rows must hold a multiple of 8 elements, 16-byte aligned, row stride a multiple of 8 (C=%lld ld=%lld)", \
               (long long)(C_), (long long)(ld_))

extern "C" int64_t mfnet_lora_pool_image_elements(int64_t C, int RP) { return C < 0 ? 0 : pool_image(C, RP); }

extern "C" int mfnet_lora_pool_pack(const void* A, const void* B, int dtype, const float* scale, int64_t n, int64_t K, int64_t N, int r, int RP,
                                    void* a_down, void* a_up, void* b_down, void* b_up, float* scale_out, hipStream_t stream) {
  MF_CHECK_ARG(A && B && a_down && a_up && b_down && b_up && scale_out, "lora_pool_pack: null pointer");
  MF_CHECK_ARG(dtype == MFNET_F32 || dtype == MFNET_BF16, "lora_pool_pack: bad dtype");
  MF_CHECK_ARG(n >= 1 && n <= 65535 && pool_rows(a_down, K, K) && pool_rows(b_down, N, N) && r >= 1 && r <= RP && pool_rp(RP),
               "lora_pool_pack: bad sizes (n=%lld K=%lld N=%lld r=%d RP=%d)", (long long)n, (long long)K, (long long)N, r, RP);
  MF_CHECK_ARG(((uintptr_t)A | (uintptr_t)B) % (dtype == MFNET_F32 ? 4 : 2) == 0 && ((uintptr_t)a_up | (uintptr_t)b_up) % 16 == 0, "lora_pool_pack: misaligned tensor");
  PoolPack p;
  p.src[0] = A; p.src[1] = B; p.down[0] = (bf16_t*)a_down; p.down[1] = (bf16_t*)b_down; p.up[0] = (bf16_t*)a_up; p.up[1] = (bf16_t*)b_up;
  p.C[0] = (int)K; p.C[1] = (int)N; p.r = r; p.RP = RP; p.scale = scale; p.scale_out = scale_out;
  const int64_t L = K > N ? K : N;
  const dim3 grid((unsigned)ceil_div64((ceil_div64(L, 64) * 64 + L) * RP / 8, 256), (unsigned)n, 2);
  if (dtype == MFNET_F32) hipLaunchKernelGGL(pool_pack_kernel<float>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(pool_pack_kernel<bf16_t>, grid, dim3(256), 0, stream, p);
  MF_LAUNCH_CHECK("lora_pool_pack");
  return MFNET_OK;
}

// Rows of a chunk of the backward sums. Up to 512 rows: every adapter's rows are one chunk, whose sums are the result (no second launch);
// above 128 rows eight waves share it. Against chunks of 128 rows and their sum: 509 rows of 2 adapters, 768 -> 768: 25.2 to 22.0 us a
// backward call; 512 of 8, 1280 -> 3840: 35.2 to 32.1, of 1: 34.7 to 35.6.
static bool pool_one_chunk(int64_t M) { return M <= TN_MAX_CH; }
// More rows: short chunks while they are few (they fill the chip), long ones where their partial sums would be bytes (both sums of K = 768,
// N = 2304, rank 8, us with chunks of 128, 256 and 512: 4000 rows 23.2, 22.8, 28.3, 8192 rows 31.8, 28.4, 30.2, 24000 rows 69.1, 64.7,
// 64.8; of K = N = 768: 15.1, 17.1, 23.1; 20.9, 20.1, 25.4; 43.7, 41.6, 37.6).
static int pool_chunk_rows(int64_t M) { return pool_one_chunk(M) || M > 12288 ? TN_MAX_CH : M > 5000 ? 256 : 128; }
extern "C" int64_t mfnet_lora_pool_chunks(int64_t M, int64_t n) {
  return M <= 0 || n <= 0 ? 0 : M / pool_chunk_rows(M) + (n < M ? n : M);
}

extern "C" int mfnet_lora_pool_plan(const int* ids, int64_t M, int64_t n, int* offs, int* perm, int* base, int* table, hipStream_t stream) {
  MF_CHECK_ARG(pool_counts(M, n), "lora_pool_plan: bad sizes (M=%lld n=%lld)", (long long)M, (long long)n);
  MF_CHECK_ARG(offs && base && (M == 0 || (ids && perm && table)), "lora_pool_plan: null pointer");
  MF_CHECK_ARG((uintptr_t)table % 16 == 0, "lora_pool_plan: table must be 16-byte aligned");
  hipLaunchKernelGGL(pool_plan_kernel, dim3((unsigned)n + 1), dim3(1024), 0, stream, ids, (int)M, (int)n, offs, perm);
  MF_LAUNCH_CHECK("lora_pool_plan");
  hipLaunchKernelGGL(pool_chunks_kernel, dim3((unsigned)n + 1), dim3(256), 0, stream, offs, (int)n, pool_chunk_rows(M), (int)mfnet_lora_pool_chunks(M, n), base, (int4*)table);
  MF_LAUNCH_CHECK("lora_pool_plan (chunks)");
  return MFNET_OK;
}

// Few rows, which the product takes 64 at a time with 16 columns per workgroup: up to 64, and more while the workgroups fill the chip at
// most once. us a call with the 64 x 64 tiles and so, 2 adapters in runs: [256, 768] -> 768 9.8, 9.6; [192, 1280] -> 1280 11.9, 12.2;
// [192, 3840] -> 1280 23.0, 24.9; 16 in random order (a tile multiplies with each in turn): 15.3, 10.0; 17.2, 12.5; 31.9, 27.5. Beyond:
// [384, 768] -> 768 10.0, 13.3 in runs, 15.0, 14.2 in random order.
static bool pool_few(int64_t M, int64_t N) { return M <= 64 || ceil_div64(M, 64) * ceil_div64(N, 16) <= 256; }

// perm / count: the rows that have an adapter, grouped by it (NULL: the rows as they come; every row of out is written)
static int pool_down(const void* X, int64_t ldx, const void* image, const float* scale, const int* ids, int64_t n, int RP, const int* perm, const int* count, const PoolDown& out, int64_t M,
                     int64_t K, hipStream_t stream) {
  // Up to 1024 rows: a workgroup per row, whatever the adapters' order; above, 16 rows that share their factor (a call on 16 adapters,
  // K = 1280, rank 16: 1024 rows in runs 13.7 us with a workgroup per row, 13.0 with 16 rows, in random order 14.1 and 25.0; 4096 rows
  // 22.7 and 15.4, 22.9 and 29.5). 32 rows per workgroup halve the factor's traffic where there are enough of them to fill the chip.
#define PDL(NR_, XR_) hipLaunchKernelGGL((pool_down_kernel<NR_, XR_>), dim3((unsigned)ceil_div64(M, 16 * XR_)), dim3(256), 0, stream, (const bf16_t*)X, ldx, (const bf16_t*)image, scale, ids, (int)n, perm, count, out, M, (int)K)
#define PD(NR_) do { \
    if (M <= 1024) hipLaunchKernelGGL((pool_down_row_kernel<NR_>), dim3((unsigned)M), dim3(256), 0, stream, (const bf16_t*)X, ldx, (const bf16_t*)image, scale, ids, (int)n, out, (int)K); \
    else if (M < 8192) PDL(NR_, 1); else PDL(NR_, 2); } while (0)
  if (RP == 16) PD(1); else if (RP == 32) PD(2); else PD(4);
#undef PD
#undef PDL
  MF_LAUNCH_CHECK("lora_pool (down)");
  return MFNET_OK;
}

static int pool_gemm(PoolGemm& p, hipStream_t stream) {
  const int64_t M = p.M, N = p.N;
  auto tiles = [&](int bm, int bn) { p.tiles_m = (int)ceil_div64(M, bm); p.tiles_n = (int)ceil_div64(N, bn); return (int64_t)p.tiles_m * p.tiles_n; };
#define PR(XF_) hipLaunchKernelGGL((pool_gemm_rows_kernel<XF_>), dim3((unsigned)ceil_div64(N, 16), (unsigned)ceil_div64(M, 16 * XF_)), dim3(256), 0, stream, p)
  if (M <= 32) PR(2);
  else if (pool_few(M, N)) PR(4);
#undef PR
  else {
    // The tile with the least modelled time, in us, as measured at K = 64 .. 8192 on 100 .. 32768 rows: a tile costs a fixed part and a
    // part per k-tile. 256 x 256: one workgroup per CU, so whole rounds of the 256 CUs count. 128 x 192 and 128 x 128: two per CU, which
    // hide each other's fixed part; an odd one runs alone. 64 x 64: three or four per CU; with no more tiles than CUs two groups of waves split K.
    const double it = (p.K + 63) / 64;
    auto rounds = [&](int bm, int bn) { return ceil((double)ceil_div64(M, bm) * (double)ceil_div64(N, bn) / 256); };
    auto paired = [&](double r, double fix, double per2, double per1) { return floor(r / 2) * (fix + 2 * per2 * it) + (r - 2 * floor(r / 2)) * (fix + per1 * it); };
    const double t64 = (double)ceil_div64(M, 64) * (double)ceil_div64(N, 64);
    const bool split = t64 <= 256 && it >= 4;
    const double cost[4] = {4.5 + (split ? 0.5 : 1.0) * it * (0.33 + 0.2 * t64 / 256), paired(rounds(128, 128), 5.3, 0.66, 0.72), paired(rounds(128, 192), 6.3, 0.70, 0.74),
                            rounds(256, 256) * (10 + 1.47 * it)};
    int best = 0;
    if (p.ldx <= (1 << 22) && p.ldw <= (1 << 22))                         // (the phased kernel's 32-bit offsets)
      for (int i = 1; i < 4; ++i) best = cost[i] < cost[best] ? i : best;
    const int64_t nwg = best == 0 ? tiles(64, 64) : best == 1 ? tiles(128, 128) : best == 2 ? tiles(128, 192) : tiles(256, 256);
    MF_CHECK_ARG(nwg < (1ll << 23), "lora_pool: too many tiles (%lld)", (long long)nwg);
    const dim3 grid((unsigned)nwg);
    if (best == 0 && split) hipLaunchKernelGGL((pool_gemm_kernel<2>), grid, dim3(512), 0, stream, p);
    else if (best == 0) hipLaunchKernelGGL((pool_gemm_kernel<1>), grid, dim3(256), 0, stream, p);
    else if (best == 1) hipLaunchKernelGGL((pool_gemm_phased_kernel<4, 2>), grid, dim3(512), 0, stream, p);
    else if (best == 2) hipLaunchKernelGGL((pool_gemm_phased_kernel<4, 3>), grid, dim3(512), 0, stream, p);
    else hipLaunchKernelGGL((pool_gemm_phased_kernel<8, 4>), grid, dim3(512), 0, stream, p);
  }
  MF_LAUNCH_CHECK("lora_pool (product)");
  return MFNET_OK;
}

// down = scale_i image_i x, out = x W^T (+ bias) + up_i down
// (down: M RP fp32 and behind them, unless there are few rows, the parts)
static int pool_products(PoolGemm& p, const void* image, const float* scale, const int* perm, const int* count, float* down, hipStream_t stream) {
  p.D = down;
  // One launch for both products saves the host 3 us, but every workgroup makes all down products again: it pays while they are few. us a
  // call, issued one by one (on the GPU alone): 16 rows, 768 -> 2304, rank 16: 11.4 (10.8) in one launch, 14.7 (7.1) in two; 8 rows,
  // 1280 -> 3840: 11.3 (10.8), 14.3 (8.1); 16 rows: 15.8 (16.1), 14.7 (8.6); 1 row, 1280 -> 5120, rank 32: 11.3 (10.6), 14.9 (10.0); 1 row,
  // 5120 -> 1280, rank 16: 21.0 (21.5), 15.8 (15.5). (64 ranks: more registers than 16 waves have.) The rule goes by calls issued one by one:
  // in a replayed graph two launches are the faster form wherever their time on the GPU is.
  const int64_t one_row = (int64_t)p.K * p.RP;
  if (p.M > 16 || p.RP > 32 || one_row > 40960 || p.M * one_row > (1 << 18)) {
    PoolDown d = {down, reinterpret_cast<bf16_t*>(down + p.M * p.RP), pool_few(p.M, p.N) ? 0 : p.out_f32 ? 3 : 2};
    p.U = d.parts;
    p.P = d.P;
    const int rc = pool_down(p.X, p.ldx, image, scale, p.ids, p.n, p.RP, perm, count, d, p.M, p.K, stream);
    return rc ? rc : pool_gemm(p, stream);
  }
  const dim3 grid((unsigned)ceil_div64(p.N, 32));
#define PF(NR_) hipLaunchKernelGGL((pool_rows_fused_kernel<NR_>), grid, dim3(1024), 0, stream, p, (const bf16_t*)image, scale, down)
  if (p.RP == 16) PF(1); else PF(2);
#undef PF
  MF_LAUNCH_CHECK("lora_pool (few rows)");
  return MFNET_OK;
}

// floats of mfnet_lora_pool_fwd's down: the product [M, RP] and workspace behind it (its parts)
extern "C" int64_t mfnet_lora_pool_down_floats(int64_t M, int RP, int out_dtype) {
  return M <= 0 ? 0 : M * RP + (M <= 64 ? 0 : M * RP * (out_dtype == MFNET_F32 ? 3 : 2) / 2);
}
extern "C" int mfnet_lora_pool_fwd(const void* X, int64_t ldx, const void* W, int64_t ldw, const float* bias, const float* scale, const void* a_down,
                                   const void* b_up, const int* ids, int64_t n, int RP, float* down, int64_t down_floats, void* out, int out_dtype,
                                   int64_t ldo, int64_t M, int64_t N, int64_t K, hipStream_t stream) {
  MF_CHECK_ARG(pool_counts(M, n) && pool_rp(RP), "lora_pool_fwd: bad sizes (M=%lld n=%lld RP=%d)", (long long)M, (long long)n, RP);
  MF_CHECK_ARG(out_dtype == MFNET_BF16 || out_dtype == MFNET_F32, "lora_pool_fwd: bad out dtype");
  if (M == 0) return MFNET_OK;
  MF_CHECK_ARG(X && W && scale && a_down && b_up && ids && down && out, "lora_pool_fwd: null pointer");
  POOL_CHECK_ROWS("lora_pool_fwd", X, ldx, K);
  POOL_CHECK_ROWS("lora_pool_fwd (weight)", W, ldw, K);
  POOL_CHECK_ROWS("lora_pool_fwd (out)", out, ldo, N);
  MF_CHECK_ARG(((uintptr_t)bias | (uintptr_t)down | (uintptr_t)a_down | (uintptr_t)b_up) % 16 == 0, "lora_pool_fwd: misaligned tensor");
  MF_CHECK_ARG(down_floats >= mfnet_lora_pool_down_floats(M, RP, out_dtype), "lora_pool_fwd: down holds too few floats (%lld)", (long long)down_floats);
  PoolGemm p;
  p.X = (const bf16_t*)X; p.ldx = ldx; p.W = (const bf16_t*)W; p.ldw = ldw; p.bias = bias;
  p.Up = (const bf16_t*)b_up; p.ids = ids; p.n = (int)n; p.RP = RP;
  p.out = out; p.ldo = ldo; p.out_f32 = out_dtype == MFNET_F32;
  p.M = M; p.N = (int)N; p.K = (int)K;
  return pool_products(p, a_down, scale, nullptr, nullptr, down, stream);
}

// floats of workspace of mfnet_lora_pool_bwd: p [M, RP] and its parts, the partial sums of dA and dB (more than one chunk per adapter)
extern "C" int64_t mfnet_lora_pool_bwd_workspace_floats(int64_t M, int64_t n, int64_t K, int64_t N, int RP) {
  return M <= 0 ? 0 : mfnet_lora_pool_down_floats(M, RP, MFNET_BF16) + (pool_one_chunk(M) ? 0 : mfnet_lora_pool_chunks(M, n) * (K + N) * RP);
}

extern "C" int mfnet_lora_pool_bwd(const void* dy, int64_t lddy, const void* X, int64_t ldx, const void* codes, const void* exps, const void* Wt, int64_t ldwt,
                                   const float* scale, const void* b_down, const void* a_up, const int* ids, const int* offs, const int* perm, const int* base,
                                   const int* table, int64_t n, int r, int RP, const float* down, void* dx, int64_t lddx, float* dA, float* dB, float* ws, int64_t ws_floats,
                                   int64_t M, int64_t N, int64_t K, hipStream_t stream) {
  MF_CHECK_ARG(pool_counts(M, n) && pool_rp(RP) && r >= 1 && r <= RP, "lora_pool_bwd: bad sizes (M=%lld n=%lld r=%d RP=%d)", (long long)M, (long long)n, r, RP);
  MF_CHECK_ARG(K >= 8 && K % 8 == 0 && K < (1 << 24) && N >= 8 && N % 8 == 0 && N < (1 << 24), "lora_pool_bwd: K=%lld and N=%lld must be multiples of 8", (long long)K, (long long)N);
  MF_CHECK_ARG(dA && dB && base, "lora_pool_bwd: null pointer");
  const int64_t chunks = mfnet_lora_pool_chunks(M, n);
  float* part_a = ws + mfnet_lora_pool_down_floats(M, RP, MFNET_BF16);
  float* part_b = part_a + chunks * K * RP;
  if (M > 0) {
    MF_CHECK_ARG(dy && scale && b_down && ids && offs && perm && table && down && ws && (!dx || (Wt && a_up)), "lora_pool_bwd: null pointer");
    MF_CHECK_ARG((X != nullptr) != (codes != nullptr) && (!codes || exps), "lora_pool_bwd: the input either as bf16 rows or as a checkpoint");
    POOL_CHECK_ROWS("lora_pool_bwd (dy)", dy, lddy, N);
    if (X) POOL_CHECK_ROWS("lora_pool_bwd (x)", X, ldx, K);
    if (dx) POOL_CHECK_ROWS("lora_pool_bwd (weight)", Wt, ldwt, N);
    if (dx) POOL_CHECK_ROWS("lora_pool_bwd (dx)", dx, lddx, K);
    MF_CHECK_ARG((uintptr_t)codes % 8 == 0 && ((uintptr_t)table | (uintptr_t)down | (uintptr_t)ws | (uintptr_t)b_down | (uintptr_t)a_up) % 16 == 0, "lora_pool_bwd: misaligned tensor");
    MF_CHECK_ARG(ws_floats >= mfnet_lora_pool_bwd_workspace_floats(M, n, K, N, RP), "lora_pool_bwd: workspace too small");
    MF_CHECK_ARG(chunks <= 65535, "lora_pool_bwd: too many chunks of rows (%lld)", (long long)chunks);
    int rc;
    if (!dx) rc = pool_down(dy, lddy, b_down, scale, ids, n, RP, perm, offs + n, PoolDown{ws, nullptr, 0}, M, N, stream);
    else {
      PoolGemm p;
      p.X = (const bf16_t*)dy; p.ldx = lddy; p.W = (const bf16_t*)Wt; p.ldw = ldwt; p.bias = nullptr;
      p.Up = (const bf16_t*)a_up; p.ids = ids; p.n = (int)n; p.RP = RP;
      p.out = dx; p.ldo = lddx; p.out_f32 = 0;
      p.M = M; p.N = (int)K; p.K = (int)N;
      rc = pool_products(p, b_down, scale, perm, offs + n, ws, stream);
    }
    if (rc) return rc;
    PoolTn a, b;
    a.Y = (const bf16_t*)X; a.ldy = ldx; a.codes = (const signed char*)codes; a.exps = (const unsigned char*)exps;
    a.U = ws; a.RP = RP; a.perm = perm; a.table = (const int4*)table; a.part = part_a; a.C = (int)K;
    b = a;
    b.Y = (const bf16_t*)dy; b.ldy = lddy; b.U = down; b.part = part_b; b.C = (int)N;
    const bool one_chunk = pool_one_chunk(M);
    a.base = b.base = base;
    a.r = b.r = r;
    a.out = one_chunk ? dA : nullptr;
    b.out = one_chunk ? dB : nullptr;
    const int strips_a = (int)ceil_div64(K, 256), strips_b = (int)ceil_div64(N, 256);
    const dim3 grid((unsigned)(strips_a + strips_b), (unsigned)(one_chunk ? n : chunks), RP == 64 ? 2 : 1);
#define PT(NR_, CK_, W_) hipLaunchKernelGGL((pool_tn_kernel<NR_, CK_, W_>), grid, dim3(64 * W_), 0, stream, a, b, strips_a)
#define PTW(W_) do { if (RP == 16) { if (codes) PT(1, true, W_); else PT(1, false, W_); } \
    else { if (codes) PT(2, true, W_); else PT(2, false, W_); } } while (0)
    if (one_chunk && M > 128) PTW(8); else PTW(4);
#undef PTW
#undef PT
    MF_LAUNCH_CHECK("lora_pool_bwd (sums over rows)");
    if (one_chunk) return MFNET_OK;
  }
  PoolSum sa, sb;
  sa.part = part_a; sa.out = dA; sa.per = K * RP; sa.ld = (int)K; sa.d0 = r; sa.d1 = (int)K;
  sb.part = part_b; sb.out = dB; sb.per = N * RP; sb.ld = RP; sb.d0 = (int)N; sb.d1 = r;
  hipLaunchKernelGGL(pool_sum_kernel, dim3((unsigned)ceil_div64((K > N ? K : N) * r, 256), (unsigned)n, 2), dim3(256), 0, stream, sa, sb, base);
  MF_LAUNCH_CHECK("lora_pool_bwd (sums of chunks)");
  return MFNET_OK;
}
