// Linear layers on 8-bit codes: dynamic quantisation of token rows and the product with per-token and per-channel scales
// (the projections and the feed-forward layers of model/modules/sparse_transformer.py:68-69,123-130 served in 8 bits).
//
//   scale[r] = max_k |x[r,k]| / 127,  q[r,k] = round-half-even(x[r,k] / scale[r])
//   out[m,n] = act(sum_k xq[m,k] wq[n,k] * xs[m] * ws[n] + bias[n])        sum exact in int32 (K <= 131072: K * 127^2 < 2^31)
//
// MFMA operand order.  v_mfma_i32_16x16x64_i8: lane l hands in 16 bytes = row l & 15, k = (l >> 4) * 16 .. + 15 of either operand and
// receives column l & 15, rows (l >> 4) * 4 + r of the product.  The weights are the row operand: a lane then holds neighbouring output
// channels of ONE token.  They are laid out once in 4 KB blocks of 64 channels x 64 k, four operand tiles of 1 KB each in lane order; row
// i of tile t is channel (t / 2) * 32 + (i / 4) * 8 + (t % 2) * 4 + i % 4 of the block, so that two tiles give every lane 8 CONSECUTIVE
// channels, a 16-byte fp16 store of which 4 lanes fill 64 bytes of a row, and a wave reads a tile as one contiguous kilobyte.
#include "common.h"

namespace pp {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------------------------------------------------------------
// codes of token rows
// ---------------------------------------------------------------------------------------------------------------------------------
// 8 elements at column c of a row of K; columns past K are 0.  `wide`: rows are 16-byte aligned.
template <typename T>
__device__ __forceinline__ void row_load8(const T* row, int c, int K, bool wide, float* v) {
  if (wide && c + 8 <= K) {
    load8<T>(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? to_f32(row[c + i]) : 0.f;
  }
}

// |v| as ordered bits: the maximum of these keeps NaN (largest) and infinity, which fmaxf would drop
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct RowScale {
  float scale;     // as stored: amax / 127, NaN if the row holds a NaN or an infinity
  float s, rcp;    // scale and its reciprocal after the power-of-two lift of rows whose quotients would leave fp32's normal range
  float lift;
  bool zero;       // every code is 0
};
__device__ __forceinline__ RowScale row_scale(unsigned amax_bits) {
  RowScale r;
  const float amax = __uint_as_float(amax_bits);
  const bool bad = amax_bits >= 0x7f800000u;
  r.scale = bad ? __uint_as_float(0x7fc00000u) : amax / 127.f;
  r.lift = amax < 1e-18f ? 18446744073709551616.f : 1.f;
  r.s = r.scale * r.lift;
  r.zero = bad || !(r.s > 0.f);
  r.rcp = 1.f / r.s;
  return r;
}
// The integer nearest to v / s: the product with the reciprocal is off by at most one step near a tie; the remainder v - q s is exact in
// fp32 (a multiple of the smaller operand's last place, not above |s|), so comparing twice its size with s decides the step.
__device__ __forceinline__ int code_of(float v, const RowScale& r) {
  v *= r.lift;
  float q = rintf(v * r.rcp);
  const float rem = fmaf(-q, r.s, v), two = 2.f * fabsf(rem);
  const float step = rem > 0.f ? 1.f : -1.f;
  if (two > r.s || (two == r.s && ((int)q & 1))) q += step;
  q = fminf(fmaxf(q, -127.f), 127.f);
  return r.zero ? 0 : (int)q;
}
__device__ __forceinline__ u32x2 codes8(const float* v, const RowScale& r) {
  unsigned w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[h] |= (unsigned)(code_of(v[h * 4 + i], r) & 0xff) << (8 * i);
  }
  return u32x2{w[0], w[1]};
}

__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o));
  return v;
}

// Codes of 8 values of a row whose scale needs no lift: v / s rounded by adding 1.5 * 2^23 (the code is the sum's low byte), the remainders'
// maximum looked at once -- a remainder of half a step or more (ties, and quotients next to one) takes code_of's comparison.
__device__ __forceinline__ u32x2 codes8_fast(const float* v, const RowScale& r, float half) {
  constexpr float magic = 12582912.f;
  float worst = 0.f;
  unsigned b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = fmaf(v[i], r.rcp, magic);
    b[i] = __float_as_uint(t);
    worst = fmaxf(worst, fabsf(fmaf(magic - t, r.s, v[i])));
  }
  u32x2 w;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const unsigned lo = __builtin_amdgcn_perm(b[h * 4 + 1], b[h * 4], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[h * 4 + 3], b[h * 4 + 2], 0x0c0c0400u);
    w[h] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  return worst >= half ? codes8(v, r) : w;
}

// abs maximum of 8 raw elements, as bits of the element type (fp16: two at a time)
template <typename T> struct Raw8;
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <> struct Raw8<_Float16> {
  u32x4 r;
  __device__ __forceinline__ void load(const _Float16* p) { r = *reinterpret_cast<const u32x4*>(p); }
  __device__ __forceinline__ void set(int i, _Float16 v) {
    const unsigned u = __builtin_bit_cast(unsigned short, v);
    r[i >> 1] = (i & 1) ? (r[i >> 1] & 0xffffu) | (u << 16) : (r[i >> 1] & 0xffff0000u) | u;
  }
  __device__ __forceinline__ void values(float* v) const {
    const _Float16* h = reinterpret_cast<const _Float16*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
  }
  __device__ __forceinline__ unsigned amax() const {      // bits of the maximum as fp32
    u16x2 m = __builtin_bit_cast(u16x2, r[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, r[i] & 0x7fff7fffu));
    const unsigned short b = m[0] > m[1] ? m[0] : m[1];
    return abs_bits((float)__builtin_bit_cast(_Float16, b));
  }
};
template <> struct Raw8<float> {
  u32x4 r[2];
  __device__ __forceinline__ void load(const float* p) { r[0] = *reinterpret_cast<const u32x4*>(p); r[1] = *reinterpret_cast<const u32x4*>(p + 4); }
  __device__ __forceinline__ void set(int i, float v) { r[i >> 2][i & 3] = __float_as_uint(v); }
  __device__ __forceinline__ void values(float* v) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i >> 2][i & 3]);
  }
  __device__ __forceinline__ unsigned amax() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, r[i >> 2][i & 3] & 0x7fffffffu);
    return m;
  }
};

// A row in the registers of WPR waves, VPL vectors of 8 a lane: one pass over memory.  4 / WPR rows a block.
template <typename T, int VPL, int WPR>
__global__ __launch_bounds__(256) void quant_kernel(const T* __restrict__ x, long long xrs, int8_t* __restrict__ q, long long qrs,
                                                    float* __restrict__ scale, long long rows, int K, int Kp, int wide) {
  __shared__ unsigned wm[4];
  const int wave = threadIdx.x >> 6, t = threadIdx.x % (64 * WPR);
  for (long long row0 = blockIdx.x * (long long)(4 / WPR); row0 < rows; row0 += gridDim.x * (long long)(4 / WPR)) {
    const long long row = row0 + wave / WPR;
    const bool on = row < rows;
    const T* xr = x + (on ? row : rows - 1) * xrs;
    Raw8<T> raw[VPL];
    unsigned m = 0;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int c = (v * 64 * WPR + t) * 8;
      if (wide && c + 8 <= K) {
        raw[v].load(xr + c);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[v].set(i, c + i < K ? xr[c + i] : (T)0.f);
      }
    }
#pragma unroll
    for (int v = 0; v < VPL; ++v) m = max(m, raw[v].amax());
    m = wave_umax(m);
    if constexpr (WPR == 4) {
      if ((threadIdx.x & 63) == 0) wm[wave] = m;
      __syncthreads();
      m = max(max(wm[0], wm[1]), max(wm[2], wm[3]));
      __syncthreads();
    }
    m = __builtin_amdgcn_readfirstlane(m);
    const RowScale r = row_scale(m);
    if (!on) continue;                                     // (WPR == 4: one row a block, always on)
    if (t == 0) scale[row] = r.scale;
    const bool plain = !r.zero && r.lift == 1.f;
    const float half = 0.5f * r.s;
    int8_t* qr = q + row * qrs;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int c = (v * 64 * WPR + t) * 8;
      if (c >= Kp) break;
      float f[8];
      raw[v].values(f);
      *reinterpret_cast<u32x2*>(qr + c) = plain ? codes8_fast(f, r, half) : codes8(f, r);
    }
  }
}

// One block of 256 threads per row, any K: the row is read twice (the second time from L2).
template <typename T>
__global__ __launch_bounds__(256) void quant_row_kernel(const T* __restrict__ x, long long xrs, int8_t* __restrict__ q, long long qrs,
                                                        float* __restrict__ scale, long long rows, int K, int Kp, int wide) {
  __shared__ unsigned wm[4];
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
  const T* xr = x + row * xrs;
  unsigned m = 0;
  for (int c = threadIdx.x * 8; c < K; c += 2048) {
    float v[8];
    row_load8<T>(xr, c, K, wide, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
  }
  m = wave_umax(m);
  if ((threadIdx.x & 63) == 0) wm[threadIdx.x >> 6] = m;
  __syncthreads();
  const RowScale r = row_scale(max(max(wm[0], wm[1]), max(wm[2], wm[3])));
  if (threadIdx.x == 0) scale[row] = r.scale;
  for (int c = threadIdx.x * 8; c < Kp; c += 2048) {
    float v[8];
    row_load8<T>(xr, c, K, wide, v);
    *reinterpret_cast<u32x2*>(q + row * qrs + c) = codes8(v, r);
  }
  __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// weight layout
// ---------------------------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void pack_i8_kernel(const int8_t* __restrict__ w, long long wrs, u32x4* __restrict__ out, int N, int K,
                                                      int ktiles, long long pieces) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < pieces; i += gridDim.x * 256ll) {
    const int lane = (int)(i & 63), t = (int)(i >> 6) & 3;
    const long long blk = i >> 8;
    const int kt = (int)(blk % ktiles);
    const long long nb = blk / ktiles;
    const int row = lane & 15;
    const long long n = nb * 64 + (t >> 1) * 32 + (row >> 2) * 8 + (t & 1) * 4 + (row & 3);
    const int k0 = kt * 64 + (lane >> 4) * 16;
    u32x4 o = {0, 0, 0, 0};
    if (n < N) {
#pragma unroll
      for (int b = 0; b < 16; ++b)
        if (k0 + b < K) o[b >> 2] |= (unsigned)(uint8_t)w[n * wrs + k0 + b] << (8 * (b & 3));
    }
    out[i] = o;
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------------------------------------------------------------
struct LinI8Params {
  const int8_t* xq;
  const float* xs;
  const u32x4* w;
  const float* ws;
  const float* bias;
  char* out;
  long long qrs, ors, M;
  int N, ktiles, act;
  float act_param;
  int wide_out;      // rows of `out` are 16-byte aligned
};

// The channels of a 64-channel block that one lane holds (8 at c0 = n0 + (lane / 16) * 8, 8 at c0 + 32) with their scales and biases
template <typename TO> struct LaneChannels {
  int c0;
  float ws[16], bias[16];
  __device__ __forceinline__ void load(const LinI8Params& p, int n0) {
    c0 = n0 + ((threadIdx.x & 63) >> 4) * 8;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int n = min(c0 + (i >> 3) * 32 + (i & 7), p.N - 1);
      ws[i] = p.ws[n];
      bias[i] = p.bias != nullptr ? p.bias[n] : 0.f;
    }
  }
  // scale, bias, activation, store of token m
  __device__ __forceinline__ void store(const LinI8Params& p, long long m, float xs, const i32x4* acc) const {
    TO* o = reinterpret_cast<TO*>(p.out) + m * p.ors + c0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf((float)acc[h * 2 + (i >> 2)][i & 3] * xs, ws[h * 8 + i], bias[h * 8 + i]);
      if (p.act != PP_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_value(v[i], p.act, p.act_param);
      }
      const int c = c0 + h * 32;
      if (p.wide_out && c + 8 <= p.N) {
        store8<TO>(o + h * 32, v);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < p.N) o[h * 32 + i] = from_f32<TO>(v[i]);
      }
    }
  }
};

// 4 waves, each 64 channels x 32 tokens, operands straight from memory.  Token rows past M repeat the last one and are not stored.
template <typename TO>
__global__ __launch_bounds__(256) void lin_i8_kernel(const LinI8Params p) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long m0 = (blockIdx.x * 4ll + wave) * 32;
  const int nb = blockIdx.y;
  const u32x4* w = p.w + (long long)nb * p.ktiles * 256 + lane;
  const int8_t* xa[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    long long m = m0 + j * 16 + (lane & 15);
    if (m >= p.M) m = p.M - 1;
    xa[j] = p.xq + m * p.qrs + (lane >> 4) * 16;
  }
  i32x4 acc[2][4];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[j][t] = i32x4{0, 0, 0, 0};
  for (int kt = 0; kt < p.ktiles; ++kt) {
    u32x4 wf[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) wf[t] = w[(long long)kt * 256 + t * 64];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u32x4 xf = *reinterpret_cast<const u32x4*>(xa[j] + (long long)kt * 64);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        acc[j][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, wf[t]), __builtin_bit_cast(i32x4, xf), acc[j][t], 0, 0, 0);
    }
  }
  LaneChannels<TO> ch;
  ch.load(p, nb * 64);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const long long m = m0 + j * 16 + (lane & 15);
    if (m < p.M) ch.store(p, m, p.xs[m], acc[j]);
  }
#endif
}

// Tiles of BM tokens x BN channels, WM x WN waves of BM / WM tokens x BN / WN channels.  Both operands go from memory into LDS without
// passing registers (16 bytes a lane, one kilobyte an instruction), S stages of 64 k deep: the weights' kilobytes are in operand order
// already, the lanes of a token piece gather 16 rows x 4 pieces so that it lands in operand order too -- fragment reads are then
// lane-linear and free of bank conflicts without any swizzle.  Token rows past M repeat the last one, channel blocks past N the last one.
typedef __attribute__((address_space(3))) void* i8_lptr;
typedef __attribute__((address_space(1))) void* i8_gptr;

template <typename TO, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN, 1) void lin_i8_tile_kernel(const LinI8Params p, const int tm, const int tn) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int NW = WM * WN, PA = BM / 16, PW = BN / 16, G = (PA + PW) / NW;      // 1 KB pieces of a stage; DMA instructions a wave
  constexpr int STAGE = (PA + PW) * 1024, TA = BM / WM / 16, TB = BN / WN / 64;    // 16-token tiles, 64-channel blocks of a wave
  static_assert((PA + PW) % NW == 0 && PA % NW == 0, "pieces are dealt out evenly");
  __shared__ __attribute__((aligned(1024))) char lds[S * STAGE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
  // block -> tile: every XCD (block id mod 8) gets a contiguous run; runs walk groups of 8 token tiles, tokens fastest, so that the blocks
  // which run together share few token and weight panels
  long long id = blockIdx.x;
  {
    const long long n = gridDim.x, per = n >> 3, extra = n & 7, x = id & 7;
    id = x * per + (x < extra ? x : extra) + (id >> 3);
  }
  const long long grp = id / (8ll * tn);
  const int gm = (int)min(8ll, tm - grp * 8);
  const int in = (int)(id - grp * 8 * tn);
  const long long m0 = (grp * 8 + in % gm) * BM;
  const int n0 = in / gm * BN;

  const int8_t* src[G];
  int step[G];
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const int piece = j * NW + wave;
    if (piece < PA) {
      long long m = m0 + piece * 16 + (lane & 15);
      if (m >= p.M) m = p.M - 1;
      src[j] = p.xq + m * p.qrs + (lane >> 4) * 16;
      step[j] = 64;
    } else {
      int nb = n0 / 64 + (piece - PA) / 4;
      const int last = (p.N + 63) / 64 - 1;
      if (nb > last) nb = last;
      src[j] = reinterpret_cast<const int8_t*>(p.w) + ((long long)nb * p.ktiles * 4 + (piece - PA) % 4) * 1024 + lane * 16;
      step[j] = 4096;
    }
  }
  auto issue = [&](int buf) {
#pragma unroll
    for (int j = 0; j < G; ++j) {
      __builtin_amdgcn_global_load_lds((i8_gptr)src[j], (i8_lptr)(lds + buf * STAGE + (j * NW + wave) * 1024), 16, 0, 0);
      src[j] += step[j];
    }
  };
  i32x4 acc[TA][TB * 4];
#pragma unroll
  for (int a = 0; a < TA; ++a)
#pragma unroll
    for (int b = 0; b < TB * 4; ++b) acc[a][b] = i32x4{0, 0, 0, 0};
  const int nk = p.ktiles;
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < nk) issue(s);
  int buf = 0, nbuf = S - 1;
  for (int ks = 0; ks < nk; ++ks) {
    const int ahead = min(S - 2, nk - 1 - ks);      // younger stages that may still be in flight
    if (ahead >= 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * G) : "memory");
    else if (ahead == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(G) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();                   // stage `buf` is there for all waves; stage `nbuf`, read one step ago, is free
    if (ks + S - 1 < nk) issue(nbuf);
    const char* st = lds + buf * STAGE + lane * 16;
    i32x4 wf[TB * 4], xf[TA];
#pragma unroll
    for (int b = 0; b < TB * 4; ++b) wf[b] = *reinterpret_cast<const i32x4*>(st + (PA + wn * TB * 4 + b) * 1024);
#pragma unroll
    for (int a = 0; a < TA; ++a) xf[a] = *reinterpret_cast<const i32x4*>(st + (wm * TA + a) * 1024);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int a = 0; a < TA; ++a)
#pragma unroll
      for (int b = 0; b < TB * 4; ++b) acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[b], xf[a], acc[a][b], 0, 0, 0);
    buf = buf + 1 == S ? 0 : buf + 1;
    nbuf = nbuf + 1 == S ? 0 : nbuf + 1;
  }
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    const int nb = n0 + (wn * TB + b) * 64;
    if (nb >= p.N) break;
    LaneChannels<TO> ch;
    ch.load(p, nb);
#pragma unroll
    for (int a = 0; a < TA; ++a) {
      const long long m = m0 + (wm * TA + a) * 16 + (lane & 15);
      if (m < p.M) ch.store(p, m, p.xs[m], &acc[a][b * 4]);
    }
  }
#endif
}

template <typename TO, int BM, int BN, int WM, int WN, int S>
static void launch_tiles(const LinI8Params& p, hipStream_t st) {
  const int tm = (int)((p.M + BM - 1) / BM), tn = (p.N + BN - 1) / BN;
  hipLaunchKernelGGL((lin_i8_tile_kernel<TO, BM, BN, WM, WN, S>), dim3((unsigned)((long long)tm * tn)), dim3(64 * WM * WN), 0, st, p, tm, tn);
}
template <typename TO>
static void launch_product(const LinI8Params& p, hipStream_t st) {
  const long long t256 = ((p.M + 255) / 256) * ((p.N + 255) / 256);
  if (p.M <= 32) hipLaunchKernelGGL((lin_i8_kernel<TO>), dim3((unsigned)((p.M + 127) / 128), (p.N + 63) / 64), dim3(256), 0, st, p);
  else if (t256 >= 256) launch_tiles<TO, 256, 256, 2, 4, 4>(p, st);
  else launch_tiles<TO, 128, 128, 2, 2, 4>(p, st);
}

}  // namespace pp

using namespace pp;

constexpr int PP_I8_MAX_N = 65535 * 64;            // grid.y
constexpr int64_t PP_I8_MAX_M = (int64_t)1 << 30;  // grid.x * 256 threads below 2^32

extern "C" int pp_i8_row_bytes(int K) {
  if (K <= 0 || K > 131072) return PP_ERR_ARG;
  return (K + 63) / 64 * 64;
}

// A row goes into the registers of one wave (K <= 2048) or of a block (K <= 16384) where it fits in 8 vectors a lane, else it is read twice.
template <typename T>
static void launch_quant(const void* x, int64_t xrs, void* q, int64_t qrs, float* scale, int64_t rows, int K, int Kp, int wide, hipStream_t st) {
  const int64_t want = K <= 2048 ? (rows + 3) / 4 : rows;
  const dim3 grid((unsigned)(want < 65536 ? want : 65536)), block(256);
#define PP_QUANT(V, W) hipLaunchKernelGGL((quant_kernel<T, V, W>), grid, block, 0, st, (const T*)x, (long long)xrs, (int8_t*)q, (long long)qrs, scale, (long long)rows, K, Kp, wide)
  if (K <= 512) PP_QUANT(1, 1);
  else if (K <= 1024) PP_QUANT(2, 1);
  else if (K <= 2048) PP_QUANT(4, 1);
  else if (K <= 4096) PP_QUANT(2, 4);
  else if (K <= 8192) PP_QUANT(4, 4);
  else if (K <= 16384) PP_QUANT(8, 4);
  else hipLaunchKernelGGL((quant_row_kernel<T>), grid, block, 0, st, (const T*)x, (long long)xrs, (int8_t*)q, (long long)qrs, scale, (long long)rows, K, Kp, wide);
#undef PP_QUANT
}

extern "C" int pp_quantize_tokens(const void* x, int64_t x_rstride, void* q, int64_t q_rstride, float* scale, int64_t rows, int K, int dtype,
                                  void* stream) {
  const int Kp = pp_i8_row_bytes(K);
  PP_REQUIRE(Kp > 0 && rows >= 0 && rows <= 0x7fffffff, PP_ERR_ARG, "pp_quantize_tokens: bad arguments (rows=%lld, K=%d, at most 131072)", (long long)rows, K);
  PP_REQUIRE(dtype == PP_F32 || dtype == PP_F16, PP_ERR_DTYPE, "pp_quantize_tokens: dtype %d", dtype);
  if (rows == 0) return 0;
  const int esz = dtype == PP_F16 ? 2 : 4;
  PP_REQUIRE(x && q && scale && x_rstride >= 0 && q_rstride >= Kp, PP_ERR_ARG, "pp_quantize_tokens: null buffer or row stride (x %lld, q %lld < %d)",
             (long long)x_rstride, (long long)q_rstride, Kp);
  PP_REQUIRE((uintptr_t)x % esz == 0 && (uintptr_t)q % 16 == 0 && q_rstride % 16 == 0 && (uintptr_t)scale % 4 == 0, PP_ERR_ALIGN,
             "pp_quantize_tokens: q and its row stride must be multiples of 16 bytes");
  const int wide = (uintptr_t)x % 16 == 0 && x_rstride * esz % 16 == 0;
  if (dtype == PP_F16) launch_quant<_Float16>(x, x_rstride, q, q_rstride, scale, rows, K, Kp, wide, (hipStream_t)stream);
  else launch_quant<float>(x, x_rstride, q, q_rstride, scale, rows, K, Kp, wide, (hipStream_t)stream);
  return launch_status("pp_quantize_tokens");
}

extern "C" int64_t pp_linear_i8_weight_bytes(int N, int K) {
  const int Kp = pp_i8_row_bytes(K);
  if (N <= 0 || N > PP_I8_MAX_N || Kp <= 0) return PP_ERR_ARG;
  return (int64_t)((N + 63) / 64) * 64 * Kp;
}

extern "C" int pp_linear_i8_pack(const void* wq, int64_t wq_rstride, void* weight, int N, int K, void* stream) {
  const int64_t bytes = pp_linear_i8_weight_bytes(N, K);
  PP_REQUIRE(bytes > 0 && wq && weight && wq_rstride >= K, PP_ERR_ARG, "pp_linear_i8_pack: bad arguments (N=%d, K=%d)", N, K);
  PP_REQUIRE((uintptr_t)weight % 16 == 0, PP_ERR_ALIGN, "pp_linear_i8_pack: weight must be 16-byte aligned");
  const long long pieces = bytes / 16;
  const long long blocks = (pieces + 255) / 256;
  hipLaunchKernelGGL(pack_i8_kernel, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, (hipStream_t)stream, (const int8_t*)wq,
                     (long long)wq_rstride, (u32x4*)weight, N, K, pp_i8_row_bytes(K) / 64, pieces);
  return launch_status("pp_linear_i8_pack");
}

extern "C" int pp_linear_i8(const void* xq, int64_t q_rstride, const float* xs, const void* weight, const float* ws, const float* bias, void* out,
                            int64_t out_rstride, int64_t M, int N, int K, int act, float act_param, int out_dtype, void* stream) {
  const int Kp = pp_i8_row_bytes(K);
  PP_REQUIRE(Kp > 0 && N > 0 && N <= PP_I8_MAX_N && M >= 0 && M <= PP_I8_MAX_M, PP_ERR_ARG, "pp_linear_i8: bad arguments (M=%lld N=%d K=%d)", (long long)M, N, K);
  PP_REQUIRE(act >= PP_ACT_NONE && act <= PP_ACT_SILU, PP_ERR_ARG, "pp_linear_i8: activation code %d", act);
  PP_REQUIRE(out_dtype == PP_F32 || out_dtype == PP_F16, PP_ERR_DTYPE, "pp_linear_i8: out_dtype %d", out_dtype);
  if (M == 0) return 0;
  PP_REQUIRE(xq && xs && weight && ws && out && q_rstride >= Kp && out_rstride >= N, PP_ERR_ARG,
             "pp_linear_i8: null buffer or row stride (q %lld < %d, out %lld < %d)", (long long)q_rstride, Kp, (long long)out_rstride, N);
  const int osz = out_dtype == PP_F16 ? 2 : 4;
  PP_REQUIRE((uintptr_t)xq % 16 == 0 && q_rstride % 16 == 0 && (uintptr_t)weight % 16 == 0 && (uintptr_t)out % osz == 0, PP_ERR_ALIGN,
             "pp_linear_i8: codes, their row stride and the weight must be multiples of 16 bytes");
  LinI8Params p;
  p.xq = (const int8_t*)xq; p.xs = xs; p.w = (const u32x4*)weight; p.ws = ws; p.bias = bias; p.out = (char*)out;
  p.qrs = q_rstride; p.ors = out_rstride; p.M = M; p.N = N; p.ktiles = Kp / 64; p.act = act; p.act_param = act_param;
  p.wide_out = (uintptr_t)out % 16 == 0 && out_rstride * osz % 16 == 0;
  hipStream_t st = (hipStream_t)stream;
  PP_REQUIRE(((M + 127) / 128) * ((N + 127) / 128) <= (1 << 23), PP_ERR_ARG, "pp_linear_i8: too many tiles (M=%lld N=%d)", (long long)M, N);
  if (out_dtype == PP_F16) launch_product<_Float16>(p, st);
  else launch_product<float>(p, st);
  return launch_status("pp_linear_i8");
}
