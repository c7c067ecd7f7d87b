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

// maximum over the wave, on the VALU: rotations inside the 16-lane rows, then the swaps of rows and half-waves
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#if defined(__HIP_DEVICE_COMPILE__)
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));      // row_ror:8, 4, 2, 1
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  u2 r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max((unsigned)r.x, (unsigned)r.y);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max((unsigned)r.x, (unsigned)r.y);
#endif
  return v;
}

// Codes of 8 values of a row whose scale needs no lift (half = s / 2; a negative half sends the others to code_of): v / s rounded by adding 1.5 * 2^23 (the code is the sum's low byte), the remainders'
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
  if (worst >= half) {
    float u[8];                                    // (opaque: the rare path's arithmetic stays in it instead of being done for everybody)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u[i] = v[i];
#if defined(__HIP_DEVICE_COMPILE__)
      asm volatile("" : "+v"(u[i]));
#endif
    }
    w = codes8(u, r);
  }
  return w;
}

// abs maximum of 8 raw elements, as bits of the element type (fp16: two at a time)
template <typename T> struct Raw8;
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <> struct Raw8<_Float16> {
  u32x4 r;
  __device__ __forceinline__ void load(const _Float16* p) { r = *reinterpret_cast<const u32x4*>(p); }
  __device__ __forceinline__ void load_any(const _Float16* p) { r = load16_any(p); }
  __device__ __forceinline__ void clear() { r = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void keep(int n) {            // elements n .. 7 become 0
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = 2 * i + 1 < n ? r[i] : 2 * i < n ? r[i] & 0xffffu : 0u;
  }
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
  __device__ __forceinline__ void load_any(const float* p) { r[0] = load16_any(p); r[1] = load16_any(p + 4); }
  __device__ __forceinline__ void clear() { r[0] = r[1] = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void keep(int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i >> 2][i & 3] = i < n ? r[i >> 2][i & 3] : 0u;
  }
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

// A row in the registers of WPR waves, VPL vectors of 8 a lane: one pass over memory, 4 / WPR rows a block.  WIDE: K a multiple of 8, rows 16-byte
// aligned.  Bound by memory: 110160 x 1960 fp16 115 us (5.6 TB/s, a copy's rate), x 512 33 us (5.2 TB/s); with the rare path's arithmetic left to
// the compiler's hoisting the latter took 45.
template <typename T, int VPL, int WPR, bool WIDE>
__global__ __launch_bounds__(256) void quant_kernel(const T* __restrict__ x, long long xrs, int8_t* __restrict__ q, long long qrs,
                                                    float* __restrict__ scale, long long rows, int K, int Kp) {
  __shared__ unsigned wm[4];
  const int wave = threadIdx.x >> 6, t = threadIdx.x % (64 * WPR);
  for (long long row0 = blockIdx.x * (long long)(4 / WPR); row0 < rows; row0 += gridDim.x * (long long)(4 / WPR)) {
    const long long row = row0 + wave / WPR;
    const T* xr = x + min(row, rows - 1) * xrs;
    const bool inside = row < rows - 1 && xrs >= 8;        // a vector past this row's end is still inside the rows
    Raw8<T> raw[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int c = (v * 64 * WPR + t) * 8;
      if constexpr (WIDE) {
        raw[v].load(xr + (c < K ? c : 0));
        if (c >= K) raw[v].clear();
      } else if (c + 8 <= K || (c < K && inside)) {
        raw[v].load_any(xr + c);
        raw[v].keep(K - c);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[v].set(i, c + i < K ? xr[c + i] : (T)0.f);
      }
    }
    unsigned m = 0;
#pragma unroll
    for (int v = 0; v < VPL; ++v) m = max(m, raw[v].amax());
    m = wave_umax(m);
    if constexpr (WPR == 4) {
      if ((threadIdx.x & 63) == 0) wm[wave] = m;
      __syncthreads();
      m = max(max(wm[0], wm[1]), max(wm[2], wm[3]));
      __syncthreads();
    }
    if (row >= rows) continue;                             // (WPR == 4: one row a block, always below)
    const RowScale r = row_scale(__builtin_amdgcn_readfirstlane(m));
    if (t == 0) scale[row] = r.scale;
    const float half = !r.zero && r.lift == 1.f ? 0.5f * r.s : -1.f;
    int8_t* qr = q + row * qrs;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int c = (v * 64 * WPR + t) * 8;
      if (c >= Kp) break;
      float f[8];
      raw[v].values(f);
      *reinterpret_cast<u32x2*>(qr + c) = codes8_fast(f, r, half);
    }
  }
}

// One block of 256 threads per row, any K: the row is read twice (the second time from L2).
template <typename T>
__global__ __launch_bounds__(256) void quant_row_kernel(const T* __restrict__ x, long long xrs, int8_t* __restrict__ q, long long qrs,
                                                        float* __restrict__ scale, long long rows, int K, int Kp) {
  __shared__ unsigned wm[4];
  auto vector = [&](const T* xr, int c) {
    Raw8<T> raw;
    if (c + 8 <= K) {
      raw.load_any(xr + c);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) raw.set(i, c + i < K ? xr[c + i] : (T)0.f);
    }
    return raw;
  };
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * xrs;
    unsigned m = 0;
    for (int c = threadIdx.x * 8; c < K; c += 2048) m = max(m, vector(xr, c).amax());
    m = wave_umax(m);
    if ((threadIdx.x & 63) == 0) wm[threadIdx.x >> 6] = m;
    __syncthreads();
    const RowScale r = row_scale(max(max(wm[0], wm[1]), max(wm[2], wm[3])));
    if (threadIdx.x == 0) scale[row] = r.scale;
    const float half = !r.zero && r.lift == 1.f ? 0.5f * r.s : -1.f;
    for (int c = threadIdx.x * 8; c < Kp; c += 2048) {
      float f[8];
      vector(xr, c).values(f);
      *reinterpret_cast<u32x2*>(q + row * qrs + c) = codes8_fast(f, r, half);
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
};

// 8 consecutive channels c .. c + 7 that a lane holds of two neighbouring operand tiles, with their scales and biases
template <typename TO> struct Lane8 {
  int c;
  float ws[8], bias[8];
  __device__ __forceinline__ void load(const LinI8Params& p, int first) {
    c = first;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = min(c + i, p.N - 1);
      ws[i] = p.ws[n];
      bias[i] = p.bias != nullptr ? p.bias[n] : 0.f;
    }
  }
  // scale, bias, activation
  __device__ __forceinline__ void value(const LinI8Params& p, float xs, const i32x4* acc, float* v) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf((float)acc[i >> 2][i & 3] * xs, ws[i], bias[i]);
    act_values<8>(v, p.act, p.act_param);
  }
  __device__ __forceinline__ void store(const LinI8Params& p, long long m, const float* v) const {
    TO* o = reinterpret_cast<TO*>(p.out) + m * p.ors + c;
    if (c + 8 <= p.N) {
      store8_any<TO>(o, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < p.N) o[i] = from_f32<TO>(v[i]);
    }
  }
};

// Few tokens: the weights' bytes are the work.  A block takes TPB operand tiles (16 channels each) of one 64-channel block and 16 MT tokens; its 8
// waves share out K, operands straight from memory, several tiles in flight, and add their exact partial sums through LDS.  Latency: 16 tokens x 1024 ->
// 16384 6.0 us (16.8 MB of weights, out of the cache).
constexpr int I8_KW = 8;
template <typename T> struct FloatTokens { const T* x; long long xrs; int K; };

// acc[t][j] += tiles kt0 .. kt1 of the weights times the tokens; tok(kt, j) gives the token operand
template <int MT, int TPB, typename F>
__device__ __forceinline__ void thin_product(const u32x4* w, int kt0, int kt1, i32x4 (&acc)[TPB][MT], F tok) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int U = TPB + MT <= 3 ? 8 : 4;
  int kt = kt0;
  for (; kt + U <= kt1; kt += U) {
    i32x4 wf[U][TPB], xf[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int t = 0; t < TPB; ++t) wf[u][t] = __builtin_bit_cast(i32x4, w[(long long)(kt + u) * 256 + t * 64]);
#pragma unroll
      for (int j = 0; j < MT; ++j) xf[u][j] = tok(kt + u, j);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < TPB; ++t)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[t][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][t], xf[u][j], acc[t][j], 0, 0, 0);
  }
  for (; kt < kt1; ++kt)
#pragma unroll
    for (int t = 0; t < TPB; ++t) {
      const i32x4 wf = __builtin_bit_cast(i32x4, w[(long long)kt * 256 + t * 64]);
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[t][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, tok(kt, j), acc[t][j], 0, 0, 0);
    }
#endif
}

// adds the waves' sums and writes the block's outputs, tokens m0 .. m_end - 1; xs_of(m) is the scale of token m
template <typename TO, int MT, int TPB, typename F>
__device__ __forceinline__ void thin_finish(const LinI8Params& p, i32x4* red, const i32x4 (&acc)[TPB][MT], int nb, int t0, long long m0, long long m_end, F xs_of) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int t = 0; t < TPB; ++t)
#pragma unroll
    for (int j = 0; j < MT; ++j) red[((t * MT + j) * I8_KW + wave) * 64 + lane] = acc[t][j];
  __syncthreads();
  for (int f = wave; f < TPB * MT; f += I8_KW) {
    i32x4 a = red[f * I8_KW * 64 + lane];
#pragma unroll
    for (int w = 1; w < I8_KW; ++w) a += red[(f * I8_KW + w) * 64 + lane];
    const int t = t0 + f / MT;
    const long long m = m0 + f % MT * 16 + (lane & 15);
    const int c = nb * 64 + (t >> 1) * 32 + (lane >> 4) * 8 + (t & 1) * 4;
    if (m >= m_end) continue;
    const float xs = xs_of(m);
    TO* o = reinterpret_cast<TO*>(p.out) + m * p.ors + c;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < p.N)
        o[i] = from_f32<TO>(act_value(fmaf((float)a[i] * xs, p.ws[c + i], p.bias != nullptr ? p.bias[c + i] : 0.f), p.act, p.act_param));
  }
}

template <typename TO, int MT, int TPB>
__global__ __launch_bounds__(512) void lin_i8_thin_kernel(const LinI8Params p) {
  __shared__ __attribute__((aligned(16))) i32x4 red[TPB * MT * I8_KW * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int nb = blockIdx.x / (4 / TPB), t0 = blockIdx.x % (4 / TPB) * TPB;
  const long long m0 = blockIdx.y * 16ll * MT;
  const u32x4* w = p.w + (long long)nb * p.ktiles * 256 + t0 * 64 + lane;
  const int8_t* xa[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    long long m = m0 + j * 16 + (lane & 15);      // token rows past M repeat the last one and are not stored
    if (m >= p.M) m = p.M - 1;
    xa[j] = p.xq + m * p.qrs + (lane >> 4) * 16;
  }
  i32x4 acc[TPB][MT];
#pragma unroll
  for (int t = 0; t < TPB; ++t)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[t][j] = i32x4{0, 0, 0, 0};
  thin_product<MT, TPB>(w, (int)((long long)p.ktiles * wave / I8_KW), (int)((long long)p.ktiles * (wave + 1) / I8_KW), acc,
                        [&](int kt, int j) { return *reinterpret_cast<const i32x4*>(xa[j] + (long long)kt * 64); });
  thin_finish<TO, MT, TPB>(p, red, acc, nb, t0, m0, p.M, [&](long long m) { return p.xs[m]; });
}

// Small calls on float tokens: a block takes up to 16 tokens (2048 vectors of 8 in all) and 16 channels and makes the tokens' codes itself, into LDS --
// they come out of L2, and a launch and a round trip of the codes are saved.  Replayed / called (us): 45 x 512 -> 1536 5.7 / 9 against 6.5 / 14.4 with
// two launches, 200 x 512 -> 512 6.6 / 9 against 7.4 / 14.6; with more blocks every one of them quantises too much: 400 x 512 -> 512 (800 blocks)
// 9.3 against 7.6 replayed.  One token is taken here up to K = 16384 (1 x 4096 -> 4096: 6.6 us kernel time, 11 a call).
constexpr int I8_FUSE_VEC = 4;                     // vectors a thread
constexpr int64_t I8_FUSE_BLOCKS = 512;            // two a CU
inline int i8_fused_rows(int64_t M, int N, int K) {  // tokens a block (0: two launches)
  int rows = 512 * I8_FUSE_VEC / ((K + 63) / 64 * 8);
  if (rows > 16) rows = 16;
  if (rows > M) rows = (int)M;
  return rows > 0 && (M == 1 || (M + rows - 1) / rows * ((N + 63) / 64 * 4) <= I8_FUSE_BLOCKS) ? rows : 0;
}
template <typename T, typename TO>
__global__ __launch_bounds__(512) void lin_i8_token_kernel(const LinI8Params p, const FloatTokens<T> x, const int rows) {
  __shared__ __attribute__((aligned(16))) i32x4 red[I8_KW * 64];
  __shared__ __attribute__((aligned(16))) int8_t codes[512 * I8_FUSE_VEC * 8 + 16 * 16];       // rows of K padded to 64, 16 bytes apart
  __shared__ unsigned rmax[16];
  __shared__ float xs[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int nb = blockIdx.x >> 2, t0 = blockIdx.x & 3;
  const long long m0 = (long long)blockIdx.y * rows;
  const int M = (int)min((long long)rows, p.M - m0), Kp = p.ktiles * 64, vr = Kp >> 3, ld = Kp + 16;
  if (threadIdx.x < 16) rmax[threadIdx.x] = 0;
  __syncthreads();
  Raw8<T> raw[I8_FUSE_VEC];
  int row[I8_FUSE_VEC];
#pragma unroll
  for (int v = 0; v < I8_FUSE_VEC; ++v) {
    const int i = v * 512 + threadIdx.x, r = i / vr, c = (i - r * vr) * 8;
    row[v] = r < M ? r : -1;
    raw[v].clear();
    if (row[v] >= 0 && c < x.K) {
      const T* xr = x.x + (m0 + r) * x.xrs + c;
      if (c + 8 <= x.K) {
        raw[v].load_any(xr);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c + k < x.K) raw[v].set(k, xr[k]);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < I8_FUSE_VEC; ++v) {
    unsigned m = raw[v].amax();                    // 8 neighbouring lanes hold one row: vr is a multiple of 8
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o));
    if ((lane & 7) == 0 && row[v] >= 0) atomicMax(&rmax[row[v]], m);      // (a maximum: the order does not matter)
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < I8_FUSE_VEC; ++v) {
    if (row[v] < 0) continue;
    const int c = (v * 512 + threadIdx.x - row[v] * vr) * 8;
    const RowScale r = row_scale(rmax[row[v]]);
    if (c == 0) xs[row[v]] = r.scale;
    float f[8];
    raw[v].values(f);
    *reinterpret_cast<u32x2*>(codes + row[v] * ld + c) = codes8_fast(f, r, !r.zero && r.lift == 1.f ? 0.5f * r.s : -1.f);
  }
  __syncthreads();
  i32x4 acc[1][1] = {{i32x4{0, 0, 0, 0}}};
  const u32x4* w = p.w + (long long)nb * p.ktiles * 256 + t0 * 64 + lane;
  const int8_t* xa = codes + ((lane & 15) < M ? lane & 15 : 0) * ld + (lane >> 4) * 16;        // (columns past M repeat row 0 and are not stored)
  thin_product<1, 1>(w, (int)((long long)p.ktiles * wave / I8_KW), (int)((long long)p.ktiles * (wave + 1) / I8_KW), acc,
                     [&](int kt, int) { return *reinterpret_cast<const i32x4*>(xa + kt * 64); });
  thin_finish<TO, 1, 1>(p, red, acc, nb, t0, m0, m0 + M, [&](long long m) { return xs[m - m0]; });
}

// Tiles of BM tokens x BN channels, WM x WN waves of BM / WM tokens x BN / WN channels.  Both operands go from memory into LDS without
// passing registers (16 bytes a lane, one kilobyte an instruction), S stages of 64 k deep: the weights' kilobytes are in operand order
// already, the lanes of a token piece gather 16 rows x 4 pieces so that it lands in operand order too -- fragment reads are then
// lane-linear and free of bank conflicts without any swizzle.  Token rows past M repeat the last one, channel blocks past N the last one.
// Bound by the matrix cores: 8192^3 488-494 us = 2.2 POP/s on a card that has been busy, 576 in the first calls on an idle one (the vendor library's
// product beside it 438-446; all fragment reads of a stage ahead of its products; in the compiler's order 597).  LDS is not what holds it: 4 waves of
// 128 x 128 with the next stage's operands read during this one's products, half the LDS bytes a product and no wait among them, took 511
// against 496, and weights from the cache straight into registers 665.
typedef __attribute__((address_space(3))) void* i8_lptr;
typedef __attribute__((address_space(1))) void* i8_gptr;

template <typename TO, int BM, int BN, int WM, int WN, int S, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void lin_i8_tile_kernel(const LinI8Params p, const int tm, const int tn) {
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
  float xs[TA];      // all scales ahead of the first store: a load between stores would wait for them (one in-order counter)
#pragma unroll
  for (int a = 0; a < TA; ++a) xs[a] = p.xs[min(m0 + (wm * TA + a) * 16 + (lane & 15), p.M - 1)];
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    Lane8<TO> ch[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) ch[h].load(p, n0 + (wn * TB + b) * 64 + h * 32 + (lane >> 4) * 8);
#pragma unroll
    for (int a = 0; a < TA; ++a) {
      const long long m = m0 + (wm * TA + a) * 16 + (lane & 15);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
        ch[h].value(p, xs[a], &acc[a][b * 4 + h * 2], v);
        if (m < p.M) ch[h].store(p, m, v);
      }
    }
  }
#endif
}

// Short K, many tokens: the output's bytes are the work.  A block of 4 waves keeps the weights of 256 channels in registers (64 a wave, KT operand
// tiles deep) for the whole launch and streams token tiles of 64 through two LDS stages.  The `panels` blocks that read the same tokens
// run next to each other on one XCD (block id mod 8).  Bound by the stores: 110160 x 512 -> 1536 in fp16 119 us (112 at best) for 338 MB of output
// and 56 MB of codes (3.3 TB/s).  With the quantiser, 137: stores past the cache 149 against 147 then, outputs held back a tile 148 against 133 then.
template <typename TO, int KT>
__global__ __launch_bounds__(256, 2) void lin_i8_stream_kernel(const LinI8Params p, const int panels, const int groups, const int tiles) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ __attribute__((aligned(1024))) char lds[2 * 4 * KT * 1024];
  __shared__ float xs[2][64];                      // scales of the tile's tokens
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);      // (scalar branches on it)
  const int panel = (int)(blockIdx.x >> 3) % panels, grp = (int)(blockIdx.x >> 3) / panels * 8 + (int)(blockIdx.x & 7);
  const int nb = panel * 4 + wave, last = (p.N + 63) / 64 - 1;
  i32x4 wf[KT][4];
  {
    const u32x4* w = p.w + (long long)(nb < last ? nb : last) * p.ktiles * 256 + lane;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int t = 0; t < 4; ++t) wf[kt][t] = kt < p.ktiles ? __builtin_bit_cast(i32x4, w[kt * 256 + t * 64]) : i32x4{0, 0, 0, 0};
  }
  Lane8<TO> ch[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) ch[h].load(p, nb * 64 + h * 32 + (lane >> 4) * 8);
  auto issue = [&](int tile, int buf) {
    long long m = tile * 64ll + wave * 16 + (lane & 15);
    if (m >= p.M) m = p.M - 1;
    const int8_t* src = p.xq + m * p.qrs + (lane >> 4) * 16;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
      if (kt < p.ktiles) __builtin_amdgcn_global_load_lds((i8_gptr)(src + kt * 64), (i8_lptr)(lds + ((buf * 4 + wave) * KT + kt) * 1024), 16, 0, 0);
    if (wave == 0) __builtin_amdgcn_global_load_lds((i8_gptr)(p.xs + min(tile * 64ll + lane, p.M - 1)), (i8_lptr)xs[buf], 4, 0, 0);
  };
  bool full = false;                               // the tile before left 8 or more stores behind this tile's loads
  int buf = 0;
  if (grp < tiles) issue(grp, 0);
  for (int tile = grp; tile < tiles; tile += groups) {
    // the tile's loads are older than the stores of the tile before: where those are at least 8 (whole tiles of whole blocks: one each for 4 x 16
    // tokens and 2 x 8 channels, two in fp32) the stores stay in flight
    if (full) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();                  // tile is there for all waves; the other stage, read one tile ago, is free
    if (tile + groups < tiles) issue(tile + groups, buf ^ 1);
    full = nb * 64 + 64 <= p.N && tile * 64ll + 64 <= p.M;
    const char* st = lds + buf * 4 * KT * 1024 + lane * 16;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      i32x4 acc[4], xf[KT];
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[t] = i32x4{0, 0, 0, 0};
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) xf[kt] = *reinterpret_cast<const i32x4*>(st + (mt * KT + kt) * 1024);      // (past the last k tile: anything, times weights of 0)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[kt][t], xf[kt], acc[t], 0, 0, 0);
      const long long m = tile * 64ll + mt * 16 + (lane & 15);
      const float xm = xs[buf][mt * 16 + (lane & 15)];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
        ch[h].value(p, xm, &acc[h * 2], v);
        if (full) store8_any<TO>(reinterpret_cast<TO*>(p.out) + m * p.ors + ch[h].c, v);
        else if (m < p.M) ch[h].store(p, m, v);
      }
    }
    buf ^= 1;
  }
#endif
}
template <typename TO, int KT>
static void launch_stream(const LinI8Params& p, hipStream_t st) {
  const int panels = (p.N + 255) / 256, tiles = (int)((p.M + 63) / 64);
  int per = 64 / panels;                           // token groups an XCD works on at a time: 64 blocks, two a CU
  if (per < 1) per = 1;
  hipLaunchKernelGGL((lin_i8_stream_kernel<TO, KT>), dim3((unsigned)(8 * panels * per)), dim3(256), 0, st, p, panels, 8 * per, tiles);
}

template <typename TO, int BM, int BN, int WM, int WN, int S, int OCC>
static void launch_tiles(const LinI8Params& p, hipStream_t st) {
  const int tm = (int)((p.M + BM - 1) / BM), tn = (p.N + BN - 1) / BN;
  hipLaunchKernelGGL((lin_i8_tile_kernel<TO, BM, BN, WM, WN, S, OCC>), dim3((unsigned)((long long)tm * tn)), dim3(64 * WM * WN), 0, st, p, tm, tn);
}
template <typename TO, int MT, int TPB>
static void launch_thin(const LinI8Params& p, hipStream_t st) {
  hipLaunchKernelGGL((lin_i8_thin_kernel<TO, MT, TPB>), dim3((unsigned)((p.N + 63) / 64 * (4 / TPB)), (unsigned)((p.M + 16 * MT - 1) / (16 * MT))), dim3(512), 0, st, p);
}
// Which form: measured at K = N = 4096 unless said otherwise (us).
//   thin, few 128 x 128 tiles (at most 64: they would leave most CUs idle) or few tokens: 16 tokens x 1024 -> 16384 6.0 against 8.5 with tiles,
//   64 tokens 10.5 against 22.7, 256 tokens 15.5 against 23.3, 512 tokens 28.7 against 23.8; 1084 x 7352 -> 760 25.4 against 30.0 with 64 x 128
//   64 x 128 tiles, at most 128 of 128 x 128 (one a CU): 512 tokens 20.5 against 26.3, 1500 x 1024 -> 1024 8.4 against 10.9, 2935 x 4207 -> 988
//   (184 tiles) 29.6 against 28.8
//   stream, K <= 512 and enough token tiles for every resident block: 110160 x 512 -> 1536 134 against 166, 10000 tokens 16.4 against 17.3,
//   5000 x 512 -> 512 7.9 against 6.8
//   256 x 256 tiles where K is long and they fill the chip twice: 8192^3 487 against 505 with 128 x 256; 4096^3 65 either way
//   128 x 256 tiles where they fill the chip: 4096^3 66 against 84 with 128 x 128; 2048^3 20.5 against 15.4
template <typename TO>
static void launch_product(const LinI8Params& p, hipStream_t st) {
  const long long t128 = ((p.M + 127) / 128) * ((p.N + 127) / 128), t256w = ((p.M + 127) / 128) * ((p.N + 255) / 256), t256 = ((p.M + 255) / 256) * ((p.N + 255) / 256);
  if (t128 <= 64 || p.M <= 32) {
    if (p.M <= 16) launch_thin<TO, 1, 1>(p, st);
    else if (p.M <= 32) launch_thin<TO, 1, 2>(p, st);
    else if (p.M <= 64) launch_thin<TO, 1, 4>(p, st);
    else launch_thin<TO, 2, 4>(p, st);
  } else if (p.ktiles <= 8 && (p.M + 63) / 64 * ((p.N + 255) / 256) >= 768) {
    if (p.ktiles <= 4) launch_stream<TO, 4>(p, st);
    else launch_stream<TO, 8>(p, st);
  } else if (p.ktiles >= 96 && t256 >= 512) {
    launch_tiles<TO, 256, 256, 2, 4, 4, 1>(p, st);
  } else if (t128 <= 128) {
    launch_tiles<TO, 64, 128, 2, 2, 4, 3>(p, st);
  } else if (t256w >= 256) {
    launch_tiles<TO, 128, 256, 2, 4, 3, 4>(p, st);
  } else {
    launch_tiles<TO, 128, 128, 4, 2, 4, 4>(p, st);
  }
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
#define PP_QUANT_FORM(V, W, F) hipLaunchKernelGGL((quant_kernel<T, V, W, F>), grid, block, 0, st, (const T*)x, (long long)xrs, (int8_t*)q, (long long)qrs, scale, (long long)rows, K, Kp)
#define PP_QUANT(V, W) do { if (wide && K % 8 == 0) PP_QUANT_FORM(V, W, true); else PP_QUANT_FORM(V, W, false); } while (0)
  if (K <= 512) PP_QUANT(1, 1);
  else if (K <= 1024) PP_QUANT(2, 1);
  else if (K <= 2048) PP_QUANT(4, 1);
  else if (K <= 4096) PP_QUANT(2, 4);
  else if (K <= 8192) PP_QUANT(4, 4);
  else if (K <= 16384) PP_QUANT(8, 4);
  else hipLaunchKernelGGL((quant_row_kernel<T>), grid, block, 0, st, (const T*)x, (long long)xrs, (int8_t*)q, (long long)qrs, scale, (long long)rows, K, Kp);
#undef PP_QUANT
#undef PP_QUANT_FORM
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

static int lin_i8_check(const char* who, const void* weight, const float* ws, const void* out, int64_t out_rstride, int64_t M, int N, int K, int act, int out_dtype) {
  PP_REQUIRE(pp_i8_row_bytes(K) > 0 && N > 0 && N <= PP_I8_MAX_N && M >= 0 && M <= PP_I8_MAX_M, PP_ERR_ARG, "%s: bad arguments (M=%lld N=%d K=%d)", who, (long long)M, N, K);
  PP_REQUIRE(act >= PP_ACT_NONE && act <= PP_ACT_SILU, PP_ERR_ARG, "%s: activation code %d", who, act);
  PP_REQUIRE(out_dtype == PP_F32 || out_dtype == PP_F16, PP_ERR_DTYPE, "%s: out_dtype %d", who, out_dtype);
  if (M == 0) return 0;
  PP_REQUIRE(weight && ws && out && out_rstride >= N, PP_ERR_ARG, "%s: null buffer or row stride (out %lld < %d)", who, (long long)out_rstride, N);
  PP_REQUIRE((uintptr_t)weight % 16 == 0 && (uintptr_t)out % (out_dtype == PP_F16 ? 2 : 4) == 0, PP_ERR_ALIGN, "%s: the weight must be 16-byte aligned", who);
  PP_REQUIRE(((M + 127) / 128) * ((N + 127) / 128) < (1 << 23), PP_ERR_ARG, "%s: too many tiles (M=%lld N=%d)", who, (long long)M, N);
  return 0;
}
static LinI8Params lin_i8_params(const void* xq, int64_t q_rstride, const float* xs, const void* weight, const float* ws, const float* bias, void* out, int64_t out_rstride,
                                 int64_t M, int N, int K, int act, float act_param) {
  LinI8Params p;
  p.xq = (const int8_t*)xq; p.xs = xs; p.w = (const u32x4*)weight; p.ws = ws; p.bias = bias; p.out = (char*)out;
  p.qrs = q_rstride; p.ors = out_rstride; p.M = M; p.N = N; p.ktiles = pp_i8_row_bytes(K) / 64; p.act = act; p.act_param = act_param;
  return p;
}

extern "C" int pp_linear_i8(const void* xq, int64_t q_rstride, const float* xs, const void* weight, const float* ws, const float* bias, void* out,
                            int64_t out_rstride, int64_t M, int N, int K, int act, float act_param, int out_dtype, void* stream) {
  const int rc = lin_i8_check("pp_linear_i8", weight, ws, out, out_rstride, M, N, K, act, out_dtype);
  if (rc != 0 || M == 0) return rc;
  const int Kp = pp_i8_row_bytes(K);
  PP_REQUIRE(xq && xs && q_rstride >= Kp, PP_ERR_ARG, "pp_linear_i8: null codes or row stride (%lld < %d)", (long long)q_rstride, Kp);
  PP_REQUIRE((uintptr_t)xq % 16 == 0 && q_rstride % 16 == 0, PP_ERR_ALIGN, "pp_linear_i8: codes and their row stride must be multiples of 16 bytes");
  const LinI8Params p = lin_i8_params(xq, q_rstride, xs, weight, ws, bias, out, out_rstride, M, N, K, act, act_param);
  if (out_dtype == PP_F16) launch_product<_Float16>(p, (hipStream_t)stream);
  else launch_product<float>(p, (hipStream_t)stream);
  return launch_status("pp_linear_i8");
}

extern "C" int64_t pp_linear_i8_tokens_workspace_bytes(int64_t M, int N, int K) {
  const int Kp = pp_i8_row_bytes(K);
  if (Kp <= 0 || N <= 0 || N > PP_I8_MAX_N || M < 0 || M > PP_I8_MAX_M) return PP_ERR_ARG;
  return M == 0 || i8_fused_rows(M, N, K) ? 0 : M * Kp + M * 4;
}

extern "C" int pp_linear_i8_tokens(const void* x, int64_t x_rstride, int x_dtype, const void* weight, const float* ws, const float* bias, void* out,
                                   int64_t out_rstride, int64_t M, int N, int K, int act, float act_param, int out_dtype, void* work,
                                   int64_t work_bytes, void* stream) {
  int rc = lin_i8_check("pp_linear_i8_tokens", weight, ws, out, out_rstride, M, N, K, act, out_dtype);
  if (rc != 0) return rc;
  PP_REQUIRE(x_dtype == PP_F32 || x_dtype == PP_F16, PP_ERR_DTYPE, "pp_linear_i8_tokens: dtype %d", x_dtype);
  if (M == 0) return 0;
  const int esz = x_dtype == PP_F16 ? 2 : 4, Kp = pp_i8_row_bytes(K);
  PP_REQUIRE(x && x_rstride >= 0, PP_ERR_ARG, "pp_linear_i8_tokens: null tokens or row stride %lld", (long long)x_rstride);
  PP_REQUIRE((uintptr_t)x % esz == 0, PP_ERR_ALIGN, "pp_linear_i8_tokens: misaligned tokens");
  const int64_t need = pp_linear_i8_tokens_workspace_bytes(M, N, K);
  PP_REQUIRE(need == 0 || (work != nullptr && work_bytes >= need && (uintptr_t)work % 16 == 0), PP_ERR_WORKSPACE,
             "pp_linear_i8_tokens: needs %lld bytes of 16-byte aligned scratch, got %lld", (long long)need, (long long)work_bytes);
  int8_t* q = (int8_t*)work;
  float* xs = (float*)(q + M * Kp);
  if (need != 0) {
    if ((rc = pp_quantize_tokens(x, x_rstride, q, Kp, xs, M, K, x_dtype, stream)) != 0) return rc;
    return pp_linear_i8(q, Kp, xs, weight, ws, bias, out, out_rstride, M, N, K, act, act_param, out_dtype, stream);
  }
  const LinI8Params p = lin_i8_params(nullptr, 0, nullptr, weight, ws, bias, out, out_rstride, M, N, K, act, act_param);
  const int rows = i8_fused_rows(M, N, K);
  const dim3 grid((unsigned)((N + 63) / 64 * 4), (unsigned)((M + rows - 1) / rows)), block(512);
#define PP_TOKEN(T, TO) \
  hipLaunchKernelGGL((lin_i8_token_kernel<T, TO>), grid, block, 0, (hipStream_t)stream, p, FloatTokens<T>{(const T*)x, (long long)x_rstride, K}, rows)
  if (x_dtype == PP_F16) { if (out_dtype == PP_F16) PP_TOKEN(_Float16, _Float16); else PP_TOKEN(_Float16, float); }
  else { if (out_dtype == PP_F16) PP_TOKEN(float, _Float16); else PP_TOKEN(float, float); }
#undef PP_TOKEN
  return launch_status("pp_linear_i8_tokens");
}
