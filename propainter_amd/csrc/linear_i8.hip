// Linear layers on 8-bit codes: dynamic quantisation of token rows and the product with per-token and per-channel scales
// (the projections and the feed-forward layers of model/modules/sparse_transformer.py:68-69,123-130 served in 8 bits).
//
//   scale[r] = max_k |x[r,k]| / 127,  q[r,k] = round-half-even(x[r,k] / scale[r])
//   out[m,n] = act(sum_k xq[m,k] wq[n,k] * xs[m] * ws[n] + bias[n])        sum exact in int32 (K <= 131072: K * 127^2 < 2^31)
//
// MFMA operand order.  v_mfma_i32_16x16x64_i8: lane l hands in 16 bytes = row l & 15, k = (l >> 4) * 16 .. + 15 of either operand and
// receives column l & 15, rows (l >> 4) * 4 + r of the product.  The weights are the row operand: a lane then holds neighbouring output
// channels of ONE token.  They are laid out once in 4 KB blocks of 64 channels x 64 k, four operand tiles of 1 KB each in lane order; row
// i of tile t is channel (i / 4) * 16 + t * 4 + i % 4 of the block, so that the 4 tiles give every lane 16 CONSECUTIVE channels (16-byte
// stores) and a wave reads a tile as one contiguous kilobyte.
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
    const long long n = nb * 64 + (row >> 2) * 16 + t * 4 + (row & 3);
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

// 16 consecutive channels n0 .. n0 + 15 of token m: scale, bias, activation, store
template <typename TO>
__device__ __forceinline__ void store_channels(const LinI8Params& p, long long m, int n0, const i32x4* acc) {
  if (m >= p.M || n0 >= p.N) return;
  const float xs = p.xs[m];
  TO* o = reinterpret_cast<TO*>(p.out) + m * p.ors + n0;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int n = min(n0 + i, p.N - 1);
    v[i] = (float)acc[i >> 2][i & 3] * xs * p.ws[n];
    if (p.bias != nullptr) v[i] += p.bias[n];
    v[i] = act_value(v[i], p.act, p.act_param);
  }
  if (p.wide_out && n0 + 16 <= p.N) {
    store8<TO>(o, v);
    store8<TO>(o + 8, v + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (n0 + i < p.N) o[i] = from_f32<TO>(v[i]);
  }
}

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
#pragma unroll
  for (int j = 0; j < 2; ++j) store_channels<TO>(p, m0 + j * 16 + (lane & 15), nb * 64 + (lane >> 4) * 16, acc[j]);
#endif
}

}  // namespace pp

using namespace pp;

constexpr int PP_I8_MAX_N = 65535 * 64;            // grid.y
constexpr int64_t PP_I8_MAX_M = (int64_t)1 << 30;  // grid.x * 256 threads below 2^32

extern "C" int pp_i8_row_bytes(int K) {
  if (K <= 0 || K > 131072) return PP_ERR_ARG;
  return (K + 63) / 64 * 64;
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
  hipStream_t st = (hipStream_t)stream;
  if (dtype == PP_F16)
    hipLaunchKernelGGL((quant_row_kernel<_Float16>), dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(256), 0, st, (const _Float16*)x, (long long)x_rstride, (int8_t*)q,
                       (long long)q_rstride, scale, (long long)rows, K, Kp, wide);
  else
    hipLaunchKernelGGL((quant_row_kernel<float>), dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(256), 0, st, (const float*)x, (long long)x_rstride, (int8_t*)q,
                       (long long)q_rstride, scale, (long long)rows, K, Kp, wide);
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
  const dim3 grid((unsigned)((M + 127) / 128), (N + 63) / 64);
  if (out_dtype == PP_F16) hipLaunchKernelGGL((lin_i8_kernel<_Float16>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((lin_i8_kernel<float>), grid, dim3(256), 0, st, p);
  return launch_status("pp_linear_i8");
}
