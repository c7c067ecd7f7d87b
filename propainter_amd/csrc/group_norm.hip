// Group norm with an activation over a channels-last map (the norm_fn == 'group' layers of RAFT/extractor.py:14-18,123-124; any C % 8 == 0).
//
//   y[n,p,c] = act((x[n,p,c] - mean[n,g]) * rstd[n,g] * gamma[c] + beta[c]),   g = c / (C / groups),
//   mean and rstd = 1 / sqrt(var + eps) over the H*W pixels and the C / groups channels of a group, var the biased variance.
//
// Statistics are held in fp32 as (count, mean, sum of squared deviations) and joined pairwise (Chan et al. 1979): no difference of large
// sums of squares, so a map whose mean is far from zero loses nothing.  The order of every sum is fixed by the sizes: no atomics.
// Bound by memory: the map is read twice (the second time partly from the cache) and written once, 4x360x640x64 fp16 in 75 us (kernels 25 + 43) =
// 4.7 TB/s of those three passes.  Every output block joins all slices of all groups of its image first, which counts where groups are many and images
// few: 1x540x960x64 fp16 in 8 / 32 / 64 groups 58 / 115 / 190 us.
#include "common.h"
#include "attn_lanes.h"
#include <type_traits>

namespace pp {

struct GnParams {
  const char* in;
  char* out;
  const float* gamma;     // [C] or NULL (1)
  const float* beta;      // [C] or NULL (0)
  float* part;            // [N][slices][groups][2] (mean, M2) of a slice
  long long in_cs, out_cs;
  int in_co, out_co;
  int HW, C, groups, cg, slices, ppslice, ppblock;   // pixels of a slice (statistics), of a block (output)
  float eps, act_param;
  int act;
};

__device__ __forceinline__ void chan_merge(float& n, float& m, float& M2, float nb, float mb, float M2b) {
  if (nb == 0.f) return;
  const float nt = n + nb, d = mb - m, f = nb / nt;
  m = fmaf(d, f, m);
  M2 = M2 + M2b + d * d * (n * f);
  n = nt;
}

// Threads s0 = 0 .. per - 1 hold parts of one group (thread s0 * ng + g of group g): joined into thread g, in a fixed order.  All threads call it.
__device__ __forceinline__ void join_parts(int per, int ng, int s0, float& cnt, float& m, float& M2, float (*lds)[256]) {
  const int t = threadIdx.x;
  lds[0][t] = cnt; lds[1][t] = m; lds[2][t] = M2;
  for (int h = per; h > 1;) {
    const int half = (h + 1) >> 1;
    __syncthreads();
    if (s0 < h - half) {
      const int o = t + half * ng;
      chan_merge(cnt, m, M2, lds[0][o], lds[1][o], lds[2][o]);
      lds[0][t] = cnt; lds[1][t] = m; lds[2][t] = M2;
    }
    h = half;
  }
  __syncthreads();
}

// 256 threads: column = 8 channels, the rest of the block walks the pixels of one slice, GN_U at a time: those are in registers, so their mean and
// squared deviations are taken in two passes, and joined to what the thread has.  Values are taken relative to the slice's first pixel (per
// channel), so that means hold deviations and not magnitudes; it may itself lie far from the rest (a border of zeros): nothing is subtracted
// from sums of squares.
constexpr int GN_U = 8;        // (2, 4 and 8 pixels: 23.9 / 25.4 / 25.4 us at 4x360x640x64 fp16, 19.0 / 18.8 / 19.4 at 2x270x480x96 fp32; most merges are saved by 8)
template <typename T>
__global__ __launch_bounds__(256) void gn_stats_kernel(const GnParams p) {
  __shared__ float s1[256 * 8], s2[256 * 8], parts[3][256];
  const int c8 = p.C >> 3, rows = 256 / c8;
  const int t = threadIdx.x, col = t % c8, pr = t / c8;
  const int slice = blockIdx.x, n = blockIdx.y;
  const int p0 = slice * p.ppslice;
  const int np = min(p.ppslice, p.HW - p0);
  const int last = pr < rows ? np : 0;               // threads past the last whole row of columns have no pixels
  const T* x = reinterpret_cast<const T*>(p.in) + ((long long)n * p.HW + p0) * p.in_cs + p.in_co + col * 8;
  float shift[8], m[8], M2[8], cnt = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i] = M2[i] = 0.f;
  if (last > 0) load8<T>(x, shift);
  // pixels q, q + rows, ..: all GN_U of them, or (FULL false) those below last
  auto batch = [&](int q, auto full) {
    constexpr bool FULL = decltype(full)::value;
    float v[GN_U][8];
    const float nb = FULL ? (float)GN_U : (float)((last - q + rows - 1) / rows);
#pragma unroll
    for (int u = 0; u < GN_U; ++u)
      if (FULL || q + u * rows < last) load8<T>(x + (long long)(q + u * rows) * p.in_cs, v[u]);
    const float nt = cnt + nb, f = nb / nt, w = cnt * f, rb = 1.f / nb;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float sum = 0.f, dev = 0.f;
#pragma unroll
      for (int u = 0; u < GN_U; ++u)
        if (FULL || q + u * rows < last) {
          v[u][i] -= shift[i];
          sum += v[u][i];
        }
      const float mb = sum * rb;
#pragma unroll
      for (int u = 0; u < GN_U; ++u)
        if (FULL || q + u * rows < last) {
          const float d = v[u][i] - mb;
          dev = fmaf(d, d, dev);
        }
      const float d = mb - m[i];
      m[i] = fmaf(d, f, m[i]);
      M2[i] = M2[i] + dev + d * w * d;
    }
    cnt = nt;
  };
  int q = pr;
  for (; q + (GN_U - 1) * rows < last; q += GN_U * rows) batch(q, std::true_type{});
  if (q < last) batch(q, std::false_type{});
  parts[0][t] = cnt;
#pragma unroll
  for (int i = 0; i < 8; ++i) { s1[t * 8 + i] = m[i]; s2[t * 8 + i] = M2[i]; }
  for (int h = rows; h > 1;) {                       // rows of the block, halved
    const int half = (h + 1) >> 1;
    __syncthreads();
    if (pr < h - half) {
      const int o = t + half * c8;
      const float nb = parts[0][o];
      if (nb > 0.f) {                                // (a row without pixels lies behind those with pixels)
        const float nt = cnt + nb, f = nb / nt, w = cnt * f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = s1[o * 8 + i] - m[i];
          m[i] = fmaf(d, f, m[i]);
          M2[i] = M2[i] + s2[o * 8 + i] + d * w * d;
          s1[t * 8 + i] = m[i];
          s2[t * 8 + i] = M2[i];
        }
        cnt = nt;
        parts[0][t] = nt;
      }
    }
    h = half;
  }
  __syncthreads();
  // per channel (mean, M2), then the channels of each group
  const T* x0 = reinterpret_cast<const T*>(p.in) + ((long long)n * p.HW + p0) * p.in_cs + p.in_co;
  for (int c = t; c < p.C; c += 256) s1[c] += to_f32(x0[c]);
  __syncthreads();
  const int per = p.groups < 256 ? 256 / p.groups : 1;   // threads that share one group's channels
  for (int g0 = 0; g0 < p.groups; g0 += 256) {
    const int ng = min(256, p.groups - g0), g = g0 + t % ng, s0 = t / ng;
    float gn = 0.f, gm = 0.f, gM2 = 0.f;
    if (s0 < per)
      for (int c = s0; c < p.cg; c += per) chan_merge(gn, gm, gM2, (float)np, s1[g * p.cg + c], s2[g * p.cg + c]);
    join_parts(per, ng, s0, gn, gm, gM2, parts);
    if (s0 == 0) {
      float* o = p.part + (((long long)n * p.slices + slice) * p.groups + g) * 2;
      o[0] = gm;
      o[1] = gM2;
    }
  }
}

// 8 values past the cache: an output that does not fit next to the input would push out what the second read wants
template <typename T> __device__ __forceinline__ void stream8(T* p, const float* v) {
  if constexpr (sizeof(T) == 2) {
    u32x4 raw;
    _Float16* h = reinterpret_cast<_Float16*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)v[i];
    __builtin_nontemporal_store(raw, reinterpret_cast<u32x4*>(p));
  } else {
    __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4*>(p));
    __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, reinterpret_cast<f32x4*>(p + 4));
  }
}

// STREAM: a template, as the two stores of a run-time choice would be merged into an ordinary one
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void gn_apply_kernel(const GnParams p) {
  __shared__ float gm[2048], gr[2048];                 // mean and rstd of every group (groups <= C <= 2048)
  __shared__ float parts[3][256];
  const int t = threadIdx.x, n = blockIdx.y;
  const float* part = p.part + (long long)n * p.slices * p.groups * 2;
  const int per = p.groups < 256 ? 256 / p.groups : 1;  // threads that share one group's slices
  for (int g0 = 0; g0 < p.groups; g0 += 256) {
    const int ng = min(256, p.groups - g0);
    const int g = t % ng, s0 = t / ng;
    float cnt = 0.f, m = 0.f, M2 = 0.f;
    if (s0 < per)
      for (int s = s0; s < p.slices; s += per) {
        const int np = min(p.ppslice, p.HW - s * p.ppslice);
        const float* e = part + ((long long)s * p.groups + g0 + g) * 2;
        chan_merge(cnt, m, M2, (float)np * (float)p.cg, e[0], e[1]);
      }
    join_parts(per, ng, s0, cnt, m, M2, parts);
    if (s0 == 0) {
      gm[g0 + g] = m;
      gr[g0 + g] = 1.f / sqrtf(M2 / cnt + p.eps);
    }
    __syncthreads();
  }
  const int c8 = p.C >> 3, rows = 256 / c8, col = t % c8, pr = t / c8;
  if (pr >= rows) return;
  float mean[8], mul[8], add[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = col * 8 + i, g = c / p.cg;
    mean[i] = gm[g];
    mul[i] = gr[g] * (p.gamma != nullptr ? p.gamma[c] : 1.f);
    add[i] = p.beta != nullptr ? p.beta[c] : 0.f;
  }
  const T* x = reinterpret_cast<const T*>(p.in) + (long long)n * p.HW * p.in_cs + p.in_co + col * 8;
  T* y = reinterpret_cast<T*>(p.out) + (long long)n * p.HW * p.out_cs + p.out_co + col * 8;
  const long long q0 = (long long)blockIdx.x * p.ppblock, q1 = min(q0 + p.ppblock, (long long)p.HW);
  constexpr int U = 2;                                  // loads in flight a thread (at 4x360x640x64 fp16 / 2x270x480x96 fp32: 1 or 2 are the same within noise, 77.5 / 66.6 and 78.5 / 66.0 us in one run; 4: 86.4 / 69.9)
  for (long long q = q0 + pr; q < q1; q += U * rows) {
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (q + u * rows < q1) load8<T>(x + (q + u * rows) * p.in_cs, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (q + u * rows < q1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = fmaf(v[u][i] - mean[i], mul[i], add[i]);
        act_values<8>(v[u], p.act, p.act_param);
        if constexpr (STREAM) stream8<T>(y + (q + u * rows) * p.out_cs, v[u]);
        else store8<T>(y + (q + u * rows) * p.out_cs, v[u]);
      }
  }
}

// Sum over the block, the same value in every thread; two barriers.
template <int BLOCK>
__device__ __forceinline__ float block_sum(float v, float* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x128, 0xf, 0xf, false));      // rotations inside 16 lanes: 8, 4, 2, 1
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x124, 0xf, 0xf, false));
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x122, 0xf, 0xf, false));
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x121, 0xf, 0xf, false));
  v = rows_sum(v);
#endif
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int w = 0; w < BLOCK / 64; ++w) v += lds[w];
  __syncthreads();
  return v;
}

// A group that fits a block's registers (channels of a group a multiple of 8): one launch, one read; the variance is a second pass over registers.
// A thread keeps one column of 8 channels and walks the pixels.
constexpr int GN_VEC = 8;         // vectors of 8 a thread
template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void gn_group_kernel(const GnParams p) {
  __shared__ float red[2][BLOCK / 64];
  const int g = blockIdx.x, n = blockIdx.y, vpp = p.cg >> 3, rows = BLOCK / vpp;
  const int pr = (int)threadIdx.x / vpp, c = ((int)threadIdx.x - pr * vpp) * 8;
  const int last = pr < rows ? p.HW : 0;            // threads past the last whole row of columns have no pixels
  const T* x = reinterpret_cast<const T*>(p.in) + (long long)n * p.HW * p.in_cs + p.in_co + g * p.cg + c;
  T* y = reinterpret_cast<T*>(p.out) + (long long)n * p.HW * p.out_cs + p.out_co + g * p.cg + c;
  float v[GN_VEC][8], gm[8], bt[8];
#pragma unroll
  for (int k = 0; k < GN_VEC; ++k)
    if (pr + k * rows < last) load8<T>(x + (pr + k * rows) * p.in_cs, v[k]);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    gm[j] = p.gamma != nullptr ? p.gamma[g * p.cg + c + j] : 1.f;
    bt[j] = p.beta != nullptr ? p.beta[g * p.cg + c + j] : 0.f;
  }
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < GN_VEC; ++k)
    if (pr + k * rows < last) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[k][j];
    }
  const float count = (float)p.HW * (float)p.cg;
  const float mean = block_sum<BLOCK>(sum, red[0]) / count;
  float dev = 0.f;
#pragma unroll
  for (int k = 0; k < GN_VEC; ++k)
    if (pr + k * rows < last) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[k][j] -= mean;
        dev = fmaf(v[k][j], v[k][j], dev);
      }
    }
  const float rstd = 1.f / sqrtf(block_sum<BLOCK>(dev, red[1]) / count + p.eps);
#pragma unroll
  for (int j = 0; j < 8; ++j) gm[j] *= rstd;
#pragma unroll
  for (int k = 0; k < GN_VEC; ++k)
    if (pr + k * rows < last) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = fmaf(v[k][j], gm[j], bt[j]);
      act_values<8>(v[k], p.act, p.act_param);
      store8<T>(y + (pr + k * rows) * p.out_cs, v[k]);
    }
}

}  // namespace pp

using namespace pp;

// A group in one block's registers where it fits: 30 x 54 x 128 in 8 groups 6.5 us in one launch, 11.7 in two.
static int gn_group_block(int64_t HW, int C, int groups) {      // threads, 0: it does not fit
  const int cg = C / groups;
  if (cg % 8 != 0) return 0;
  for (int block = 256; block <= 1024; block *= 2)
    if (cg / 8 <= block && HW <= (int64_t)GN_VEC * (block / (cg / 8))) return block;
  return 0;
}

static void gn_split(int N, int HW, int C, int* slices, int* ppslice) {
  // enough blocks to fill the chip, but no slice under 4 pixels a thread (the joins would cost more than the pixels)
  const int rows = 256 / (C / 8) > 0 ? 256 / (C / 8) : 1;
  int want = 1024 / N;
  if (want < 1) want = 1;
  int64_t pp = ((int64_t)HW + want - 1) / want;
  if (pp < 4 * rows) pp = 4 * rows;
  *ppslice = (int)(pp < HW ? pp : HW);
  *slices = ceil_div(HW, *ppslice);
}

extern "C" int64_t pp_group_norm_workspace_floats(int N, int H, int W, int C, int groups) {
  if (N <= 0 || H <= 0 || W <= 0 || C <= 0 || C % 8 != 0 || C > 2048 || groups <= 0 || C % groups != 0 || (int64_t)H * W > 0x7fffffff) return PP_ERR_ARG;
  if (gn_group_block((int64_t)H * W, C, groups)) return 0;
  int slices, pps;
  gn_split(N, H * W, C, &slices, &pps);
  return (int64_t)N * slices * groups * 2;
}

extern "C" int pp_group_norm(const void* in, int in_cstride, int in_choff, void* out, int out_cstride, int out_choff, const float* gamma,
                             const float* beta, float* stats_ws, int N, int H, int W, int C, int groups, float eps, int act, float act_param,
                             int dtype, void* stream) {
  PP_REQUIRE(in && out && N > 0 && N <= 65535 && H > 0 && W > 0 && (int64_t)H * W <= 0x7fffffff, PP_ERR_ARG,
             "pp_group_norm: bad arguments (N=%d H=%d W=%d)", N, H, W);
  PP_REQUIRE(C > 0 && C % 8 == 0 && C <= 2048 && groups > 0 && C % groups == 0, PP_ERR_ARG,
             "pp_group_norm: C=%d must be a multiple of 8, <= 2048, and of groups=%d", C, groups);
  PP_REQUIRE(act >= PP_ACT_NONE && act <= PP_ACT_SILU, PP_ERR_ARG, "pp_group_norm: activation code %d", act);
  PP_REQUIRE(eps >= 0.f, PP_ERR_ARG, "pp_group_norm: eps must not be negative");
  PP_REQUIRE(dtype == PP_F32 || dtype == PP_F16, PP_ERR_DTYPE, "pp_group_norm: dtype %d", dtype);
  PP_REQUIRE(in_choff >= 0 && out_choff >= 0 && in_cstride >= in_choff + C && out_cstride >= out_choff + C, PP_ERR_ARG,
             "pp_group_norm: channel windows %d+%d of %d, %d+%d of %d", in_choff, C, in_cstride, out_choff, C, out_cstride);
  PP_REQUIRE((in_cstride | in_choff | out_cstride | out_choff) % 8 == 0 && (uintptr_t)in % 16 == 0 && (uintptr_t)out % 16 == 0 &&
                 (uintptr_t)stats_ws % 8 == 0,
             PP_ERR_ALIGN, "pp_group_norm: strides and channel offsets must be multiples of 8, the buffers 16-byte aligned");
  const int HW = H * W;
  const int one = gn_group_block(HW, C, groups);
  PP_REQUIRE(one || stats_ws, PP_ERR_WORKSPACE, "pp_group_norm: needs %lld floats of scratch", (long long)pp_group_norm_workspace_floats(N, H, W, C, groups));
  GnParams p;
  p.in = (const char*)in; p.out = (char*)out; p.gamma = gamma; p.beta = beta; p.part = stats_ws;
  p.in_cs = in_cstride; p.out_cs = out_cstride; p.in_co = in_choff; p.out_co = out_choff;
  p.HW = HW; p.C = C; p.groups = groups; p.cg = C / groups; p.eps = eps; p.act = act; p.act_param = act_param;
  hipStream_t st = (hipStream_t)stream;
  if (one) {
    const dim3 grid(groups, N);
#define PP_GN_GROUP(T)                                                                                \
  if (one == 256) hipLaunchKernelGGL((gn_group_kernel<T, 256>), grid, dim3(256), 0, st, p);           \
  else if (one == 512) hipLaunchKernelGGL((gn_group_kernel<T, 512>), grid, dim3(512), 0, st, p);      \
  else hipLaunchKernelGGL((gn_group_kernel<T, 1024>), grid, dim3(1024), 0, st, p)
    if (dtype == PP_F16) { PP_GN_GROUP(_Float16); }
    else { PP_GN_GROUP(float); }
#undef PP_GN_GROUP
    return launch_status("pp_group_norm");
  }
  gn_split(N, HW, C, &p.slices, &p.ppslice);
  const int rows = 256 / (C / 8);
  int blocks = ceil_div(HW, 4 * rows);
  const int most = 2048 / N > 1 ? 2048 / N : 1;
  if (blocks > most) blocks = most;
  p.ppblock = ceil_div(HW, blocks);
  blocks = ceil_div(HW, p.ppblock);
  // maps of 64 MB and more: 4x360x640x64 fp16 75 us against 86, 2x270x480x96 fp32 67 against 75; smaller outputs stay in the cache for their reader
  const bool past = (int64_t)N * HW * C * (dtype == PP_F16 ? 2 : 4) >= (64 << 20);
  if (dtype == PP_F16) {
    hipLaunchKernelGGL((gn_stats_kernel<_Float16>), dim3(p.slices, N), dim3(256), 0, st, p);
    if (past) hipLaunchKernelGGL((gn_apply_kernel<_Float16, true>), dim3(blocks, N), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((gn_apply_kernel<_Float16, false>), dim3(blocks, N), dim3(256), 0, st, p);
  } else {
    hipLaunchKernelGGL((gn_stats_kernel<float>), dim3(p.slices, N), dim3(256), 0, st, p);
    if (past) hipLaunchKernelGGL((gn_apply_kernel<float, true>), dim3(blocks, N), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((gn_apply_kernel<float, false>), dim3(blocks, N), dim3(256), 0, st, p);
  }
  return launch_status("pp_group_norm");
}
