// Attention of a batch of sequences over the keys of a shared prefix and of their own suffix, in one softmax.
//
//   out[b,i,h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q[b,i,h] . k_j - m),   m = max_j
//   j over prefix_lens[g] shared keys of group g = b / (B / G), then over lens[b] (causal: the first lens[b] - Lq + i + 1) own keys
//
// One wave per (query, head): the kernel every other form is checked against.  fp32 arithmetic, online maximum and sum.
#include "common.h"

namespace pp {

struct PaParams {
  const char *q, *pk, *pv, *k, *v;
  char* out;
  const int *plens, *lens;
  long long qs[3], pks[3], pvs[3], ks[3], vs[3], os[3];
  int B, G, nseq, Lq, Hq, Hkv, rep, P, S, causal;
  float sc2;      // scale * log2(e)
};

__device__ __forceinline__ int clamp_len(const int* lens, int i, int most) {
  const int n = lens != nullptr ? lens[i] : most;
  return n < 0 ? 0 : (n > most ? most : n);
}

template <typename T, int D>
__global__ __launch_bounds__(256) void pa_simple_kernel(const PaParams p) {
  const int lane = threadIdx.x & 63;
  const long long id = blockIdx.x * 4ll + (threadIdx.x >> 6);
  if (id >= (long long)p.B * p.Lq * p.Hq) return;
  const int h = (int)(id % p.Hq);
  const int i = (int)(id / p.Hq % p.Lq);
  const int b = (int)(id / ((long long)p.Hq * p.Lq));
  const int g = b / p.nseq, hk = h / p.rep;
  constexpr int E = D / 64;
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.qs[0] + i * p.qs[1] + h * p.qs[2] + lane;
  float qv[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) { qv[e] = to_f32(q[e * 64]) * p.sc2; acc[e] = 0.f; }
  const int np = clamp_len(p.plens, g, p.P);
  int ns = clamp_len(p.lens, b, p.S);
  if (p.causal) ns = max(0, min(ns, ns - p.Lq + i + 1));
  float m = -3.4028235e38f, l = 0.f;
  for (int j = 0; j < np + ns; ++j) {
    const T *kr, *vr;
    if (j < np) {
      kr = reinterpret_cast<const T*>(p.pk) + g * p.pks[0] + j * p.pks[1] + hk * p.pks[2] + lane;
      vr = reinterpret_cast<const T*>(p.pv) + g * p.pvs[0] + j * p.pvs[1] + hk * p.pvs[2] + lane;
    } else {
      kr = reinterpret_cast<const T*>(p.k) + b * p.ks[0] + (j - np) * p.ks[1] + hk * p.ks[2] + lane;
      vr = reinterpret_cast<const T*>(p.v) + b * p.vs[0] + (j - np) * p.vs[1] + hk * p.vs[2] + lane;
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(qv[e], to_f32(kr[e * 64]), s);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    const float mn = fmaxf(m, s);
    const float alpha = __builtin_amdgcn_exp2f(m - mn), pe = __builtin_amdgcn_exp2f(s - mn);
    l = l * alpha + pe;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(pe, to_f32(vr[e * 64]), acc[e] * alpha);
    m = mn;
  }
  T* o = reinterpret_cast<T*>(p.out) + b * p.os[0] + i * p.os[1] + h * p.os[2] + lane;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e * 64] = from_f32<T>(np + ns > 0 ? acc[e] / l : 0.f);
}

}  // namespace pp

using namespace pp;

extern "C" int pp_sizeof_prefix_attn_args(void) { return (int)sizeof(pp_prefix_attn_args_t); }

static int pa_check_sizes(const pp_prefix_attn_args_t* a) {
  PP_REQUIRE(a != nullptr, PP_ERR_ARG, "pp_shared_prefix_attention: null args");
  PP_REQUIRE(a->dtype == PP_F32 || a->dtype == PP_F16, PP_ERR_DTYPE, "pp_shared_prefix_attention: dtype %d", a->dtype);
  PP_REQUIRE(a->D == 64 || a->D == 128, PP_ERR_ARG, "pp_shared_prefix_attention: head dim %d (64 or 128)", a->D);
  PP_REQUIRE(a->B >= 0 && a->G > 0 && a->B % a->G == 0 && a->Lq >= 0 && a->P >= 0 && a->S >= 0 && a->Hkv > 0 && a->Hq > 0 && a->Hq % a->Hkv == 0,
             PP_ERR_ARG, "pp_shared_prefix_attention: bad sizes (B=%d G=%d Lq=%d Hq=%d Hkv=%d P=%d S=%d)", a->B, a->G, a->Lq, a->Hq, a->Hkv, a->P, a->S);
  PP_REQUIRE((int64_t)a->B * a->Lq * a->Hq <= (1 << 28) && (int64_t)a->B * a->Hkv <= (1 << 24) && (int64_t)a->P + a->S <= 0x40000000, PP_ERR_ARG,
             "pp_shared_prefix_attention: too many queries or keys (B=%d Lq=%d Hq=%d P=%d S=%d)", a->B, a->Lq, a->Hq, a->P, a->S);
  return 0;
}

extern "C" int64_t pp_shared_prefix_attention_workspace_bytes(const pp_prefix_attn_args_t* a) {
  const int rc = pa_check_sizes(a);
  return rc != 0 ? rc : 0;
}

static int pa_check_tensor(const char* name, const void* ptr, const int64_t* st, int n0, int n1, int n2, int D, int dtype) {
  const int per = dtype == PP_F16 ? 8 : 4;
  PP_REQUIRE(ptr != nullptr && (uintptr_t)ptr % 16 == 0, ptr == nullptr ? PP_ERR_ARG : PP_ERR_ALIGN, "pp_shared_prefix_attention: %s must be 16-byte aligned device memory",
             name);
  const int64_t n[3] = {n0, n1, n2};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1) {
      PP_REQUIRE(st[i] >= 0 && st[i] % per == 0, PP_ERR_ALIGN, "pp_shared_prefix_attention: %s stride %lld (dimension %d) must be a multiple of %d", name,
                 (long long)st[i], i, per);
      PP_REQUIRE(i != 1 || (st[i] >= D && st[i] <= (1 << 22)), PP_ERR_ARG, "pp_shared_prefix_attention: %s token stride %lld (%d to 2^22)", name, (long long)st[i], D);
    }
  return 0;
}

extern "C" int pp_shared_prefix_attention(const pp_prefix_attn_args_t* a, void* stream) {
  int rc = pa_check_sizes(a);
  if (rc != 0) return rc;
  if (a->B == 0 || a->Lq == 0) return 0;
  PP_REQUIRE(a->causal == 0 || a->causal == 1, PP_ERR_ARG, "pp_shared_prefix_attention: causal %d", a->causal);
  PP_REQUIRE(isfinite(a->scale), PP_ERR_ARG, "pp_shared_prefix_attention: scale is not finite");
  if ((rc = pa_check_tensor("q", a->q, a->q_stride, a->B, a->Lq, a->Hq, a->D, a->dtype)) != 0) return rc;
  if ((rc = pa_check_tensor("out", a->out, a->out_stride, a->B, a->Lq, a->Hq, a->D, a->dtype)) != 0) return rc;
  PP_REQUIRE((a->B == 1 || a->out_stride[0] > 0) && (a->Hq == 1 || a->out_stride[2] >= a->D), PP_ERR_ARG, "pp_shared_prefix_attention: out repeats elements");
  if (a->P > 0) {
    if ((rc = pa_check_tensor("pk", a->pk, a->pk_stride, a->G, a->P, a->Hkv, a->D, a->dtype)) != 0) return rc;
    if ((rc = pa_check_tensor("pv", a->pv, a->pv_stride, a->G, a->P, a->Hkv, a->D, a->dtype)) != 0) return rc;
  }
  if (a->S > 0) {
    if ((rc = pa_check_tensor("k", a->k, a->k_stride, a->B, a->S, a->Hkv, a->D, a->dtype)) != 0) return rc;
    if ((rc = pa_check_tensor("v", a->v, a->v_stride, a->B, a->S, a->Hkv, a->D, a->dtype)) != 0) return rc;
  }
  const int64_t need = pp_shared_prefix_attention_workspace_bytes(a);
  PP_REQUIRE(need == 0 || (a->work != nullptr && a->work_bytes >= need && (uintptr_t)a->work % 16 == 0), PP_ERR_WORKSPACE,
             "pp_shared_prefix_attention: needs %lld bytes of 16-byte aligned scratch, got %lld", (long long)need, (long long)a->work_bytes);
  PaParams p;
  p.q = (const char*)a->q; p.pk = (const char*)a->pk; p.pv = (const char*)a->pv; p.k = (const char*)a->k; p.v = (const char*)a->v;
  p.out = (char*)a->out; p.plens = a->prefix_lens; p.lens = a->lens;
  const int64_t* from[6] = {a->q_stride, a->pk_stride, a->pv_stride, a->k_stride, a->v_stride, a->out_stride};
  long long* to[6] = {p.qs, p.pks, p.pvs, p.ks, p.vs, p.os};
  for (int t = 0; t < 6; ++t)
    for (int i = 0; i < 3; ++i) to[t][i] = from[t][i];
  p.B = a->B; p.G = a->G; p.nseq = a->B / a->G; p.Lq = a->Lq; p.Hq = a->Hq; p.Hkv = a->Hkv; p.rep = a->Hq / a->Hkv; p.P = a->P; p.S = a->S;
  p.causal = a->causal;
  p.sc2 = a->scale * 1.4426950408889634f;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(((long long)a->B * a->Lq * a->Hq + 3) / 4));
  if (grid.x > (1u << 23)) { set_error("pp_shared_prefix_attention: too many queries"); return PP_ERR_ARG; }
#define PA_LAUNCH(T, DD) hipLaunchKernelGGL((pa_simple_kernel<T, DD>), grid, dim3(256), 0, st, p)
  if (a->dtype == PP_F16) { if (a->D == 128) PA_LAUNCH(_Float16, 128); else PA_LAUNCH(_Float16, 64); }
  else { if (a->D == 128) PA_LAUNCH(float, 128); else PA_LAUNCH(float, 64); }
#undef PA_LAUNCH
  return launch_status("pp_shared_prefix_attention");
}
