// fp16 GEMM for the short-K linears (1x1 convolutions, K <= 512): A-STATIONARY.
//
// The transformer's Linear layers (qkv 512->1536, proj 512->512, fc1 512->1960, SoftComp embedding 512->6272, pooled
// k/v) and RAFT's 1x1 correlation encoder have K = 384..512: 6-8 K steps per 128x128 tile.  In the tiled kernels
// (conv_gemm_v2.hip) such a tile spends as long in its prologue (first DMA round trip) and epilogue as in its K loop,
// and every M tile is re-gathered once per N tile.  Here a block owns 128 pixels for ALL output channels:
//   * each wave loads its 32 pixels x K activations ONCE, straight from global memory into the MFMA fragment layout
//     (128 VGPRs at K = 512) -- no LDS, no re-reads;
//   * the packed weights stream through LDS in [64 couts][128 k] steps (two 64x64 sub-tiles in the v2 swizzled
//     image, LDS-DMA, double buffered) as ONE continuous pipeline over (64-cout chunk, k step): no per-tile prologue;
//   * after the last k step of a chunk the 32 x 64 accumulators go through the shared lean epilogue
//     (conv_epilogue.h, wave-private staging tile) while the next chunk's weights are already in flight; the
//     chunk's bias is fetched at the start of its K loop.
// Same K order and MFMA sequence per output as the other kernels: bit-identical results.
#include "conv_epilogue.h"

namespace pp {

typedef __attribute__((address_space(3))) void* lptr4_t;

template <int KMAX, int DIAG = 0>
__global__ __launch_bounds__(256, 2) void conv_ast_kernel(const ConvParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef _Float16 T;
  constexpr int NW = 4;
  constexpr int BM = 128, WM = 32, TM = 2;            // 4 waves x 32 pixels
  constexpr int CN = 64, TN = 4;                      // couts per chunk
  constexpr int KS32 = KMAX / 32;                     // 32-wide MFMA k steps held in registers
  constexpr int SUB = CN * 128;                       // one 64x64 fp16 sub-tile (128-byte rows)
  constexpr int STAGE = 2 * SUB;                      // 128 k per pipeline step
  constexpr int EPI_W = WM * (CN + 4) * 4;            // wave-private epilogue staging (fp32 worst case)
  constexpr int LDS_BYTES = 2 * STAGE + NW * EPI_W;
  static_assert(LDS_BYTES <= 80 * 1024, "lds");

  __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];
  char* const epi = lds + 2 * STAGE;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l15 = lane & 15, l4 = lane >> 4;
  const long long m0 = (long long)blockIdx.x * BM;
  const int K = p.kchunks * 8;
  const int nk32 = K / 32;                            // <= KS32
  const int nsteps = (K + 127) / 128;                 // 128-k pipeline steps per chunk (the last may be half: K % 128 == 64)
  const int nchunks = (p.cout_g + CN - 1) / CN;

  // ---- A: this wave's 32 pixels x K, loaded once in fragment layout (row = l15 of tile t, 8 k at (s*4 + l4)*8)
  f16x8 af[TM][KS32];
  {
    const T* src = reinterpret_cast<const T*>(p.src[0].ptr) + p.src[0].choff;
    const long long cs = p.src[0].cstride;
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      long long m = m0 + wave * WM + t * 16 + l15;
      if (m >= p.M) m = p.M - 1;                      // rows past M are computed but never stored
      const T* rp = src + m * cs + l4 * 8;
#pragma unroll
      for (int s = 0; s < KS32; ++s)
        af[t][s] = s < nk32 ? *reinterpret_cast<const f16x8*>(rp + s * 32) : f16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }

  // ---- B DMA roles (v2 image: 8 rows of 128 B per instruction, slot ^ ((row >> 1) & 7))
  const int rin = lane >> 3, slot = lane & 7;
  const int lc = slot ^ ((4 * (wave & 1) + (rin >> 1)) & 7);
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p.weight), 0, p.cout_pad * p.kchunks * 16, 0x00020000);
  // one pipeline step = 16 instructions (2 sub-tiles x 8 row groups): wave w issues row groups w and w + 4 of each sub-tile
  // (a macro, not a capturing lambda: see conv_gemm_v3.hip)
  const int Kb = K * 2;
#define AST_ISSUE(chunk_, step_, buf_)                                                                             \
  do {                                                                                                              \
    char* st_ = lds + (buf_) * STAGE;                                                                               \
    _Pragma("unroll") for (int h_ = 0; h_ < 2; ++h_) {                                                              \
      const int kb_ = (step_) * 128 + h_ * 64;                                                                      \
      _Pragma("unroll") for (int j_ = 0; j_ < 2; ++j_) {                                                            \
        const int q_ = j_ * NW + wave;                                                                              \
        int row_ = (chunk_) * CN + q_ * 8 + rin;                                                                    \
        if (row_ >= p.cout_pad) row_ = p.cout_pad - 1;                                                              \
        const int voff_ = kb_ < K ? row_ * Kb + kb_ * 2 + lc * 16 : (int)0x80000000;                                \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lptr4_t)(st_ + h_ * SUB + q_ * 1024), 16, voff_, 0, 0, 0);    \
      }                                                                                                             \
    }                                                                                                               \
  } while (0)

  f32x4 acc[TN][TM];
  const int b_off = l15 * 128;
  const int bswz = (l15 >> 1) & 7;
  const int total = nchunks * nsteps;
  AST_ISSUE(0, 0, 0);
  int chunk = 0, step = 0, buf = 0;
  bool prewaited = false;
  f32x4 bias4[TN];
  for (int it = 0; it < total; ++it) {
    if (step == 0) {
#pragma unroll
      for (int a = 0; a < TN; ++a) {
#pragma unroll
        for (int b = 0; b < TM; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
        // the chunk's bias, in flight during its K loop
        const int c0 = chunk * CN + a * 16 + l4 * 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) bias4[a][r] = (p.bias != nullptr && c0 + r < p.cout_g) ? p.bias[c0 + r] : 0.f;
      }
    }
    if (!prewaited) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    prewaited = false;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // this wave's fragment reads of stage buf^1 are back
    __builtin_amdgcn_s_barrier();                     // stage `buf` landed for all waves; stage buf^1 is free
    {
      int nc = chunk, ns = step + 1;
      if (ns == nsteps) { ns = 0; ++nc; }
      if (it + 1 < total) AST_ISSUE(nc, ns, buf ^ 1);
    }
    const char* sb = lds + buf * STAGE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        f16x8 bf[TN];
#pragma unroll
        for (int f = 0; f < TN; ++f)
          bf[f] = *reinterpret_cast<const f16x8*>(sb + h * SUB + b_off + f * 16 * 128 + (((kk * 4 + l4) ^ bswz) << 4));
        // af is indexed with a loop-carried `step`: select the fragment with compile-time indices per step value
#pragma unroll
        for (int sv = 0; sv < KS32 / 4; ++sv) {
          if (step == sv) {
#pragma unroll
            for (int a = 0; a < TN; ++a)
#pragma unroll
              for (int b = 0; b < TM; ++b)
                acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bf[a], af[b][sv * 4 + h * 2 + kk], acc[a][b], 0, 0, 0);
          }
        }
      }
    }
    buf ^= 1;
    if (++step == nsteps) {
      // ---- chunk done: epilogue of 32 px x 64 couts per wave (weights of the next chunk are already in flight)
      struct RowMap {
        long long m_base, M;
        __device__ __forceinline__ long long operator()(int prow) const {
          const long long m = m_base + prow;
          return m < M ? m : -1ll;
        }
      };
      const RowMap rowmap{m0 + wave * WM, p.M};
      // retire the next stage's DMA BEFORE the epilogue: vmcnt is in-order and also counts stores, so waiting at the top of
      // the next step would drain this chunk's output stores; this way they complete in the shadow of the next K step
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      prewaited = true;
      if constexpr (DIAG == 0) {
        conv_epilogue<WM, CN, CN / 16, 0, false, false>(p, acc, epi + wave * EPI_W, lane, chunk * CN, 0, p.out, rowmap, bias4);
      } else {                                        // [diagnostic] no epilogue: keep the accumulators alive only
        float sacc = 0.f;
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
          for (int b = 0; b < TM; ++b) sacc += acc[a][b][0] + bias4[a][0];
        if (sacc == 123456.789f) reinterpret_cast<float*>(p.out)[lane] = sacc;
      }
      step = 0;
      ++chunk;
    }
  }
#undef AST_ISSUE
#endif
}

// Returns -1000 when the layer is not a short-K single-source 1x1 fp16 convolution (caller falls back to v2).
// cfg: 0 = auto, 80 = force.
int conv_ast_dispatch(const ConvParams& p, int cfg, hipStream_t stream) {
  const int K = p.kchunks * 8;
  if (p.preadd != nullptr || p.fuse != PP_FUSE_NONE) return -1000;      // the fused recurrent-cell epilogue lives in the tiled kernels
  if (p.tap_h != 1 || p.tap_w != 1 || p.nsrc != 1 || p.groups != 1 || p.sh != 1 || p.sw != 1 || p.ph != 0 || p.pw != 0) return -1000;
  if (K > 512 || K % 64 != 0 || !(p.ktable_uniform & 8) || p.pad_mode != 0 || p.src_gstride != 0 || p.out_gstride != 0 || p.OH != p.H || p.OW != p.W) return -1000;
  if ((long long)p.cout_pad * p.kchunks * 16 >= (1ll << 31) || p.M >= (1ll << 31)) return -1000;
  if (cfg == 0 && (p.cout_g < 256 || p.M < 128 * 256)) return -1000;       // needs enough couts to amortise the A load, enough rows to fill the GPU
  const unsigned nblk = (unsigned)((p.M + 127) / 128);
#if defined(PP_DIAG)
  if (cfg == 81) hipLaunchKernelGGL((conv_ast_kernel<512, 1>), dim3(nblk), dim3(256), 0, stream, p);   // diagnostic: no epilogue
  else
#endif
  hipLaunchKernelGGL((conv_ast_kernel<512>), dim3(nblk), dim3(256), 0, stream, p);
  return launch_status("pp_conv2d(ast)");
}

}  // namespace pp
