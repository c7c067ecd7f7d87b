// Attention of a batch of sequences over the keys of a shared prefix and of their own suffix, in one softmax.
//
//   out[b,i,h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q[b,i,h] . k_j - m),   m = max_j
//   j over prefix_lens[g] shared keys of group g = b / (B / G), then over lens[b] (causal: the first lens[b] - Lq + i + 1) own keys
//
// Rows.  The queries that read one key head form rows: Lq * rep of a sequence (rep = Hq / Hkv query heads a key head), or, packed, those of
// ALL sequences of a group, which is how a prefix is read once for the whole batch.  A part of the work is a set of row spaces with the keys
// they walk; a call is one part (every sequence walks prefix and suffix) or two (packed rows walk the prefix, single sequences their
// suffix).  Where a row's keys are split over several blocks, each leaves (max, sum, unnormalised output) in fp32 scratch and
// pa_join_kernel joins them in a fixed order.
//
// S^T = K Q^T and O^T += V^T P^T on 16x16 MFMA tiles: a lane holds scores of ONE query (column l & 15), so the row maximum takes two lane
// swaps, and its scores are the second product's operand as they are, keys relabelled.  Maximum, sum and output stay in fp32 registers.
// fp16 calls round every weight once to fp16: the matrix instructions take both operands in one type, and weights in two fp16 parts would double the second
// product.  It costs 2^-11 of a weight at most; over the shapes below the error against 64 bits is 2.4e-4 to 2.6e-4 of the outputs' size, 2.1e-4 of
// which is the rounding of the outputs themselves.
//
// Forms (4 waves a block).  Many rows: a wave owns 16 QT rows and every key of a tile of 64 that lies in LDS (K and V swizzled, fp32 V
// skewed), the next tile's loads in flight during the products.  Few rows (WK): the four waves share 16 QT rows and take different keys,
// joined through LDS at the end; in fp16 every wave streams keys of its own (pa_stream_block).
//   rows: 24 sequences x 765 queries, 4 heads of 128, 2430 shared + 1158 own keys, fp16: 181 us = 750 TFLOP/s (181 and a join of 10 under the profiler).  Products alone would be 102 us at the
//     rate of a large matrix product; the softmax' vector instructions take 190 of 407 thousand cycles a CU next to 130 of MFMA, and two blocks a
//     CU overlap them in part.  LDS conflicts: none.  Two LDS tiles (one barrier a tile, one block a CU): 193.
//   single tokens: 64 sequences, 8192 shared + up to 1024 own keys, 32 heads on 8 key heads of 128, fp16: 54-59 us for 171 MB (68.7 with every suffix full, 48.9 half full); the two parts run in one launch
//     (44 us: the suffixes out of memory next to the packed rows' products), 6 us of joining, the rest launches.
//   fp32: 16 sequences x 4 queries, 16 heads on 2 key heads of 64, 4096 + up to 512 keys: 26 us, of which 6.6 are products at the fp32 matrix
//     rate; few waves, so the latency of a tile's loads and dependent products, and the join's 6 us.
#include "common.h"
#include "attn_lanes.h"

namespace pp {

struct PaPart {
  int nper;              // sequences a row space packs (1 or nseq)
  int rows, rowblocks;   // rows of a space, blocks that cover them
  int prefix, suffix;    // keys it walks
  int items, whole;      // row blocks over all spaces and key heads; the first `whole` walk all their keys and write the output
  int nsplit, slot0;     // the others: blocks that share the keys; first scratch slot
  int by_row;            // scratch rows: 1 = query rows of the call (two parts join there), 0 = rows of the split items alone
  int blocks;            // whole + (items - whole) * nsplit
};
struct PaParams {
  const char *q, *pk, *pv, *k, *v;
  char* out;
  const int *plens, *lens;
  float* part_o;         // scratch [slots][prows][D]: unnormalised outputs
  float* part_ml;        // scratch [slots][prows][2]: maximum and sum
  long long prows;
  long long qs[3], pks[3], pvs[3], ks[3], vs[3], os[3];
  int B, G, nseq, Lq, Hq, Hkv, rep, P, S, causal, slots;
  float sc2;             // |scale| * log2(e)  (1 if scale is 0)
  float qsign;           // sign of scale (0 if it is 0), taken into the queries
  PaPart part[2];
};

// blocks 8 apart share an XCD: give each XCD one contiguous run of 0 .. n - 1, so that blocks that read the same keys meet in one L2
__device__ __forceinline__ int xcd_run(int id, int n) {
  const int per = n >> 3, extra = n & 7, x = id & 7;
  return x * per + min(x, extra) + (id >> 3);
}
// query row r of row space `space` and key head hk -> sequence, token, head
struct PaRow { int b, i, h; };
__device__ __forceinline__ PaRow pa_row(int Lq, int rep, int nper, int space, int hk, int r) {
  const int rpseq = Lq * rep, sq = r / rpseq, rest = r - sq * rpseq, i = rest / rep;
  return {space * nper + sq, i, hk * rep + (rest - i * rep)};
}

constexpr float PA_NONE = -3.4028235e38f;   // running maximum before the first key: finite, so that masked scores (-inf) weigh 0

// A weight is exp2((s - m) sc2 + lift) for the score s and the row's maximum m, both as the products left them.  fp16 weights are lifted: 2^15 for the
// maximum, so that one of 2^-29 of it still has its 11 bits and one of 2^-39 is not lost (unlifted 2^-14 and 2^-24: behind a million keys the tail of a
// softmax would be).  Sums and outputs carry the same factor, which the last division takes out.
template <typename T> constexpr float pa_lift() { return sizeof(T) == 2 ? 15.f : 0.f; }
// s sc2 + c with c = lift - m sc2 is one operation a score; c's own rounding scales all weights of the row alike.  Past 2^20 that factor could
// leave the weights' range, so there the scores' differences are taken first (by the whole wave; such scores are that uncertain anyway).
constexpr float PA_BIG = 1048576.f;
template <int QT> struct PaRows { float m[QT], l[QT]; };      // running maximum, sum of the weights of this lane's keys
template <int QT, int DT>
__device__ __forceinline__ void pa_rows_start(PaRows<QT>& w, f32x4 (&oacc)[QT][DT]) {
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    w.m[qt] = PA_NONE;
    w.l[qt] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) oacc[qt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}
// c of a row's new maximum
template <typename T, int N>
__device__ __forceinline__ float pa_base(const float m_new, const float sc2, f32x4 (&s)[N]) {
#if defined(__HIP_DEVICE_COMPILE__)
  const float c = fminf(fmaf(-m_new, sc2, pa_lift<T>()), -PA_NONE);
  if (__builtin_amdgcn_ballot_w64(fabsf(c) > PA_BIG && m_new > PA_NONE) == 0ull) return c;
#pragma unroll
  for (int kt = 0; kt < N; ++kt) s[kt] -= m_new;
#endif
  return pa_lift<T>();
}
// adds a tile's weights to a row's sum; what is summed so far is scaled to the new maximum
template <int QT, int DT>
__device__ __forceinline__ void pa_rows_add(PaRows<QT>& w, f32x4 (&oacc)[QT][DT], const int qt, const float m_new, const float psum, const float sc2) {
#if defined(__HIP_DEVICE_COMPILE__)
  if (__builtin_amdgcn_ballot_w64(m_new > w.m[qt]) != 0ull) {
    const float alpha = __builtin_amdgcn_exp2f((w.m[qt] - m_new) * sc2);
    w.l[qt] *= alpha;
#pragma unroll
    for (int d = 0; d < DT; ++d) oacc[qt][d] *= alpha;
  }
  w.m[qt] = m_new;
  w.l[qt] += psum;
#endif
}

__device__ __forceinline__ int clamp_len(const int* lens, int i, int most) {
  const int n = lens != nullptr ? lens[i] : most;
  return n < 0 ? 0 : (n > most ? most : n);
}

#if defined(__HIP_DEVICE_COMPILE__)
// 16 bytes of a row: 8 consecutive fp16 channels, or 4 of fp32, one contraction slot of 4 products
template <typename T> struct PaFrag { typedef f16x8 type; };
template <> struct PaFrag<float> { typedef f32x4 type; };
#endif

template <typename T, int D, bool WK> struct PaTile {
  static constexpr bool F16 = sizeof(T) == 2;
  static constexpr int KT = 64;                               // keys of a tile
  static constexpr int NK = WK ? 1 : 4;                       // 16-key tiles of a wave
  static constexpr int SLOTS = D * (int)sizeof(T) / 16;       // 16-byte slots of a key row
  static constexpr int STEPS = SLOTS / 4;                     // fragments of a row
  static constexpr int VLD = F16 ? D : D + 16;                // V row stride (elements); fp16 rows are swizzled (v_at), fp32 rows skewed
  static constexpr int LOADS = KT * SLOTS / 256;              // 16-byte pieces a thread stages of K and of V
  static constexpr int KBYTES = KT * D * (int)sizeof(T), VBYTES = KT * VLD * (int)sizeof(T);
};

// fp16 V rows: 16-byte slot s (8 channels) of key k lies in slot s ^ f(k), its 8-byte halves swapped where k & 4 -- the 8 keys x 4 halves that 32
// lanes of a transposing read take then cover all 64 banks once.
template <int D> __device__ __forceinline__ int v_slot(int key, int s) { return s ^ (D == 128 ? (key & 3) << 2 : (key & 2) << 1); }

template <typename T, int D, int QT, bool WK> struct PaLds {
  typedef PaTile<T, D, WK> C;
  static constexpr int JOIN = WK ? 4 * 16 * QT * (D + 4) * 4 : 0;
  static constexpr int BYTES = C::KBYTES + C::VBYTES > JOIN ? C::KBYTES + C::VBYTES : JOIN;
};

// channel of position `pos` (of 4 neighbours) of an accumulator row: see the product with V
template <bool F16> __device__ __forceinline__ int pa_channel(int pos) {
  const int d = pos >> 4, g = (pos >> 2) & 3;
  return F16 ? (d >> 1) * 32 + g * 8 + (d & 1) * 4 + (pos & 3) : pos;
}

// block -> item (row block fastest, key head, row space) and key split
struct PaItem { bool whole; int item, split, rb, hk, space; };
__device__ __forceinline__ PaItem pa_item(const PaParams& p, const PaPart& pt, const int bid) {
  int item, split = 0;
  const bool whole = bid < pt.whole;
  if (whole) {
    item = xcd_run(bid, pt.whole);
  } else {
    const int x = xcd_run(bid - pt.whole, pt.blocks - pt.whole), rest = pt.items - pt.whole;
    if (pt.whole == 0) {      // row blocks of one space and split are neighbours
      const int rb = x % pt.rowblocks, y = x / pt.rowblocks;
      split = y % pt.nsplit;
      item = y / pt.nsplit * pt.rowblocks + rb;
    } else {
      split = x / rest;
      item = pt.whole + x % rest;
    }
  }
  return {whole, item, split, item % pt.rowblocks, item / pt.rowblocks % p.Hkv, item / pt.rowblocks / p.Hkv};
}

// The four waves of a block hold the same 16 QT rows for different keys: joined through LDS, then written out (or left in the scratch)
template <typename T, int D, int QT>
__device__ __forceinline__ void pa_join_waves(const PaParams& p, const PaPart& pt, char* lds, float* wave_ml, const f32x4 (&oacc)[QT][D / 16], const PaRows<QT>& w,
                                              const long long (&rowid)[QT], char* const (&optr)[QT], const bool whole, const int split,
                                              const bool any) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr bool F16 = sizeof(T) == 2;
  constexpr int DT = D / 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lg = lane >> 4, lc = lane & 15;
  // every wave scales its rows to the common maximum, LDS holds [wave][row][D + 4] floats
  float* jo = reinterpret_cast<float*>(lds);
  constexpr int JLD = D + 4;
  float l[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    l[qt] = rows_sum(w.l[qt]);
    if (lg == 0) {
      wave_ml[(wave * 16 * QT + qt * 16 + lc) * 2] = w.m[qt];
      wave_ml[(wave * 16 * QT + qt * 16 + lc) * 2 + 1] = l[qt];
    }
  }
  __syncthreads();
  float mj[QT], lj[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float* e = wave_ml + (qt * 16 + lc) * 2;
    constexpr int W = 16 * QT * 2;
    mj[qt] = fmaxf(fmaxf(e[0], e[W]), fmaxf(e[2 * W], e[3 * W]));
    lj[qt] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) lj[qt] += e[i * W + 1] * __builtin_amdgcn_exp2f((e[i * W] - mj[qt]) * p.sc2);
    const float f = __builtin_amdgcn_exp2f((w.m[qt] - mj[qt]) * p.sc2);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(jo + (wave * 16 * QT + qt * 16 + lc) * JLD + d * 16 + lg * 4) = oacc[qt][d] * f;
  }
  __syncthreads();
  // wave w finishes positions w * D / 4 .. of rows lc: 16 rows x 4 lane groups x D / 64 pieces of 4
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    if (rowid[qt] < 0) continue;
    const float* e = jo + (qt * 16 + lc) * JLD;
    constexpr int W = 16 * QT * JLD;
    const float inv = lj[qt] != 0.f ? 1.f / lj[qt] : 0.f;
    const long long at = (pt.slot0 + split) * p.prows + rowid[qt];
    if (!whole && wave == 0 && lg == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mj[qt], lj[qt]);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const int pos = wave * (D / 4) + c * 16 + lg * 4;
      f32x4 v = *reinterpret_cast<const f32x4*>(e + pos);
#pragma unroll
      for (int i = 1; i < 4; ++i) v += *reinterpret_cast<const f32x4*>(e + i * W + pos);
      if (!whole) {
        if (any) *reinterpret_cast<f32x4*>(p.part_o + at * D + pos) = v;
      } else if constexpr (F16) {
        const f16x4 o = {(_Float16)(v[0] * inv), (_Float16)(v[1] * inv), (_Float16)(v[2] * inv), (_Float16)(v[3] * inv)};
        *reinterpret_cast<f16x4*>(reinterpret_cast<T*>(optr[qt]) + pa_channel<F16>(pos)) = o;
      } else {
        *reinterpret_cast<f32x4*>(reinterpret_cast<T*>(optr[qt]) + pos) = v * inv;
      }
    }
  }
#endif
}

// block `bid` of part `pt`, key tiles of 64 through LDS (fp16: WK = false alone, few rows go to pa_stream_block)
template <typename T, int D, int QT, bool WK>
__device__ __forceinline__ void pa_block(const PaParams& p, const PaPart& pt, const int bid, char* lds, float* wave_ml) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef PaTile<T, D, WK> C;
  typedef typename PaFrag<T>::type frag;
  constexpr int KT = C::KT, NK = C::NK, STEPS = C::STEPS, DT = D / 16;
  static_assert(!(C::F16 && WK), "fp16 blocks of few rows are streamed");
  T* Ks = reinterpret_cast<T*>(lds);
  T* Vs = reinterpret_cast<T*>(lds + C::KBYTES);

  const PaItem it = pa_item(p, pt, bid);
  const bool whole = it.whole;
  const int item = it.item, split = it.split, nsplit = whole ? 1 : pt.nsplit, rb = it.rb, hk = it.hk, space = it.space;
  const int b0 = space * pt.nper, g = b0 / p.nseq;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lg = lane >> 4, lc = lane & 15;
  const int row0 = rb * 16 * QT * (WK ? 1 : 4);
  const int row_end = min(pt.rows, row0 + 16 * QT * (WK ? 1 : 4));

  const int np = pt.prefix ? clamp_len(p.plens, g, p.P) : 0;
  const int ns = pt.suffix ? clamp_len(p.lens, b0, p.S) : 0;
  int vis_min = ns, vis_max = ns;                 // suffix keys the block's first / last row sees
  if (pt.suffix && p.causal) {
    vis_min = min(ns, max(0, ns - p.Lq + row0 / p.rep + 1));
    vis_max = min(ns, max(0, ns - p.Lq + (row_end - 1) / p.rep + 1));
  }
  const int ptiles = (np + KT - 1) / KT;
  const int tiles = ptiles + (vis_max + KT - 1) / KT;
  const int t0 = (int)((long long)tiles * split / nsplit), t1 = (int)((long long)tiles * (split + 1) / nsplit);

  // ---- this lane's queries (column lane & 15 of the wave's row tiles)
  frag qf[QT][STEPS];
  long long rowid[QT];
  int vis[QT];
  char* optr[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int rl = (WK ? qt : wave * QT + qt) * 16 + lc, r = row0 + rl;
    const bool ok = r < pt.rows;
    const PaRow w = pa_row(p.Lq, p.rep, pt.nper, space, hk, ok ? r : 0);
    // row of the scratch (-1: no row)
    rowid[qt] = !ok ? -1 : pt.by_row ? ((long long)w.b * p.Lq + w.i) * p.Hq + w.h : (long long)(item - pt.whole) * (16 * QT * (WK ? 1 : 4)) + rl;
    if (ok && whole) rowid[qt] = 0;
    vis[qt] = p.causal ? max(0, ns - p.Lq + w.i + 1) : ns;
    optr[qt] = p.out + (w.b * p.os[0] + w.i * p.os[1] + w.h * p.os[2]) * (long long)sizeof(T);
    const T* qp = reinterpret_cast<const T*>(p.q) + w.b * p.qs[0] + w.i * p.qs[1] + w.h * p.qs[2];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      frag f = *reinterpret_cast<const frag*>(qp + (s * 4 + lg) * (16 / sizeof(T)));
      if (p.qsign != 1.f) f *= (T)p.qsign;
      qf[qt][s] = f;
    }
  }

  f32x4 oacc[QT][DT];
  PaRows<QT> run;
  pa_rows_start(run, oacc);

  // ---- staging: a tile's valid keys lie inside the buffer descriptor built for it, the rest (token strides are at least D) comes back as zeros,
  // so that nothing behind a length is used; 64-bit base per tile, 32-bit offsets inside it
  u32x4 kr[C::LOADS], vr[C::LOADS];
  auto tile_keys = [&](int t) {                    // valid keys of tile t
    return t < ptiles ? min(KT, np - t * KT) : min(KT, vis_max - (t - ptiles) * KT);
  };
  auto load_tile = [&](int t) {
    const bool pre = t < ptiles;
    const long long j0 = (long long)(pre ? t : t - ptiles) * KT;
    const long long kts = pre ? p.pks[1] : p.ks[1], vts = pre ? p.pvs[1] : p.vs[1];
    const T* kb = pre ? reinterpret_cast<const T*>(p.pk) + g * p.pks[0] + hk * p.pks[2] : reinterpret_cast<const T*>(p.k) + b0 * p.ks[0] + hk * p.ks[2];
    const T* vb = pre ? reinterpret_cast<const T*>(p.pv) + g * p.pvs[0] + hk * p.pvs[2] : reinterpret_cast<const T*>(p.v) + b0 * p.vs[0] + hk * p.vs[2];
    const unsigned kp = (unsigned)kts * sizeof(T), vp = (unsigned)vts * sizeof(T);
    const int n = tile_keys(t);
    const __amdgpu_buffer_rsrc_t rk = uniform_buffer_rsrc(kb + j0 * kts, (int)((n - 1) * kp + D * sizeof(T)));
    const __amdgpu_buffer_rsrc_t rv = uniform_buffer_rsrc(vb + j0 * vts, (int)((n - 1) * vp + D * sizeof(T)));
#pragma unroll
    for (int i = 0; i < C::LOADS; ++i) {
      const int c = tid + 256 * i, key = c / C::SLOTS, sl = c % C::SLOTS;
      kr[i] = __builtin_amdgcn_raw_buffer_load_b128(rk, (int)(key * kp + sl * 16), 0, 0);
      vr[i] = __builtin_amdgcn_raw_buffer_load_b128(rv, (int)(key * vp + sl * 16), 0, 0);
    }
  };
  auto swz = [](int key) { return C::SLOTS >= 16 ? key & 15 : (key >> 1) & 7; };
  auto store_tile = [&]() {
#pragma unroll
    for (int i = 0; i < C::LOADS; ++i) {
      const int c = tid + 256 * i, key = c / C::SLOTS, sl = c % C::SLOTS;
      *reinterpret_cast<u32x4*>(&Ks[key * D + (sl ^ swz(key)) * (16 / sizeof(T))]) = kr[i];
      if constexpr (C::F16) {
        const u32x4 v = key & 4 ? u32x4{vr[i][2], vr[i][3], vr[i][0], vr[i][1]} : vr[i];
        *reinterpret_cast<u32x4*>(&Vs[key * C::VLD + v_slot<D>(key, sl) * 8]) = v;
      } else {
        *reinterpret_cast<u32x4*>(&Vs[key * C::VLD + sl * 4]) = vr[i];
      }
    }
  };

  const int wkey = WK ? wave * NK * 16 : 0;        // first key of the wave inside a tile
  if (t0 < t1) load_tile(t0);
  for (int t = t0; t < t1; ++t) {
    store_tile();
    __syncthreads();
    if (t + 1 < t1) load_tile(t + 1);
    // ---- scores: sacc[qt][kt][r] = key wkey + kt * 16 + lg * 4 + r, query lc of row tile qt
    f32x4 sacc[QT][NK];
    auto key_frag = [&](int kt, int st) {
      const int key = wkey + kt * 16 + lc;
      return *reinterpret_cast<const frag*>(&Ks[key * D + ((st * 4 + lg) ^ swz(key)) * (16 / sizeof(T))]);
    };
    if constexpr (C::F16) {
#pragma unroll
      for (int kt = 0; kt < NK; ++kt) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) sacc[qt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          const frag kf = key_frag(kt, st);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) sacc[qt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[qt][st], sacc[qt][kt], 0, 0, 0);
        }
      }
    } else {
      // fp32 products take twice as long and leave registers: the next operand is requested ahead of this one's products
      frag cur = key_frag(0, 0);
#pragma unroll
      for (int i = 0; i < NK * STEPS; ++i) {
        const int kt = i / STEPS, st = i % STEPS;
        frag next = cur;
        if (i + 1 < NK * STEPS) next = key_frag((i + 1) / STEPS, (i + 1) % STEPS);
        __builtin_amdgcn_sched_barrier(0);
        if (st == 0)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) sacc[qt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) sacc[qt][kt] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)cur[j], (float)qf[qt][st][j], sacc[qt][kt], 0, 0, 0);
        cur = next;
      }
    }
    // ---- online softmax in the exp2 domain
    const int n = tile_keys(t), j0 = (t - ptiles) * KT;
    const bool cut = p.causal && t >= ptiles && j0 + n > vis_min;      // rows of the block see different parts of the tile
    constexpr int NP = C::F16 ? NK / 2 : 1;
    f16x8 pfr[QT][NP];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      if (n < KT || cut) {
        const int most = cut ? min(n, vis[qt] - j0) : n;
#pragma unroll
        for (int kt = 0; kt < NK; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (wkey + kt * 16 + lg * 4 + r >= most) sacc[qt][kt][r] = -INFINITY;
      }
      float tmax = sacc[qt][0][0];
#pragma unroll
      for (int kt = 0; kt < NK; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) tmax = fmaxf(tmax, sacc[qt][kt][r]);
      tmax = rows_max(tmax);
      const float m_new = fmaxf(run.m[qt], tmax), base = pa_base<T>(m_new, p.sc2, sacc[qt]);
      float psum = 0.f;
#pragma unroll
      for (int kt = 0; kt < NK; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(fmaf(sacc[qt][kt][r], p.sc2, base));
          psum += e;
          if constexpr (C::F16) pfr[qt][kt >> 1][(kt & 1) * 4 + r] = (_Float16)e;    // weights in the values' type: the product's operand
          else sacc[qt][kt][r] = e;
        }
      pa_rows_add(run, oacc, qt, m_new, psum, p.sc2);      // (this lane's keys; the four lane groups are summed at the end)
    }
    // ---- O^T += V^T P^T
    if constexpr (C::F16) {
      // contraction slot lg * 8 + e of a 32-key step is key (e >> 2) * 16 + lg * 4 + (e & 3); accumulator row i of tile d is channel
      // (d / 2) * 32 + (i / 4) * 8 + (d % 2) * 4 + i % 4: two tiles give a lane 8 consecutive channels, four lanes 64 bytes of a row
      const int key = wkey + lg * 4 + (lc >> 2);          // (+ 16, + 32: the swizzle looks at its low bits only)
      const _Float16* vb = reinterpret_cast<const _Float16*>(Vs) + key * C::VLD;
#pragma unroll
      for (int j = 0; j < NK / 2; ++j)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const int at = v_slot<D>(key, (d >> 1) * 4 + (lane & 3)) * 8 + (((d & 1) ^ ((key >> 2) & 1)) << 2);
          const f16x4 v0 = lds_read_tr16(vb + 32 * j * C::VLD + at);
          const f16x4 v1 = lds_read_tr16(vb + (32 * j + 16) * C::VLD + at);
          const f16x8 vf = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) oacc[qt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pfr[qt][j], oacc[qt][d], 0, 0, 0);
        }
    } else {
      // one key a lane group: slot lg is key kt * 16 + lg * 4 + r; accumulator row i of tile d is channel d * 16 + i
      const float* vb = reinterpret_cast<const float*>(Vs) + (wkey + lg * 4) * C::VLD + lc;
      float cur[DT], next[DT];
#pragma unroll
      for (int d = 0; d < DT; ++d) cur[d] = vb[d * 16];
#pragma unroll
      for (int i = 0; i < NK * 4; ++i) {
        if (i + 1 < NK * 4)
#pragma unroll
          for (int d = 0; d < DT; ++d) next[d] = vb[((i + 1) / 4 * 16 + (i + 1) % 4) * C::VLD + d * 16];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) oacc[qt][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(cur[d], sacc[qt][i / 4][i % 4], oacc[qt][d], 0, 0, 0);
#pragma unroll
        for (int d = 0; d < DT; ++d) cur[d] = next[d];
      }
    }
    __syncthreads();
  }

  // Accumulator element (d, r) of lane group lg is position d * 16 + lg * 4 + r of its row; scratch rows are kept in that order.
  if constexpr (!WK) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const float l = rows_sum(run.l[qt]);
      if (rowid[qt] < 0) continue;
      if (!whole) {
        const long long at = (pt.slot0 + split) * p.prows + rowid[qt];
        if (lg == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(run.m[qt], l);
        if (t0 < t1) {
#pragma unroll
          for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(p.part_o + at * D + d * 16 + lg * 4) = oacc[qt][d];
        }
      } else {
        const float inv = l != 0.f ? 1.f / l : 0.f;           // no keys: zeros
        T* o = reinterpret_cast<T*>(optr[qt]);
        if constexpr (C::F16) {
#pragma unroll
          for (int d = 0; d < DT; d += 2) {
            float v[8];
#pragma unroll
            for (int r = 0; r < 4; ++r) { v[r] = oacc[qt][d][r] * inv; v[4 + r] = oacc[qt][d + 1][r] * inv; }
            store8<T>(o + pa_channel<C::F16>(d * 16 + lg * 4), v);
          }
        } else {
#pragma unroll
          for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(o + d * 16 + lg * 4) = oacc[qt][d] * inv;
        }
      }
    }
  } else {
    pa_join_waves<T, D, QT>(p, pt, lds, wave_ml, oacc, run, rowid, optr, whole, split, t0 < t1);
  }
#endif
}

// fp16, few rows: every wave streams 32-key chunks of its own (chunk t0 + wave, then every fourth), with no barrier until the end.  K goes from
// memory into the operand registers as it is (a chunk's keys are read by one wave only), V through 8 KB of the wave's own LDS for the
// transposing read; the loads of the next DEPTH chunks are in flight during a chunk's products.
template <int D, int QT> struct PaStream {
  static constexpr int DEPTH = QT == 1 ? 2 : 1;
  static constexpr int VBYTES = 32 * D * 2;
  static constexpr int JOIN = 4 * 16 * QT * (D + 4) * 4;
  static constexpr int BYTES = 4 * VBYTES > JOIN ? 4 * VBYTES : JOIN;
};
template <int D, int QT>
__device__ __forceinline__ void pa_stream_block(const PaParams& p, const PaPart& pt, const int bid, char* lds, float* wave_ml) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef _Float16 T;
  typedef PaStream<D, QT> C;
  constexpr int STEPS = D / 32, DT = D / 16, SLOTS = D / 8, VL = 32 * SLOTS / 64, KT = 32;     // VL: V loads a lane and chunk
  const PaItem it = pa_item(p, pt, bid);
  const bool whole = it.whole;
  const int nsplit = whole ? 1 : pt.nsplit, b0 = it.space * pt.nper, g = b0 / p.nseq, hk = it.hk;
  const int lane = threadIdx.x & 63, lg = lane >> 4, lc = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);      // provably uniform: chunks, descriptors and branches stay scalar
  const int row0 = it.rb * 16 * QT, row_end = min(pt.rows, row0 + 16 * QT);
  T* Vs = reinterpret_cast<T*>(lds + wave * C::VBYTES);

  const int np = pt.prefix ? clamp_len(p.plens, g, p.P) : 0;
  const int ns = pt.suffix ? clamp_len(p.lens, b0, p.S) : 0;
  int vis_min = ns, vis_max = ns;                 // suffix keys the block's first / last row sees
  if (pt.suffix && p.causal) {
    vis_min = min(ns, max(0, ns - p.Lq + row0 / p.rep + 1));
    vis_max = min(ns, max(0, ns - p.Lq + (row_end - 1) / p.rep + 1));
  }
  const int ptiles = (np + KT - 1) / KT, tiles = ptiles + (vis_max + KT - 1) / KT;
  const int t0 = (int)((long long)tiles * it.split / nsplit), t1 = (int)((long long)tiles * (it.split + 1) / nsplit);

  f16x8 qf[QT][STEPS];
  long long rowid[QT];
  int vis[QT];
  char* optr[QT];
  f32x4 oacc[QT][DT];
  PaRows<QT> run;
  pa_rows_start(run, oacc);
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int rl = qt * 16 + lc, r = row0 + rl;
    const bool ok = r < pt.rows;
    const PaRow w = pa_row(p.Lq, p.rep, pt.nper, it.space, hk, ok ? r : 0);
    rowid[qt] = !ok ? -1 : whole ? 0 : pt.by_row ? ((long long)w.b * p.Lq + w.i) * p.Hq + w.h : (long long)(it.item - pt.whole) * (16 * QT) + rl;
    vis[qt] = p.causal ? max(0, ns - p.Lq + w.i + 1) : ns;
    optr[qt] = p.out + (w.b * p.os[0] + w.i * p.os[1] + w.h * p.os[2]) * 2;
    const T* qp = reinterpret_cast<const T*>(p.q) + w.b * p.qs[0] + w.i * p.qs[1] + w.h * p.qs[2];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      f16x8 f = *reinterpret_cast<const f16x8*>(qp + (s * 4 + lg) * 8);
      if (p.qsign != 1.f) f *= (T)p.qsign;
      qf[qt][s] = f;
    }
  }

  u32x4 kf[C::DEPTH][2][STEPS], vr[C::DEPTH][VL];
  auto keys_of = [&](int t) { return t >= t1 ? 0 : t < ptiles ? min(KT, np - t * KT) : min(KT, vis_max - (t - ptiles) * KT); };
  // (issued for every chunk, those past the last one with an empty descriptor: with a load that may or may not be there the wait for an older
  // one would be a wait for all)
  auto load = [&](int t, int set) {
    const bool pre = t < ptiles;
    const long long j0 = t < t1 ? (long long)(pre ? t : t - ptiles) * KT : 0;
    const long long kts = pre ? p.pks[1] : p.ks[1], vts = pre ? p.pvs[1] : p.vs[1];
    const T* kb = pre ? reinterpret_cast<const T*>(p.pk) + g * p.pks[0] + hk * p.pks[2] : reinterpret_cast<const T*>(p.k) + b0 * p.ks[0] + hk * p.ks[2];
    const T* vb = pre ? reinterpret_cast<const T*>(p.pv) + g * p.pvs[0] + hk * p.pvs[2] : reinterpret_cast<const T*>(p.v) + b0 * p.vs[0] + hk * p.vs[2];
    const unsigned kp = (unsigned)kts * 2, vp = (unsigned)vts * 2;
    const int n = keys_of(t);
    const __amdgpu_buffer_rsrc_t rk = uniform_buffer_rsrc(kb + j0 * kts, n > 0 ? (int)((n - 1) * kp + D * 2) : 0);
    const __amdgpu_buffer_rsrc_t rv = uniform_buffer_rsrc(vb + j0 * vts, n > 0 ? (int)((n - 1) * vp + D * 2) : 0);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int key = kt * 16 + lc;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        kf[set][kt][s] = __builtin_amdgcn_raw_buffer_load_b128(rk, (int)(key * kp + (s * 4 + lg) * 16), 0, 0);
    }
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int key = (i * 64 + lane) / SLOTS, sl = lane % SLOTS;
      vr[set][i] = __builtin_amdgcn_raw_buffer_load_b128(rv, (int)(key * vp + sl * 16), 0, 0);
    }
  };
  auto chunk = [&](int t, int set) {
    // V of the chunk: rows into the wave's own LDS (its earlier reads are ahead of these writes in the LDS queue)
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int key = (i * 64 + lane) / SLOTS, sl = lane % SLOTS;
      const u32x4 v = key & 4 ? u32x4{vr[set][i][2], vr[set][i][3], vr[set][i][0], vr[set][i][1]} : vr[set][i];
      *reinterpret_cast<u32x4*>(&Vs[key * D + v_slot<D>(key, sl) * 8]) = v;
    }
    // its operands, all requested here: they arrive during the scores and the softmax (read one by one ahead of each product they made up most
    // of a chunk's time)
    f16x8 vf[DT];
    {
      const int key = lg * 4 + (lc >> 2);
      const _Float16* vb = Vs + key * D;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int at = v_slot<D>(key, (d >> 1) * 4 + (lane & 3)) * 8 + (((d & 1) ^ ((key >> 2) & 1)) << 2);
        const f16x4 v0 = lds_read_tr16(vb + at);
        const f16x4 v1 = lds_read_tr16(vb + 16 * D + at);
        vf[d] = f16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    f32x4 sacc[QT][2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        sacc[qt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
          sacc[qt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, kf[set][kt][s]), qf[qt][s], sacc[qt][kt], 0, 0, 0);
      }
    const int n = keys_of(t), j0 = (t - ptiles) * KT;
    const bool cut = p.causal && t >= ptiles && j0 + n > vis_min;
    f16x8 pfr[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      if (n < KT || cut) {
        const int most = cut ? min(n, vis[qt] - j0) : n;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (kt * 16 + lg * 4 + r >= most) sacc[qt][kt][r] = -INFINITY;
      }
      float tmax = sacc[qt][0][0];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) tmax = fmaxf(tmax, sacc[qt][kt][r]);
      tmax = rows_max(tmax);
      const float m_new = fmaxf(run.m[qt], tmax), base = pa_base<T>(m_new, p.sc2, sacc[qt]);
      float psum = 0.f;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(fmaf(sacc[qt][kt][r], p.sc2, base));
          psum += e;
          pfr[qt][kt * 4 + r] = (_Float16)e;             // weights in the values' type: the product's operand
        }
      pa_rows_add(run, oacc, qt, m_new, psum, p.sc2);
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) oacc[qt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[d], pfr[qt], oacc[qt][d], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    load(t + 4 * C::DEPTH, set);
  };
#pragma unroll
  for (int i = 0; i < C::DEPTH; ++i) load(t0 + wave + 4 * i, i);
  for (int t = t0 + wave; t < t1; t += 4 * C::DEPTH) {
    chunk(t, 0);
    if constexpr (C::DEPTH == 2) chunk(t + 4, 1);         // (a chunk past the last one has no keys)
  }
  __syncthreads();                                         // every wave is done with its V rows: the join takes their place
  pa_join_waves<T, D, QT>(p, pt, lds, wave_ml, oacc, run, rowid, optr, whole, it.split, t0 < t1);
#endif
}

// the form of a part: see PaPlan
template <typename T, int D, int QT, bool WK> constexpr int pa_lds_bytes() { return WK && sizeof(T) == 2 ? PaStream<D, QT>::BYTES : PaLds<T, D, QT, WK>::BYTES; }
template <typename T, int D, int QT, bool WK>
__device__ __forceinline__ void pa_run(const PaParams& p, const PaPart& pt, const int bid, char* lds, float* wave_ml) {
  if constexpr (WK && sizeof(T) == 2) pa_stream_block<D, QT>(p, pt, bid, lds, wave_ml);
  else pa_block<T, D, QT, WK>(p, pt, bid, lds, wave_ml);
}

// waves a SIMD the registers are to allow: two blocks a CU, but for fp32 heads of 128 in two row tiles, which do not fit
template <typename T, int D, int QT> constexpr int pa_waves() { return sizeof(T) == 4 && D == 128 && QT == 2 ? 1 : 2; }

template <typename T, int D, int QT, bool WK>
__global__ __launch_bounds__(256, (pa_waves<T, D, QT>())) void pa_tile_kernel(const PaParams p) {
  __shared__ __attribute__((aligned(16))) char lds[(pa_lds_bytes<T, D, QT, WK>())];
  __shared__ float wave_ml[WK ? 4 * 16 * QT * 2 : 1];
  pa_run<T, D, QT, WK>(p, p.part[0], (int)blockIdx.x, lds, wave_ml);
}
template <typename T, int D, int QT0, bool WK0, int QT1, bool WK1>
__global__ __launch_bounds__(256, (pa_waves<T, D, (QT0 > QT1 ? QT0 : QT1)>())) void pa_pair_kernel(const PaParams p) {
  constexpr int B0 = pa_lds_bytes<T, D, QT0, WK0>(), B1 = pa_lds_bytes<T, D, QT1, WK1>();
  __shared__ __attribute__((aligned(16))) char lds[B0 > B1 ? B0 : B1];
  __shared__ float wave_ml[4 * 16 * 2 * 2];
  if ((int)blockIdx.x < p.part[1].blocks) pa_run<T, D, QT1, WK1>(p, p.part[1], (int)blockIdx.x, lds, wave_ml);
  else pa_run<T, D, QT0, WK0>(p, p.part[0], (int)blockIdx.x - p.part[1].blocks, lds, wave_ml);
}

// One wave per split row: the slots' outputs, weighted by exp2(max - common max), over the weighted sum.  A slot without keys (sum 0) left no output:
// what the scratch holds there is read and dropped.
template <typename T, int D>
__global__ __launch_bounds__(256) void pa_join_kernel(const PaParams p, const int per) {
  const int lane = threadIdx.x & 63;
  const PaPart& pt = p.part[0];
  for (long long row = blockIdx.x * 4ll + (threadIdx.x >> 6); row < p.prows; row += gridDim.x * 4ll) {
    PaRow w;
    if (pt.by_row) {
      w = {(int)(row / p.Hq / p.Lq), (int)(row / p.Hq % p.Lq), (int)(row % p.Hq)};
    } else {
      const int item = pt.whole + (int)(row / per), rb = item % pt.rowblocks, r = rb * per + (int)(row % per);
      if (r >= pt.rows) continue;
      w = pa_row(p.Lq, p.rep, pt.nper, item / pt.rowblocks / p.Hkv, item / pt.rowblocks % p.Hkv, r);
    }
    constexpr int E = D / 64, U = 8;
    float m = PA_NONE, l = 0.f;                      // slots <= 64: one a lane
    if (lane < p.slots) {
      const float2 e = *reinterpret_cast<const float2*>(p.part_ml + (lane * p.prows + row) * 2);
      m = e.x;
      l = e.y;
    }
    float mj = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mj = fmaxf(mj, __shfl_xor(mj, o));
    const float wt = l != 0.f ? __builtin_amdgcn_exp2f((m - mj) * p.sc2) : 0.f;
    float total = l != 0.f ? l * wt : 0.f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    const float* src = p.part_o + row * D + lane * E;
    for (int s0 = 0; s0 < p.slots; s0 += U) {
      float v[U][E];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) v[u][e] = src[(long long)min(s0 + u, p.slots - 1) * p.prows * D + e];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int sl = min(s0 + u, 63);
        const float ls = __shfl(l, sl), ws = __shfl(wt, sl);       // (lanes past the last slot: sum 0; a NaN sum is not 0 and stays)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = s0 + u < p.slots && ls != 0.f ? fmaf(ws, v[u][e], acc[e]) : acc[e];
      }
    }
    T* o = reinterpret_cast<T*>(p.out) + w.b * p.os[0] + w.i * p.os[1] + w.h * p.os[2] + pa_channel<sizeof(T) == 2>(lane * E);
    const float inv = total != 0.f ? 1.f / total : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = from_f32<T>(acc[e] * inv);
  }
}

// ---- the plan of a call: which parts, which tile form, how many key splits.  A function of sizes and types alone (lengths stay on the device).
struct PaPlan {
  int nparts, slots;
  long long prows;       // rows of the scratch
  PaPart part[2];
  int qt[2], wk[2];
  bool ok;
};

constexpr int PA_SLOTS = 512;         // blocks that run at a time: two a CU
constexpr long long PA_JOIN_ROWS = 1 << 24;      // rows a join launch has waves for (a grid has less than 2^32 threads); more take turns

// two row tiles a wave where they leave two blocks a CU (fp32 heads of 128: 24 sequences of 413 queries over 77 + 622 keys 74 us with two, 50 with one)
constexpr bool pa_two_row_tiles(int esz, int D) { return !(esz == 4 && D == 128); }

inline PaPlan pa_plan(const pp_prefix_attn_args_t* a) {
  PaPlan r{};
  r.ok = true;
  const int nseq = a->B / a->G, rep = a->Hq / a->Hkv, esz = a->dtype == PP_F16 ? 2 : 4;
  const long long R = (long long)a->Lq * rep;
  // rows of several sequences are packed where one sequence's do not fill a tile and re-reading the prefix for each would move 16 MB or more
  const bool packed = a->P > 0 && nseq > 1 && R <= 32 && (long long)(a->B - a->G) * a->Hkv * a->P * a->D * 2 * esz >= (16 << 20);
  auto add = [&](int nper, int prefix, int suffix, int most, bool both) {
    const int i = r.nparts++;
    PaPart& t = r.part[i];
    t.nper = nper; t.prefix = prefix; t.suffix = suffix; t.by_row = both;
    t.rows = (int)(R * nper);
    r.wk[i] = t.rows <= 32;
    r.qt[i] = t.rows <= 16 ? 1 : t.rows <= 32 ? 2 : t.rows <= 64 || !pa_two_row_tiles(esz, a->D) ? 1 : 2;
    const int per = 16 * r.qt[i] * (r.wk[i] ? 1 : 4);
    t.rowblocks = ceil_div(t.rows, per);
    const long long items = (long long)(a->B / nper) * a->Hkv * t.rowblocks;
    if (items > (1 << 22)) { r.ok = false; return; }
    t.items = (int)items;
    const int kt = a->dtype == PP_F16 && r.wk[i] ? 128 : 64;
    const int tiles = (prefix ? ceil_div(a->P, kt) : 0) + (suffix ? ceil_div(a->S, kt) : 0);
    // items that fill whole rounds walk their keys alone; those of the last, incomplete round are split until it is full too, four tiles a block at least
    const int rest = both ? t.items : t.items % PA_SLOTS;
    int n = rest > 0 ? most / rest : 1;
    const int least = r.wk[i] ? 1 : a->dtype == PP_F16 ? 4 : 2;
    if (n > tiles / least) n = tiles / least;
    if (!both && tiles < 8) n = 1;      // (a second launch costs more than what is left to split)
    if (n > 32) n = 32;
    if (n < 1) n = 1;
    t.nsplit = n;
    t.whole = both ? 0 : n == 1 ? t.items : t.items - rest;
    t.slot0 = r.slots;
    t.blocks = t.whole + (t.items - t.whole) * n;
    if (both) r.prows = (long long)a->B * a->Lq * a->Hq;
    else r.prows = (long long)(t.items - t.whole) * per;
    if (t.whole < t.items) r.slots += n;
  };
  if (packed && a->S > 0) {
    add(1, 0, 1, PA_SLOTS, true);
    // Blocks for the packed rows: every split leaves outputs to join, and their blocks take the place of suffix walks, so no more than finish their
    // products while the suffixes (taken as half full: the plan knows sizes, the lengths stay on the device) come out of memory, and at most one a CU.  A tile's products take about 2 us (two fp16
    // row tiles of 16; fp32 four times that), the suffixes come at 4.3 TB/s.  Against 256 always (us): 64 sequences behind 8192 keys, suffixes up to
    // 1024: 54 / 64.5, behind 2048: 46 / 50; 16 sequences behind 32768 keys, suffixes up to 512, where 128 blocks are too few: 50 with 256, 71.5.
    const long long prows = R * nseq;
    const long long units = ((prows + 63) / 64) * a->G * a->Hkv * ceil_div(a->P, 64) * (esz == 2 ? 1 : 4);      // us of products
    const long long suffix = (long long)a->B * a->Hkv * a->S * a->D * esz / 4300000 + 1;                        // us of half of the suffix bytes
    long long most = (units + suffix - 1) / suffix;
    if (most < 32) most = 32;
    if (most > PA_SLOTS / 2) most = PA_SLOTS / 2;
    add(nseq, 1, 0, (int)most, true);
  } else if (packed) {
    add(nseq, 1, 0, PA_SLOTS, false);
  } else {
    add(1, a->P > 0, a->S > 0, PA_SLOTS, false);
  }
  return r;
}
inline int64_t pa_scratch(const PaPlan& plan, int D) { return plan.slots * plan.prows * (D + 2) * 4; }

template <typename T, int D>
static void pa_launch(const PaPlan& plan, const PaParams& p, hipStream_t st) {
  const dim3 block(256);
  constexpr bool TWO = pa_two_row_tiles((int)sizeof(T), D);
  if (plan.nparts == 2) {
    const dim3 grid((unsigned)(plan.part[0].blocks + plan.part[1].blocks));
    const int form = plan.wk[1] ? plan.qt[1] - 1 : 1 + plan.qt[1];      // of the packed part: wk 1, wk 2, rows 1, rows 2; the suffix part is always wk
#define PA_PAIR(Q0, Q1, W1) hipLaunchKernelGGL((pa_pair_kernel<T, D, Q0, true, Q1, W1>), grid, block, 0, st, p)
    if (plan.qt[0] == 1) {
      if (form == 0) PA_PAIR(1, 1, true);
      else if (form == 1) PA_PAIR(1, 2, true);
      else if (form == 2) PA_PAIR(1, 1, false);
      else if constexpr (TWO) PA_PAIR(1, 2, false);
    } else {
      if (form == 2) PA_PAIR(2, 1, false);
      else if constexpr (TWO) PA_PAIR(2, 2, false);
    }
#undef PA_PAIR
  } else {
    const dim3 grid((unsigned)plan.part[0].blocks);
    if (plan.wk[0]) {
      if (plan.qt[0] == 1) hipLaunchKernelGGL((pa_tile_kernel<T, D, 1, true>), grid, block, 0, st, p);
      else hipLaunchKernelGGL((pa_tile_kernel<T, D, 2, true>), grid, block, 0, st, p);
    } else {
      if (plan.qt[0] == 1) hipLaunchKernelGGL((pa_tile_kernel<T, D, 1, false>), grid, block, 0, st, p);
      else if constexpr (TWO) hipLaunchKernelGGL((pa_tile_kernel<T, D, 2, false>), grid, block, 0, st, p);
    }
  }
  if (plan.slots > 0)
    hipLaunchKernelGGL((pa_join_kernel<T, D>), dim3((unsigned)(plan.prows < PA_JOIN_ROWS ? (plan.prows + 3) / 4 : PA_JOIN_ROWS / 4)), block, 0, st, p, 16 * plan.qt[0] * (plan.wk[0] ? 1 : 4));
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
  if (rc != 0) return rc;
  if (a->B == 0 || a->Lq == 0) return 0;
  const PaPlan plan = pa_plan(a);
  PP_REQUIRE(plan.ok, PP_ERR_ARG, "pp_shared_prefix_attention: too many blocks of work");
  return pa_scratch(plan, a->D);
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
  if (need < 0) return (int)need;
  PP_REQUIRE(need == 0 || (a->work != nullptr && a->work_bytes >= need && (uintptr_t)a->work % 16 == 0), PP_ERR_WORKSPACE,
             "pp_shared_prefix_attention: needs %lld bytes of 16-byte aligned scratch, got %lld", (long long)need, (long long)a->work_bytes);
  PaParams p;
  p.q = (const char*)a->q; p.pk = (const char*)a->pk; p.pv = (const char*)a->pv; p.k = (const char*)a->k; p.v = (const char*)a->v;
  p.out = (char*)a->out; p.plens = a->prefix_lens; p.lens = a->lens;
  const int64_t* from[6] = {a->q_stride, a->pk_stride, a->pv_stride, a->k_stride, a->v_stride, a->out_stride};
  long long* to[6] = {p.qs, p.pks, p.pvs, p.ks, p.vs, p.os};
  for (int t = 0; t < 6; ++t)
    for (int i = 0; i < 3; ++i) to[t][i] = from[t][i];
  // (the stride of a single token is free: keys past it have to lie outside)
  if (a->P <= 1) p.pks[1] = p.pvs[1] = a->D;
  if (a->S <= 1) p.ks[1] = p.vs[1] = a->D;
  p.B = a->B; p.G = a->G; p.nseq = a->B / a->G; p.Lq = a->Lq; p.Hq = a->Hq; p.Hkv = a->Hkv; p.rep = a->Hq / a->Hkv; p.P = a->P; p.S = a->S;
  p.causal = a->causal;
  p.sc2 = a->scale != 0.f ? fabsf(a->scale) * 1.4426950408889634f : 1.f;
  p.qsign = a->scale > 0.f ? 1.f : a->scale < 0.f ? -1.f : 0.f;
  const PaPlan plan = pa_plan(a);
  p.slots = plan.slots;
  p.prows = plan.prows;
  p.part[0] = plan.part[0];
  p.part[1] = plan.part[1];
  p.part_o = (float*)a->work;
  p.part_ml = (float*)a->work + plan.slots * plan.prows * a->D;
  hipStream_t st = (hipStream_t)stream;
  if (a->dtype == PP_F16) {
    if (a->D == 128) pa_launch<_Float16, 128>(plan, p, st);
    else pa_launch<_Float16, 64>(plan, p, st);
  } else {
    if (a->D == 128) pa_launch<float, 128>(plan, p, st);
    else pa_launch<float, 64>(plan, p, st);
  }
  return launch_status("pp_shared_prefix_attention");
}
