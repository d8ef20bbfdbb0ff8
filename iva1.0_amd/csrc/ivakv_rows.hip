// Attention of blocks of query rows over pages that every row of the block sees, for gfx950:
// cross attention (a decoder's rows over an encoder's states of another length) and decode
// attention of sequences that share their first pages.
//
// A unit is (group, kv head).  Its rows are the group's query rows times the G = Hq / Hkv
// heads of the kv head, r = i * G + g; its keys are the group's shared pages:
//   cross    rows query_start[b] .., keys 0 .. context_lens[b] - 1 of sequence b
//   prefix   rows group_start[g] .. (one per sequence), the full pages of the first
//            prefix_lens[g] tokens, which the sequences' tables have in common
// No mask depends on the row, so a page's K and V enter registers once and serve every row
// block of the wave:
//   S^T[key][row]  = K_page(16 x D) . Q^T(D x 16)          v_mfma 16x16x32, per page
//   O^T[dim][row] += V^T_pair(D x 32) . P^T(32 x 16)       v_mfma 16x16x32, per two pages
// The pools' page layout is the operand layout, and the lanes' scores (keys 4 (l / 16) .. + 3 of
// both pages) are the PV product's B operand, so nothing passes through LDS but the end of
// the walk.  The softmax runs online in fp32 in the log2 domain.
//
// Split: a workgroup takes a chunk of 16 NR rows and a segment of the unit's pages, its waves the page
// pairs in turn; their states meet in LDS and leave one partial (running max, sum, unnormalized
// rows).  Segments are sized on the device from the groups' pages, so that ragged groups fill the
// CUs evenly.  The prefix op's own pages are walked in the same launch by workgroups behind those:
// waves with equal shares of all (sequence, kv head, page pair) tiles, as the decode walk has them.  A
// second launch joins a row's partials.
//
// Bound: the K and V bytes of the shared pages, read once for up to 16 NR rows, and of the own
// pages; from a few hundred rows on the matrix and vector pipes (4 D operations per key and row).
// Measured per call, 32 / 8 heads of 128: 16 rows behind 8192 shared tokens (fp16, 50 MB) 19.3 us; 9
// ragged groups (bf16, 277 MB) 71 us, 3.9 TB/s; 64 rows behind 4000 tokens on FP8 pages (149 MB) 53 us;
// 256 rows behind 16384 120 us; beams of 5 rows on 16 sequences of 301 .. 1500 keys (60 MB) 18.3 us.  16
// heads of 64: 16 sequences of 97 .. 448 rows on 700 .. 1500 keys 40 us, 445 TFLOP/s, by the vector pipe.
#include <type_traits>

#include "ivakv_rows.h"

namespace ivakv {
namespace {

// Log2-domain headroom of the lazy row max, as in the prefill: p = exp2(s - m) stays <= 2^8.
constexpr float kLazyMax = 8.f;

// Register tile of one page (lane = 16 lq + ln) and its products, for pools of the queries' type.
template <int DT, int D, bool kFp8>
struct PageOps {
  using Tr = Traits<DT>;
  using E = typename Tr::E;
  using VChunk = typename Tr::VChunk;
  static constexpr int kPages = DT == IVAKV_F32 ? 1 : 2;  // pages of one PV product
  static constexpr int X = 16 / (int)sizeof(E);
  static constexpr int NQ = D / X / 4;   // 16-byte query chunks per lane
  static constexpr int NB = D / 16;
  static constexpr int64_t kTile = (int64_t)D * kBS;
  struct QReg {
    Chunk16 c[NQ];
  };
  static constexpr int VW = (int)sizeof(VChunk) / 4;  // words of four keys of one dim
  // The pages of one PV product: per page the K words, and per dim block the V words of all pages
  // (keys 4lq .. 4lq+3 of page 0, then of page 1), the operand in order.
  struct Set {
    uint32_t k[kPages][4 * NQ];
    uint32_t v[NB][VW * kPages];
  };
  // Element of the row that chunk j of lane group lq starts at.
  static IVAKV_INLINE __device__ inline int q_at(int j, int lq) { return (4 * j + lq) * X; }
  // (The empty asm keeps the loads here, ahead of their first use.)
  template <bool NT>
  static IVAKV_INLINE __device__ inline void load_k(const RowArgs& a, int id, int h, int g, int ln, int lq, Set& t) {
    const E* kp = static_cast<const E*>(a.k_pool) + ((int64_t)id * a.Hkv + h) * kTile;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      const Chunk16 c = ld<NT, Chunk16>(kp + ((4 * j + lq) * kBS + ln) * X);
#pragma unroll
      for (int i = 0; i < 4; ++i) t.k[g][4 * j + i] = c.w[i];
    }
    __asm__ volatile("" ::: "memory");
  }
  template <bool NT>
  static IVAKV_INLINE __device__ inline void load_v(const RowArgs& a, int id, int h, int g, int ln, int lq, Set& t) {
    const E* vp = static_cast<const E*>(a.v_pool) + ((int64_t)id * a.Hkv + h) * kTile;
#pragma unroll
    for (int m = 0; m < NB; ++m) {
      const VChunk c = ld<NT, VChunk>(vp + (16 * m + ln) * kBS + 4 * lq);
#pragma unroll
      for (int i = 0; i < VW; ++i) t.v[m][VW * g + i] = c.w[i];
    }
    __asm__ volatile("" ::: "memory");
  }
  static IVAKV_INLINE __device__ inline Chunk16 key(const Set& t, int g, int j) {
    return Chunk16{{t.k[g][4 * j], t.k[g][4 * j + 1], t.k[g][4 * j + 2], t.k[g][4 * j + 3]}};
  }
  static IVAKV_INLINE __device__ inline void mask_v(Set& t, int g, const bool vis[4]) {
    uint32_t keep[VW];
    if constexpr (VW == 2) {
      keep[0] = (vis[0] ? 0x0000FFFFu : 0u) | (vis[1] ? 0xFFFF0000u : 0u);
      keep[1] = (vis[2] ? 0x0000FFFFu : 0u) | (vis[3] ? 0xFFFF0000u : 0u);
    } else {
#pragma unroll
      for (int i = 0; i < VW; ++i) keep[i] = vis[i] ? ~0u : 0u;
    }
#pragma unroll
    for (int m = 0; m < NB; ++m)
#pragma unroll
      for (int i = 0; i < VW; ++i) t.v[m][VW * g + i] &= keep[i];
  }
};

// FP8 pages (e4m3fn codes, value = code / factor; layouts as in the decode walk): codes become
// the queries' type exactly for QK, 1 / factor of a key joins its scores and its weight.  The
// PV product is bf16 for either query type: a weight over a factor can leave fp16's range.
template <int DT, int D>
struct PageOps<DT, D, true> {
  using Tr = Traits<DT>;
  using E = typename Tr::E;
  static constexpr int kPages = 2;
  static constexpr int NQ = D / 32;
  static constexpr int NB = D / 16;
  static constexpr int KL = D / 64;
  static constexpr int64_t kTile = (int64_t)D * kBS;
  struct QReg {
    Chunk16 c[NQ];
  };
  struct Set {
    uint32_t k[2][4 * KL];
    uint32_t v[NB][2];  // keys 4lq .. 4lq+3 of dim 16m + ln, per page
    float ks[2][4], vs[2][4];
  };
  static IVAKV_INLINE __device__ inline int q_at(int j, int lq) { return 16 * (4 * (j >> 1) + lq) + 8 * (j & 1); }
  template <bool NT>
  static IVAKV_INLINE __device__ inline void load_k(const RowArgs& a, int id, int h, int g, int ln, int lq, Set& t) {
    const int64_t tile = (int64_t)id * a.Hkv + h;
    const uint8_t* kp = static_cast<const uint8_t*>(a.k_pool) + tile * kTile;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const Chunk16 c = ld<NT, Chunk16>(kp + ((4 * i + lq) * kBS + ln) * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) t.k[g][4 * i + j] = c.w[j];
    }
    const f32x4 f = ld<NT, f32x4>(a.k_scale + tile * kBS + 4 * lq);
#pragma unroll
    for (int r = 0; r < 4; ++r) t.ks[g][r] = f[r];
    __asm__ volatile("" ::: "memory");
  }
  template <bool NT>
  static IVAKV_INLINE __device__ inline void load_v(const RowArgs& a, int id, int h, int g, int ln, int lq, Set& t) {
    const int64_t tile = (int64_t)id * a.Hkv + h;
    const uint8_t* vp = static_cast<const uint8_t*>(a.v_pool) + tile * kTile + fp8_v_offset(ln, 4 * lq, D);
#pragma unroll
    for (int m = 0; m < NB; m += 4) {
      const Chunk16 c = ld<NT, Chunk16>(vp + 4 * m);
#pragma unroll
      for (int j = 0; j < 4; ++j) t.v[m + j][g] = c.w[j];
    }
    const f32x4 f = ld<NT, f32x4>(a.v_scale + tile * kBS + 4 * lq);
#pragma unroll
    for (int r = 0; r < 4; ++r) t.vs[g][r] = f[r];
    __asm__ volatile("" ::: "memory");
  }
  static IVAKV_INLINE __device__ inline void mask_v(Set& t, int g, const bool vis[4]) {
    const uint32_t keep = (vis[0] ? 0xFFu : 0u) | (vis[1] ? 0xFF00u : 0u) | (vis[2] ? 0xFF0000u : 0u) |
                          (vis[3] ? 0xFF000000u : 0u);
#pragma unroll
    for (int m = 0; m < NB; ++m) t.v[m][g] &= keep;
#pragma unroll
    for (int r = 0; r < 4; ++r) t.vs[g][r] = vis[r] ? t.vs[g][r] : 1.f;  // (may be anything too)
  }
  // Operand j of the QK product: half of a 16-byte chunk of codes, in the queries' type.
  static IVAKV_INLINE __device__ inline Chunk16 key(const Set& t, int g, int j) {
    const uint32_t w0 = t.k[g][2 * j], w1 = t.k[g][2 * j + 1];
    return Chunk16{{cvt2<DT, false>(w0), cvt2<DT, true>(w0), cvt2<DT, false>(w1), cvt2<DT, true>(w1)}};
  }
  template <int T, bool HI>
  static IVAKV_INLINE __device__ inline uint32_t cvt2(uint32_t w) {
    if constexpr (T == IVAKV_F16)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  }
};

// What a walk reads of its unit: which logical pages, and which of their keys.
struct KeyList {
  const int32_t* row;  // block-table row
  int num_pages;
  int na, c0;          // list entry v: logical page v below na, then c0 + v - na
  int len, win_start, n_sink;  // keys < len, and >= win_start or < n_sink
  IVAKV_INLINE __device__ inline int page(int v) const { return v < na ? v : c0 + (v - na); }
  IVAKV_INLINE __device__ inline bool full(int lp) const {
    return lp * kBS + kBS <= len && (lp * kBS >= win_start || lp * kBS + kBS <= n_sink);
  }
  IVAKV_INLINE __device__ inline void visible(int lp, bool ok, int lq, bool vis[4]) const {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int pos = lp * kBS + 4 * lq + r;
      vis[r] = ok && pos < len && (pos >= win_start || pos < n_sink);
    }
  }
};

// kRegs: the registers of a lane that the kernel's occupancy leaves it.
template <int DT, int D, bool kFp8, int NR, int kRegs>
struct Walk {
  using Ops = PageOps<DT, D, kFp8>;
  using Tr = typename Ops::Tr;
  using E = typename Ops::E;
  static constexpr int NB = Ops::NB, PG = Ops::kPages;
  // 16-bit pages: the row sums come from the same rounded weights as the rows, by one more
  // product with ones, so the rounding of P (2^-9 relative in bf16, 2^-12 in fp16) cancels
  // where one key dominates.  FP8 and fp32 sum the weights in fp32.
  static constexpr bool kSumMfma = !kFp8 && DT != IVAKV_F32;
  // With many row blocks, or long rows, the rows' operands stay in LDS, in lane order (one copy per workgroup), and
  // leave their registers to the accumulators.
  static constexpr bool kQLds = NR >= 4 || (NR >= 2 && D * sizeof(E) >= 512);
  static constexpr int kQBytes = kQLds ? 16 * NR * D * (int)sizeof(E) : 0;
  typename Ops::QReg q[kQLds ? 1 : NR];
  const Chunk16* q_lds;
  f32x4 acc[NR][NB];
  f32x4 lacc[kSumMfma ? NR : 1];
  float m[NR], l[NR], grow_at[NR], neg_m[NR];
  float c, inv_c;  // |scale| log2(e)

  // Rows r0 .. r0 + 16 NR - 1 of n (row r: query row row0 + r / G, head r % G of kv head h).  Every
  // wave of the workgroup calls it; with kQLds it ends in a barrier.
  template <int W>
  IVAKV_INLINE __device__ inline void init(const RowArgs& a, int64_t row0, int n, int h, int r0, int wave,
                                           int ln, int lq, Chunk16* lds) {
    c = fmaxf(fabsf(a.scale_log2), 1.17549435e-38f);
    inv_c = 1.f / c;
    q_lds = lds + 16 * lq + ln;
    const int Hq = a.Hkv * a.G;
    // a negative scale negates q instead (exact)
    const uint32_t sign = a.scale_log2 >= 0.f ? 0u : sizeof(E) == 2 ? 0x80008000u : 0x80000000u;
    auto chunk = [&](int rb, int j) IVAKV_INLINE -> Chunk16 {
      const int r = min(r0 + 16 * rb + ln, n - 1);  // rows past the end repeat the last one
      const E* p = static_cast<const E*>(a.q) + ((row0 + r / a.G) * Hq + h * a.G + r % a.G) * D;
      Chunk16 x = *reinterpret_cast<const Chunk16*>(p + Ops::q_at(j, lq));
#pragma unroll
      for (int i = 0; i < 4; ++i) x.w[i] ^= sign;
      return x;
    };
    if constexpr (kQLds) {
      for (int rb = wave; rb < NR; rb += W)
#pragma unroll
        for (int j = 0; j < Ops::NQ; ++j) lds[(rb * Ops::NQ + j) * 64 + 16 * lq + ln] = chunk(rb, j);
    } else {
#pragma unroll
      for (int rb = 0; rb < NR; ++rb)
#pragma unroll
        for (int j = 0; j < Ops::NQ; ++j) q[rb].c[j] = chunk(rb, j);
    }
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
      m[rb] = grow_at[rb] = kNegInf;
      l[rb] = neg_m[rb] = 0.f;
      if constexpr (kSumMfma) lacc[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[rb][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (kQLds) __syncthreads();
  }
  IVAKV_INLINE __device__ inline Chunk16 row(int rb, int j) const {
    if constexpr (kQLds) return q_lds[(rb * Ops::NQ + j) * 64];
    else return q[rb].c[j];
  }

  using Scores = f32x4[NR][PG];
  // Raw products of the loaded K with the rows (FP8: over the keys' factors).
  IVAKV_INLINE __device__ inline void scores(const typename Ops::Set& t, Scores& s) {
#pragma unroll
    for (int i = 0; i < PG; ++i) {
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) s[rb][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < Ops::NQ; ++j) {
        const Chunk16 k = Ops::key(t, i, j);
#pragma unroll
        for (int rb = 0; rb < NR; ++rb) s[rb][i] = Tr::qk(k, row(rb, j), s[rb][i]);
      }
      if constexpr (kFp8) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float kf = __builtin_amdgcn_rcpf(t.ks[i][r]);
#pragma unroll
          for (int rb = 0; rb < NR; ++rb) s[rb][i][r] *= kf;
        }
      }
    }
  }

  // Scores -inf for page i's hidden keys, and zeroes their V.
  template <class I>
  IVAKV_INLINE __device__ inline void hide(Scores& s, typename Ops::Set& t, const KeyList& kl,
                                           const int (&lp)[PG], const bool (&ok)[PG], int lq, I) {
    constexpr int i = I::value;
    bool vis[4];
    kl.visible(lp[i], ok[i], lq, vis);
    Ops::mask_v(t, i, vis);
#pragma unroll
    for (int rb = 0; rb < NR; ++rb)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[rb][i][r] = vis[r] ? s[rb][i][r] : kNegInf;
  }

  // Folds the scores and the loaded V of PG pages (logical pages lp, ok[i] false: not attended).
  IVAKV_INLINE __device__ inline void fold(Scores& s, typename Ops::Set& t,
                                                            const KeyList& kl, const int (&lp)[PG],
                                                            const bool (&ok)[PG], int lq) {
    // Hidden keys (past the length, outside the window, on an invalid page) score -inf, and
    // their V, which may hold any bits, is zeroed; pages without any skip this (uniform).
    bool whole = true;
#pragma unroll
    for (int i = 0; i < PG; ++i) whole = whole && ok[i] && kl.full(lp[i]);
    if (!whole) {
      hide(s, t, kl, lp, ok, lq, std::integral_constant<int, 0>{});
      if constexpr (PG == 2) hide(s, t, kl, lp, ok, lq, std::integral_constant<int, 1>{});
    }
    // Lazy rescaling: a row's reference max moves, with a rescale of its sums, only when a
    // score passes it by more than kLazyMax; one test covers all row blocks.  (The maximum that
    // keeps a NaN is one instruction for two scores; fmaxf would quiet each score first: 16 sequences
    // of 97 .. 448 rows on 700 .. 1500 keys, 16 heads of 64, 49 us against 52.)
    bool grow = false;
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
      float mx = grow_at[rb];
#pragma unroll
      for (int i = 0; i < PG; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = __builtin_elementwise_maximum(mx, s[rb][i][r]);
      grow = grow || mx > grow_at[rb];
    }
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        float mx = kNegInf;
#pragma unroll
        for (int i = 0; i < PG; ++i)
          mx = fmaxf(fmaxf(mx, fmaxf(s[rb][i][0], s[rb][i][1])), fmaxf(s[rb][i][2], s[rb][i][3]));
        mx *= c;
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m_new = fmaxf(m[rb], mx);
        const float f = m_new == kNegInf ? 1.f : exp2_fast(m[rb] - m_new);
        // (the first keys of a walk find sums of zero: nothing to scale)
        if (__builtin_amdgcn_ballot_w64(m[rb] != kNegInf) != 0) {
          l[rb] *= f;
          if constexpr (kSumMfma) lacc[rb] *= f;
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[rb][b] *= f;
        }
        m[rb] = m_new;
        grow_at[rb] = (m_new + kLazyMax) * inv_c;
        neg_m[rb] = m_new == kNegInf ? 0.f : -m_new;
      }
    }
    if constexpr (kFp8) {
      float vf[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) vf[i][r] = __builtin_amdgcn_rcpf(t.vs[i][r]);
      Chunk16 hi[NR], lo[NR];
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        // A weight over its factor, as a pair of bf16 values (to about 16 bits).
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            const float p0 = exp2_fast(__builtin_fmaf(s[rb][i][r], c, neg_m[rb]));
            const float p1 = exp2_fast(__builtin_fmaf(s[rb][i][r + 1], c, neg_m[rb]));
            l[rb] += p0 + p1;
            const float w0 = p0 * vf[i][r], w1 = p1 * vf[i][r + 1];
            const uint32_t h2 = Traits<IVAKV_BF16>::pack2(w0, w1);
            hi[rb].w[2 * i + r / 2] = h2;
            lo[rb].w[2 * i + r / 2] = Traits<IVAKV_BF16>::pack2(w0 - __uint_as_float(h2 << 16),
                                                                w1 - __uint_as_float(h2 & 0xFFFF0000u));
          }
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const Chunk16 v{{Ops::template cvt2<IVAKV_BF16, false>(t.v[b][0]), Ops::template cvt2<IVAKV_BF16, true>(t.v[b][0]),
                         Ops::template cvt2<IVAKV_BF16, false>(t.v[b][1]), Ops::template cvt2<IVAKV_BF16, true>(t.v[b][1])}};
#pragma unroll
        for (int rb = 0; rb < NR; ++rb) {
          acc[rb][b] = Traits<IVAKV_BF16>::qk(v, hi[rb], acc[rb][b]);
          acc[rb][b] = Traits<IVAKV_BF16>::qk(v, lo[rb], acc[rb][b]);
        }
      }
    } else if constexpr (PG == 2) {
      typename Tr::PP8 p8[NR];
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        float pa[4], pb[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          pa[r] = exp2_fast(__builtin_fmaf(s[rb][0][r], c, neg_m[rb]));
          pb[r] = exp2_fast(__builtin_fmaf(s[rb][1][r], c, neg_m[rb]));
        }
        p8[rb] = Tr::pack_pp8(pa, pb);
        const uint32_t one = DT == IVAKV_F16 ? 0x3C003C00u : 0x3F803F80u;
        lacc[rb] = Tr::pv_pair(Chunk16{{one, one, one, one}}, p8[rb], lacc[rb]);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const Chunk16 v{{t.v[b][0], t.v[b][1], t.v[b][2], t.v[b][3]}};
#pragma unroll
        for (int rb = 0; rb < NR; ++rb) acc[rb][b] = Tr::pv_pair(v, p8[rb], acc[rb][b]);
      }
    } else {
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = exp2_fast(__builtin_fmaf(s[rb][0][r], c, neg_m[rb]));
        l[rb] += (p[0] + p[1]) + (p[2] + p[3]);
        const typename Tr::PVec pv = Tr::pack_p(p);
#pragma unroll
        for (int b = 0; b < NB; ++b)
          acc[rb][b] = Tr::pv(Chunk16{{t.v[b][0], t.v[b][1], t.v[b][2], t.v[b][3]}}, pv, acc[rb][b]);
      }
    }
  }

  // Sets of PG pages in flight in registers: two, or one where a second does not fit beside NR row
  // blocks; K of the set after next is loaded as soon as this set's scores are there, V as soon as
  // its rows are.
  static constexpr int kSetRegs = 2 * (int)sizeof(typename Ops::Set) / 4;
  static constexpr int kRowRegs = NR * (4 * NB + (kQLds ? 0 : 4 * Ops::NQ) + 4 * PG + 8);
  static constexpr int kSets = kSetRegs + kRowRegs <= (kRegs > 256 ? 300 : 180) ? 2 : 1;

  // Walks list entries [v0, v1) PG at a time: this wave the sets w, w + W, ...  Loads past the end
  // repeat the last entry and are not folded.
  template <bool NT, int W>
  IVAKV_INLINE __device__ inline void run(const RowArgs& a, const KeyList& kl, int h, int v0,
                                                           int v1, int w, int ln, int lq) {
    const int sets = (v1 - v0 + PG - 1) / PG;
    const int mine = sets > w ? (sets - w + W - 1) / W : 0;
    if (mine <= 0) return;
    typename Ops::Set t[kSets];
    int lp[kSets][PG], id[kSets][PG];
    bool ok[kSets][PG];
    auto issue_k = [&](int s, int i) IVAKV_INLINE {
#pragma unroll
      for (int g = 0; g < PG; ++g) {
        const int v = v0 + PG * (w + W * min(i, mine - 1)) + g;
        lp[s][g] = kl.page(min(v, v1 - 1));
        const int p = kl.row[lp[s][g]];
        const bool in_pool = (uint32_t)p < (uint32_t)kl.num_pages;
        ok[s][g] = v < v1 && i < mine && in_pool;
        id[s][g] = in_pool ? p : 0;
        Ops::template load_k<NT>(a, id[s][g], h, g, ln, lq, t[s]);
      }
    };
    auto issue_v = [&](int s) IVAKV_INLINE {
#pragma unroll
      for (int g = 0; g < PG; ++g) Ops::template load_v<NT>(a, id[s][g], h, g, ln, lq, t[s]);
    };
    auto step = [&](auto more, int s, int i) IVAKV_INLINE {
      Scores sc;
      scores(t[s], sc);
      int lp_now[PG];
      bool ok_now[PG];
#pragma unroll
      for (int g = 0; g < PG; ++g) {
        lp_now[g] = lp[s][g];
        ok_now[g] = ok[s][g];
      }
      if constexpr (decltype(more)::value) issue_k(s, i + kSets);
      fold(sc, t[s], kl, lp_now, ok_now, lq);
      if constexpr (decltype(more)::value) issue_v(s);
    };
    issue_k(0, 0);
    issue_v(0);
    int i = 0;
    if constexpr (kSets == 2) {
      issue_k(1, 1);
      issue_v(1);
      for (; i + 2 < mine; i += 2) {
        step(std::true_type{}, 0, i);
        step(std::true_type{}, 1, i + 1);
      }
      step(std::false_type{}, 0, i);
      if (i + 1 < mine) step(std::false_type{}, 1, i + 1);
    } else {
      for (; i + 1 < mine; ++i) step(std::true_type{}, 0, i);
      step(std::false_type{}, 0, i);
    }
  }

  // Row sum of row ln of a block.
  __device__ inline float total(int rb) const {
    if constexpr (kSumMfma) return lacc[rb][0];
    float t = l[rb] + __shfl_xor(l[rb], 16);
    return t + __shfl_xor(t, 32);
  }
};

// LDS of a workgroup's join: per wave and row max and sum, then the rows [wave][16 NR][D + 4].
template <int D, int NR, int W>
constexpr size_t join_floats() { return (size_t)W * 16 * NR * (2 + D + 4); }

// Brings the W waves' states to the rows' common max in LDS: afterwards s_fin holds (max, sum) of
// each row and the sum over the waves of s_acc its unnormalized elements.
template <class WalkT, int D, int NR, int W>
__device__ inline void join_waves(const WalkT& wk, float* smem, int wave, int ln, int lq, float* s_fin) {
  constexpr int R = 16 * NR;
  float* s_m = smem;
  float* s_l = smem + W * R;
  float* s_acc = smem + 2 * W * R;
#pragma unroll
  for (int rb = 0; rb < NR; ++rb) {
    const float t = wk.total(rb);
    if (lq == 0) {
      s_m[wave * R + 16 * rb + ln] = wk.m[rb];
      s_l[wave * R + 16 * rb + ln] = t;
    }
  }
  __syncthreads();
#pragma unroll
  for (int rb = 0; rb < NR; ++rb) {
    const int row = 16 * rb + ln;
    float M = kNegInf;
#pragma unroll
    for (int u = 0; u < W; ++u) M = fmaxf(M, s_m[u * R + row]);
    const float M_use = M == kNegInf ? 0.f : M;
    const float f = exp2_fast(wk.m[rb] - M_use);
    float* dst = s_acc + (wave * R + row) * (D + 4) + 4 * lq;
#pragma unroll
    for (int b = 0; b < D / 16; ++b) *reinterpret_cast<f32x4*>(dst + 16 * b) = wk.acc[rb][b] * f;
    if (wave == 0 && lq == 0) {
      float L = 0.f;
#pragma unroll
      for (int u = 0; u < W; ++u) L += s_l[u * R + row] * exp2_fast(s_m[u * R + row] - M_use);
      s_fin[2 * row] = M;
      s_fin[2 * row + 1] = L;
    }
  }
  __syncthreads();
}

// Workgroups of the walks: four waves of 256 registers, two workgroups per CU (a shared one and one
// of the own walk, say); rows of 512 bytes need 512 registers.
template <int DT, int D, bool kFp8, int NR>
struct Shape {
  static constexpr int kRow = D * (DT == IVAKV_F32 ? 4 : 2);  // bytes of a query row
  static constexpr bool kWide = kRow >= 512;
  static constexpr int W = 4;
  static constexpr int kRegs = kWide ? 512 : 256;
  using WalkT = Walk<DT, D, kFp8, NR, kRegs>;
  static constexpr int kLds = (int)(join_floats<D, NR, W>() * sizeof(float)) + WalkT::kQBytes;
};

// One segment of one group for a chunk of rows.
template <int DT, int D, bool kFp8, int NR, bool NT>
__device__ inline void shared_walk(const RowArgs& a, const int32_t* __restrict__ bt, int wg, float* smem,
                                   float* s_fin) {
  using S = Shape<DT, D, kFp8, NR>;
  using WalkT = typename S::WalkT;
  using E = typename WalkT::E;
  constexpr int R = 16 * NR, W = S::W;
  const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4;
  const int wave = uni(threadIdx.x >> 6);
  const Group own = load_group(a, lane);
  const Pieces pc(a, own, lane);
  // Each XCD takes a contiguous run of the workgroups, so that a piece's chunks are on one XCD, one
  // after the other (chunks past the first find the pages in its L2), and all groups of a kv head.
  const int n_wg = pc.items * a.Hkv;
  if (wg >= n_wg) return;
  wg = (int)xcd_contiguous_block(wg, n_wg);
  Group group;
  int g, piece, h, chunk, slot;
  if (!pc.find(a, own, wg, lane, group, g, piece, h, chunk, slot)) return;
  const int rows = min(group.r1 - group.r0, a.max_rows) * a.G;  // (at most n_rows * Hq, which the entry checks)
  KeyList kl;
  kl.num_pages = a.num_pages;
  kl.win_start = kl.n_sink = kl.na = kl.c0 = 0;
  int table = g;
  kl.len = group.pages * kBS;
  if (a.prefix) table = prefix_row(a, group.pages, group.r0, group.r1, lane);
  else kl.len = a.ctx[g];
  if (table < 0) return;
  kl.row = bt + (int64_t)table * a.max_blocks;
  const int v0 = piece * pc.len, v1 = min(v0 + pc.len, group.pages);
  WalkT wk;
  wk.template init<W>(a, group.r0, rows, h, chunk * R, wave, ln, lq,
                      reinterpret_cast<Chunk16*>(smem + join_floats<D, NR, W>()));
  wk.template run<NT, W>(a, kl, h, v0, v1, wave, ln, lq);
  join_waves<WalkT, D, NR, W>(wk, smem, wave, ln, lq, s_fin);
  const float* s_acc = smem + 2 * W * R;
  const bool whole = !a.prefix && pc.of(group) == 1;
  const int Hq = a.Hkv * a.G;
  for (int e = threadIdx.x; e < R * (D / 4); e += 64 * W) {
    const int row = e / (D / 4), d = 4 * (e % (D / 4)), r = chunk * R + row;
    if (r >= rows) break;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < W; ++u) o += *reinterpret_cast<const f32x4*>(s_acc + (u * R + row) * (D + 4) + d);
    if (whole) {
      const float L = s_fin[2 * row + 1], inv = L > 0.f ? 1.f / L : 0.f;
      E* dst = static_cast<E*>(a.out) + ((int64_t)(group.r0 + r / a.G) * Hq + h * a.G + r % a.G) * D + d;
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[i] = WalkT::Tr::from_float(o[i] * inv);
    } else {
      *reinterpret_cast<f32x4*>(a.part_acc + ((int64_t)slot * R + row) * D + d) = o;
      if (d == 0) *reinterpret_cast<f32x2*>(a.part_ml + ((int64_t)slot * R + row) * 2) = f32x2{s_fin[2 * row], s_fin[2 * row + 1]};
    }
  }
}

// The group that query row `row` (of this thread) belongs to: its pages (0: none) and first row.
__device__ inline int row_pages(const RowArgs& a, int row, int& r0) {
  int lo = 0, hi = a.n_groups;  // the last group that starts at or before the row
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.start[mid] <= row) lo = mid + 1;
    else hi = mid;
  }
  r0 = 0;
  if (lo == 0) return 0;
  const Group x = load_group(a, lo - 1);
  if (row < x.r0 || row >= x.r1 || row - x.r0 >= a.max_rows) return 0;
  r0 = x.r0;
  return x.pages;
}

// A sequence's own pages: of one that takes part in a shared walk those after the prefix, else all that
// its window and sinks leave.  `blocks`: shared pages of its group, 0 when it has none.
struct OwnPages {
  KeyList kl;
  int n;
  bool part;
  __device__ inline OwnPages(const RowArgs& a, int len, int blocks) {
    const PageWalk w = make_walk(len, a.window, a.n_sink, kBS);
    part = blocks > 0 && takes_part(a, len, blocks);
    kl.len = w.L;
    kl.num_pages = a.num_pages;
    if (part) {
      kl.win_start = kl.n_sink = kl.na = 0;
      kl.c0 = blocks;
      n = max(min(cdiv(w.L, kBS), a.max_blocks) - blocks, 0);
    } else {
      kl.win_start = w.win_start;
      kl.n_sink = a.n_sink;
      kl.na = w.sink_pages;
      kl.c0 = w.win_first;
      n = table_pages(w, a.max_blocks, kBS);
    }
  }
};

// Own walk: tile t of T is a set of PG own pages, in the order (sequence, kv head, set); wave k of W
// owns tiles [k T / W, (k + 1) T / W).  What it leaves of unit u (sequence * Hkv + kv head) goes to
// own slot k + u, which rises along the tiles.
struct OwnSplit {
  uint32_t T, W;
  __device__ inline OwnSplit(uint32_t tiles, const RowArgs& a) : T(tiles) {
    // two tiles a wave at least: a walk of one has nothing in flight beside it
    W = min(max((T + 1) / 2, 1u), (uint32_t)a.own_waves);
  }
  __device__ inline uint32_t start(uint32_t k) const { return div((uint64_t)k * T, W); }
  // The wave k with start(k) <= t < start(k + 1).
  __device__ inline uint32_t owner(uint32_t t) const { return div((uint64_t)(t + 1) * W - 1, T); }
  // (a 64-bit division takes long on the walk's way to its first load)
  static __device__ inline uint32_t div(uint64_t x, uint32_t y) {
    return x >> 32 == 0 ? (uint32_t)x / y : (uint32_t)(x / y);
  }
};

template <int DT, int D, bool kFp8, int kRegs>
__device__ inline void own_walk(const RowArgs& a, const int32_t* __restrict__ bt, int wg, int32_t* s_pref) {
  using WalkT = Walk<DT, D, kFp8, 1, kRegs>;
  constexpr int PG = WalkT::PG, W = 4;
  const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4;
  const int wave = uni(threadIdx.x >> 6);
  __shared__ int s_wave[W];
  // Prefix of the sequences' sets (a contiguous run per thread, a scan per wave, the waves' totals), with
  // their shared pages packed beside: s_pref[b] sets before b, s_pref[n + 1 + b] pages it shares.
  const int n = a.n_rows, each = (n + 64 * W - 1) / (64 * W);
  const int b0 = min((int)threadIdx.x * each, n), b1 = min(b0 + each, n);
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    int r0;
    const int blocks = row_pages(a, b, r0);
    const OwnPages own(a, a.ctx[b], blocks);
    const int sets = (own.n + PG - 1) / PG;
    s_pref[b + 1] = sets;
    s_pref[n + 1 + b] = own.part ? blocks : 0;
    mine += sets;
  }
  const int incl = wave_scan(mine);
  if (lane == 63) s_wave[wave] = incl;
  __syncthreads();
  int run = incl - mine;
  for (int w = 0; w < wave; ++w) run += s_wave[w];
  if (threadIdx.x == 0) s_pref[0] = 0;
  for (int b = b0; b < b1; ++b) {
    run += s_pref[b + 1];
    s_pref[b + 1] = run;
  }
  __syncthreads();
  if (wg == 0)
    for (int b = threadIdx.x; b <= n; b += 64 * W) a.own_pref[b] = s_pref[b];
  const uint32_t T = (uint32_t)uni(s_pref[n]) * (uint32_t)a.Hkv;
  if (T == 0) return;
  const OwnSplit split(T, a);
  const uint32_t k = (uint32_t)(wg * W + wave);
  if (k >= split.W) return;
  uint32_t t = split.start(k);
  const uint32_t end = split.start(k + 1);
  const int Hq = a.Hkv * a.G;
  // the last sequence with s_pref <= t / Hkv (it has sets)
  int b = 0, hi = n;
  const int key = (int)(t / (uint32_t)a.Hkv);
  while (hi - b > 1) {
    const int mid = (b + hi) >> 1;
    if (s_pref[mid] <= key) b = mid;
    else hi = mid;
  }
  b = uni(b);
  while (t < end) {
    while (s_pref[b + 1] == s_pref[b]) ++b;  // (a sequence without sets: some later one has, as t < T)
    b = uni(b);
    const uint32_t sets = (uint32_t)uni(s_pref[b + 1] - s_pref[b]), base = (uint32_t)uni(s_pref[b]) * (uint32_t)a.Hkv;
    const int h = (int)((t - base) / sets);
    const uint32_t first = base + (uint32_t)h * sets, stop = min(end, first + sets);
    OwnPages own(a, a.ctx[b], uni(s_pref[n + 1 + b]));
    own.kl.row = bt + (int64_t)b * a.max_blocks;
    const int v0 = (int)(t - first) * PG, v1 = min((int)(stop - first) * PG, own.n);
    const int64_t slot = (int64_t)k + (int64_t)b * a.Hkv + h;
    for (int g0 = 0; g0 < a.G; g0 += 16) {
      WalkT wk;
      wk.template init<1>(a, b, a.G, h, g0, 0, ln, lq, nullptr);
      wk.template run<true, 1>(a, own.kl, h, v0, v1, 0, ln, lq);
      const float l = wk.total(0);
      if (g0 + ln < a.G) {
        float* dst = a.own_acc + (slot * a.G + g0 + ln) * D + 4 * lq;
#pragma unroll
        for (int m = 0; m < D / 16; ++m) *reinterpret_cast<f32x4*>(dst + 16 * m) = wk.acc[0][m];
        if (lq == 0) *reinterpret_cast<f32x2*>(a.own_ml + (slot * a.G + g0 + ln) * 2) = f32x2{wk.m[0], l};
      }
    }
    t = stop;
    if (h == a.Hkv - 1 && stop == first + sets) ++b;
  }
}

// The walks: workgroups [0, shared_wgs) the shared segments, the others the own pages.
template <int DT, int D, bool kFp8, int NR, bool NT>
__global__ __launch_bounds__(256, (512 / Shape<DT, D, kFp8, NR>::kRegs)) void rows_walk_kernel(
    RowArgs a, const int32_t* __restrict__ bt) {
  extern __shared__ __align__(16) float smem[];
  __shared__ float s_fin[32 * NR];
  if ((int)blockIdx.x < a.shared_wgs) shared_walk<DT, D, kFp8, NR, NT>(a, bt, blockIdx.x, smem, s_fin);
  else own_walk<DT, D, kFp8, Shape<DT, D, kFp8, NR>::kRegs>(a, bt, blockIdx.x - a.shared_wgs,
                                                              reinterpret_cast<int32_t*>(smem));
}

// Log-sum-exp fold of one more state into (M, L, O).
__device__ inline void fold_state(float& M, float& L, f32x4& O, float m, float l, const f32x4& o) {
  const float mc = fmaxf(M, m), m_use = mc == kNegInf ? 0.f : mc;
  const float fa = exp2_fast(M - m_use), fb = exp2_fast(m - m_use);
  L = L * fa + l * fb;
  O = O * fa + o * fb;
  M = mc;
}

// Log-sum-exp fold of `count` partials at(i) (state index of a row) at elements d .. d + 3 into
// (M, L, O), U at a time.
template <int D, class At>
__device__ inline void fold_partials(const float* acc, const float* mls, int count, int d, At at, float& M,
                                     float& L, f32x4& O) {
  constexpr int U = 8;
  for (int s0 = 0; s0 < count; s0 += U) {
    f32x2 ml[U];
    f32x4 av[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = at(min(s0 + u, count - 1));
      ml[u] = *reinterpret_cast<const f32x2*>(mls + i * 2);
      av[u] = *reinterpret_cast<const f32x4*>(acc + i * D + d);
    }
    float mc = M;
#pragma unroll
    for (int u = 0; u < U; ++u) mc = fmaxf(mc, ml[u][0]);  // (a repeated one changes no max)
    const float m_use = mc == kNegInf ? 0.f : mc;
    const float f = exp2_fast(M - m_use);
    L *= f;
    O *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = exp2_fast(ml[u][0] - m_use);
      if (s0 + u < count) {
        L += ml[u][1] * w;
        O += av[u] * w;
      }
    }
    M = mc;
  }
}

// The join: a workgroup per (query row, kv head).  Its elements (four dims of a head) are dealt to
// as many threads each as there are, every one folding a run of the row's partials.
template <int DT, int D>
__global__ __launch_bounds__(256) void rows_join_kernel(RowArgs a) {
  using E = typename Traits<DT>::E;
  __shared__ float smem[6 * 256];
  const int h = blockIdx.x % a.Hkv, row = blockIdx.x / a.Hkv, lane = threadIdx.x & 63, tid = threadIdx.x;
  // (what does not wait for the group is loaded beside it; without an own walk, of any length)
  const bool walked = a.own_waves > 0;
  const int32_t* pref = walked ? a.own_pref : a.ctx;
  const uint32_t p0 = (uint32_t)pref[walked ? row : 0], p1 = (uint32_t)pref[walked ? row + 1 : 0];
  const uint32_t p_all = (uint32_t)pref[walked ? a.n_rows : 0];
  const int len = a.ctx[a.prefix ? row : 0];
  const Group mine = load_group(a, lane);
  // the group of the row (uniform)
  int g = -1, r0 = 0, pages = 0, chunks = 0;
  for (int g0 = 0; g0 < a.n_groups && g < 0; g0 += 64) {
    const Group x = g0 == 0 ? mine : load_group(a, g0 + lane);
    const uint64_t in = __builtin_amdgcn_ballot_w64(x.r0 <= row && row < x.r1);
    if (in != 0) {
      const int w = __builtin_ctzll(in);
      g = g0 + w;
      r0 = __builtin_amdgcn_readlane(x.r0, w);
      pages = __builtin_amdgcn_readlane(x.pages, w);
      chunks = __builtin_amdgcn_readlane(x.chunks, w);
    }
  }
  if (g >= 0 && row - r0 >= a.max_rows) g = -1;
  int64_t first = 0;
  int count = 0;
  if (!a.prefix) {
    if (g < 0) return;  // no sequence's row, or one the launch was not sized for: left as it is
    Pieces(a, mine, lane).of_group(a, mine, g, lane, first, count);
    if (count == 1) return;  // written by the walk
  } else if (g >= 0 && pages > 0 && takes_part(a, len, pages)) {
    Pieces(a, mine, lane).of_group(a, mine, g, lane, first, count);
  }
  // the own walk's partials: slots k + u of the waves that had tiles of this unit
  int64_t own_first = 0;
  int own_count = 0;
  if (walked) {
    const uint32_t sets = p1 - p0;
    if (sets > 0) {
      const OwnSplit split(p_all * (uint32_t)a.Hkv, a);
      const uint32_t t0 = p0 * (uint32_t)a.Hkv + (uint32_t)h * sets;
      const uint32_t k0 = split.owner(t0), k1 = split.owner(t0 + sets - 1);
      own_first = (int64_t)k0 + (int64_t)row * a.Hkv + h;
      own_count = (int)(k1 - k0) + 1;
    }
  }
  const int n_el = a.G * (D / 4), total = count + own_count;
  E* out = static_cast<E*>(a.out) + ((int64_t)row * a.Hkv + h) * a.G * D;
  int split = 1;
  while (split < 16 && 2 * split * n_el <= 256 && split < total) split *= 2;
  // partials [i0, i1) of one element: the shared ones, then the own
  auto fold = [&](int e, int i0, int i1, float& M, float& L, f32x4& O) IVAKV_INLINE {
    const int head = e / (D / 4), d = 4 * (e % (D / 4)), r = (row - r0) * a.G + head;
    const int at = r & ((1 << a.rows_shift) - 1);
    const int64_t slot = first + (int64_t)h * chunks + (r >> a.rows_shift), step = (int64_t)a.Hkv * chunks;
    const int s1 = min(i1, count), o0 = max(i0 - count, 0);
    fold_partials<D>(a.part_acc, a.part_ml, s1 - i0, d,
                     [&](int i) { return ((slot + (i0 + i) * step) << a.rows_shift) + at; }, M, L, O);
    fold_partials<D>(a.own_acc, a.own_ml, i1 - count - o0, d,
                     [&](int i) { return (own_first + o0 + i) * a.G + head; }, M, L, O);
  };
  auto emit = [&](int e, float L, const f32x4& O) IVAKV_INLINE {
    const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[4 * e + i] = Traits<DT>::from_float(O[i] * inv);
  };
  if (split == 1) {
    for (int e = tid; e < n_el; e += 256) {
      float M = kNegInf, L = 0.f;
      f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
      fold(e, 0, total, M, L, O);
      emit(e, L, O);
    }
    return;
  }
  const int e = tid % n_el, part = tid / n_el, each = (total + split - 1) / split;
  float M = kNegInf, L = 0.f;
  f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
  if (part < split) fold(e, min(part * each, total), min((part + 1) * each, total), M, L, O);
  if (part > 0 && part < split) {
    smem[6 * tid] = M;
    smem[6 * tid + 1] = L;
#pragma unroll
    for (int i = 0; i < 4; ++i) smem[6 * tid + 2 + i] = O[i];
  }
  __syncthreads();
  if (part > 0) return;
  for (int p = 1; p < split; ++p) {
    const float* x = smem + 6 * (tid + p * n_el);
    fold_state(M, L, O, x[0], x[1], f32x4{x[2], x[3], x[4], x[5]});
  }
  emit(e, L, O);
}

// Row blocks of a wave: as many as the rows need, up to what the registers hold beside the pages in
// flight.
constexpr int max_row_blocks(int row_bytes) { return row_bytes >= 1024 ? 1 : row_bytes >= 256 ? 2 : 4; }
int row_blocks(int row_bytes, int64_t rows) {
  const int most = max_row_blocks(row_bytes), want = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  return want < most ? want : most;
}

// The largest dynamic LDS a walk takes: the joins' 135 KiB, or the own walk's prefix of kMaxBatch rows.
constexpr int kMaxLds = 150 * 1024;
constexpr int kMaxBatch = 8192;

int num_cus() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1)
    cus = 256;
  return cus;
}

struct Plan {
  int nr, rows_chunk, chunks, items, own_waves;
  bool split, wide;
};

// Whether a group's shared walk goes through LDS in chunks of up to 256 rows (wide) rather than through
// the waves' own registers in chunks of 32.  It reads the pages from the L2 once for eight times the
// rows, but leaves a partial of all rows per piece and has one workgroup per CU to hide a piece's
// start and end.  So it takes cross attention where whole chunks need no cutting into pieces (bf16,
// D 128, walk : wide in us: 8 sequences of 200 x 2000, 32 / 8 heads 100 : 73, 16 of 97 .. 448 x 700 ..
// 1500 154 : 119, 16 of 300 x 1000 .. 1500, 16 heads 114 : 99; cut in two, 16 of 64 x 1000 .. 1500 50 :
// 71), and a prefix long for its rows (768 rows on 8192 tokens 77 : 68, 1024 on 16384 155 : 128; 512 on
// 8192 48 : 57, 1024 on 2048 47 : 58).  At head_dim 64 the softmax bounds both (16 of 448 x 1500, 16
// heads 79 : 87).  FP8 pages would be rounded to the queries' type on the way.
bool wide_walk(int head_dim, int dtype, bool fp8, bool prefix, int n_groups, int64_t rows, int hkv, int max_blocks) {
  if (fp8 || dtype == IVAKV_F32 || head_dim < 128 || rows < 256) return false;
  const int64_t chunk = wide_rows(head_dim);
  return prefix ? rows * max_blocks >= 5 << 16 : n_groups * ((rows + chunk - 1) / chunk) * hkv >= num_cus();
}

// Row chunks and items of a launch: a shared workgroup per CU, at least one per group and chunk (then
// nothing is cut).  The own walk (own_sets > 0: the sets of pages it has at most) gets a wave per
// SIMD, the other half of the CU (two: 64 rows on FP8 pages 55.6 against 51.6 us, 256 rows 154
// against 142), or two in a launch of its own.
Plan make_plan(int head_dim, int dtype, bool fp8, bool prefix, int n_groups, int64_t max_rows, int hkv, int g,
               int64_t own_sets, int max_blocks) {
  Plan p;
  const int64_t rows = n_groups > 0 ? max_rows * g : 0;
  const int row_bytes = head_dim * dtype_size(dtype);
  p.wide = wide_walk(head_dim, dtype, fp8, prefix, n_groups, rows, hkv, max_blocks);
  p.nr = row_blocks(row_bytes, p.wide ? 1 : rows);
  p.rows_chunk = p.wide ? wide_rows(head_dim) : 16 * p.nr;
  p.chunks = (int)((rows + p.rows_chunk - 1) / p.rows_chunk);
  const int64_t least = (int64_t)n_groups * p.chunks, most = num_cus() / hkv;
  p.split = p.chunks > 0 && most > least && most * max_blocks < 0x7fffffff;
  p.items = p.split ? (int)most : least < 0x7fffffff ? (int)least : 0x7fffffff;
  const int64_t waves = (int64_t)num_cus() * (p.wide ? 8 : 4), want = ((own_sets + 1) / 2 + 3) & ~3ll;
  p.own_waves = (int)(want < waves ? want : waves);
  return p;
}

// Workspace layout in floats: shared partials, own partials, the own walk's prefix.
struct Layout {
  size_t part_ml, own_acc, own_ml, own_pref, total;
};
Layout make_layout(const Plan& p, int n_rows, int hkv, int g, int d) {
  Layout l;
  const size_t rows = p.split || p.own_waves > 0 ? (size_t)p.items * hkv * p.rows_chunk : 0;
  const size_t own = p.own_waves > 0 ? ((size_t)p.own_waves + (size_t)n_rows * hkv) * g : 0;
  l.part_ml = rows * d;
  l.own_acc = l.part_ml + rows * 2;
  l.own_ml = l.own_acc + own * d;
  l.own_pref = l.own_ml + own * 2;
  l.total = l.own_pref + (p.own_waves > 0 ? (size_t)n_rows + 1 : 0);
  return l;
}

template <int DT, int D, bool kFp8, int NR, bool NT>
void launch_walk_n(RowArgs a, hipStream_t stream) {
  using S = Shape<DT, D, kFp8, NR>;
  const int pref = a.own_waves > 0 ? (2 * a.n_rows + 1) * (int)sizeof(int32_t) : 0;
  const int lds = a.shared_wgs > 0 && S::kLds > pref ? S::kLds : pref;
  static std::atomic<uint64_t> done{0};
  allow_lds(reinterpret_cast<const void*>(&rows_walk_kernel<DT, D, kFp8, NR, NT>), kMaxLds, done);
  rows_walk_kernel<DT, D, kFp8, NR, NT><<<a.shared_wgs + a.own_waves / 4, 256, lds, stream>>>(a, a.bt);
}

template <int DT, int D, bool kFp8>
void launch_d(const Plan& p, RowArgs a, hipStream_t stream) {
  const int nr = p.nr;
  const bool shared_chunks = p.chunks > 1;
  constexpr int most = max_row_blocks(Shape<DT, D, kFp8, 1>::kRow);
  a.unit = 4 * PageOps<DT, D, kFp8>::kPages;
  a.shared_wgs = a.items * a.Hkv;
  if (p.wide) {  // the shared walk in a launch of its own
    a.unit = 4;  // (two page pairs: the staged walk starts at even ones)
    launch_rows_wide(DT, D, a, stream);
    a.shared_wgs = 0;
  }
  // One chunk reads every page once: streaming loads.  Several share them through the L2.
  if (a.shared_wgs + a.own_waves == 0) {
    // nothing (more) to walk
  } else if (nr == most && shared_chunks && !p.wide) {
    launch_walk_n<DT, D, kFp8, most, false>(a, stream);
  } else if (nr == 1) {
    launch_walk_n<DT, D, kFp8, 1, true>(a, stream);
  } else if constexpr (most >= 2) {
    if (nr == 2) launch_walk_n<DT, D, kFp8, 2, true>(a, stream);
    else launch_walk_n<DT, D, kFp8, most, true>(a, stream);
  }
  if (a.prefix || a.split)
    rows_join_kernel<DT, D><<<(unsigned)a.n_rows * a.Hkv, 256, 0, stream>>>(a);
}

template <int DT, bool kFp8>
void launch_t(int head_dim, const Plan& p, const RowArgs& a, hipStream_t stream) {
  switch (head_dim) {
    case 64: launch_d<DT, 64, kFp8>(p, a, stream); break;
    case 128: launch_d<DT, 128, kFp8>(p, a, stream); break;
    default: launch_d<DT, 256, kFp8>(p, a, stream); break;
  }
}

void launch(int dtype, bool fp8, int head_dim, const Plan& p, const RowArgs& a, hipStream_t stream) {
  if (fp8) {
    if (dtype == IVAKV_F16) launch_t<IVAKV_F16, true>(head_dim, p, a, stream);
    else launch_t<IVAKV_BF16, true>(head_dim, p, a, stream);
    return;
  }
  switch (dtype) {
    case IVAKV_F16: launch_t<IVAKV_F16, false>(head_dim, p, a, stream); break;
    case IVAKV_BF16: launch_t<IVAKV_BF16, false>(head_dim, p, a, stream); break;
    default: launch_t<IVAKV_F32, false>(head_dim, p, a, stream); break;
  }
}

// Geometry checks that the entry points and their workspace queries share.
int check_geometry(const char* name, int n_groups, int num_q_heads, int num_kv_heads, int head_dim,
                   int max_rows, int dtype) {
  if (dtype_size(dtype) == 0) return fail(IVAKV_E_DTYPE, "%s: unknown dtype code %d", name, dtype);
  if (n_groups < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || max_rows < 0)
    return fail(IVAKV_E_ARG, "%s: bad sizes groups=%d Hq=%d Hkv=%d rows=%d", name, n_groups, num_q_heads,
                num_kv_heads, max_rows);
  if (num_q_heads % num_kv_heads != 0)
    return fail(IVAKV_E_SHAPE, "%s: num_q_heads %d not a multiple of num_kv_heads %d", name, num_q_heads,
                num_kv_heads);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(IVAKV_E_SHAPE, "%s: head_dim %d not in {64,128,256}", name, head_dim);
  return IVAKV_OK;
}

Plan plan_of(int n_groups, int n_rows, int num_q_heads, int num_kv_heads, int head_dim, int max_rows, int dtype,
             bool fp8, int max_blocks, bool prefix) {
  return make_plan(head_dim, dtype, fp8, prefix, n_groups, max_rows, num_kv_heads, num_q_heads / num_kv_heads,
                   prefix ? (int64_t)n_rows * num_kv_heads * max_blocks : 0, max_blocks);
}

// Workgroups of a launch: with up to 512 threads each, a grid of less than 2^32 threads.
constexpr int64_t kMaxGrid = 0x7fffff;

int check_plan(const char* name, const Plan& p, int n_rows, int num_kv_heads, bool prefix) {
  if ((int64_t)p.items * num_kv_heads + p.own_waves > kMaxGrid ||
      ((prefix || p.split) && (int64_t)n_rows * num_kv_heads > kMaxGrid))
    return fail(IVAKV_E_SHAPE, "%s: launch too large", name);
  return IVAKV_OK;
}

int rows_entry(const char* name, RowArgs a, int batch, int num_q_heads, int head_dim, int block_size,
               float scale, int dtype, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const int err = check_geometry(name, a.n_groups, num_q_heads, a.Hkv, head_dim, a.max_rows, dtype);
  if (err != IVAKV_OK) return err;
  const bool fp8 = a.k_scale != nullptr || a.v_scale != nullptr;
  if (fp8 && dtype != IVAKV_F16 && dtype != IVAKV_BF16)
    return fail(IVAKV_E_DTYPE, "%s: FP8 pools take fp16 or bf16 queries (dtype %d)", name, dtype);
  if (batch < 0 || a.n_rows < 0 || a.max_blocks < 0 || a.n_sink < 0)
    return fail(IVAKV_E_ARG, "%s: bad sizes batch=%d rows=%d max_blocks=%d n_sink=%d", name, batch, a.n_rows,
                a.max_blocks, a.n_sink);
  if (block_size != kBS) return fail(IVAKV_E_SHAPE, "%s: block_size %d != %d", name, block_size, kBS);
  if (a.n_rows == 0 || (!a.prefix && (a.n_groups == 0 || a.max_rows == 0))) return IVAKV_OK;
  if (a.num_pages < 1) return fail(IVAKV_E_ARG, "%s: num_pages must be >= 1", name);
  if (!a.q || !a.k_pool || !a.v_pool || !a.ctx || !a.out || (a.n_groups > 0 && !a.start) ||
      (a.prefix && a.n_groups > 0 && !a.shared) || (a.max_blocks > 0 && !a.bt))
    return fail(IVAKV_E_ARG, "%s: null pointer argument", name);
  if (!aligned16(a.q) || !aligned16(a.k_pool) || !aligned16(a.v_pool) || !aligned16(a.out))
    return fail(IVAKV_E_ARG, "%s: q, pools and out must be 16-byte aligned", name);
  if (fp8 && (!a.k_scale || !a.v_scale || !aligned16(a.k_scale) || !aligned16(a.v_scale)))
    return fail(IVAKV_E_ARG, "%s: k_scale / v_scale must be 16-byte aligned device pointers", name);
  if (!(scale == scale)) return fail(IVAKV_E_ARG, "%s: scale is NaN", name);
  a.G = num_q_heads / a.Hkv;
  if ((int64_t)a.n_rows * num_q_heads > 0x7fffffff)
    return fail(IVAKV_E_SHAPE, "%s: launch too large", name);
  if (a.prefix && (a.n_rows > kMaxBatch || (int64_t)a.n_rows * a.max_blocks > 0x7fffffff / a.Hkv))
    return fail(IVAKV_E_SHAPE, "%s: at most %d rows, and rows x max_blocks x num_kv_heads below 2^31 (got %d, %d, %d)",
                name, kMaxBatch, a.n_rows, a.max_blocks, a.Hkv);
  a.max_rows = a.max_rows < a.n_rows ? a.max_rows : a.n_rows;
  const Plan p = plan_of(a.n_groups, a.n_rows, num_q_heads, a.Hkv, head_dim, a.max_rows, dtype, fp8,
                         a.max_blocks, a.prefix);
  const int bad = check_plan(name, p, a.n_rows, a.Hkv, a.prefix);
  if (bad != IVAKV_OK) return bad;
  const Layout l = make_layout(p, a.n_rows, a.Hkv, a.G, head_dim);
  const size_t need = l.total * sizeof(float);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(IVAKV_E_WORKSPACE, "%s: workspace of %zu bytes (16-byte aligned) required, got %zu", name, need,
                workspace ? workspace_bytes : (size_t)0);
  a.rows_shift = 0;
  while ((1 << a.rows_shift) < p.rows_chunk) ++a.rows_shift;
  a.items = p.items;
  a.split = p.split;
  a.own_waves = p.own_waves;
  a.part_acc = static_cast<float*>(workspace);
  a.part_ml = a.part_acc + l.part_ml;
  a.own_acc = a.part_acc + l.own_acc;
  a.own_ml = a.part_acc + l.own_ml;
  a.own_pref = reinterpret_cast<int32_t*>(a.part_acc + l.own_pref);
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.window = a.window > 0 ? a.window : 0;
  launch(dtype, fp8, head_dim, p, a, stream);
  return launch_status(name);
}

int workspace_size(const char* name, int n_groups, int n_rows, int num_q_heads, int num_kv_heads, int head_dim,
                   int max_rows, int dtype, bool fp8, int max_blocks, bool prefix, size_t* bytes) {
  if (!bytes) return fail(IVAKV_E_ARG, "%s: null bytes", name);
  *bytes = 0;
  const int err = check_geometry(name, n_groups, num_q_heads, num_kv_heads, head_dim, max_rows, dtype);
  if (err != IVAKV_OK) return err;
  if (n_rows < 0 || max_blocks < 0)
    return fail(IVAKV_E_ARG, "%s: bad sizes rows=%d max_blocks=%d", name, n_rows, max_blocks);
  const Plan p = plan_of(n_groups, n_rows, num_q_heads, num_kv_heads, head_dim,
                         max_rows < n_rows ? max_rows : n_rows, dtype, fp8, max_blocks, prefix);
  const int bad = check_plan(name, p, n_rows, num_kv_heads, prefix);
  if (bad != IVAKV_OK) return bad;
  *bytes = make_layout(p, n_rows, num_kv_heads, num_q_heads / num_kv_heads, head_dim).total * sizeof(float);
  return IVAKV_OK;
}

}  // namespace
}  // namespace ivakv

using namespace ivakv;

extern "C" int ivakv_prefix_workspace_size(int batch, int n_groups, int max_group, int num_q_heads,
                                           int num_kv_heads, int head_dim, int max_blocks, int dtype, int fp8,
                                           size_t* bytes) {
  return workspace_size("ivakv_prefix_workspace_size", n_groups, batch, num_q_heads, num_kv_heads, head_dim,
                        max_group, dtype, fp8 != 0, max_blocks, true, bytes);
}

extern "C" int ivakv_prefix_decode_attn(const void* q, const void* k_pool, const void* v_pool,
                                        const float* k_scale, const float* v_scale, const int32_t* block_tables,
                                        const int32_t* context_lens, const int32_t* group_start,
                                        const int32_t* prefix_lens, int n_groups, void* out, void* workspace,
                                        size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads,
                                        int head_dim, int block_size, int max_blocks, int num_pages,
                                        int max_group, float scale, int window, int n_sink, int dtype,
                                        hipStream_t stream) {
  RowArgs a{};
  a.q = q;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.out = out;
  a.bt = block_tables;
  a.ctx = context_lens;
  a.start = group_start;
  a.shared = prefix_lens;
  a.n_groups = n_groups;
  a.n_rows = batch;
  a.Hkv = num_kv_heads;
  a.max_blocks = max_blocks;
  a.num_pages = num_pages;
  a.prefix = 1;
  a.max_rows = max_group;
  a.window = window;
  a.n_sink = n_sink;
  return rows_entry("ivakv_prefix_decode_attn", a, batch, num_q_heads, head_dim, block_size, scale, dtype,
                    workspace, workspace_bytes, stream);
}

extern "C" int ivakv_cross_workspace_size(int batch, int n_tok, int max_query_len, int num_q_heads,
                                          int num_kv_heads, int head_dim, int max_blocks, int dtype, int fp8,
                                          size_t* bytes) {
  return workspace_size("ivakv_cross_workspace_size", batch, n_tok, num_q_heads, num_kv_heads, head_dim,
                        max_query_len, dtype, fp8 != 0, max_blocks, false, bytes);
}

extern "C" int ivakv_cross_attn(const void* q, const void* k_pool, const void* v_pool, const float* k_scale,
                                const float* v_scale, const int32_t* block_tables, const int32_t* context_lens,
                                const int32_t* query_start, int n_tok, void* out, void* workspace,
                                size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads,
                                int head_dim, int block_size, int max_blocks, int num_pages, int max_query_len,
                                float scale, int dtype, hipStream_t stream) {
  RowArgs a{};
  a.q = q;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.out = out;
  a.bt = block_tables;
  a.ctx = context_lens;
  a.start = query_start;
  a.n_groups = batch;
  a.n_rows = n_tok;
  a.Hkv = num_kv_heads;
  a.max_blocks = max_blocks;
  a.num_pages = num_pages;
  a.max_rows = max_query_len;
  return rows_entry("ivakv_cross_attn", a, batch, num_q_heads, head_dim, block_size, scale, dtype, workspace,
                    workspace_bytes, stream);
}
