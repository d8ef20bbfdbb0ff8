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
// Split: a workgroup of four waves takes a chunk of 16 NR rows and a segment of the unit's pages,
// wave w the page pairs w, w + 4, ...; the four states meet in LDS and leave one partial (running
// max, sum, unnormalized rows).  Segments are sized on the device from the groups' pages, so that
// ragged groups fill the CUs evenly; a second launch joins a row's partials.  For the prefix that
// launch walks each sequence's own pages first (prefix_own_kernel).
//
// Bound: the K and V bytes of the shared pages, read once for up to 16 NR rows; from a few
// hundred rows on the matrix and vector pipes (4 D operations per key and row).
#include <type_traits>

#include "ivakv_tile.h"

namespace ivakv {
namespace {

// Log2-domain headroom of the lazy row max, as in the prefill: p = exp2(s - m) stays <= 2^8.
constexpr float kLazyMax = 8.f;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;

struct RowArgs {
  const void* q;  // [n_rows, Hq, D]
  const void* k_pool;
  const void* v_pool;
  const float* k_scale;  // FP8 pools
  const float* v_scale;
  void* out;             // like q
  const int32_t* bt;     // [tables, max_blocks]
  const int32_t* ctx;    // cross: keys of each group; prefix: length of each row's sequence
  const int32_t* start;  // [n_groups + 1] first query row of each group
  const int32_t* shared; // prefix: [n_groups] shared tokens
  float* part_acc;       // [slot][16 NR][D]
  float* part_ml;        // [slot][16 NR][2]  (running max, sum)
  int n_groups, n_rows, Hkv, G, max_blocks, num_pages;
  int prefix;            // 1: prefix groups, 0: cross
  int max_rows;          // query rows of the largest group
  int chunks, rows_chunk;  // its row chunks, rows of a chunk (16 NR)
  int segments;          // segments of all groups the grid holds
  float scale_log2;
  int window, n_sink;
};

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
  // Logical page of list entry v: three runs of consecutive pages.
  int a0, na, b0, nb, c0;
  int len, win_start, n_sink;  // keys < len, and >= win_start or < n_sink
  IVAKV_INLINE __device__ inline int page(int v) const {
    return v < na ? a0 + v : v < na + nb ? b0 + (v - na) : c0 + (v - na - nb);
  }
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

// The online softmax of NR blocks of 16 rows and its walk over a list of pages.
template <int DT, int D, bool kFp8, int NR>
struct Walk {
  using Ops = PageOps<DT, D, kFp8>;
  using Tr = typename Ops::Tr;
  using E = typename Ops::E;
  static constexpr int NB = Ops::NB, PG = Ops::kPages;
  // 16-bit pages: the row sums come from the same rounded weights as the rows, by one more
  // product with ones, so the rounding of P (2^-9 relative in bf16, 2^-12 in fp16) cancels
  // where one key dominates.  FP8 and fp32 sum the weights in fp32.
  static constexpr bool kSumMfma = !kFp8 && DT != IVAKV_F32;
  typename Ops::QReg q[NR];
  f32x4 acc[NR][NB];
  f32x4 lacc[kSumMfma ? NR : 1];
  float m[NR], l[NR], grow_at[NR], neg_m[NR];
  float c, inv_c;  // |scale| log2(e)

  IVAKV_INLINE __device__ inline void init(const RowArgs& a, int64_t row0, int n, int h,
                                                            int r0, int ln, int lq) {
    c = fmaxf(fabsf(a.scale_log2), 1.17549435e-38f);
    inv_c = 1.f / c;
    const int Hq = a.Hkv * a.G;
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
      const int r = min(r0 + 16 * rb + ln, n - 1);  // rows past the end repeat the last one
      const E* p = static_cast<const E*>(a.q) + ((row0 + r / a.G) * Hq + h * a.G + r % a.G) * D;
#pragma unroll
      for (int j = 0; j < Ops::NQ; ++j) q[rb].c[j] = *reinterpret_cast<const Chunk16*>(p + Ops::q_at(j, lq));
      m[rb] = grow_at[rb] = kNegInf;
      l[rb] = neg_m[rb] = 0.f;
      if constexpr (kSumMfma) lacc[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[rb][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (a.scale_log2 < 0.f) {  // a negative scale negates q instead (exact)
      const uint32_t sign = sizeof(E) == 2 ? 0x80008000u : 0x80000000u;
#pragma unroll
      for (int rb = 0; rb < NR; ++rb)
#pragma unroll
        for (int j = 0; j < Ops::NQ; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) q[rb].c[j].w[i] ^= sign;
    }
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
        for (int rb = 0; rb < NR; ++rb) s[rb][i] = Tr::qk(k, q[rb].c[j], s[rb][i]);
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
    // score passes it by more than kLazyMax; one test covers all row blocks.
    bool grow = false;
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
      float mx = grow_at[rb];
#pragma unroll
      for (int i = 0; i < PG; ++i)
        mx = fmaxf(fmaxf(mx, fmaxf(s[rb][i][0], s[rb][i][1])), fmaxf(s[rb][i][2], s[rb][i][3]));
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
        l[rb] *= f;
        if constexpr (kSumMfma) lacc[rb] *= f;
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[rb][b] *= f;
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
  static constexpr int kRowRegs = NR * (4 * NB + 4 * Ops::NQ + 4 * PG + 8);
  static constexpr int kSets = kSetRegs + kRowRegs <= 320 ? 2 : 1;

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

// Full pages of the first tokens of group g that its sequences share, inside the table.
__device__ inline int shared_blocks(const RowArgs& a, int g) {
  const int p = a.shared[g] / kBS;
  return p < 0 ? 0 : p < a.max_blocks ? p : a.max_blocks;
}

// Rows [r0, r1) of group g, inside [0, n_rows].
__device__ inline void group_rows(const RowArgs& a, int g, int& r0, int& r1) {
  r0 = min(max(a.start[g], 0), a.n_rows);
  r1 = min(max(a.start[g + 1], r0), a.n_rows);
}

// The part of a prefix group's shared pages that is walked for all rows.  Without a window
// all of them.  With one, every row that has the whole prefix (length >= 16 blocks) sees the full
// sink pages, [0, sinks), and what its own window, length - window on, leaves: the pages from
// lo on lie in every row's window.  [base, lo) and the rest belong to the rows' own walks, as does
// everything of a row shorter than the prefix.
struct SharedPages {
  int blocks, sinks, base, lo;
  __device__ inline int listed() const { return sinks + blocks - base; }
};

__device__ inline SharedPages shared_pages(const RowArgs& a, int g) {
  SharedPages s;
  s.blocks = shared_blocks(a, g);
  s.sinks = s.base = 0;
  if (a.window > 0) {
    s.base = max(0, s.blocks - cdiv(a.window, kBS));
    s.sinks = min(a.n_sink / kBS, s.base);
  }
  s.lo = s.base;
  return s;
}

// Sets lo: the first shared page inside every row's window (uniform over the wave).
__device__ inline void window_start(const RowArgs& a, SharedPages& s, int r0, int r1, int lane) {
  if (a.window <= 0) return;
  int longest = 0;
  for (int r = r0 + lane; r < r1; r += 64) longest = max(longest, a.ctx[r]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) longest = max(longest, __shfl_xor(longest, o));
  s.lo = min(s.blocks, max(s.base, cdiv(max(uni(longest) - a.window, 0), kBS)));
}

// The first row of [r0, r1) that has the whole prefix, whose table the shared walk reads (-1: none, and
// then no row asks for the walk's partials).
__device__ inline int prefix_row(const RowArgs& a, const SharedPages& s, int r0, int r1, int lane) {
  for (int r = r0; r < r1; r += 64) {
    const uint64_t has = __builtin_amdgcn_ballot_w64(r + lane < r1 && a.ctx[min(r + lane, r1 - 1)] >= s.blocks * kBS);
    if (has != 0) return r + __builtin_ctzll(has);
  }
  return -1;
}

// List entries (pages) of group g, -1 for a group without rows.
__device__ inline int group_pages(const RowArgs& a, int g) {
  int r0, r1;
  group_rows(a, g, r0, r1);
  if (r1 <= r0) return -1;
  if (a.prefix) return shared_pages(a, g).listed();
  const int n = a.ctx[g];
  return min(cdiv(n < 0 ? 0 : n, kBS), a.max_blocks);
}

// Segments: every group's list is cut into pieces of `len` pages, a multiple of the eight pages that
// a workgroup's waves take at once, sized so that all groups' pieces number at most `segments`:
// whole pieces are at most segments - n_groups, and a group has at most one that is not whole.
// A cross group without keys has one empty piece, which writes its rows' zeros.
struct Segments {
  int len, least;
  __device__ inline int of(int pages) const { return pages < 0 ? 0 : max((pages + len - 1) / len, least); }
};

// The segment length: each wave sums the groups' pages, 64 at a time.
__device__ inline Segments segment_len(const RowArgs& a, int lane) {
  int64_t total = 0;
  for (int g0 = 0; g0 < a.n_groups; g0 += 64) {
    int n = g0 + lane < a.n_groups ? max(group_pages(a, g0 + lane), 0) : 0;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o);
    total += uni(n);
  }
  const int parts = max(a.segments - a.n_groups, 1);
  const int64_t len = (total + parts - 1) / parts;
  Segments s;
  s.len = (int)min<int64_t>(max<int64_t>((len + 7) & ~7ll, 8), 1 << 28);
  s.least = a.prefix ? 0 : 1;
  return s;
}

// The group of segment `seg` and which piece of the group it is (group -1: no such segment).
__device__ inline void find_segment(const RowArgs& a, const Segments& sg, int seg, int lane, int& group,
                                    int& piece) {
  int before = 0;
  group = -1;
  piece = 0;
  for (int g0 = 0; g0 < a.n_groups; g0 += 64) {
    const int n = g0 + lane < a.n_groups ? sg.of(group_pages(a, g0 + lane)) : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(incl, o);
      if (lane >= o) incl += u;
    }
    const uint64_t has = __builtin_amdgcn_ballot_w64(seg < before + incl);
    if (has != 0) {
      const int w = __builtin_ctzll(has);
      group = g0 + w;
      piece = seg - before - (__shfl(incl, w) - __shfl(n, w));
      return;
    }
    before += __shfl(incl, 63);
  }
}

// First segment of group g, and how many it has.
__device__ inline void group_segments(const RowArgs& a, const Segments& sg, int group, int lane, int& first,
                                      int& count) {
  int before = 0;
  count = 0;
  for (int g0 = 0; g0 <= group; g0 += 64) {
    const int n = g0 + lane <= group ? sg.of(group_pages(a, g0 + lane)) : 0;
    int sum = n;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    before += sum;
    if (group < g0 + 64) count = __shfl(n, group - g0);
  }
  first = uni(before - count);
  count = uni(count);
}

// Slot of a partial: segment, kv head, row chunk.
__device__ inline int64_t slot_of(const RowArgs& a, int seg, int h, int chunk) {
  return ((int64_t)seg * a.Hkv + h) * a.chunks + chunk;
}

// Shared walk.  Grid: (segment, kv head) x row chunk, a pair's chunks on one XCD (ids equal mod 8)
// one after the other, so that chunks past the first find the pages in its L2.
template <int DT, int D, bool kFp8, int NR, bool NT>
__global__ __launch_bounds__(kThreads) void rows_walk_kernel(RowArgs a, const int32_t* __restrict__ bt) {
  using WalkT = Walk<DT, D, kFp8, NR>;
  using E = typename WalkT::E;
  constexpr int R = 16 * NR;
  extern __shared__ float smem[];
  __shared__ float s_fin[2 * R];
  const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
  const int chunk = at % a.chunks, sh = (at / a.chunks) * 8 + xcd;
  if (sh >= a.segments * a.Hkv) return;
  const int seg = sh / a.Hkv, h = sh % a.Hkv;
  const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4;
  const int wave = uni(threadIdx.x >> 6);
  const Segments sg = segment_len(a, lane);
  int g, piece;
  find_segment(a, sg, seg, lane, g, piece);
  g = uni(g);
  piece = uni(piece);
  if (g < 0) return;
  int r0, r1;
  group_rows(a, g, r0, r1);
  const int rows = (r1 - r0) * a.G;  // (at most 2^31 / Hkv: the entry checks n_rows * Hq)
  if (chunk * R >= rows) return;
  KeyList kl;
  kl.num_pages = a.num_pages;
  kl.win_start = kl.n_sink = kl.a0 = kl.na = kl.b0 = kl.nb = 0;
  int n;
  if (a.prefix) {
    SharedPages s = shared_pages(a, g);
    window_start(a, s, r0, r1, lane);
    const int row = prefix_row(a, s, r0, r1, lane);
    if (row < 0) return;
    n = s.listed();
    kl.row = bt + (int64_t)row * a.max_blocks;
    kl.na = s.sinks;
    kl.c0 = s.base;
    kl.len = s.blocks * kBS;
    // pages [base, lo) of the list are left to the rows' own walks
    kl.win_start = s.lo * kBS;
    kl.n_sink = s.sinks * kBS;
  } else {
    n = group_pages(a, g);
    kl.row = bt + (int64_t)g * a.max_blocks;
    kl.c0 = 0;
    kl.len = a.ctx[g];
  }
  const int v0 = piece * sg.len, v1 = min(v0 + sg.len, n);
  WalkT wk;
  wk.init(a, r0, rows, h, chunk * R, ln, lq);
  wk.template run<NT, kWaves>(a, kl, h, v0, v1, wave, ln, lq);
  join_waves<WalkT, D, NR, kWaves>(wk, smem, wave, ln, lq, s_fin);
  const float* s_acc = smem + 2 * kWaves * R;
  const bool whole = !a.prefix && sg.of(n) == 1;
  const int64_t slot = slot_of(a, seg, h, chunk);
  const int Hq = a.Hkv * a.G;
  for (int e = threadIdx.x; e < R * (D / 4); e += kThreads) {
    const int row = e / (D / 4), d = 4 * (e % (D / 4)), r = chunk * R + row;
    if (r >= rows) break;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < kWaves; ++u) o += *reinterpret_cast<const f32x4*>(s_acc + (u * R + row) * (D + 4) + d);
    if (whole) {
      const float L = s_fin[2 * row + 1], inv = L > 0.f ? 1.f / L : 0.f;
      E* dst = static_cast<E*>(a.out) + ((int64_t)(r0 + r / a.G) * Hq + h * a.G + r % a.G) * D + d;
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[i] = WalkT::Tr::from_float(o[i] * inv);
    } else {
      *reinterpret_cast<f32x4*>(a.part_acc + (slot * R + row) * D + d) = o;
      if (d == 0) *reinterpret_cast<f32x2*>(a.part_ml + (slot * R + row) * 2) = f32x2{s_fin[2 * row], s_fin[2 * row + 1]};
    }
  }
}

// Log-sum-exp fold of the partials of segments [first, first + count) of row r (kv head h) at
// elements d .. d + 3 into (M, L, O), U at a time.
template <int D>
__device__ inline void fold_segments(const RowArgs& a, int first, int count, int h, int r, int d, float& M,
                                     float& L, f32x4& O) {
  constexpr int U = 4;
  const int chunk = r / a.rows_chunk, row = r % a.rows_chunk;
  for (int s0 = 0; s0 < count; s0 += U) {
    float mv[U], lv[U];
    f32x4 av[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = slot_of(a, first + min(s0 + u, count - 1), h, chunk) * a.rows_chunk + row;
      const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + at * 2);
      mv[u] = s0 + u < count ? ml[0] : kNegInf;
      lv[u] = ml[1];
      av[u] = *reinterpret_cast<const f32x4*>(a.part_acc + at * D + d);
    }
    float mc = M;
#pragma unroll
    for (int u = 0; u < U; ++u) mc = fmaxf(mc, mv[u]);
    const float m_use = mc == kNegInf ? 0.f : mc;
    const float f = exp2_fast(M - m_use);
    L *= f;
    O *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = exp2_fast(mv[u] - m_use);
      if (s0 + u < count) {
        L += lv[u] * w;
        O += av[u] * w;
      }
    }
    M = mc;
  }
}

// The group that query row `row` belongs to and the group's rows; false when there is none, or the
// row lies past the largest group the launch was sized for (uniform over the wave).
__device__ inline bool row_group(const RowArgs& a, int row, int lane, int& g, int& r0, int& r1) {
  g = -1;
  for (int g0 = 0; g0 < a.n_groups; g0 += 64) {  // the last group that starts at or before it
    const uint64_t le = __builtin_amdgcn_ballot_w64(g0 + lane < a.n_groups && a.start[min(g0 + lane, a.n_groups)] <= row);
    if (le == 0) break;
    g = g0 + 63 - __builtin_clzll(le);
  }
  r0 = r1 = 0;
  if (g < 0) return false;
  group_rows(a, g, r0, r1);
  return row >= r0 && row < r1 && row - r0 < a.max_rows;
}

// Cross attention's second launch: rows of groups cut into more than one segment.  Grid (kv head,
// query row).
template <int DT, int D>
__global__ __launch_bounds__(kThreads) void rows_merge_kernel(RowArgs a) {
  using E = typename Traits<DT>::E;
  const int h = blockIdx.x % a.Hkv, row = blockIdx.x / a.Hkv, lane = threadIdx.x & 63;
  int g, r0, r1;
  if (!row_group(a, row, lane, g, r0, r1)) return;
  const Segments sg = segment_len(a, lane);
  int first, count;
  group_segments(a, sg, g, lane, first, count);
  if (count == 1) return;  // written by the walk
  const int Hq = a.Hkv * a.G;
  for (int e = threadIdx.x; e < a.G * (D / 4); e += kThreads) {
    const int head = e / (D / 4), d = 4 * (e % (D / 4));
    float M = kNegInf, L = 0.f;
    f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
    fold_segments<D>(a, first, count, h, (row - r0) * a.G + head, d, M, L, O);
    const float inv = L > 0.f ? 1.f / L : 0.f;
    E* dst = static_cast<E*>(a.out) + ((int64_t)row * Hq + h * a.G + head) * D + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = Traits<DT>::from_float(O[i] * inv);
  }
}

// The prefix op's second launch: a workgroup walks one sequence's own pages for up to 16 heads of
// a kv head and joins the shared segments' partials.  Grid (kv head x block of 16 heads, sequence).
template <int DT, int D, bool kFp8, int W>
__global__ __launch_bounds__(64 * W) void prefix_own_kernel(RowArgs a, const int32_t* __restrict__ bt) {
  using WalkT = Walk<DT, D, kFp8, 1>;
  using E = typename WalkT::E;
  extern __shared__ float smem[];
  __shared__ float s_fin[32];
  const int head_blocks = (a.G + 15) / 16, per_row = a.Hkv * head_blocks;
  const int b = blockIdx.x / per_row, h = blockIdx.x % per_row / head_blocks, g0 = 16 * (blockIdx.x % head_blocks);
  const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4;
  const int wave = uni(threadIdx.x >> 6);
  const int L = max(a.ctx[b], 0);
  int g, r0, r1, first = 0, count = 0;
  SharedPages s{0, 0, 0, 0};
  if (row_group(a, b, lane, g, r0, r1)) {
    s = shared_pages(a, g);
    if (L >= s.blocks * kBS) {
      window_start(a, s, r0, r1, lane);
      group_segments(a, segment_len(a, lane), g, lane, first, count);
    } else {
      s = SharedPages{0, 0, 0, 0};  // shorter than the prefix: its own walk takes everything
    }
  }
  // Own pages: the sink pages before the window, then the window's, without those of the shared
  // walk, [0, sinks) and [lo, blocks).
  const PageWalk w = make_walk(L, a.window, a.n_sink, kBS);
  const int n_log = min(cdiv(L, kBS), a.max_blocks);
  KeyList kl;
  kl.row = bt + (int64_t)b * a.max_blocks;
  kl.num_pages = a.num_pages;
  kl.len = L;
  kl.win_start = w.win_start;
  kl.n_sink = a.n_sink;
  kl.a0 = s.sinks;
  kl.na = max(min(w.sink_pages, n_log) - s.sinks, 0);
  kl.b0 = w.win_first;
  kl.nb = max(min(s.lo, n_log) - w.win_first, 0);
  kl.c0 = max(w.win_first, s.blocks);
  const int n = kl.na + kl.nb + max(n_log - kl.c0, 0);
  WalkT wk;
  wk.init(a, b, a.G, h, g0, ln, lq);
  wk.template run<true, W>(a, kl, h, 0, n, wave, ln, lq);
  join_waves<WalkT, D, 1, W>(wk, smem, wave, ln, lq, s_fin);
  const float* s_acc = smem + 2 * W * 16;
  const int heads = min(a.G - g0, 16), Hq = a.Hkv * a.G;
  for (int e = threadIdx.x; e < heads * (D / 4); e += 64 * W) {
    const int head = e / (D / 4), d = 4 * (e % (D / 4));
    f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < W; ++u) O += *reinterpret_cast<const f32x4*>(s_acc + (u * 16 + head) * (D + 4) + d);
    float M = s_fin[2 * head], Ls = s_fin[2 * head + 1];
    fold_segments<D>(a, first, count, h, (b - r0) * a.G + g0 + head, d, M, Ls, O);
    const float inv = Ls > 0.f ? 1.f / Ls : 0.f;
    E* dst = static_cast<E*>(a.out) + ((int64_t)b * Hq + h * a.G + g0 + head) * D + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = WalkT::Tr::from_float(O[i] * inv);
  }
}

// Row blocks of a wave: as many as the rows need, up to what the registers hold beside two sets
// of pages in flight.
constexpr int max_row_blocks(bool fp8, int d) {
  return fp8 ? (d == 256 ? 2 : 4) : d == 64 ? 4 : d == 128 ? 2 : 1;
}
int row_blocks(bool fp8, int d, int64_t rows) {
  const int most = max_row_blocks(fp8, d);
  const int want = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  return want < most ? want : most;
}

// Workgroups of the shared walk that run at once.
int walk_slots(int nr) {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1)
    cus = 256;
  return nr == 4 ? cus : 2 * cus;
}

struct Plan {
  int nr, chunks, segments;
  int64_t rows() const { return 16 * nr; }
};

// Row chunks and segments of a launch: as many segments as fill the workgroup slots once, and one
// per group for the pieces that are not whole.
Plan make_plan(bool fp8, int d, int n_groups, int64_t max_rows, int hkv, int g) {
  Plan p;
  const int64_t rows = max_rows * g;
  p.nr = row_blocks(fp8, d, rows);
  p.chunks = (int)((rows + 16 * p.nr - 1) / (16 * p.nr));
  const int64_t per = (int64_t)hkv * p.chunks;
  const int64_t parts = walk_slots(p.nr) / (per > 0 ? per : 1);
  p.segments = n_groups + (int)(parts > n_groups ? parts : 0);
  return p;
}

size_t plan_bytes(const Plan& p, int hkv, int d) {
  return (size_t)p.segments * hkv * p.chunks * 16 * p.nr * (d + 2) * sizeof(float);
}

template <int DT, int D, bool kFp8, int NR, bool NT>
void launch_walk_n(const RowArgs& a, hipStream_t stream) {
  constexpr int lds = (int)(join_floats<D, NR, kWaves>() * sizeof(float));
  static std::atomic<uint64_t> done{0};
  allow_lds(reinterpret_cast<const void*>(&rows_walk_kernel<DT, D, kFp8, NR, NT>), lds, done);
  const unsigned n = ((unsigned)(a.segments * a.Hkv) + 7) / 8 * 8 * (unsigned)a.chunks;
  rows_walk_kernel<DT, D, kFp8, NR, NT><<<n, kThreads, lds, stream>>>(a, a.bt);
}

template <int DT, int D, bool kFp8>
void launch_walk_d(int nr, const RowArgs& a, hipStream_t stream) {
  constexpr int most = max_row_blocks(kFp8, D);
  // One chunk reads every page once: streaming loads.  Several share them through the L2.
  if (nr == most && a.chunks > 1) return launch_walk_n<DT, D, kFp8, most, false>(a, stream);
  if constexpr (most >= 4) {
    if (nr == 4) return launch_walk_n<DT, D, kFp8, 4, true>(a, stream);
  }
  if constexpr (most >= 2) {
    if (nr == 2) return launch_walk_n<DT, D, kFp8, 2, true>(a, stream);
  }
  launch_walk_n<DT, D, kFp8, 1, true>(a, stream);
}

template <int DT, int D, bool kFp8, int W>
void launch_own_w(const RowArgs& a, int batch, hipStream_t stream) {
  constexpr int lds = (int)(join_floats<D, 1, W>() * sizeof(float));
  static std::atomic<uint64_t> done{0};
  allow_lds(reinterpret_cast<const void*>(&prefix_own_kernel<DT, D, kFp8, W>), lds, done);
  const unsigned n = (unsigned)batch * a.Hkv * ((a.G + 15) / 16);
  prefix_own_kernel<DT, D, kFp8, W><<<n, 64 * W, lds, stream>>>(a, a.bt);
}

template <int DT, int D, bool kFp8>
void launch_d(int nr, const RowArgs& a, hipStream_t stream) {
  if (a.n_groups > 0 && a.chunks > 0) launch_walk_d<DT, D, kFp8>(nr, a, stream);
  if (a.prefix) {
    launch_own_w<DT, D, kFp8, 4>(a, a.n_rows, stream);
  } else if (a.segments > a.n_groups) {
    rows_merge_kernel<DT, D><<<(unsigned)a.n_rows * a.Hkv, kThreads, 0, stream>>>(a);
  }
}

template <int DT, bool kFp8>
void launch_t(int head_dim, int nr, const RowArgs& a, hipStream_t stream) {
  switch (head_dim) {
    case 64: launch_d<DT, 64, kFp8>(nr, a, stream); break;
    case 128: launch_d<DT, 128, kFp8>(nr, a, stream); break;
    default: launch_d<DT, 256, kFp8>(nr, a, stream); break;
  }
}

void launch(int dtype, bool fp8, int head_dim, int nr, const RowArgs& a, hipStream_t stream) {
  if (fp8) {
    if (dtype == IVAKV_F16) launch_t<IVAKV_F16, true>(head_dim, nr, a, stream);
    else launch_t<IVAKV_BF16, true>(head_dim, nr, a, stream);
    return;
  }
  switch (dtype) {
    case IVAKV_F16: launch_t<IVAKV_F16, false>(head_dim, nr, a, stream); break;
    case IVAKV_BF16: launch_t<IVAKV_BF16, false>(head_dim, nr, a, stream); break;
    default: launch_t<IVAKV_F32, false>(head_dim, nr, a, stream); break;
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

int check_plan(const char* name, const Plan& p, int num_kv_heads) {
  if ((int64_t)(p.segments + 8) * num_kv_heads > 0x7fffffff ||
      ((int64_t)p.segments * num_kv_heads + 8) * p.chunks > 0x7fffffff)
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
  if ((int64_t)a.n_rows * num_q_heads > 0x7fffffff) return fail(IVAKV_E_SHAPE, "%s: launch too large", name);
  a.max_rows = a.max_rows < a.n_rows ? a.max_rows : a.n_rows;
  const Plan p = make_plan(fp8, head_dim, a.n_groups, a.max_rows, a.Hkv, a.G);
  const int bad = check_plan(name, p, a.Hkv);
  if (bad != IVAKV_OK) return bad;
  const size_t need = plan_bytes(p, a.Hkv, head_dim);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(IVAKV_E_WORKSPACE, "%s: workspace of %zu bytes (16-byte aligned) required, got %zu", name, need,
                workspace ? workspace_bytes : (size_t)0);
  a.chunks = p.chunks;
  a.rows_chunk = 16 * p.nr;
  a.segments = p.segments;
  a.part_acc = static_cast<float*>(workspace);
  a.part_ml = a.part_acc + (size_t)p.segments * a.Hkv * p.chunks * 16 * p.nr * head_dim;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.window = a.window > 0 ? a.window : 0;
  launch(dtype, fp8, head_dim, p.nr, a, stream);
  return launch_status(name);
}

int workspace_size(const char* name, int n_groups, int n_rows, int num_q_heads, int num_kv_heads, int head_dim,
                   int max_rows, int dtype, int fp8, size_t* bytes) {
  if (!bytes) return fail(IVAKV_E_ARG, "%s: null bytes", name);
  *bytes = 0;
  const int err = check_geometry(name, n_groups, num_q_heads, num_kv_heads, head_dim, max_rows, dtype);
  if (err != IVAKV_OK) return err;
  if (n_rows < 0) return fail(IVAKV_E_ARG, "%s: negative row count", name);
  const Plan p = make_plan(fp8 != 0, head_dim, n_groups, max_rows < n_rows ? max_rows : n_rows, num_kv_heads,
                           num_q_heads / num_kv_heads);
  const int bad = check_plan(name, p, num_kv_heads);
  if (bad != IVAKV_OK) return bad;
  *bytes = plan_bytes(p, num_kv_heads, head_dim);
  return IVAKV_OK;
}

}  // namespace
}  // namespace ivakv

using namespace ivakv;

extern "C" int ivakv_prefix_workspace_size(int batch, int n_groups, int max_group, int num_q_heads,
                                           int num_kv_heads, int head_dim, int dtype, int fp8,
                                           size_t* bytes) {
  return workspace_size("ivakv_prefix_workspace_size", n_groups, batch, num_q_heads, num_kv_heads, head_dim,
                        max_group, dtype, fp8, bytes);
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
                                          int num_kv_heads, int head_dim, int dtype, int fp8,
                                           size_t* bytes) {
  return workspace_size("ivakv_cross_workspace_size", batch, n_tok, num_q_heads, num_kv_heads, head_dim,
                        max_query_len, dtype, fp8, bytes);
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
