// Log probabilities of given tokens, the entropy and the most likely tokens of rows of logits, and
// the gradient of the first two (and of the tops' log probabilities) by the logits, for gfx950.
//
// Row z of V logits, m = max z, S = sum_j e^(z_j - m), W = sum_j e^(z_j - m) (z_j - m):
//   logp_j  = (z_j - m) - log S            H = log S - W / S   (both terms >= 0: no cancellation)
//   top k   by value, equal values by index
//   dz_j    = g [j = t] + sum_i gk_i [j = top_i] - p_j (g + sum_i gk_i + gH (logp_j + H))
// One pass: every thread keeps (m, S, W) relative to its own running max; a new max m' takes
// W to e^(m - m') (W + (m - m') S).  The differences z - m are exact to fp32, so a large
// common offset of the logits costs no accuracy.
//
// Top k, by keys (value, -index), which are unique.  The lanes' maxima bound the k-th key from
// below: by the k-th largest of one wave's maxima, and by the least over the W waves of their
// ceil(k / W)-th largest, found bit by bit with ballots.  A row of one block is still in registers
// then; of a longer one only the blocks of a lane whose maximum reaches the bound are read again.
// The few vectors with a logit that reaches the bound are listed in LDS, then their logits, and
// there each logit counts those above it.  Where too many reach it (a constant row, say), every
// wave keeps its k best in one register per lane, sorted, inserts what passes the k-th, and the
// waves' lists meet in LDS, where every entry finds its rank by a binary search in each other
// list.  (Looking for single logits among the registers at once, 64 unrolled tests, was slower:
// 15.0 us against 11.5 at 4 rows of 32000, bf16, top 20, for the code that each wave had to fetch.)
//
// Bound: reading the logits once (forward), and again with one write (backward).  8192 rows of
// 32000, bf16: 83 us without tops (6.3 TB/s), 130 us with the top 5; 512 rows of 131072, fp32: 45
// and 53 us; a row of 32000: 6 us without tops, 11 us with 20, the latencies of the load, the
// bound, the barriers and the lists.  Both passes of 4096 rows of 32000, bf16: 131 us.
#include "ivakv_tile.h"

namespace ivakv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;
// A difference z - m below this has weight 0 in fp32 (and keeps 0 * inf out of W).
constexpr float kNoWeight = -1000.f;
constexpr int kMaxTop = 64;
constexpr int64_t kMaxRows = 0xffffff;  // (a grid has less than 2^32 threads, a row 256)

struct LogprobArgs {
  const void* logits;
  int64_t stride;          // elements between rows
  const int64_t* tokens;   // [n]
  int64_t n;
  int vocab, top;
  float* logprobs;         // [n]
  float* entropy;          // [n]
  float* stats;            // [n][2] m, log S (for the backward pass; may be null)
  float* top_logprobs;     // [n][top]
  int64_t* top_tokens;     // [n][top]
};

struct Moments {
  float m, s, w;
  IVAKV_INLINE __device__ inline void to_max(float mx) {  // mx >= m
    const float d = fmaxf(m - mx, kNoWeight);
    const float f = exp2_fast(d * kLog2e);
    w = f * (w + d * s);
    s *= f;
    m = mx;
  }
  IVAKV_INLINE __device__ inline void add(float z) {  // z <= m, or NaN, or both infinite
    const float d = z - m;
    const float e = exp2_fast(d * kLog2e);
    s += e;
    w = __builtin_fmaf(e, fmaxf(d, kNoWeight), w);
  }
  IVAKV_INLINE __device__ inline void join(float om, float os, float ow) {
    const float mx = fmaxf(m, om);
    Moments o{om, os, ow};
    o.to_max(mx);
    to_max(mx);
    s += o.s;
    w += o.w;
  }
};

template <int DT>
struct Elem;
template <>
struct Elem<IVAKV_F32> {
  using T = float;
  static constexpr int kVec = 4;
  static constexpr int kKeyBits = 24;  // of a sort key that bound the tops
  static IVAKV_INLINE __device__ inline float at(const Chunk16& c, int j) { return __uint_as_float(c.w[j]); }
  static __device__ inline float one(const float* p) { return *p; }
};
template <>
struct Elem<IVAKV_F16> {
  using T = _Float16;
  static constexpr int kVec = 8;
  static constexpr int kKeyBits = 19;
  static IVAKV_INLINE __device__ inline float at(const Chunk16& c, int j) {
    return (float)__builtin_bit_cast(f16x2, c.w[j >> 1])[j & 1];
  }
  static __device__ inline float one(const _Float16* p) { return (float)*p; }
};
template <>
struct Elem<IVAKV_BF16> {
  using T = __bf16;
  static constexpr int kVec = 8;
  static constexpr int kKeyBits = 16;
  static IVAKV_INLINE __device__ inline float at(const Chunk16& c, int j) {
    return __uint_as_float(j & 1 ? c.w[j >> 1] & 0xFFFF0000u : c.w[j >> 1] << 16);
  }
  static __device__ inline float one(const __bf16* p) { return (float)*p; }
};

// Sort key of a value: unsigned order is numeric order, -0 as +0 and every NaN above +inf; 0 is no
// value's key.
__device__ inline uint32_t key_of(float z) {
  const uint32_t u = __float_as_uint(z + 0.f);
  if (z != z) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The value of the lane below (lane 0: any).
__device__ inline uint32_t from_lane_below(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x138, 0xF, 0xF, false);
}

// A wave's k best: lane i < k the i-th.
struct TopList {
  uint32_t key, idx;
  uint32_t kth_key, kth_idx;  // of lane k - 1 (uniform)
  __device__ inline void reset() {
    key = kth_key = 0;
    idx = kth_idx = 0xFFFFFFFFu;
  }
  static __device__ inline bool beats(uint32_t ka, uint32_t ia, uint32_t kb, uint32_t ib) {
    return ka > kb || (ka == kb && ia < ib);
  }
  __device__ inline void insert(uint32_t k, uint32_t i, int top, int lane) {  // (k, i) uniform
    const int p = __popcll(__builtin_amdgcn_ballot_w64(beats(key, idx, k, i)));
    const uint32_t up_k = from_lane_below(key), up_i = from_lane_below(idx);
    key = lane > p ? up_k : lane == p ? k : key;
    idx = lane > p ? up_i : lane == p ? i : idx;
    kth_key = __builtin_amdgcn_readlane(key, top - 1);
    kth_idx = __builtin_amdgcn_readlane(idx, top - 1);
  }
  // Offers one (key, index) per lane where `has`: inserted in lane order while they beat the k-th.
  __device__ inline void offer(bool has, uint32_t k, uint32_t i, int top, int lane) {
    uint64_t todo = __builtin_amdgcn_ballot_w64(has && beats(k, i, kth_key, kth_idx));
    while (todo != 0) {
      const int l = __builtin_ctzll(todo);
      insert(__builtin_amdgcn_readlane(k, l), __builtin_amdgcn_readlane(i, l), top, lane);
      todo &= todo - 1;
      todo &= __builtin_amdgcn_ballot_w64(beats(k, i, kth_key, kth_idx));
    }
  }
};

// The k-th and the j-th largest of the lanes' keys to BITS bits, rounded down, or 0 when fewer
// lanes hold one.
template <int BITS>
__device__ inline void kth_of_lanes(uint32_t key, int k, int j, uint32_t& kth, uint32_t& jth) {
  kth = jth = 0;
#pragma unroll 4
  for (int bit = 31; bit > 31 - BITS; --bit) {
    const uint32_t c = kth | (1u << bit), d = jth | (1u << bit);
    if (__popcll(__builtin_amdgcn_ballot_w64(key >= c)) >= k) kth = c;
    if (__popcll(__builtin_amdgcn_ballot_w64(key >= d)) >= j) jth = d;
  }
}

// The entries of a sorted list of `top` in LDS that beat (k, i).
__device__ inline int beating(const uint32_t* keys, const uint32_t* idx, int top, uint32_t k, uint32_t i) {
  int lo = 0, hi = top;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (TopList::beats(keys[mid], idx[mid], k, i)) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

__device__ inline float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

constexpr int kCandidates = 512;
constexpr int kMaxBlocks = 16;  // blocks of a row whose lanes' maxima are kept

// One workgroup of W waves per row.
template <int DT, bool kTop, int W>
__global__ __launch_bounds__(64 * W) void logprob_kernel(LogprobArgs a) {
  using El = Elem<DT>;
  using T = typename El::T;
  constexpr int VEC = El::kVec, STEPS = 8, kThreads = 64 * W;
  __shared__ float s_m[W], s_s[W], s_w[W];
  __shared__ float s_bmax[kTop ? kMaxBlocks : 1][kTop ? kThreads : 1];
  __shared__ uint32_t s_key[kTop ? kCandidates : 1], s_idx[kTop ? kCandidates : 1];  // candidates, or W lists
  static_assert(W * kMaxTop <= kCandidates, "the waves' lists fit");
  __shared__ int s_hit[kTop ? kCandidates : 1];  // vectors that hold candidates
  __shared__ uint32_t s_kth[W], s_least[W], s_n, s_hits;
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + row * a.stride;
  const int V = a.vocab, tid = threadIdx.x;
  const int lane = tid & 63, wave = uni(tid >> 6);
  // Elements before the first 16-byte boundary and after the last are taken one by one.
  const int head = min(V, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(T));
  const int vecs = (V - head) / VEC, tail = head + vecs * VEC;
  const Chunk16* zv = reinterpret_cast<const Chunk16*>(z + head);
  if (kTop && tid == 0) s_n = s_hits = 0;
  // A block: STEPS vectors per lane, the threads' loads side by side.
  constexpr int kBlock = STEPS * kThreads;
  const int blocks = (vecs + kBlock - 1) / kBlock;
  auto vec_at = [&](int v0, int i) IVAKV_INLINE -> int { return v0 + i * kThreads + tid; };
  Moments mo{kLowest, 0.f, 0.f};
  Chunk16 c[STEPS];
  float mx = kNegInf;  // of this lane's logits
  for (int b = 0; b < blocks; ++b) {
    const int v0 = b * kBlock;
    // A backward pass reads the row again: then it is left in the caches (4096 rows of 32000, bf16,
    // both passes 131 us against 149; the forward pass alone is faster past them, 83 against 94).
    if (a.stats) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) c[i] = zv[min(vec_at(v0, i), vecs - 1)];
    } else {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) c[i] = load_nt<Chunk16>(zv + min(vec_at(v0, i), vecs - 1));
    }
    float bm = kNegInf;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      float t = El::at(c[i], 0);
#pragma unroll
      for (int j = 1; j < VEC; ++j) t = fmaxf(t, El::at(c[i], j));
      bm = fmaxf(bm, vec_at(v0, i) < vecs ? t : kNegInf);
    }
    if constexpr (kTop)
      if (b < kMaxBlocks) s_bmax[b][tid] = bm;
    mx = fmaxf(mx, bm);
    mo.to_max(fmaxf(mo.m, bm));
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (vec_at(v0, i) < vecs) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) mo.add(El::at(c[i], j));
      }
    }
  }
  // The row's ends, on wave 0: at most VEC - 1 elements each.
  const int e_at = lane < head ? lane : tail + (lane - head);
  const bool e_in = wave == 0 && (lane < head || e_at < V);
  const float e_x = e_in ? El::one(z + e_at) : kNegInf;
  mo.to_max(fmaxf(mo.m, e_x));
  if (e_in) mo.add(e_x);
  if constexpr (kTop) {
    const uint32_t mine = e_in || tid < vecs ? key_of(fmaxf(mx, e_x)) : 0u;
    uint32_t kth, least;
    kth_of_lanes<El::kKeyBits>(mine, a.top, (a.top + W - 1) / W, kth, least);
    if (lane == 0) {
      s_kth[wave] = kth;
      s_least[wave] = least;
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1)
    mo.join(__shfl_xor(mo.m, o), __shfl_xor(mo.s, o), __shfl_xor(mo.w, o));
  if (lane == 0) {
    s_m[wave] = mo.m;
    s_s[wave] = mo.s;
    s_w[wave] = mo.w;
  }
  __syncthreads();
  Moments all{s_m[0], s_s[0], s_w[0]};
#pragma unroll
  for (int u = 1; u < W; ++u) all.join(s_m[u], s_s[u], s_w[u]);
  // No finite logit: no distribution; log probabilities -inf, entropy 0.
  const bool none = all.s == 0.f;
  const float log_s = none ? 0.f : logf(all.s);
  if (tid == 0) {
    const int64_t t = a.tokens[row];
    const bool given = t >= 0 && t < V;
    a.logprobs[row] = given ? (El::one(z + (given ? t : 0)) - all.m) - log_s : 0.f;
    a.entropy[row] = none ? 0.f : log_s - all.w / all.s;
    if (a.stats) {
      a.stats[2 * row] = all.m;
      a.stats[2 * row + 1] = none ? kNegInf : log_s;
    }
  }
  if constexpr (kTop) {
    auto emit = [&](int rank, uint32_t k, uint32_t i) IVAKV_INLINE {
      if (rank >= a.top) return;
      a.top_logprobs[row * a.top + rank] = (value_of(k) - all.m) - log_s;
      a.top_tokens[row * a.top + rank] = i;
    };
    uint32_t bound = s_kth[0], least = s_least[0];
#pragma unroll
    for (int u = 1; u < W; ++u) {
      bound = max(bound, s_kth[u]);
      least = min(least, s_least[u]);
    }
    bound = max(bound, least);
    const bool nan = all.s != all.s;  // (the maxima drop a NaN: such a row is searched whole)
    auto gather = [&](float x, int at) IVAKV_INLINE {
      const uint32_t k = key_of(x);
      if (k >= bound) {
        const uint32_t n = atomicAdd(&s_n, 1u);
        if (n < kCandidates) {
          s_key[n] = k;
          s_idx[n] = (uint32_t)at;
        }
      }
    };
    auto hits_of = [&](int v0) IVAKV_INLINE {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        float t = El::at(c[i], 0);
#pragma unroll
        for (int j = 1; j < VEC; ++j) t = fmaxf(t, El::at(c[i], j));
        const int v = vec_at(v0, i);
        if (v < vecs && (nan || key_of(t) >= bound)) {
          const uint32_t n = atomicAdd(&s_hits, 1u);
          if (n < kCandidates) s_hit[n] = v;
        }
      }
    };
    if (blocks <= kMaxBlocks) {
      if (blocks == 1) {
        if (nan || key_of(mx) >= bound) hits_of(0);
      } else {
        for (int b = 0; b < blocks; ++b) {
          if (!nan && key_of(s_bmax[b][tid]) < bound) continue;
#pragma unroll
          for (int i = 0; i < STEPS; ++i) c[i] = zv[min(vec_at(b * kBlock, i), vecs - 1)];
          hits_of(b * kBlock);
        }
      }
      __syncthreads();
      const int hits = (int)s_hits;
      if (hits <= kCandidates) {
        for (int e = tid; e < hits * VEC; e += kThreads) {
          const int at = head + s_hit[e / VEC] * VEC + e % VEC;
          gather(El::one(z + at), at);
        }
        if (e_in) gather(e_x, e_at);
      }
      __syncthreads();
      const int n = hits <= kCandidates ? (int)s_n : hits;
      if (n <= kCandidates) {
        // Every wave holds the candidates, 64 to a register, and ranks each W-th.
        constexpr int M = kCandidates / 64;
        uint32_t ck[M], ci[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const bool in = 64 * m + lane < n;
          ck[m] = in ? s_key[64 * m + lane] : 0u;
          ci[m] = in ? s_idx[64 * m + lane] : 0u;
        }
        for (int e = wave; e < n; e += W) {
          const uint32_t k = s_key[e], i = s_idx[e];
          int rank = 0;
#pragma unroll
          for (int m = 0; m < M; ++m)
            if (64 * m < n) rank += __popcll(__builtin_amdgcn_ballot_w64(TopList::beats(ck[m], ci[m], k, i)));
          if (lane == 0) emit(rank, k, i);
        }
        return;
      }
      __syncthreads();
    }
    TopList list;
    list.reset();
    for (int b = 0; b < blocks; ++b) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int v = vec_at(b * kBlock, i);
        const Chunk16 x = zv[min(v, vecs - 1)];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const uint32_t k = key_of(El::at(x, j));
          list.offer(v < vecs && k >= bound, k, (uint32_t)(head + v * VEC + j), a.top, lane);
        }
      }
    }
    list.offer(e_in, key_of(e_x), (uint32_t)e_at, a.top, lane);
    if (lane < a.top) {
      s_key[wave * kMaxTop + lane] = list.key;
      s_idx[wave * kMaxTop + lane] = list.idx;
    }
    __syncthreads();
    for (int e = tid; e < W * a.top; e += kThreads) {
      const int u = e / a.top, at = e % a.top;
      const uint32_t k = s_key[u * kMaxTop + at], i = s_idx[u * kMaxTop + at];
      if (k == 0) continue;  // an empty place
      int rank = at;
      for (int o = 0; o < W; ++o)
        if (o != u) rank += beating(s_key + o * kMaxTop, s_idx + o * kMaxTop, a.top, k, i);
      emit(rank, k, i);
    }
  }
}

struct LogprobGradArgs {
  const void* logits;
  int64_t stride;
  const int64_t* tokens;
  const float* entropy;
  const float* stats;
  const int64_t* top_tokens;
  const float* g;      // [n] of the log probabilities
  const float* gh;     // [n] of the entropy
  const float* gt;     // [n][top] of the tops' log probabilities
  void* grad;          // [n][vocab]
  int64_t n;
  int vocab, top;
};

template <int DT>
__global__ __launch_bounds__(256) void logprob_grad_kernel(LogprobGradArgs a) {
  using El = Elem<DT>;
  using Tr = Traits<DT>;
  using T = typename El::T;
  constexpr int VEC = El::kVec;
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + row * a.stride;
  T* dz = static_cast<T*>(a.grad) + row * a.vocab;
  const int V = a.vocab;
  const float m = a.stats[2 * row], log_s = a.stats[2 * row + 1];
  const bool none = log_s == kNegInf;
  const int64_t t = a.tokens[row];
  const float g = t >= 0 && t < V ? a.g[row] : 0.f, gh = a.gh[row], h = a.entropy[row];
  float all = g;
  for (int i = 0; i < a.top; ++i) all += a.gt[row * a.top + i];
  auto base = [&](float x) IVAKV_INLINE -> float {
    const float lp = (x - m) - log_s;
    const float p = exp2_fast(lp * kLog2e);
    return none ? 0.f : -p * __builtin_fmaf(gh, fmaxf(lp, kNoWeight) + h, all);
  };
  // Vectors where both rows lie alike on 16 bytes, else element by element.
  const bool alike = (((uintptr_t)z ^ (uintptr_t)dz) & 15) == 0;
  const int head = alike ? min(V, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(T)) : V;
  const int vecs = (V - head) / VEC, tail = head + vecs * VEC;
  for (int v = threadIdx.x; v < vecs; v += 256) {
    const Chunk16 c = load_nt<Chunk16>(z + head + (int64_t)v * VEC);
    Chunk16 o;
#pragma unroll
    for (int j = 0; j < VEC; j += 16 / (int)sizeof(T) / 4) {
      if constexpr (DT == IVAKV_F32) o.w[j] = __float_as_uint(base(El::at(c, j)));
      else o.w[j / 2] = Tr::pack2(base(El::at(c, j)), base(El::at(c, j + 1)));
    }
    store_nt<Chunk16>(dz + head + (int64_t)v * VEC, o);
  }
  for (int e = threadIdx.x; e < head; e += 256) dz[e] = Tr::from_float(base(El::one(z + e)));
  for (int e = tail + threadIdx.x; e < V; e += 256) dz[e] = Tr::from_float(base(El::one(z + e)));
  // The given token's and the tops' own terms, after the row is written: each of their places is
  // computed whole again (equal places get equal values).
  __syncthreads();
  if (threadIdx.x <= a.top && !none) {
    const int64_t j = (int)threadIdx.x < a.top ? a.top_tokens[row * a.top + threadIdx.x] : t;
    if (j >= 0 && j < V) {
      float x = base(El::one(z + j)) + (j == t ? g : 0.f);
      for (int i = 0; i < a.top; ++i)
        if (a.top_tokens[row * a.top + i] == j) x += a.gt[row * a.top + i];
      dz[j] = Tr::from_float(x);
    }
  }
}

int check_logits(const char* name, const void* logits, int64_t stride, int64_t n, int vocab, int top, int dtype) {
  if (dtype_size(dtype) == 0) return fail(IVAKV_E_DTYPE, "%s: unknown dtype code %d", name, dtype);
  if (n < 0 || vocab < 0 || stride < 0 || top < 0)
    return fail(IVAKV_E_ARG, "%s: bad sizes n=%lld vocab=%d stride=%lld top=%d", name, (long long)n, vocab,
                (long long)stride, top);
  if (n > kMaxRows) return fail(IVAKV_E_SHAPE, "%s: %lld rows, at most %lld", name, (long long)n, (long long)kMaxRows);
  if (top > kMaxTop || top > vocab)
    return fail(IVAKV_E_SHAPE, "%s: top %d exceeds %d", name, top, vocab < kMaxTop ? vocab : kMaxTop);
  if (n > 0 && vocab < 1) return fail(IVAKV_E_SHAPE, "%s: rows without logits", name);
  if (n > 0 && (!logits || (reinterpret_cast<uintptr_t>(logits) & (dtype_size(dtype) - 1))))
    return fail(IVAKV_E_ARG, "%s: logits must be a device pointer aligned to its elements", name);
  return IVAKV_OK;
}

// Waves of a row: one where one holds it in its registers (8192 rows of 512, bf16, top 5: 19 us;
// four waves 47); eight for few rows, whose time is latency (4 rows of 131072, fp32, top 20: 27 us
// against 37; 512 rows of 32000, bf16: 18 against 20); else four (1024 rows: 27 us against 30;
// 8192: 130 against 163).
constexpr int kFewRows = 512;

template <int DT, bool kTop>
void launch_logprob(const LogprobArgs& a, hipStream_t stream) {
  if (a.vocab <= 512 * Elem<DT>::kVec) logprob_kernel<DT, kTop, 1><<<(unsigned)a.n, 64, 0, stream>>>(a);
  else if (a.n <= kFewRows) logprob_kernel<DT, kTop, 8><<<(unsigned)a.n, 512, 0, stream>>>(a);
  else logprob_kernel<DT, kTop, 4><<<(unsigned)a.n, 256, 0, stream>>>(a);
}

template <int DT>
void launch_logprob_t(const LogprobArgs& a, hipStream_t stream) {
  if (a.top > 0) launch_logprob<DT, true>(a, stream);
  else launch_logprob<DT, false>(a, stream);
}

}  // namespace
}  // namespace ivakv

using namespace ivakv;

extern "C" int ivakv_token_logprobs(const void* logits, int64_t row_stride, const int64_t* tokens, int64_t n,
                                    int vocab, int top, float* logprobs, float* entropy, float* stats,
                                    float* top_logprobs, int64_t* top_tokens, int dtype, hipStream_t stream) {
  const char* name = "ivakv_token_logprobs";
  const int err = check_logits(name, logits, row_stride, n, vocab, top, dtype);
  if (err != IVAKV_OK || n == 0) return err;
  if (!tokens || !logprobs || !entropy || (top > 0 && (!top_logprobs || !top_tokens)))
    return fail(IVAKV_E_ARG, "%s: null pointer argument", name);
  const LogprobArgs a{logits, row_stride, tokens, n, vocab, top, logprobs, entropy, stats, top_logprobs, top_tokens};
  switch (dtype) {
    case IVAKV_F16: launch_logprob_t<IVAKV_F16>(a, stream); break;
    case IVAKV_BF16: launch_logprob_t<IVAKV_BF16>(a, stream); break;
    default: launch_logprob_t<IVAKV_F32>(a, stream); break;
  }
  return launch_status(name);
}

extern "C" int ivakv_token_logprobs_grad(const void* logits, int64_t row_stride, const int64_t* tokens,
                                         const float* entropy, const float* stats, const int64_t* top_tokens,
                                         const float* grad_logprobs, const float* grad_entropy,
                                         const float* grad_top, int64_t n, int vocab, int top, void* grad,
                                         int dtype, hipStream_t stream) {
  const char* name = "ivakv_token_logprobs_grad";
  const int err = check_logits(name, logits, row_stride, n, vocab, top, dtype);
  if (err != IVAKV_OK || n == 0) return err;
  if (!tokens || !entropy || !stats || !grad_logprobs || !grad_entropy || !grad ||
      (top > 0 && (!top_tokens || !grad_top)))
    return fail(IVAKV_E_ARG, "%s: null pointer argument", name);
  if (reinterpret_cast<uintptr_t>(grad) & (dtype_size(dtype) - 1))
    return fail(IVAKV_E_ARG, "%s: grad must be aligned to its elements", name);
  const LogprobGradArgs a{logits, row_stride, tokens, entropy, stats, top_tokens, grad_logprobs, grad_entropy,
                          grad_top, grad, n, vocab, top};
  switch (dtype) {
    case IVAKV_F16: logprob_grad_kernel<IVAKV_F16><<<(unsigned)n, 256, 0, stream>>>(a); break;
    case IVAKV_BF16: logprob_grad_kernel<IVAKV_BF16><<<(unsigned)n, 256, 0, stream>>>(a); break;
    default: logprob_grad_kernel<IVAKV_F32><<<(unsigned)n, 256, 0, stream>>>(a); break;
  }
  return launch_status(name);
}
