// label_logprobs.hip -- log probabilities of given labels, entropies and the top alternatives of rows of logits (fp32 / bf16 / fp16),
// and the gradient of all three.  No [n, C] intermediate is written.
//
// With the row's maximum M and u = (x - M) log2(e), the exponent's own unit:
//     S = sum 2^u,  T = sum u 2^u        (one pass: S and T are rescaled when the maximum moves)
//     log p_c = ln2 (u_c - log2 S),   H = ln2 (log2 S - T / S)
//     dx_c = a (1[c = label] - p_c) - h p_c (log p_c + H) + sum_j t_j (1[c = top_j] - p_c)
// with a, h, t the gradients of the label's log probability, of the entropy and of the alternatives' log probabilities.  The backward
// pass needs M, log2 S and H of a row only, so it is elementwise: logits read once, gradient written once.  (M and log2 S are kept apart:
// their sum would cost large logits the bits of the difference.)  u is held above -1000, where 2^u has long been zero: a logit of
// -inf or of the type's lowest value then adds 0 to T instead of 0 * inf.
// A logit of -inf has probability 0 (and adds 0 to the entropy); a row without a finite logit answers -inf, H = 0 and gradient 0;
// +inf or NaN anywhere makes the row NaN.  Alternatives are ordered by (value, lowest index first), NaN above +inf.
//
// Two forms of the forward pass (forward_in_registers() has the rule): rows of up to 1024 classes stay in the registers of 4 to 64
// lanes; longer ones are streamed by a workgroup each -- by several, joined by a second kernel, where there are few rows.
// 289127 x 172 fp32: forward 32 to 39 us without alternatives (6.2 to 5.1 TB/s), 68 to 72 with five (each is a round of compares over the
// row's registers); backward 70 us (5.7 TB/s).  289127 x 47 fp32 (one element per load): 17 and 26 us.  2048 x 131072 bf16: forward 99 us
// (5.4 TB/s; eleven operations per element run beside the loads), 190 with ten alternatives (their lists leave no registers for loads ahead);
// backward 177 us (6.1 TB/s).  1 x 131072 fp16 with ten alternatives: 8.4 + 7.0 us, the latency of two launches and of the lists.
#include "elem.h"

using namespace shadow;

namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr uint32_t kMaxTop = 64;
constexpr int32_t kNoKey = INT32_MIN;         // below every value's key (-inf has 0x807FFFFF)

struct LpArgs {
  const void *x;
  int64_t ldx;
  const void *label;
  int label64;
  uint32_t n, C, k;
  float *logprob, *entropy;                   // [n]
  float2 *stat;                               // [n]: M, log2 S
  float *top_lp;                              // [n, k]
  int64_t *top_idx;
  // streaming form: partials of the splits of a row
  uint32_t splits;
  float *part;                                // [n, splits, 4]: M, S, T, -
  int2 *part_top;                             // [n, splits, 4 wavefronts, k]: key, index
};

__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }      // NaN wins

// order-preserving integer of a value: -0 = +0, NaN on top
__device__ __forceinline__ int32_t key_of(float x) {
  const int32_t b = __float_as_int(x + 0.f);
  return x != x ? INT32_MAX : b ^ ((b >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float value_of(int32_t key) {
  return key == INT32_MAX ? __int_as_float(0x7FC00000) : __int_as_float(key ^ ((key >> 31) & 0x7FFFFFFF));
}

// all-reduce over aligned groups of LS lanes with a commutative, idempotent op, on the DPP network (group_sum's steps; through the LDS
// crossbar the five alternatives of 289127 rows of 172 alone took 45 us)
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false); }
template <int LS, typename Op>
__device__ __forceinline__ uint32_t group_all(uint32_t v, Op op) {
  if (LS >= 2) v = op(v, dpp<0xB1>(v));
  if (LS >= 4) v = op(v, dpp<0x4E>(v));
  if (LS >= 8) v = op(v, dpp<0x141>(v));
  if (LS >= 16) v = op(v, dpp<0x140>(v));
  if (LS >= 32) {
    const auto sw = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(sw[0], sw[1]);
  }
  if (LS >= 64) {
    const auto sw = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(sw[0], sw[1]);
  }
  return v;
}
template <int LS>
__device__ __forceinline__ float group_nan_max(float v) {
  return __uint_as_float(group_all<LS>(__float_as_uint(v), [](uint32_t p, uint32_t q) { return __float_as_uint(nan_max(__uint_as_float(p), __uint_as_float(q))); }));
}

// u of a logit (M = -inf: no finite logit, NaN difference -> -1000; a row with +inf or NaN is told by log2 S = NaN)
__device__ __forceinline__ float unit_of(float x, float M) { return fmaxf((x - M) * kLog2e, -1000.f); }

// log probability of a logit: -inf for a masked one, also in a row without a finite one
__device__ __forceinline__ float logprob_of(float x, float2 st) {
  return x == -INFINITY && !(st.y != st.y) ? -INFINITY : (x - st.x) - kLn2 * st.y;
}

// (M, S, T) -> what the row keeps, and its entropy
__device__ __forceinline__ float2 finish_stats(float M, float S, float T, float &H) {
  const bool lost = M != M || M == INFINITY;                 // NaN or +inf in the row
  const float ls = lost ? __int_as_float(0x7FC00000) : S == 0.f ? 0.f : __builtin_amdgcn_logf(S);       // (log2; S = 0: no finite logit)
  H = S == 0.f && !lost ? 0.f : kLn2 * (ls - T / S);
  return make_float2(M, ls);
}

// the scores of a row, by one lane
template <typename T>
__device__ __forceinline__ void answer_row(const LpArgs &a, uint64_t row, const T *x, float2 st, float H) {
  const int64_t label = a.label64 ? static_cast<const int64_t *>(a.label)[row] : (int64_t) static_cast<const int32_t *>(a.label)[row];
  a.stat[row] = st;
  a.entropy[row] = H;
  a.logprob[row] = label < 0 ? 0.f : label >= (int64_t)a.C ? __int_as_float(0x7FC00000) : logprob_of((float)x[label], st);
}

// ------------------------------------------------------------------------------------------------ rows in registers
template <typename T, int V, int L, int NC>
__global__ void __launch_bounds__(256) lp_rows_kernel(LpArgs a) {
  constexpr int G = 256 / L;
  const uint32_t sub = threadIdx.x % L, nch = a.C / V;
  const uint64_t row = (uint64_t)blockIdx.x * G + threadIdx.x / L;
  if (row >= a.n) return;                                    // (whole groups of L lanes leave: the reductions stay inside a group)
  const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.ldx;
  float v[NC][V], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const uint32_t c = sub + i * L;
#pragma unroll
    for (int j = 0; j < V; j++) v[i][j] = -INFINITY;
    if (c < nch) ldv<T, V>(x + c * V, v[i]);
#pragma unroll
    for (int j = 0; j < V; j++) m = nan_max(m, v[i][j]);
  }
  m = group_nan_max<L>(m);
  float S = 0.f, Tt = 0.f;
#pragma unroll
  for (int i = 0; i < NC; i++)
#pragma unroll
    for (int j = 0; j < V; j++) {
      const float u = unit_of(v[i][j], m), e = __builtin_amdgcn_exp2f(u);
      S += e;
      Tt = __builtin_fmaf(u, e, Tt);
    }
  S = group_sum<L>(S);
  Tt = group_sum<L>(Tt);
  float H;
  const float2 st = finish_stats(m, S, Tt, H);
  if (sub == 0) answer_row(a, row, x, st, H);
  if (a.k == 0) return;
  // k rounds: the best remaining key of the group, then the lowest index that has it
  const uint32_t rows = (uint32_t)__popcll(__ballot(true)) / L;         // of this wavefront
  int32_t key[NC][V];
#pragma unroll
  for (int i = 0; i < NC; i++)
#pragma unroll
    for (int j = 0; j < V; j++) key[i][j] = sub + i * L < nch ? key_of(v[i][j]) : kNoKey;
  for (uint32_t r = 0; r < a.k; r++) {
    int32_t best = kNoKey;
#pragma unroll
    for (int i = 0; i < NC; i++)
#pragma unroll
      for (int j = 0; j < V; j++) best = max(best, key[i][j]);
    best = (int32_t)group_all<L>((uint32_t)best, [](uint32_t p, uint32_t q) { return (uint32_t)max((int32_t)p, (int32_t)q); });
    uint32_t at = 0xFFFFFFFFu, hits = 0;                     // this lane's lowest index that has it; hits of the wavefront
    bool hit[NC][V];
#pragma unroll
    for (int i = NC - 1; i >= 0; i--)
#pragma unroll
      for (int j = V - 1; j >= 0; j--) {
        hit[i][j] = key[i][j] == best;
        hits += (uint32_t)__popcll(__ballot(hit[i][j]));
        at = hit[i][j] ? (sub + i * L) * V + j : at;
      }
    bool mine = at != 0xFFFFFFFFu;
    if (hits == rows) {                                      // (uniform) no ties: the compares above tell what to take out, its lane answers
#pragma unroll
      for (int i = 0; i < NC; i++)
#pragma unroll
        for (int j = 0; j < V; j++) key[i][j] = hit[i][j] ? kNoKey : key[i][j];
    } else {
      const uint32_t first = group_all<L>(at, [](uint32_t p, uint32_t q) { return min(p, q); });
      mine = at == first;
#pragma unroll
      for (int i = 0; i < NC; i++)
#pragma unroll
        for (int j = 0; j < V; j++) key[i][j] = (sub + i * L) * V + j == first ? kNoKey : key[i][j];
    }
    if (mine) {
      a.top_lp[row * a.k + r] = logprob_of(value_of(best), st);
      a.top_idx[row * a.k + r] = at;
    }
  }
}

// ------------------------------------------------------------------------------------------------ streamed rows
// Running statistics of one lane, and the wavefront's k best (lane j holds the j-th: key descending, index ascending).
struct Best {
  int32_t key;
  int32_t idx;
  int32_t thr_key, thr_idx;                   // the k-th (uniform)
  int32_t floor;                              // a key that the k-th reaches, known before the list is full
  float thr;                                  // max(floor, k-th) as a float for the quick test (NaN-safe: !(x < thr))
};

__device__ __forceinline__ bool better(int32_t k, int32_t i, int32_t k2, int32_t i2) { return k > k2 || (k == k2 && i < i2); }

__device__ __forceinline__ void best_init(Best &b) {
  b.key = kNoKey; b.idx = INT32_MAX; b.thr_key = kNoKey; b.thr_idx = INT32_MAX; b.floor = kNoKey; b.thr = -INFINITY;
}
__device__ __forceinline__ void best_quick(Best &b) {
  const int32_t t = max(b.thr_key, b.floor);
  b.thr = t == kNoKey ? -INFINITY : value_of(t);
}

// offer one (key, idx) per lane; every lane of the wavefront calls it
__device__ __forceinline__ void best_offer(Best &b, int32_t key, int32_t idx, uint32_t k) {
  uint64_t cand = __ballot(key != kNoKey && better(key, idx, b.thr_key, b.thr_idx));
  while (cand) {                              // (one candidate leaves per trip)
    const int src = __builtin_ctzll(cand);
    const int32_t ck = __builtin_amdgcn_readlane(key, src), ci = __builtin_amdgcn_readlane(idx, src);
    const uint32_t lane = lane_id();
    const int at = __popcll(__ballot(better(b.key, b.idx, ck, ci)));            // entries that stay in front
    const int32_t pk = (int32_t)dpp<0x138>((uint32_t)b.key), pi = (int32_t)dpp<0x138>((uint32_t)b.idx);        // (wave_shr:1: the lane below)
    b.key = (int)lane < at ? b.key : (int)lane == at ? ck : pk;
    b.idx = (int)lane < at ? b.idx : (int)lane == at ? ci : pi;
    b.thr_key = __builtin_amdgcn_readlane(b.key, (int)k - 1);
    b.thr_idx = __builtin_amdgcn_readlane(b.idx, (int)k - 1);
    cand &= ~(1ull << src);
    cand &= __ballot(better(key, idx, b.thr_key, b.thr_idx));
  }
  best_quick(b);
}

// joins (M, S, T) of two disjoint parts (M = -inf: one without a finite logit, S = T = 0)
__device__ __forceinline__ void join_stats(float &M, float &S, float &T, float M2, float S2, float T2) {
  const float m = nan_max(M, M2);
  const float d1 = unit_of(M, m), d2 = unit_of(M2, m), f1 = __builtin_amdgcn_exp2f(d1), f2 = __builtin_amdgcn_exp2f(d2);
  T = f1 * __builtin_fmaf(S, d1, T) + f2 * __builtin_fmaf(S2, d2, T2);
  S = f1 * S + f2 * S2;
  M = m;
}

// one trip: W words of V values (padding: -inf) into the running statistics
template <int W, int V>
__device__ __forceinline__ void feed_stats(const float (&v)[W][V], float &M, float &S, float &T) {
  float m = M;
#pragma unroll
  for (int w = 0; w < W; w++)
#pragma unroll
    for (int j = 0; j < V; j++) m = nan_max(m, v[w][j]);
  if (!(m == M)) {                            // the maximum moved
    const float d = unit_of(M, m), f = __builtin_amdgcn_exp2f(d);
    T = f * __builtin_fmaf(S, d, T);
    S *= f;
    M = m;
  }
#pragma unroll
  for (int w = 0; w < W; w++)
#pragma unroll
    for (int j = 0; j < V; j++) {
      const float u = unit_of(v[w][j], M), e = __builtin_amdgcn_exp2f(u);
      S += e;
      T = __builtin_fmaf(u, e, T);
    }
}

// A lower bound for the k-th best from one value per lane (the lanes' maxima): the k-th largest of them -- at least k values reach it.
// A wavefront's first trip uses it, when the list is still empty and nearly everything would be offered: 2048 values then offer some
// k + 5 instead of k (1 + ln(2048 / k)).  Found by counting, for each lane, the lanes that beat it.
__device__ __forceinline__ int32_t kth_of_lanes(int32_t key, uint32_t k) {
  uint32_t above = 0;
#pragma unroll 8
  for (int l = 0; l < 64; l++) above += __builtin_amdgcn_readlane(key, l) > key ? 1u : 0u;
  return (int32_t)group_all<64>((uint32_t)(above < k ? key : INT32_MAX), [](uint32_t p, uint32_t q) { return (uint32_t)min((int32_t)p, (int32_t)q); });
}

// Collects candidates of a wavefront into 64 places of LDS; more than 64 do not fit (the caller then offers them one by one).
struct Collect {
  int2 *place;
  uint32_t total;
};
__device__ __forceinline__ void collect(Collect &c, bool valid, int32_t key, int32_t idx) {
  const uint64_t mask = __ballot(valid);
  const uint32_t pos = c.total + (uint32_t)__popcll(mask & lanemask_lt());
  if (valid && pos < 64) c.place[pos] = make_int2(key, idx);
  c.total += (uint32_t)__popcll(mask);
}
// ... and makes them the list: every candidate's rank is the number that beat it (all distinct).  An insertion costs some 180 ns, this
// 0.5 us for fifteen of them.
__device__ __forceinline__ void rank_collected(const Collect &c, Best &b, uint32_t k) {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const uint32_t lane = lane_id();
  const int2 q = lane < c.total ? c.place[lane] : make_int2(kNoKey, INT32_MAX);
  uint32_t rank = 0;
  for (uint32_t l = 0; l < c.total; l++)
    rank += better(__builtin_amdgcn_readlane(q.x, (int)l), __builtin_amdgcn_readlane(q.y, (int)l), q.x, q.y) ? 1u : 0u;
  if (lane < c.total) c.place[rank] = q;      // (each has been read)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int2 e = lane < c.total && lane < k ? c.place[lane] : make_int2(kNoKey, INT32_MAX);
  b.key = e.x; b.idx = e.y;
  b.thr_key = __builtin_amdgcn_readlane(b.key, (int)k - 1);
  b.thr_idx = __builtin_amdgcn_readlane(b.idx, (int)k - 1);
  best_quick(b);
}

// the k best of `count` entries (key kNoKey: none), by one wavefront; place: 64 entries of LDS of its own
template <typename Get>
__device__ __forceinline__ Best best_of(uint32_t count, uint32_t k, int2 *place, Get get) {
  Best b;
  best_init(b);
  int32_t most = kNoKey;
#pragma unroll 4
  for (uint32_t e = lane_id(); e < count; e += 64) most = max(most, get(e).x);
  b.floor = kth_of_lanes(most, k);
  Collect c = {place, 0};
  for (uint32_t e0 = 0; e0 < count; e0 += 64) {
    const uint32_t e = e0 + lane_id();
    const int2 q = e < count ? get(e) : make_int2(kNoKey, INT32_MAX);
    collect(c, q.x != kNoKey && q.x >= b.floor, q.x, q.y);
  }
  if (c.total <= 64) {
    rank_collected(c, b, k);
    return b;
  }
  for (uint32_t e0 = 0; e0 < count; e0 += 64) {
    const uint32_t e = e0 + lane_id();
    const int2 q = e < count ? get(e) : make_int2(kNoKey, INT32_MAX);
    best_offer(b, q.x >= b.floor ? q.x : kNoKey, q.y, k);
  }
  return b;
}

template <int W, int V>
__device__ __forceinline__ void feed_top(const float (&v)[W][V], uint32_t base, uint32_t stride, uint32_t C, Best &b, uint32_t k) {
#pragma unroll
  for (int w = 0; w < W; w++) {
    float m = v[w][0];
#pragma unroll
    for (int j = 1; j < V; j++) m = nan_max(m, v[w][j]);
    const uint32_t c = base + w * stride;
    if (!__any(c < C && !(m < b.thr))) continue;                // (uniform) nothing of this word reaches the k-th
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int32_t key = key_of(v[w][j]);
      best_offer(b, c + j < C && key >= b.floor ? key : kNoKey, (int32_t)(c + j), k);
    }
  }
}

constexpr int kStreamThreads = 256, kStreamWords = 4;

// TOP: with alternatives.  Without them the next trip's words are on their way while a trip is summed (2048 x 131072 bf16: 99 us, 117
// through the form with lists, whose registers have no room for it).
template <typename T, bool TOP>
__global__ void __launch_bounds__(kStreamThreads, 4) lp_stream_kernel(LpArgs a) {
  constexpr int V = kVec<T>, W = kStreamWords, NW = kStreamThreads / 64;
  __shared__ float st[NW][3];
  __shared__ int2 lists[TOP ? NW * kMaxTop : 1], places[TOP ? NW : 1][64];
  const uint64_t row = blockIdx.x / a.splits;
  const uint32_t split = blockIdx.x % a.splits;
  const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.ldx;
  // [0, head) and the elements behind the last whole word are taken one by one, the words between by their index
  const uint32_t mis = (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T);
  const uint32_t head = mis ? min(a.C, (uint32_t)(V - mis)) : 0u;
  const uint32_t words = (a.C - head) / V, tail0 = head + words * V;
  const uint32_t per = (words + a.splits - 1) / a.splits, w0 = min(words, split * per), w1 = min(words, w0 + per);
  float M = -INFINITY, S = 0.f, Tt = 0.f;
  Best b;
  best_init(b);
  if constexpr (!TOP) {
    const Vec<T, V> *src = reinterpret_cast<const Vec<T, V> *>(x + head);
    Vec<T, V> ahead[W];
    auto fetch = [&](uint32_t w) {            // (past w1 the last word again: it is not used)
#pragma unroll
      for (int i = 0; i < W; i++) ahead[i] = src[min(w + i * kStreamThreads + threadIdx.x, w1 - 1)];
    };
    if (w0 < w1) fetch(w0);
    for (uint32_t w = w0; w < w1; w += kStreamThreads * W) {
      float v[W][V];
#pragma unroll
      for (int i = 0; i < W; i++)
#pragma unroll
        for (int j = 0; j < V; j++) v[i][j] = (float)ahead[i].v[j];
      if (w + kStreamThreads * W < w1) {
        fetch(w + kStreamThreads * W);
      } else {
#pragma unroll
        for (int i = 0; i < W; i++)
          if (w + i * kStreamThreads + threadIdx.x >= w1) {
#pragma unroll
            for (int j = 0; j < V; j++) v[i][j] = -INFINITY;
          }
      }
      feed_stats<W, V>(v, M, S, Tt);
    }
  } else {
    for (uint32_t w = w0; w < w1; w += kStreamThreads * W) {      // (uniform trips: the wavefront's list needs every lane)
      float v[W][V];
#pragma unroll
      for (int i = 0; i < W; i++) {
        const uint32_t c = w + i * kStreamThreads + threadIdx.x;
#pragma unroll
        for (int j = 0; j < V; j++) v[i][j] = -INFINITY;
        if (c < w1) ldv<T, V>(x + head + (uint64_t)c * V, v[i]);
      }
      feed_stats<W, V>(v, M, S, Tt);
      // (words past w1 are padding here: their index is put past C)
      {
        if (w == w0) {                                            // (uniform) the first trip
          float best = -INFINITY;
#pragma unroll
          for (int i = 0; i < W; i++)
#pragma unroll
            for (int j = 0; j < V; j++) best = nan_max(best, v[i][j]);
          b.floor = kth_of_lanes(w + threadIdx.x < w1 ? key_of(best) : kNoKey, a.k);
          best_quick(b);
          Collect col = {places[wave_id()], 0};
#pragma unroll
          for (int i = 0; i < W; i++) {
            const uint32_t c = w + i * kStreamThreads + threadIdx.x;
#pragma unroll
            for (int j = 0; j < V; j++) {
              const int32_t key = key_of(v[i][j]);
              collect(col, c < w1 && key >= b.floor, key, (int32_t)(head + c * V + j));
            }
          }
          if (col.total <= 64) {
            rank_collected(col, b, a.k);
            continue;
          }
        }
#pragma unroll
        for (int i = 0; i < W; i++) {
          const uint32_t c = w + i * kStreamThreads + threadIdx.x;
          float one[1][V];
#pragma unroll
          for (int j = 0; j < V; j++) one[0][j] = v[i][j];
          feed_top<1, V>(one, c < w1 ? head + c * V : a.C, 0, a.C, b, a.k);
        }
      }
    }
  }
  if (split == 0 && (head || tail0 < a.C)) {                    // at most 2 (V - 1) single elements: one per lane
    const uint32_t t = threadIdx.x, c = t < head ? t : tail0 + (t - head);
    float one[1][1] = {{c < a.C && t < 2 * V ? (float)x[c < a.C ? c : 0] : -INFINITY}};
    feed_stats<1, 1>(one, M, S, Tt);
    if (TOP) feed_top<1, 1>(one, t < 2 * V ? c : a.C, 0, a.C, b, a.k);
  }
  // lanes -> wavefront -> workgroup
#pragma unroll
  for (int off = 1; off < 64; off <<= 1)
    join_stats(M, S, Tt, __shfl_xor(M, off, 64), __shfl_xor(S, off, 64), __shfl_xor(Tt, off, 64));
  if (lane_id() == 0) { st[wave_id()][0] = M; st[wave_id()][1] = S; st[wave_id()][2] = Tt; }
  if (!TOP) {
  } else if (a.splits > 1) {                  // (the wavefronts' lists go to the join as they are)
    if (lane_id() < a.k) a.part_top[((row * a.splits + split) * NW + wave_id()) * a.k + lane_id()] = make_int2(b.key, b.idx);
  } else if (lane_id() < a.k) {
    lists[wave_id() * a.k + lane_id()] = make_int2(b.key, b.idx);
  }
  __syncthreads();
  if (wave_id() != 0) return;
  for (int w = 1; w < NW; w++) join_stats(M, S, Tt, st[w][0], st[w][1], st[w][2]);
  if (a.splits > 1) {
    if (lane_id() == 0) {
      float *p = a.part + (row * a.splits + split) * 4;
      p[0] = M; p[1] = S; p[2] = Tt;
    }
    return;
  }
  if (TOP) b = best_of(NW * a.k, a.k, places[0], [&](uint32_t e) { return lists[e]; });
  float H;
  const float2 stat = finish_stats(M, S, Tt, H);
  if (lane_id() == 0) answer_row(a, row, x, stat, H);
  if (TOP && lane_id() < a.k) {
    a.top_lp[row * a.k + lane_id()] = logprob_of(value_of(b.key), stat);
    a.top_idx[row * a.k + lane_id()] = b.idx;
  }
}

// joins the splits of a row: one workgroup per row, each wavefront a quarter of the lists
template <typename T>
__global__ void __launch_bounds__(kStreamThreads) lp_join_kernel(LpArgs a) {
  constexpr uint32_t NW = kStreamThreads / 64;
  __shared__ int2 lists[NW * kMaxTop], places[NW][64];
  const uint64_t row = blockIdx.x;
  if (a.k) {
    const uint32_t count = a.splits * a.k;    // (a quarter: as many lists as there are splits)
    const int2 *mine = a.part_top + (row * NW + wave_id()) * count;
    const Best b = best_of(count, a.k, places[wave_id()], [&](uint32_t e) { return mine[e]; });
    if (lane_id() < a.k) lists[wave_id() * a.k + lane_id()] = make_int2(b.key, b.idx);
    __syncthreads();
  }
  if (wave_id() != 0) return;
  float M = -INFINITY, S = 0.f, Tt = 0.f;
#pragma unroll 4
  for (uint32_t s = lane_id(); s < a.splits; s += 64) {
    const float *p = a.part + (row * a.splits + s) * 4;
    join_stats(M, S, Tt, p[0], p[1], p[2]);
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1)
    join_stats(M, S, Tt, __shfl_xor(M, off, 64), __shfl_xor(S, off, 64), __shfl_xor(Tt, off, 64));
  float H;
  const float2 stat = finish_stats(M, S, Tt, H);
  if (lane_id() == 0) answer_row(a, row, static_cast<const T *>(a.x) + (int64_t)row * a.ldx, stat, H);
  if (!a.k) return;
  const Best b = best_of(NW * a.k, a.k, places[0], [&](uint32_t e) { return lists[e]; });
  if (lane_id() < a.k) {
    a.top_lp[row * a.k + lane_id()] = logprob_of(value_of(b.key), stat);
    a.top_idx[row * a.k + lane_id()] = b.idx;
  }
}

// ------------------------------------------------------------------------------------------------ backward
struct LpBwdArgs {
  const void *x;
  int64_t ldx;
  const void *label;
  int label64;
  uint32_t n, C, k;
  const float2 *stat;
  const float *entropy, *dlp, *dent, *dtop;              // gradients may be null
  const int64_t *top_idx;
  void *dx;
  int64_t lddx;
};

struct RowGrad {
  float M, ls, H, neg, h;                                // neg: a + sum of the alternatives' gradients
  float a;
  int64_t label;
  bool dead;                                             // no finite logit: gradient 0
};

__device__ __forceinline__ RowGrad row_grad(const LpBwdArgs &a, uint64_t row) {
  RowGrad g;
  g.label = a.label64 ? static_cast<const int64_t *>(a.label)[row] : (int64_t) static_cast<const int32_t *>(a.label)[row];
  const float2 st = a.stat[row];
  g.M = st.x; g.ls = st.y; g.H = a.entropy[row];
  g.a = a.dlp && g.label >= 0 ? (g.label < (int64_t)a.C ? a.dlp[row] : __int_as_float(0x7FC00000)) : 0.f;
  g.h = a.dent ? a.dent[row] : 0.f;
  g.neg = g.a;
  if (a.dtop)
    for (uint32_t j = 0; j < a.k; j++) g.neg += a.dtop[row * a.k + j];
  g.dead = g.M == -INFINITY;
  if (g.dead) g.a = g.h = g.neg = 0.f;                   // (a loss may hand such a row's -inf an infinite gradient: no 0 * inf)
  return g;
}
// the gradient of one element without its one-hot terms
__device__ __forceinline__ float grad_of(const RowGrad &g, float x) {
  const float u = unit_of(x, g.M) - g.ls, p = __builtin_amdgcn_exp2f(u);
  return -p * __builtin_fmaf(g.h, __builtin_fmaf(kLn2, u, g.H), g.neg);
}

// V elements per step; `lanes` lanes (a power of two) walk a row, workgroups walk (row, part) pairs.  The one-hot terms of the
// alternatives go in before the one rounding: every word is held against the row's k indices, which are read again for each (289127 x 172
// fp32: 72 us without their gradient, 192 with that of five).
template <typename T, int V>
__global__ void __launch_bounds__(256) lp_bwd_kernel(LpBwdArgs a, uint32_t lanes, uint32_t parts, uint32_t per) {
  const uint32_t nch = a.C / V, sub = threadIdx.x & (lanes - 1), G = 256 / lanes;
  const uint64_t items = (uint64_t)a.n * parts;
  for (uint64_t it = (uint64_t)blockIdx.x * G + threadIdx.x / lanes; it < items; it += (uint64_t)gridDim.x * G) {
    const uint64_t row = it / parts;
    const uint32_t c0 = (uint32_t)(it % parts) * per, c1 = min(nch, c0 + per);
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.ldx;
    T *dx = static_cast<T *>(a.dx) + (int64_t)row * a.lddx;
    const RowGrad g = row_grad(a, row);
    const uint32_t lab = g.label >= 0 && g.label < (int64_t)a.C && !g.dead ? (uint32_t)g.label : 0xFFFFFFFFu;
    for (uint32_t c = c0 + sub; c < c1; c += lanes) {
      float v[V];
      ldv<T, V>(x + (uint64_t)c * V, v);
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float d = grad_of(g, v[j]);
        v[j] = c * V + j == lab ? d + g.a : d;
      }
      bool hit = false;                                   // an alternative in this word: its one-hot term goes in before the rounding
      if (a.dtop && !g.dead) {
        for (uint32_t q = 0; q < a.k; q++) {
          const uint32_t at = (uint32_t)a.top_idx[row * a.k + q];
          hit = at / V == c;
          if (hit) {
#pragma unroll
            for (int j = 0; j < V; j++) v[j] += at % V == (uint32_t)j ? a.dtop[row * a.k + q] : 0.f;
          }
        }
      }
      stv<T, V>(dx + (uint64_t)c * V, v);
    }
  }
}

// the rule: a row that 64 lanes hold at 16 elements each
bool forward_in_registers(uint32_t C) { return C <= 1024; }

// parts of a streamed row: enough workgroups for two per CU, at least one trip's words each.  (64 rows of 131072 bf16 with ten
// alternatives take 31 us with one workgroup per CU, 25 so and 22 with four; without alternatives 9.4, 9.6 and 9.8; 256 rows 14.5, 17 and
// 18, 512 rows 28, 28 and 34.)
uint32_t splits_of(uint32_t n, uint32_t C, int dtype) {
  const uint32_t trip = kStreamThreads * kStreamWords * (16u / elem_bytes(dtype));
  const uint32_t most = (C + trip - 1) / trip, want = (512u + n - 1) / n;
  return want < most ? (want ? want : 1u) : most;
}

template <typename T, int V, int L>
void rows_launch(const LpArgs &a, hipStream_t st) {
  const dim3 g((uint32_t)(((uint64_t)a.n + 256 / L - 1) / (256 / L))), b(256);
  const uint32_t need = (a.C / V + L - 1) / L;            // words per lane
  constexpr int kMost = 16 / V;
  if (kMost >= 4 && need * 4 <= (uint32_t)kMost) hipLaunchKernelGGL((lp_rows_kernel<T, V, L, (kMost / 4 ? kMost / 4 : 1)>), g, b, 0, st, a);
  else if (kMost >= 2 && need * 2 <= (uint32_t)kMost) hipLaunchKernelGGL((lp_rows_kernel<T, V, L, (kMost / 2 ? kMost / 2 : 1)>), g, b, 0, st, a);
  else if (kMost >= 4 && need * 4 <= (uint32_t)kMost * 3) hipLaunchKernelGGL((lp_rows_kernel<T, V, L, (kMost * 3 / 4 ? kMost * 3 / 4 : 1)>), g, b, 0, st, a);
  else hipLaunchKernelGGL((lp_rows_kernel<T, V, L, kMost>), g, b, 0, st, a);
}

template <typename T, int V>
void rows_dispatch(const LpArgs &a, hipStream_t st) {
  if (a.C <= 4 * 16) rows_launch<T, V, 4>(a, st);
  else if (a.C <= 16 * 16) rows_launch<T, V, 16>(a, st);
  else rows_launch<T, V, 64>(a, st);
}

template <typename T>
void stream_launch(const LpArgs &a, hipStream_t st) {
  if (a.k) hipLaunchKernelGGL((lp_stream_kernel<T, true>), dim3(a.n * a.splits), dim3(kStreamThreads), 0, st, a);
  else hipLaunchKernelGGL((lp_stream_kernel<T, false>), dim3(a.n * a.splits), dim3(kStreamThreads), 0, st, a);
  if (a.splits > 1) hipLaunchKernelGGL((lp_join_kernel<T>), dim3(a.n), dim3(kStreamThreads), 0, st, a);
}

template <typename T, int V>
void bwd_launch(const LpBwdArgs &a, hipStream_t st) {
  const uint32_t nch = a.C / V;
  // lanes of a row: four trips each (the power of two that covers a row of 43 words leaves a third of its lanes idle: 100 us for
  // 289127 rows of 172 fp32)
  uint32_t lanes = 4;
  while (lanes * 4 < nch && lanes < 256) lanes <<= 1;
  // a long row is cut into parts of 8 trips, so that few rows still fill the chip
  const uint32_t per = lanes * 8, parts = (nch + per - 1) / per;
  const uint64_t need = ((uint64_t)a.n * parts + 256 / lanes - 1) / (256 / lanes);
  hipLaunchKernelGGL((lp_bwd_kernel<T, V>), dim3((uint32_t)(need < 16384 ? need : 16384)), dim3(256), 0, st, a, lanes, parts, per);
}

int check(const char *who, int dtype, uint32_t n, uint32_t C, uint32_t k) {
  if (!elem_dtype_ok(dtype)) return set_error(SG_ERR_INVALID, "%s: type %d", who, dtype);
  if (C < 1 || C > 0x7FFFFF00u || k > kMaxTop || k > C) return set_error(SG_ERR_INVALID, "%s: %u classes, %u alternatives (at most 64, at most the classes)", who, C, k);
  if (n > 0x7FFFFFu * 8) return set_error(SG_ERR_INVALID, "%s: %u rows", who, n);
  return SG_OK;
}

}  // namespace

extern "C" size_t sl_label_logprobs_scratch_bytes(int dtype, uint32_t n, uint32_t C, uint32_t k) {
  if (!elem_dtype_ok(dtype) || n == 0 || C == 0 || k > kMaxTop || forward_in_registers(C)) return 0;
  const uint32_t s = splits_of(n, C, dtype);
  return s > 1 ? (size_t)n * s * (16 + 8 * (kStreamThreads / 64) * (size_t)k) : 0;
}

extern "C" int sl_label_logprobs_fwd(int dtype, const void *d_x, int64_t ldx, const void *d_label, int label_i64, uint32_t n, uint32_t C,
                                     uint32_t k, float *d_logprob, float *d_entropy, float *d_stat, float *d_top_lp, int64_t *d_top_idx,
                                     void *d_scratch, void *stream) {
  if (const int rc = check("sl_label_logprobs_fwd", dtype, n, C, k)) return rc;
  if (n == 0) return SG_OK;
  if (!d_x || !d_label || ldx < (int64_t)C || !d_logprob || !d_entropy || !d_stat || (k && (!d_top_lp || !d_top_idx)))
    return set_error(SG_ERR_INVALID, "sl_label_logprobs_fwd: operands");
  hipStream_t st = (hipStream_t)stream;
  LpArgs a = {};
  a.x = d_x; a.ldx = ldx; a.label = d_label; a.label64 = label_i64; a.n = n; a.C = C; a.k = k; a.logprob = d_logprob; a.entropy = d_entropy;
  a.stat = reinterpret_cast<float2 *>(d_stat); a.top_lp = d_top_lp; a.top_idx = d_top_idx; a.splits = 1;
  SHD_PROF_FMT((double)n * C * elem_bytes(dtype), 0, st, "label_logprobs_fwd_C%u", C);
  if (forward_in_registers(C)) {
    const bool words = rows_of_words(d_x, ldx, C, dtype);
    SHD_DISPATCH_ELEM(dtype, if (words) rows_dispatch<T, kVec<T>>(a, st); else rows_dispatch<T, 1>(a, st));
  } else {
    a.splits = splits_of(n, C, dtype);
    if (a.splits > 1) {
      if (!d_scratch) return set_error(SG_ERR_INVALID, "sl_label_logprobs_fwd: scratch");
      a.part = static_cast<float *>(d_scratch);
      a.part_top = reinterpret_cast<int2 *>(a.part + (size_t)n * a.splits * 4);
    }
    if ((uint64_t)n * a.splits > 0xFFFFFFull) return set_error(SG_ERR_INVALID, "sl_label_logprobs_fwd: %u rows of %u classes", n, C);
    SHD_DISPATCH_ELEM(dtype, stream_launch<T>(a, st));
  }
  SHD_HIP(hipGetLastError());
  return SG_OK;
}

extern "C" int sl_label_logprobs_bwd(int dtype, const void *d_x, int64_t ldx, const void *d_label, int label_i64, uint32_t n, uint32_t C,
                                     uint32_t k, const float *d_stat, const float *d_entropy, const int64_t *d_top_idx, const float *d_dlogprob,
                                     const float *d_dentropy, const float *d_dtop, void *d_dx, int64_t lddx, void *stream) {
  if (const int rc = check("sl_label_logprobs_bwd", dtype, n, C, k)) return rc;
  if (n == 0) return SG_OK;
  if (!d_x || !d_label || ldx < (int64_t)C || lddx < (int64_t)C || !d_stat || !d_entropy || !d_dx || (d_dtop && !d_top_idx))
    return set_error(SG_ERR_INVALID, "sl_label_logprobs_bwd: operands");
  hipStream_t st = (hipStream_t)stream;
  LpBwdArgs a = {};
  a.x = d_x; a.ldx = ldx; a.label = d_label; a.label64 = label_i64; a.n = n; a.C = C; a.k = d_dtop ? k : 0; a.stat = reinterpret_cast<const float2 *>(d_stat);
  a.entropy = d_entropy; a.dlp = d_dlogprob; a.dent = d_dentropy; a.dtop = k ? d_dtop : nullptr; a.top_idx = d_top_idx; a.dx = d_dx; a.lddx = lddx;
  SHD_PROF_FMT((double)2 * n * C * elem_bytes(dtype), 0, st, "label_logprobs_bwd_C%u", C);
  const bool words = rows_of_words(d_x, ldx, C, dtype) && rows_of_words(d_dx, lddx, C, dtype);
  SHD_DISPATCH_ELEM(dtype, if (words) bwd_launch<T, kVec<T>>(a, st); else bwd_launch<T, 1>(a, st));
  SHD_HIP(hipGetLastError());
  return SG_OK;
}
