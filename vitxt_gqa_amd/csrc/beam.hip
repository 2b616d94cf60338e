// Beam search's two operators for gfx950.
//
//  * t2s_beam_select   scores[b, n, v] = cum[b, n] + logits[b, n, v] - log sum_v' exp(logits[b, n, v']), the `select` best of the N V
//                      candidates of a sequence in descending order, ties to the lowest n V + v
//  * t2s_beam_reorder  state[.., b, n, ..] <- state[.., b, parents[b, n], ..] in place
//
// The greedy loop they widen is T2S._forward_mmt_and_output's eval branch (pythia/models/t2s.py:315-354: argmax over the
// [vocabulary | OCR pointer] logits feeds back).
//
// Selection reads the logits once.  A candidate is a 64-bit key, (logit in an order-preserving integer form) << 32 | ~index: keys are
// unique, so "descending, ties to the lowest index" is plain integer order, and there is no tie to handle anywhere.  A workgroup
// holds a stretch of a row in registers, keeps its running maximum / sum of exponentials and its `select` best keys; a second kernel
// joins the stretches of a sequence and orders the candidates of its N rows by their scores, compared in 64 bits (in 32, cum - log-sum-exp
// plus different logits of a row would often round to one number: a false tie).  A row's log-sum-exp itself has fp32's accuracy: 64-bit sums of 16 to 32
// exponentials each that were made and summed in fp32, within 160 2^-24 of the exact one (terms e^d: 2 |d| + 2 halves of a step, |d| no more than log V
// on their weighted average; 31 for a lane's sum, 2 for the logarithm).  It is the same number for all candidates of a row and for all rows of the
// same logits in a call, so nothing within a row and no tie of equal beams depends on it; candidates of unequal beams that are closer than that come in either
// order.  Sequences of few logits are one workgroup's, in one launch (below).
//
// Latencies bound all of it at a beam search's sizes: a stretch of 4 096 logits takes a workgroup 4 us on its own (its logits 2 500 cycles, maxima and
// sums 600, the bound 800, listing 2 300, ranking 1 500).  Rows and join, us: 64 x 5 x 15 000
// fp32 11.4 + 4.6 (15.4 MB), 48 x 8 x 30 522 bf16 16.1 + 6.8 (21.1 MB).  Requesting the next stretch's logits while one is worked on costs a CU one of
// its six workgroups: 19.5 where the rows then took 16.4.
#include <algorithm>

#include "common.h"
#include "lanes.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int BS_MAX = T2S_BEAM_MAX;               // beams, and candidates to select
constexpr int BS_EPT = 16;                         // elements of a thread per stretch
constexpr int BS_SUB = 256 * BS_EPT;
constexpr int BS_CHUNKS = 32;                      // workgroups of a row at most
constexpr int BS_WGS = 2048;                       // workgroups about (384 rows of 30 522 bf16 logits: 3 to a row 17.6 us, 4 16.4, 8 22.0)
constexpr int BS_LIST = 256;                       // logits of a wave that are ranked without more ado

// order-preserving unsigned form of a float (-inf < ... < -0 = +0 < ... < max)
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);          // -0 -> +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// NaN counts as a masked word, +inf as the largest number
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : fminf(x, 3.402823466e38f); }

// VEC consecutive logits of a row (16 bytes) from x[v] on; past its end: -inf.  A row may start at any element: the card takes 16 bytes in one load
// from there as well.
template <typename TX, int VEC>
__device__ __forceinline__ void load_logits(const TX* __restrict__ x, uint32_t v, uint32_t V, float* o) {
  typedef TX Piece __attribute__((ext_vector_type(VEC), aligned(sizeof(TX))));
  if (v + VEC <= V) {
    const Piece f = *(const Piece*)(x + v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = (float)f[i];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = v + i < V ? (float)x[v + i] : -INFINITY;
  }
}

// A bound that the K largest of a wave's 64 keys reach and, where keys are unique, no others do; 1 where fewer than K are not zero.  Two bits
// at a time from the top, the lanes at or above the three trial values counted by ballots; done as soon as exactly K are left (some 10
// steps on random logits, 32 at most).  `least`: 1 as well where fewer than K are above it.
__device__ __forceinline__ uint64_t wave_kth(uint64_t key, int K, uint64_t least) {
  if (__popcll(__ballot(key > least)) < K) return 1;
  uint64_t t = 0;
  for (int bit = 62; bit >= 0; bit -= 2) {
    const uint64_t t1 = t | 1ull << bit, t2 = t | 2ull << bit, t3 = t | 3ull << bit;
    const int c1 = __popcll(__ballot(key >= t1)), c2 = __popcll(__ballot(key >= t2)), c3 = __popcll(__ballot(key >= t3));
    t = c3 >= K ? t3 : c2 >= K ? t2 : c1 >= K ? t1 : t;
    if (c1 == K || c2 == K || c3 == K) break;
  }
  return t;
}

template <typename TX>
__global__ __launch_bounds__(256) void beam_rows_kernel(const TX* __restrict__ logits, int64_t l_bs, int64_t l_ns, const float* __restrict__ cum,
                                                        const uint8_t* __restrict__ finished, uint64_t* __restrict__ keys, double* __restrict__ sums,
                                                        float* __restrict__ maxs, int N, int V, int K, int pad, int chunks, int subs) {
  constexpr int VEC = 16 / sizeof(TX);
  __shared__ uint64_t list_s[4 * BS_MAX * (BS_EPT + 1)];
  __shared__ uint64_t top_s[BS_MAX];
  __shared__ uint32_t low_s[4];
  __shared__ int cnt_s, rank_s[64];
  __shared__ float m_s[4];
  __shared__ double s_s[4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, chunk = blockIdx.x % chunks;
  const int64_t row = blockIdx.x / chunks;
  const int b = (int)(row / N), n = (int)(row % N);
  const TX* x = logits + (int64_t)b * l_bs + (int64_t)n * l_ns;
  // (Stretches begin at the row's first element, not at a 16-byte boundary: which logits a lane sums must not depend on where the row lies, or rows of the
  // same logits would differ in the last bit of their sums, and equal beams would no longer tie.)
  // the first logits are on their way before it is known whether the row's are wanted at all
  float val[BS_EPT];
#pragma unroll
  for (int i = 0; i < BS_EPT; i += VEC) load_logits<TX, VEC>(x, (uint32_t)(chunk * subs) * BS_SUB + i * 256 + tid * VEC, V, val + i);
  const float c = cum[row];
  const bool dead = !(c > -INFINITY);                                  // -inf or NaN: every candidate of the row is -inf
  const bool ended = finished && finished[row];
  const int64_t out_at = row * chunks + chunk;
  auto key_of = [](float x, uint32_t v) { return (uint64_t)ordered(x) << 32 | (0xffffffffu - v); };
  if (dead || ended) {
    // nothing of the row's logits counts: an ended row offers `pad` at its own score; all else is at -inf, the lowest words first
    if (tid < K) {
      const int v = dead ? tid : tid - 1 + (tid - 1 >= pad ? 1 : 0);
      keys[out_at * K + tid] = chunk != 0 ? 0 : ended && !dead && tid == 0 ? key_of(0.f, pad) : v < V ? key_of(-INFINITY, v) : 0;
    }
    if (tid == 0) {
      maxs[out_at] = -INFINITY;
      sums[out_at] = 0.0;
    }
    return;
  }
  if (tid < BS_MAX) top_s[tid] = 0;
  const int lg = K <= 1 ? 0 : 32 - __builtin_clz(K - 1);                // 2^lg = G
  float m = -INFINITY;
  double sum = 0.0;
  for (int sub = chunk * subs; sub < (chunk + 1) * subs; ++sub) {
    const uint32_t v0 = (uint32_t)sub * BS_SUB;                         // (up to a stretch past V: below 2^32)
    if (v0 >= (uint32_t)V) break;
    if (sub != chunk * subs)
#pragma unroll
      for (int i = 0; i < BS_EPT; i += VEC) load_logits<TX, VEC>(x, v0 + i * 256 + tid * VEC, V, val + i);
    auto index = [&](int i) { return v0 + (i / VEC) * VEC * 256 + tid * VEC + i % VEC; };       // rises with i
    // maximum and sum of this lane's logits; a NaN or +inf among the wave's shows as a NaN sum, and is taken out (`clean`) then and only then
    float mx, mn, s;
    for (int pass = 0;; ++pass) {
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < BS_EPT; ++i) mx = fmaxf(mx, val[i]);
      mn = fmaxf(m, mx);
      const float mu = mn > -INFINITY ? mn : 0.f;
      s = 0.f;
#pragma unroll
      for (int i = 0; i < BS_EPT; ++i) s += __expf(val[i] - mu);
      if (pass || !__any(s != s)) break;
#pragma unroll
      for (int i = 0; i < BS_EPT; ++i) val[i] = clean(val[i]);
    }
    if (mn > m) {
      sum *= (double)__expf(m - mn);
      m = mn;
    }
    sum += (double)s;
    // ---- the K best of (this stretch, what is kept of the former ones).  A number that K lanes' best logits reach bounds the K-th largest from
    // below: the least of the maxima of G >= K lane groups of the workgroup (in a row's last stretch, where waves may be without logits, of a wave, and the
    // largest of the four waves' numbers), or the K-th of what is kept already.  That leaves little more than K logits to rank.
    const bool whole = v0 + BS_SUB <= (uint32_t)V;
    __syncthreads();
    const uint64_t kept = tid < K ? top_s[tid] : 0;
    const uint32_t low = wave_group_bound(ordered(mx), whole ? 6 - max(lg - 2, 0) : 6 - lg);
    if (lane == 0) low_s[wave] = low;
    if (tid == 0) cnt_s = 0;
    if (tid < 64) rank_s[tid] = 0;
    __syncthreads();
    // (below -inf's form there is no number: everything passes)
    const uint32_t low01 = whole && lg >= 2 ? min(low_s[0], low_s[1]) : max(low_s[0], low_s[1]), low23 = whole && lg >= 2 ? min(low_s[2], low_s[3]) : max(low_s[2], low_s[3]);
    const uint32_t low4 = max(whole && lg >= 1 ? min(low01, low23) : max(low01, low23), (uint32_t)(top_s[K - 1] >> 32));
    // (a bound of zero as -0: x - -0 has the sign bit of neither zero, -0 - 0 would have it)
    const float tv = low4 == 0x80000000u ? -0.0f : low4 > 0x7fffffu ? from_ordered(low4) : -INFINITY;
    uint32_t below = 0;                                                 // bit i: this lane's logit i does not reach it (the sign of the difference)
    if (tv > -INFINITY)
#pragma unroll
      for (int i = BS_EPT - 1; i >= 0; --i) below = __builtin_amdgcn_alignbit(below, as_u(val[i] - tv), 31);
    uint32_t mask = ~below & ((1u << BS_EPT) - 1u);
    int cnt = (int)wave_sum_u(__popc(mask)) + __popcll(__ballot(kept != 0));
    // Many of them (logits in an order that defeats the bound, equal ones, lanes without any): only those that reach the wave's K-th best
    // of one key a lane, at most K (BS_EPT + 1); those are unique.
    uint64_t thr = 1;
    if (cnt > BS_LIST) {
      int at = 0;                                                       // the lane's best: its first logit, or a larger one
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < BS_EPT; ++i)
        if (val[i] > top) {
          top = val[i];
          at = i;
        }
      const uint32_t v_at = v0 + (at / VEC) * VEC * 256 + tid * VEC + at % VEC;
      const uint64_t best = v_at < (uint32_t)V ? key_of(top, v_at) : 0;
      thr = wave_kth(kept > best ? kept : best, K, 0);
      cnt = __popcll(__ballot(kept >= thr));
      mask = 0;
#pragma unroll
      for (int i = 0; i < BS_EPT; ++i) {
        const bool in = index(i) < (uint32_t)V && key_of(val[i], index(i)) >= thr;
        cnt += __popcll(__ballot(in));
        mask |= in ? 1u << i : 0u;
      }
    }
    int to = 0;
    if (lane == 0 && cnt) to = atomicAdd(&cnt_s, cnt);
    to = __builtin_amdgcn_readfirstlane(to);
    const int end = to + cnt;
    {
      const uint64_t who = __ballot(kept >= thr);
      if (kept >= thr) list_s[to + __popcll(who & ((1ull << lane) - 1))] = kept;
      to += __popcll(who);
    }
    for (uint64_t who = __ballot(mask != 0); who; who = __ballot(mask != 0)) {
      const int i = __builtin_ctz(mask | 1u << BS_EPT);
      float x = val[0];
#pragma unroll
      for (int j = 1; j < BS_EPT; ++j) x = i == j ? val[j] : x;
      const uint32_t v = v0 + (i / VEC) * VEC * 256 + tid * VEC + i % VEC;
      if (mask) list_s[to + __popcll(who & ((1ull << lane) - 1))] = v < (uint32_t)V ? key_of(x, v) : 0;
      mask &= mask - 1;
      to += __popcll(who);
    }
    for (int i = to + lane; i < end; i += 64) list_s[i] = 0;
    __syncthreads();
    const int total = cnt_s;
    if (total <= 64) {                             // a lane to a key, a quarter of the others to a wave
      const uint64_t mine = lane < total ? list_s[lane] : 0;
      const int each = (total + 3) >> 2, to_j = min(total, (wave + 1) * each);
      int rank = 0;
#pragma unroll 8
      for (int j = wave * each; j < to_j; ++j) rank += list_s[j] > mine;
      if (rank) atomicAdd(rank_s + lane, rank);
      __syncthreads();
      if (tid < total && rank_s[tid] < K) top_s[rank_s[tid]] = mine;     // (empty places rank behind all keys)
    } else {
      for (int i = tid; i < total; i += 256) {
        const uint64_t mine = list_s[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < total; ++j) rank += list_s[j] > mine;
        if (rank < K) top_s[rank] = mine;
      }
    }
  }
  // ---- the row's maximum and sum over this workgroup
  const float mw = wave_max(m);
  const double sw = wave_sum64(m > -INFINITY ? sum * (double)__expf(m - mw) : 0.0);
  if (lane == 0) {
    m_s[wave] = mw;
    s_s[wave] = sw;
  }
  __syncthreads();
  if (tid < K) keys[out_at * K + tid] = top_s[tid];
  if (tid == 0) {
    const float m4 = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3]));
    double s4 = 0.0;
    for (int w = 0; w < 4; ++w)
      if (m_s[w] > -INFINITY) s4 += s_s[w] * (double)__expf(m_s[w] - m4);
    maxs[out_at] = m4;
    sums[out_at] = s4;
  }
}

// A candidate in two integers: its score in an order-preserving form (0: no candidate), and ~(n << 32 | v), so that equal scores are in the
// order of n V + v, lowest first, when the larger pair is the better one.
struct __attribute__((aligned(16))) Cand {
  uint64_t score, place;
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.score > b.score || (a.score == b.score && a.place > b.place); }

constexpr int BJ_PER = 4;                          // candidates of a thread at a time

// order-preserving unsigned form of a double, never 0
__device__ __forceinline__ uint64_t ordered64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double from_ordered64(uint64_t k) { return __builtin_bit_cast(double, k >> 63 ? k ^ 1ull << 63 : ~k); }

// log s of a normal s > 0, off by 2^-23 at most (s has fp32's accuracy, see above), 0 for 1: the 64-bit function takes a workgroup a microsecond
__device__ __forceinline__ double log_of(double s) {
  return ((double)__builtin_amdgcn_frexp_exp(s) + (double)__builtin_amdgcn_logf((float)__builtin_amdgcn_frexp_mant(s))) * 0.69314718055994531;
}

// one workgroup per sequence: joins the stretches, orders the N rows' candidates, 256 BJ_PER of them at a time
__global__ __launch_bounds__(256) void beam_join_kernel(const uint64_t* __restrict__ keys, const double* __restrict__ sums, const float* __restrict__ maxs,
                                                        const float* __restrict__ cum, const uint8_t* __restrict__ finished, float* __restrict__ out_scores,
                                                        int64_t* __restrict__ out_parents, int64_t* __restrict__ out_tokens, int N, int K, int chunks) {
  __shared__ double off_s[BS_MAX], part_s[BS_MAX * BS_CHUNKS];
  __shared__ float top_m[BS_MAX], part_m[BS_MAX * BS_CHUNKS];
  __shared__ Cand list_s[256 * BJ_PER + BS_MAX], top_s[BS_MAX];
  __shared__ uint64_t thr_s[4];
  __shared__ int cnt_s, rank_s[64];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, b = blockIdx.x;
  const int per_row = chunks * K, M = N * per_row;                     // (32 * 32 * 32 at most)
  const float per_inv = 1.0f / (float)per_row;
  const Cand none{0, 0};
  const uint64_t* kb = keys + (int64_t)b * M;
  uint64_t raw[BJ_PER];                            // (in flight beside the rows' sums)
#pragma unroll
  for (int j = 0; j < BJ_PER; ++j) raw[j] = tid + j * 256 < M ? kb[tid + j * 256] : 0;
  for (int i = tid; i < N * chunks; i += 256) {
    part_m[i] = maxs[(int64_t)b * N * chunks + i];
    part_s[i] = sums[(int64_t)b * N * chunks + i];
  }
  const int64_t row = (int64_t)b * N + min(tid, N - 1);
  const float c0 = cum[row];
  const bool ended = finished && finished[row];
  __syncthreads();
  if (tid < N) {
    float m = part_m[tid * chunks];
    for (int i = 1; i < chunks; ++i) m = fmaxf(m, part_m[tid * chunks + i]);
    double s = 0.0;
    for (int i = 0; i < chunks; ++i) {
      const float mi = part_m[tid * chunks + i];
      if (mi > -INFINITY) s += part_s[tid * chunks + i] * (double)__expf(mi - m);
    }
    const double cd = c0 > -INFINITY ? (double)fminf(c0, 3.402823466e38f) : -INFINITY;
    top_m[tid] = ended ? 0.f : m;
    off_s[tid] = ended || !(s > 0.0) ? cd : cd - log_of(s);
  }
  if (tid < K) top_s[tid] = none;
  __syncthreads();
  for (int m0 = 0; m0 < M; m0 += 256 * BJ_PER) {
    Cand c[BJ_PER];
    const Cand kept = tid < K ? top_s[tid] : none;
    uint64_t best = kept.score;
#pragma unroll
    for (int j = 0; j < BJ_PER; ++j) {
      const int i = m0 + tid + j * 256;
      const uint64_t k = m0 == 0 ? raw[j] : (i < M ? kb[i] : 0);
      c[j] = none;
      if (k) {
        const int n = (int)(((float)i + 0.5f) * per_inv);              // i / per_row: half a step from every border, 2^-23 relative off
        const float x = from_ordered((uint32_t)(k >> 32));
        const double sc = x > -INFINITY ? off_s[n] + ((double)x - (double)top_m[n]) : -INFINITY;
        c[j].score = ordered64(sc);
        c[j].place = ~((uint64_t)n << 32 | (0xffffffffu - (uint32_t)k));
        best = max(best, c[j].score);
      }
    }
    // a lower bound for the K-th best score, as in the rows' kernel; equal scores are all listed (the list holds everything there is)
    if (tid == 0) cnt_s = 0;
    if (tid < 64) rank_s[tid] = 0;
    uint64_t thr = 1;
    if (M > 64) {
      thr = wave_kth(best, K, 0x000fffffffffffffull);          // (-inf's form: a wave of few numbers leaves the bound to the others)
      if (lane == 0) thr_s[wave] = thr;
    }
    __syncthreads();
    if (M > 64)
      for (int w = 0; w < 4; ++w) thr = max(thr, thr_s[w]);
    if (best >= thr) {
#pragma unroll
      for (int j = 0; j < BJ_PER; ++j)
        if (c[j].score >= thr) list_s[atomicAdd(&cnt_s, 1)] = c[j];
      if (kept.score >= thr) list_s[atomicAdd(&cnt_s, 1)] = kept;
    }
    __syncthreads();
    const int cnt = cnt_s;
    if (cnt <= 64) {                               // a lane to a candidate, a quarter of the others to a wave
      const Cand mine = lane < cnt ? list_s[lane] : none;
      const int each = (cnt + 3) >> 2, to_j = min(cnt, (wave + 1) * each);
      int rank = 0;
#pragma unroll 4
      for (int j = wave * each; j < to_j; ++j) rank += before(list_s[j], mine);
      if (rank) atomicAdd(rank_s + lane, rank);
      __syncthreads();
      if (tid < cnt && rank_s[tid] < K) top_s[rank_s[tid]] = mine;
    } else {
      for (int i = tid; i < cnt; i += 256) {
        const Cand mine = list_s[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < cnt; ++j) rank += before(list_s[j], mine);
        if (rank < K) top_s[rank] = mine;
      }
    }
    __syncthreads();
  }
  if (tid < K) {
    const Cand r = top_s[tid];
    const int64_t at = (int64_t)b * K + tid;
    out_scores[at] = (float)from_ordered64(r.score);
    out_parents[at] = (int64_t)(~r.place >> 32);
    out_tokens[at] = (int64_t)(~r.place & 0xffffffffu);
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// Few logits to a sequence: one launch, one workgroup of 16 waves per sequence, which holds all of its logits in registers.  A wave has up to 2 048
// consecutive logits of a row, 32 to a lane, 64 apart (every lane has some also of a short row).  With the rows' sums known, the least of the best scores
// of G >= K lane groups is a bound that K scores reach: groups of the whole workgroup where its rows are alike, of one wave where a row is far ahead,
// whichever is larger (where groups have no number, the K-th largest itself of 64 groups' best scores, or of a wave's lanes').  Only what reaches it is
// listed and ranked.  Where the list does not hold that (ties, hardly a logit left) there are two slower ways.
// The code is run once, by few workgroups: a good part of the time goes into fetching it, so what need not be unrolled is not.
constexpr int BW_WAVES = 16, BW_EPT = 32, BW_PIECE = 64 * BW_EPT, BW_LIST = 64 * BW_WAVES;

// A bound that the K largest of the wave's 64 numbers reach, and no others unless they equal the K-th; 0 where fewer than K are not zero
__device__ __forceinline__ uint32_t wave_kth32(uint32_t key, int K) {
  uint32_t t = 0;
#pragma unroll 1
  for (int bit = 30; bit >= 0; bit -= 2) {
    const uint32_t t1 = t | 1u << bit, t2 = t | 2u << bit, t3 = t | 3u << bit;
    const int c1 = __popcll(__ballot(key >= t1)), c2 = __popcll(__ballot(key >= t2)), c3 = __popcll(__ballot(key >= t3));
    t = c3 >= K ? t3 : c2 >= K ? t2 : c1 >= K ? t1 : t;
    if (c1 == K || c2 == K || c3 == K) break;
  }
  return t;
}

template <typename TX>
__global__ __launch_bounds__(64 * BW_WAVES) void beam_whole_kernel(const TX* __restrict__ logits, int64_t l_bs, int64_t l_ns, const float* __restrict__ cum,
                                                                   const uint8_t* __restrict__ finished, float* __restrict__ out_scores,
                                                                   int64_t* __restrict__ out_parents, int64_t* __restrict__ out_tokens, int N, int V, int K,
                                                                   int pad, int pieces) {
  __shared__ Cand list_s[BW_LIST], best_s[BW_WAVES];
  __shared__ double part_s[BW_WAVES];
  __shared__ float part_m[BW_WAVES];
  __shared__ uint32_t low_s[64], most_s, lanes_s;
  __shared__ int cnt_s, rank_s[BW_LIST];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, b = blockIdx.x;
  const bool busy = wave < N * pieces;             // (the same for the whole wave, like row, at, c, ended, dead)
  const int row = busy ? wave / pieces : 0, at = busy ? (wave - row * pieces) * BW_PIECE : V;
  const TX* x = logits + (int64_t)b * l_bs + (int64_t)row * l_ns;
  float val[BW_EPT];
#pragma unroll
  for (int i = 0; i < BW_EPT; ++i) {
    const int v = at + i * 64 + lane;
    val[i] = v < V ? (float)x[v] : -INFINITY;
  }
  const float c = cum[(int64_t)b * N + row];
  const bool dead = !(c > -INFINITY), ended = finished && finished[(int64_t)b * N + row] && !dead;
  rank_s[tid] = 0;
  if (tid == 0) {
    cnt_s = 0;
    most_s = lanes_s = 0;
  }
  // An ended row is one of a single word, a dead one of none.  The word changes places with word 0: it is the first logit of the row's first lane.
  if (dead || ended) {
#pragma unroll
    for (int i = 0; i < BW_EPT; ++i) val[i] = -INFINITY;
    if (ended && at + lane == 0) val[0] = 0.f;
  }
  auto word = [&](int i) {
    const int v = at + i * 64 + lane;
    return ended ? (v == 0 ? pad : v == pad ? 0 : v) : v;
  };
  float m = -INFINITY, mx = -INFINITY;
  double sum = 0.0;
  if (busy) {
#pragma unroll 1
    for (int pass = 0;; ++pass) {                  // (NaN and +inf are taken out where a NaN sum shows them, as above)
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < BW_EPT; ++i) mx = fmaxf(mx, val[i]);
      m = wave_max(mx);
      const float mu = m > -INFINITY ? m : 0.f;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < BW_EPT; ++i) s += __expf(val[i] - mu);
      sum = wave_sum64((double)s);
      if (pass || sum == sum) break;
#pragma unroll
      for (int i = 0; i < BW_EPT; ++i) val[i] = clean(val[i]);
    }
  }
  if (lane == 0) {
    part_m[wave] = m;
    part_s[wave] = sum;
  }
  __syncthreads();
  // the row's maximum and sum from its waves', and what its logits' scores are relative to
  const float m_part = lane < pieces ? part_m[row * pieces + lane] : -INFINITY, m_row = wave_max(m_part);
  const double s_row = wave_sum64(m_part > -INFINITY ? part_s[row * pieces + lane] * (double)__expf(m_part - m_row) : 0.0);
  const double cd = dead ? -INFINITY : (double)fminf(c, 3.402823466e38f), top = m_row, off = s_row > 0.0 ? cd - log_of(s_row) : cd;
  auto score = [&](float x) { return x > -INFINITY ? off + ((double)x - top) : -INFINITY; };
  const uint32_t mine = ordered((float)score(mx));
  const int most = 6 - (K <= 1 ? 0 : 32 - __builtin_clz(K - 1));       // (64 / 2^most = G)
  uint32_t low = wave_group_bound(mine, most), group = mine;
  group = max(group, as_u(dpp<DPP_XOR1>(as_f(group))));
  group = max(group, as_u(dpp<DPP_XOR2>(as_f(group))));
  group = max(group, as_u(dpp<DPP_ROR4>(as_f(group))));
  group = max(group, as_u(dpp<DPP_ROR8>(as_f(group))));
  if ((lane & 15) == 0) low_s[wave * 4 + (lane >> 4)] = group;
  if (lane == 0) atomicMax(&most_s, low);
  __syncthreads();
  group = low_s[lane];
  low = max(wave_group_bound(group, most), most_s);
  if (low <= 0x7fffffu && 4 * N * pieces >= K) low = wave_kth32(group, K);
  if (low <= 0x7fffffu) {                          // (-inf's form; the same for all waves)
    low = wave_kth32(mine, K);                     // (not into most_s: a wave behind this one still has to decide by it)
    if (lane == 0) atomicMax(&lanes_s, low);
    __syncthreads();
    low = lanes_s;
  }
  // (read once more: taking it from the registers is a choice among all of them)
  auto logit = [&](int i) { return dead || ended ? (ended && at + lane + i == 0 ? 0.f : -INFINITY) : clean((float)x[at + i * 64 + lane]); };
  auto list = [&](uint32_t mask) {
    int to = 0;
    if (mask) to = atomicAdd(&cnt_s, __popc(mask));
#pragma unroll 1
    for (; mask; mask &= mask - 1, ++to) {
      const int i = __builtin_ctz(mask);
      const uint64_t sc = ordered64(score(logit(i)));
      if (to < BW_LIST) list_s[to] = Cand{sc, ~((uint64_t)row << 32 | (uint32_t)word(i))};
    }
  };
  bool listed = low > 0x7fffffu;                   // (or no wave has K numbers)
  if (listed) {
    // Scores of 64 bits whose fp32 rounding reaches `low` belong to logits above thr: low's half step, and the roundings of thr itself, are taken off it
    const double f = (double)from_ordered(low), t = top + (f - off);
    float thr = (float)(t - (fabs(f) * 0x1p-23 + (fabs(t) + fabs(off) + fabs(top)) * 0x1p-50));
    thr = thr == 0.f ? -0.0f : fmaxf(thr, -3.402823466e38f);           // (the sign of x - thr: -0 - 0 would have one, -inf - -inf need not)
    uint32_t below = 0;
#pragma unroll
    for (int i = BW_EPT - 1; i >= 0; --i) below = __builtin_amdgcn_alignbit(below, as_u(val[i] - thr), 31);
    list(off > -INFINITY ? ~below : 0);
    __syncthreads();
    listed = cnt_s <= BW_LIST;
  }
  uint32_t left = 0;                               // the lane's logits that are there and not taken
#pragma unroll
  for (int i = 0; i < BW_EPT; ++i) left |= at + i * 64 + lane < V ? 1u << i : 0u;
  // the best of them: the largest logit, of equal ones the first word (in an ended row word 0 is ahead of the lane's other masked words); -1: none left
  auto look = [&]() {
    float bx = -INFINITY;
    int bi = -1;
#pragma unroll
    for (int i = 0; i < BW_EPT; ++i)
      if ((left >> i & 1) && (bi < 0 || val[i] > bx)) {
        bx = val[i];
        bi = i;
      }
    const int swapped = pad - at - lane;
    if (ended && bx == -INFINITY && swapped >= 0 && swapped < BW_PIECE && swapped % 64 == 0 && (left >> swapped / 64 & 1)) bi = swapped / 64;
    return bi;
  };
  if (!listed) {
    // Second try, with words for ties: of each wave what reaches its K-th best of one key a lane (keys are unique: K lanes do), and the best wave's K-th score
    __syncthreads();
    const int bi = look();
    auto key_of = [&](int i, float x) { return (uint64_t)ordered(x) << 32 | (0xffffffffu - (uint32_t)word(i)); };
    const uint64_t thr = wave_kth(bi < 0 ? 0 : key_of(bi, logit(bi)), K, 0);
    const uint32_t hi = (uint32_t)(thr >> 32);
    if (lane == 0) best_s[wave].score = thr == 1 ? 0 : ordered64(hi > 0x7fffffu ? score(from_ordered(hi)) : -INFINITY);
    if (tid == 0) cnt_s = 0;
    __syncthreads();
    uint64_t kth = 0;
#pragma unroll
    for (int w = 0; w < BW_WAVES; ++w) kth = max(kth, best_s[w].score);
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < BW_EPT; ++i) mask |= (left >> i & 1) && key_of(i, val[i]) >= thr && ordered64(score(val[i])) >= kth ? 1u << i : 0u;
    list(mask);
    __syncthreads();
    listed = cnt_s <= BW_LIST;
  }
  if (listed) {
    // a lane to a candidate, the others to compare it with shared by as many waves as there are
    const int cnt = cnt_s, across = (cnt + 63) >> 6, share = wave / across, shares = BW_WAVES / across, at = (wave - share * across) * 64 + lane;
    if (share < shares && at < cnt) {
      const Cand x = list_s[at];
      const int each = (cnt + shares - 1) / shares, to_j = min(cnt, (share + 1) * each);
      int rank = 0;
#pragma unroll 4
      for (int j = share * each; j < to_j; ++j) rank += before(list_s[j], x);
      if (rank) atomicAdd(rank_s + at, rank);
    }
    __syncthreads();
    if (tid < cnt && rank_s[tid] < K) {
      const Cand r = list_s[tid];
      const int64_t to = (int64_t)b * K + rank_s[tid];
      out_scores[to] = (float)from_ordered64(r.score);
      out_parents[to] = (int64_t)(~r.place >> 32);
      out_tokens[to] = (int64_t)(~r.place & 0xffffffffu);
    }
    return;
  }
  // third try, where a few lanes have most of the best logits: one by one
  Cand own{0, 0};
  int bi = -1;
  bool stale = true;                               // the lane's best has been taken (its wave looks again, the others' bests stand)
#pragma unroll 1
  for (int k = 0; k < K; ++k) {
    if (__any(stale)) {
      if (stale) {
        bi = look();
        own = bi < 0 ? Cand{0, 0} : Cand{ordered64(score(logit(bi))), ~((uint64_t)row << 32 | (uint32_t)word(bi))};
        stale = false;
      }
      Cand y = own;
#pragma unroll 1
      for (int i = 32; i > 0; i >>= 1) {
        const Cand z{__shfl_xor(y.score, i, 64), __shfl_xor(y.place, i, 64)};
        if (before(z, y)) y = z;
      }
      if (lane == 0) best_s[wave] = y;
    }
    __syncthreads();
    Cand y = best_s[0];
#pragma unroll
    for (int w = 1; w < BW_WAVES; ++w)
      if (before(best_s[w], y)) y = best_s[w];
    if (bi >= 0 && own.place == y.place) {
      left &= ~(1u << bi);
      stale = true;
    }
    if (tid == 0) {
      const int64_t to = (int64_t)b * K + k;
      out_scores[to] = (float)from_ordered64(y.score);
      out_parents[to] = (int64_t)(~y.place >> 32);
      out_tokens[to] = (int64_t)(~y.place & 0xffffffffu);
    }
    __syncthreads();                               // (best_s is written again)
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// in place: a thread owns one unit of bytes of every beam of a sequence, loads all of them from where they come and only then stores.  Bound by
// bandwidth where there is much (64 x 5 beams of 3 x 36 KB: 8.7 us for 57 MB that the caches hold, 17.4 when the beams went through scratch memory), by
// the chain parents - load - store otherwise (2.9 us).
template <typename U, int NT>
__global__ __launch_bounds__(256) void beam_reorder_kernel(U* __restrict__ state, const int64_t* __restrict__ parents, int B, int N, int64_t row_units,
                                                           int64_t used_units) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int b = blockIdx.y;
  if (u >= used_units) return;
  U* base = state + ((int64_t)blockIdx.z * B + b) * N * row_units + u;
  int from[NT];                                    // the beam a beam comes from; itself where it stays (or is none)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int64_t p = n < N ? parents[(int64_t)b * N + n] : n;
    from[n] = n >= N ? n : (int)(p < 0 ? 0 : (p >= N ? N - 1 : p));
  }
  U val[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) val[n] = from[n] != n ? base[from[n] * row_units] : U{};
#pragma unroll
  for (int n = 0; n < NT; ++n)
    if (from[n] != n) base[n * row_units] = val[n];
}

template <typename U>
int launch_reorder(void* state, const int64_t* parents, int outer, int B, int N, int64_t row_bytes, int64_t used_bytes, hipStream_t st) {
  const int64_t ru = row_bytes / (int64_t)sizeof(U), uu = used_bytes / (int64_t)sizeof(U);
  const int64_t gx = (uu + 255) / 256;
  T2S_CHECK_ARG(gx < ((int64_t)1 << 24), "beam_reorder: rows too long");
  dim3 grid((unsigned)gx, (unsigned)B, (unsigned)outer), block(256);
  if (N <= 4) hipLaunchKernelGGL((beam_reorder_kernel<U, 4>), grid, block, 0, st, (U*)state, parents, B, N, ru, uu);
  else if (N <= 8) hipLaunchKernelGGL((beam_reorder_kernel<U, 8>), grid, block, 0, st, (U*)state, parents, B, N, ru, uu);
  else if (N <= 16) hipLaunchKernelGGL((beam_reorder_kernel<U, 16>), grid, block, 0, st, (U*)state, parents, B, N, ru, uu);
  else hipLaunchKernelGGL((beam_reorder_kernel<U, BS_MAX>), grid, block, 0, st, (U*)state, parents, B, N, ru, uu);
  T2S_CHECK_LAUNCH("beam_reorder");
  return 0;
}

// Workgroups of a row and the stretches each walks: one stretch each while that makes no more than BS_WGS workgroups (later stretches are
// cheaper, they have a bound to start from).  At most BS_CHUNKS workgroups.
void beam_chunks(int64_t rows, int64_t V, int* chunks, int* subs) {
  const int n = (int)((V + BS_SUB - 1) / BS_SUB);
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(BS_CHUNKS, (BS_WGS + rows - 1) / rows));
  *subs = (int)((n + most - 1) / most);
  *chunks = (n + *subs - 1) / *subs;
}

// Waves of a row where a sequence is a workgroup's, 0 where it has too many logits for one.  Measured, us, one workgroup and rows + join (and a launch
// less, 3 us of the host's): 1 x 5 beams of 5 600 logits 7.4 and 5.9 + 3.3, 64 of them 9.7 and 7.4 + 4.4, 1 024 37.0 and 31.9 + 4.6; 64 x 16 x 2 048 12.7 and
// 11.5 + 4.6; 8 x 1 x 32 768, 32 best 9.7 and 8.6 + 8.1; 1 x 1 x 50 5.2 and 4.1 + 2.7.  All of 1 x 5 x 5 600 logits equal: 31 and 31 + 4.7.
int beam_pieces(int64_t N, int64_t V) {
  const int64_t pieces = (V + BW_PIECE - 1) / BW_PIECE;
  return N * pieces <= BW_WAVES ? (int)pieces : 0;
}

}  // namespace

extern "C" int64_t t2s_beam_select_workspace_bytes(int B, int N, int V, int n_select) {
  if (B <= 0 || N <= 0 || V <= 0 || n_select <= 0 || beam_pieces(N, V)) return 0;
  int chunks, subs;
  beam_chunks((int64_t)B * N, V, &chunks, &subs);
  return (int64_t)B * N * chunks * (8 * (int64_t)n_select + 8 + 4);
}

extern "C" int t2s_beam_select(const void* logits, int64_t batch_stride, int64_t beam_stride, const float* scores, const uint8_t* finished,
                               int pad, float* out_scores, int64_t* out_parents, int64_t* out_tokens, void* workspace, int64_t workspace_bytes,
                               int B, int N, int V, int n_select, int dtype, t2s_stream_t stream) {
  T2S_CHECK_ARG(logits && scores && out_scores && out_parents && out_tokens && (workspace || !workspace_bytes), "beam_select: null pointer");
  T2S_CHECK_ARG(B > 0 && N > 0 && N <= BS_MAX && V > 0 && V <= 0x7ffffff0, "beam_select: bad shape B=%d N=%d V=%d (at most %d beams)", B, N, V, BS_MAX);
  T2S_CHECK_ARG(n_select > 0 && n_select <= BS_MAX && n_select <= (int64_t)N * V, "beam_select: %d of %d x %d candidates (at most %d)", n_select, N, V, BS_MAX);
  T2S_CHECK_ARG(pad >= 0 && pad < V, "beam_select: pad %d outside the vocabulary of %d", pad, V);
  T2S_CHECK_ARG(dtype == T2S_F32 || dtype == T2S_BF16, "beam_select: bad dtype %d", dtype);
  T2S_CHECK_ARG((uintptr_t)logits % (dtype == T2S_F32 ? 4 : 2) == 0, "beam_select: logits not aligned to their type");
  T2S_CHECK_ARG((uintptr_t)workspace % 8 == 0 && workspace_bytes >= t2s_beam_select_workspace_bytes(B, N, V, n_select), "beam_select: workspace of %lld bytes is too small",
                (long long)workspace_bytes);
  hipStream_t st = (hipStream_t)stream;
  if (const int pieces = beam_pieces(N, V)) {
    T2S_CHECK_ARG(B < (1 << 22), "beam_select: too many sequences");
    if (dtype == T2S_BF16)
      hipLaunchKernelGGL(beam_whole_kernel<bf16_t>, dim3((unsigned)B), dim3(64 * BW_WAVES), 0, st, (const bf16_t*)logits, batch_stride, beam_stride, scores, finished, out_scores,
                         out_parents, out_tokens, N, V, n_select, pad, pieces);
    else
      hipLaunchKernelGGL(beam_whole_kernel<float>, dim3((unsigned)B), dim3(64 * BW_WAVES), 0, st, (const float*)logits, batch_stride, beam_stride, scores, finished, out_scores,
                         out_parents, out_tokens, N, V, n_select, pad, pieces);
    T2S_CHECK_LAUNCH("beam_select");
    return 0;
  }
  int chunks, subs;
  beam_chunks((int64_t)B * N, V, &chunks, &subs);
  const int64_t rows = (int64_t)B * N, grid = rows * chunks;
  T2S_CHECK_ARG(grid < ((int64_t)1 << 24), "beam_select: too many rows");
  uint64_t* keys = (uint64_t*)workspace;
  double* sums = (double*)(keys + grid * n_select);
  float* maxs = (float*)(sums + grid);
  if (dtype == T2S_BF16)
    hipLaunchKernelGGL(beam_rows_kernel<bf16_t>, dim3((unsigned)grid), dim3(256), 0, st, (const bf16_t*)logits, batch_stride, beam_stride, scores, finished, keys, sums, maxs,
                       N, V, n_select, pad, chunks, subs);
  else
    hipLaunchKernelGGL(beam_rows_kernel<float>, dim3((unsigned)grid), dim3(256), 0, st, (const float*)logits, batch_stride, beam_stride, scores, finished, keys, sums, maxs,
                       N, V, n_select, pad, chunks, subs);
  T2S_CHECK_LAUNCH("beam_select");
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)B), dim3(256), 0, st, keys, sums, maxs, scores, finished, out_scores, out_parents, out_tokens, N, n_select, chunks);
  T2S_CHECK_LAUNCH("beam_join");
  return 0;
}

extern "C" int t2s_beam_reorder(void* state, const int64_t* parents, int outer, int B, int N, int64_t row_bytes, int64_t used_bytes, t2s_stream_t stream) {
  T2S_CHECK_ARG(state && parents, "beam_reorder: null pointer");
  T2S_CHECK_ARG(outer > 0 && outer <= 65535 && B > 0 && B <= 65535 && N > 0 && N <= BS_MAX, "beam_reorder: bad shape outer=%d B=%d N=%d (at most %d beams)", outer, B, N, BS_MAX);
  T2S_CHECK_ARG(used_bytes > 0 && used_bytes <= row_bytes, "beam_reorder: %lld of %lld bytes", (long long)used_bytes, (long long)row_bytes);
  hipStream_t st = (hipStream_t)stream;
  const uint64_t al = (uint64_t)(uintptr_t)state | (uint64_t)row_bytes | (uint64_t)used_bytes;
  if (al % 16 == 0) return launch_reorder<u32x4>(state, parents, outer, B, N, row_bytes, used_bytes, st);
  if (al % 8 == 0) return launch_reorder<u32x2>(state, parents, outer, B, N, row_bytes, used_bytes, st);
  if (al % 4 == 0) return launch_reorder<uint32_t>(state, parents, outer, B, N, row_bytes, used_bytes, st);
  if (al % 2 == 0) return launch_reorder<uint16_t>(state, parents, outer, B, N, row_bytes, used_bytes, st);
  return launch_reorder<uint8_t>(state, parents, outer, B, N, row_bytes, used_bytes, st);
}
