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
// joins the stretches of a sequence and orders the candidates of its N rows by their scores in 64 bits (rows differ by
// cum - log-sum-exp, which 32 bits would merge into false ties).
#include "common.h"

namespace {

constexpr int BS_MAX = T2S_BEAM_MAX;               // beams, and candidates to select
constexpr int BS_EPT = 16;                         // elements of a thread per stretch
constexpr int BS_SUB = 256 * BS_EPT;
constexpr int BS_CHUNKS = 32;                      // stretches of a row at most; longer ones walk several in turn

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

template <typename TX>
__global__ __launch_bounds__(256) void beam_rows_kernel(const TX* __restrict__ logits, int64_t l_bs, int64_t l_ns, const float* __restrict__ cum,
                                                        const uint8_t* __restrict__ finished, uint64_t* __restrict__ keys, double* __restrict__ sums,
                                                        float* __restrict__ maxs, int N, int V, int K, int pad, int chunks, int subs) {
  __shared__ uint64_t best_s[256];
  __shared__ uint64_t list_s[BS_MAX * (BS_EPT + 1)];
  __shared__ uint64_t top_s[BS_MAX];
  __shared__ uint64_t thr_s;
  __shared__ int cnt_s;
  __shared__ float m_s[4];
  __shared__ double s_s[4];
  const int tid = threadIdx.x, chunk = blockIdx.x % chunks;
  const int64_t row = blockIdx.x / chunks;
  const int b = (int)(row / N), n = (int)(row % N);
  const TX* x = logits + (int64_t)b * l_bs + (int64_t)n * l_ns;
  const float c = cum[row];
  const bool dead = !(c > -INFINITY);                                  // -inf or NaN: every candidate of the row is -inf
  const bool ended = finished && finished[row];
  const bool virt = dead || ended;                                     // nothing of the row's logits is read
  const int only = dead ? -1 : pad;                                    // an ended row offers `pad` at its own score
  if (tid < BS_MAX) top_s[tid] = 0;
  float m = -INFINITY;
  double sum = 0.0;
  for (int sub = chunk * subs; sub < (chunk + 1) * subs; ++sub) {
    const int64_t v0 = (int64_t)sub * BS_SUB;
    if (v0 >= V) break;
    // of a row without logits only its first words (all -inf, lowest index first) and `pad` can be selected
    if (virt && sub != 0 && !(only >= v0 && only < v0 + BS_SUB)) continue;
    uint64_t key[BS_EPT];
    float val[BS_EPT];
    float mx = -INFINITY;
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < BS_EPT; ++i) {
      const int64_t v = v0 + i * 256 + tid;
      val[i] = -INFINITY;
      if (v < V) {
        if (!virt) val[i] = clean((float)x[v]);
        else if (v == only) val[i] = 0.f;
      }
      key[i] = v < V ? (uint64_t)ordered(val[i]) << 32 | (0xffffffffu - (uint32_t)v) : 0;
    }
#pragma unroll
    for (int i = 0; i < BS_EPT; ++i) {
      mx = fmaxf(mx, val[i]);
      best = key[i] > best ? key[i] : best;
    }
    if (mx > m) {
      sum *= (double)__expf(m - mx);
      m = mx;
    }
    if (m > -INFINITY) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < BS_EPT; ++i) s += __expf(val[i] - m);
      sum += (double)s;
    }
    // ---- the K best of (this stretch, what is kept of the former ones).  The K-th largest of the threads' best keys bounds the K-th
    // largest key from below, and only the K threads at or above it hold keys that count: at most K (BS_EPT + 1) of them.
    __syncthreads();
    const uint64_t kept = tid < K ? top_s[tid] : 0;
    best = kept > best ? kept : best;
    best_s[tid] = best;
    if (tid == 0) {
      thr_s = 1;
      cnt_s = 0;
    }
    __syncthreads();
    if (best) {
      int rank = 0;
#pragma unroll 16
      for (int i = 0; i < 256; ++i) rank += best_s[i] > best;
      if (rank == K - 1) thr_s = best;
    }
    __syncthreads();
    const uint64_t thr = thr_s;
    if (best >= thr) {
#pragma unroll
      for (int i = 0; i < BS_EPT; ++i)
        if (key[i] >= thr) list_s[atomicAdd(&cnt_s, 1)] = key[i];
      if (kept >= thr) list_s[atomicAdd(&cnt_s, 1)] = kept;
    }
    __syncthreads();
    const int cnt = cnt_s;
    for (int i = tid; i < cnt; i += 256) {
      const uint64_t mine = list_s[i];
      int rank = 0;
      for (int j = 0; j < cnt; ++j) rank += list_s[j] > mine;
      if (rank < K) top_s[rank] = mine;
    }
  }
  // ---- the row's maximum and sum over this workgroup
  float mw = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mw = fmaxf(mw, __shfl_xor(mw, o, 64));
  double sw = m > -INFINITY ? sum * exp((double)m - (double)mw) : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sw += __shfl_xor(sw, o, 64);
  if ((tid & 63) == 0) {
    m_s[tid >> 6] = mw;
    s_s[tid >> 6] = sw;
  }
  __syncthreads();
  const int64_t at = row * chunks + chunk;
  if (tid < K) keys[at * K + tid] = top_s[tid];
  if (tid == 0) {
    const float m4 = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3]));
    double s4 = 0.0;
    for (int w = 0; w < 4; ++w)
      if (m_s[w] > -INFINITY) s4 += s_s[w] * exp((double)m_s[w] - (double)m4);
    maxs[at] = m4;
    sums[at] = s4;
  }
}

struct Cand {
  double score;
  int64_t flat;       // n V + v; INT64_MAX: no candidate
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.score > b.score || (a.score == b.score && a.flat < b.flat); }

// one workgroup per sequence: joins the stretches, orders the N rows' candidates
__global__ __launch_bounds__(256) void beam_join_kernel(const uint64_t* __restrict__ keys, const double* __restrict__ sums, const float* __restrict__ maxs,
                                                        const float* __restrict__ cum, const uint8_t* __restrict__ finished, float* __restrict__ out_scores,
                                                        int64_t* __restrict__ out_parents, int64_t* __restrict__ out_tokens, int N, int V, int K, int chunks) {
  __shared__ double off_s[BS_MAX], score_s[256];
  __shared__ float top_m[BS_MAX];
  __shared__ int64_t flat_s[256];
  __shared__ int list_s[BS_MAX * BS_MAX * BS_CHUNKS * BS_MAX / 256];
  __shared__ int cnt_s;
  __shared__ Cand thr_s;
  const int tid = threadIdx.x, b = blockIdx.x;
  if (tid < N) {
    const int64_t row = (int64_t)b * N + tid;
    const float c = cum[row];
    float m = -INFINITY;
    for (int i = 0; i < chunks; ++i) m = fmaxf(m, maxs[row * chunks + i]);
    double s = 0.0;
    for (int i = 0; i < chunks; ++i) {
      const float mi = maxs[row * chunks + i];
      if (mi > -INFINITY) s += sums[row * chunks + i] * exp((double)mi - (double)m);
    }
    const bool ended = finished && finished[row];
    const double cd = c > -INFINITY ? (double)fminf(c, 3.402823466e38f) : -INFINITY;
    top_m[tid] = ended ? 0.f : m;
    off_s[tid] = ended || !(s > 0.0) ? cd : cd - log(s);
  }
  if (tid == 0) {
    cnt_s = 0;
    thr_s = Cand{-INFINITY, INT64_MAX};
  }
  __syncthreads();
  const int M = N * chunks * K;
  const uint64_t* kb = keys + (int64_t)b * M;
  auto cand = [&](int i) {
    const uint64_t k = kb[i];
    const int n = i / (chunks * K);
    if (!k) return Cand{-INFINITY, INT64_MAX};
    const float x = from_ordered((uint32_t)(k >> 32));
    const double sc = x > -INFINITY ? off_s[n] + ((double)x - (double)top_m[n]) : -INFINITY;
    return Cand{sc, (int64_t)n * V + (0xffffffffu - (uint32_t)k)};
  };
  Cand best{-INFINITY, INT64_MAX};
  for (int i = tid; i < M; i += 256) {
    const Cand c = cand(i);
    if (before(c, best)) best = c;
  }
  score_s[tid] = best.score;
  flat_s[tid] = best.flat;
  __syncthreads();
  if (best.flat != INT64_MAX) {
    int rank = 0;
    for (int i = 0; i < 256; ++i) rank += before(Cand{score_s[i], flat_s[i]}, best);
    if (rank == K - 1) thr_s = best;
  }
  __syncthreads();
  const Cand thr = thr_s;
  // the K best are among the candidates that do not come behind `thr`: those of at most K threads
  if (best.flat != INT64_MAX && !before(thr, best))
    for (int i = tid; i < M; i += 256) {
      const Cand c = cand(i);
      if (c.flat != INT64_MAX && !before(thr, c)) list_s[atomicAdd(&cnt_s, 1)] = i;
    }
  __syncthreads();
  const int cnt = cnt_s;
  for (int i = tid; i < cnt; i += 256) {
    const Cand mine = cand(list_s[i]);
    int rank = 0;
    for (int j = 0; j < cnt; ++j) rank += before(cand(list_s[j]), mine);
    if (rank < K) {
      const int64_t at = (int64_t)b * K + rank;
      out_scores[at] = (float)mine.score;
      out_parents[at] = mine.flat / V;
      out_tokens[at] = mine.flat % V;
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// in place: a thread owns one unit of bytes of every beam of a sequence, loads all of them from where they come and only then stores
template <typename U, int NT>
__global__ __launch_bounds__(256) void beam_reorder_kernel(U* __restrict__ state, const int64_t* __restrict__ parents, int B, int N, int64_t row_units,
                                                           int64_t used_units) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int b = blockIdx.y;
  if (u >= used_units) return;
  U* base = state + ((int64_t)blockIdx.z * B + b) * N * row_units + u;
  const int64_t* pb = parents + (int64_t)b * N;
  U val[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    if (n < N) {
      int64_t p = pb[n];
      p = p < 0 ? 0 : (p >= N ? N - 1 : p);
      if (p != n) val[n] = base[p * row_units];
    }
#pragma unroll
  for (int n = 0; n < NT; ++n)
    if (n < N) {
      int64_t p = pb[n];
      p = p < 0 ? 0 : (p >= N ? N - 1 : p);
      if (p != n) base[n * row_units] = val[n];
    }
}

template <typename U>
int launch_reorder(void* state, const int64_t* parents, int outer, int B, int N, int64_t row_bytes, int64_t used_bytes, hipStream_t st) {
  const int64_t ru = row_bytes / (int64_t)sizeof(U), uu = used_bytes / (int64_t)sizeof(U);
  const int64_t gx = (uu + 255) / 256;
  T2S_CHECK_ARG(gx < ((int64_t)1 << 31), "beam_reorder: rows too long");
  dim3 grid((unsigned)gx, (unsigned)B, (unsigned)outer), block(256);
  if (N <= 4) hipLaunchKernelGGL((beam_reorder_kernel<U, 4>), grid, block, 0, st, (U*)state, parents, B, N, ru, uu);
  else if (N <= 8) hipLaunchKernelGGL((beam_reorder_kernel<U, 8>), grid, block, 0, st, (U*)state, parents, B, N, ru, uu);
  else if (N <= 16) hipLaunchKernelGGL((beam_reorder_kernel<U, 16>), grid, block, 0, st, (U*)state, parents, B, N, ru, uu);
  else hipLaunchKernelGGL((beam_reorder_kernel<U, BS_MAX>), grid, block, 0, st, (U*)state, parents, B, N, ru, uu);
  T2S_CHECK_LAUNCH("beam_reorder");
  return 0;
}

// stretches of a row, and how many sub-stretches each walks
void beam_chunks(int V, int* chunks, int* subs) {
  const int n = (int)(((int64_t)V + BS_SUB - 1) / BS_SUB);
  *subs = (n + BS_CHUNKS - 1) / BS_CHUNKS;
  *chunks = (n + *subs - 1) / *subs;
}

}  // namespace

extern "C" int64_t t2s_beam_select_workspace_bytes(int B, int N, int V, int n_select) {
  if (B <= 0 || N <= 0 || V <= 0 || n_select <= 0) return 0;
  int chunks, subs;
  beam_chunks(V, &chunks, &subs);
  return (int64_t)B * N * chunks * (8 * (int64_t)n_select + 8 + 4);
}

extern "C" int t2s_beam_select(const void* logits, int64_t batch_stride, int64_t beam_stride, const float* scores, const uint8_t* finished,
                               int pad, float* out_scores, int64_t* out_parents, int64_t* out_tokens, void* workspace, int64_t workspace_bytes,
                               int B, int N, int V, int n_select, int dtype, t2s_stream_t stream) {
  T2S_CHECK_ARG(logits && scores && out_scores && out_parents && out_tokens && workspace, "beam_select: null pointer");
  T2S_CHECK_ARG(B > 0 && N > 0 && N <= BS_MAX && V > 0 && V <= 0x7ffffff0, "beam_select: bad shape B=%d N=%d V=%d (at most %d beams)", B, N, V, BS_MAX);
  T2S_CHECK_ARG(n_select > 0 && n_select <= BS_MAX && n_select <= (int64_t)N * V, "beam_select: %d of %d x %d candidates (at most %d)", n_select, N, V, BS_MAX);
  T2S_CHECK_ARG(pad >= 0 && pad < V, "beam_select: pad %d outside the vocabulary of %d", pad, V);
  T2S_CHECK_ARG(dtype == T2S_F32 || dtype == T2S_BF16, "beam_select: bad dtype %d", dtype);
  T2S_CHECK_ARG((uintptr_t)workspace % 8 == 0 && workspace_bytes >= t2s_beam_select_workspace_bytes(B, N, V, n_select), "beam_select: workspace of %lld bytes is too small",
                (long long)workspace_bytes);
  int chunks, subs;
  beam_chunks(V, &chunks, &subs);
  const int64_t rows = (int64_t)B * N, grid = rows * chunks;
  T2S_CHECK_ARG(grid < ((int64_t)1 << 31), "beam_select: too many rows");
  uint64_t* keys = (uint64_t*)workspace;
  double* sums = (double*)(keys + grid * n_select);
  float* maxs = (float*)(sums + grid);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == T2S_BF16)
    hipLaunchKernelGGL(beam_rows_kernel<bf16_t>, dim3((unsigned)grid), dim3(256), 0, st, (const bf16_t*)logits, batch_stride, beam_stride, scores, finished, keys, sums, maxs,
                       N, V, n_select, pad, chunks, subs);
  else
    hipLaunchKernelGGL(beam_rows_kernel<float>, dim3((unsigned)grid), dim3(256), 0, st, (const float*)logits, batch_stride, beam_stride, scores, finished, keys, sums, maxs,
                       N, V, n_select, pad, chunks, subs);
  T2S_CHECK_LAUNCH("beam_select");
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)B), dim3(256), 0, st, keys, sums, maxs, scores, finished, out_scores, out_parents, out_tokens, N, V, n_select, chunks);
  T2S_CHECK_LAUNCH("beam_join");
  return 0;
}

extern "C" int t2s_beam_reorder(void* state, const int64_t* parents, int outer, int B, int N, int64_t row_bytes, int64_t used_bytes, t2s_stream_t stream) {
  T2S_CHECK_ARG(state && parents, "beam_reorder: null pointer");
  T2S_CHECK_ARG(outer > 0 && outer <= 65535 && B > 0 && B <= 65535 && N > 0 && N <= BS_MAX, "beam_reorder: bad shape outer=%d B=%d N=%d (at most %d beams)", outer, B, N, BS_MAX);
  T2S_CHECK_ARG(used_bytes > 0 && used_bytes <= row_bytes, "beam_reorder: %lld of %lld bytes", (long long)used_bytes, (long long)row_bytes);
  hipStream_t st = (hipStream_t)stream;
  const uint64_t al = (uint64_t)(uintptr_t)state | (uint64_t)row_bytes | (uint64_t)used_bytes;
  if (al % 16 == 0) return launch_reorder<uint4>(state, parents, outer, B, N, row_bytes, used_bytes, st);
  if (al % 8 == 0) return launch_reorder<uint2>(state, parents, outer, B, N, row_bytes, used_bytes, st);
  if (al % 4 == 0) return launch_reorder<uint32_t>(state, parents, outer, B, N, row_bytes, used_bytes, st);
  if (al % 2 == 0) return launch_reorder<uint16_t>(state, parents, outer, B, N, row_bytes, used_bytes, st);
  return launch_reorder<uint8_t>(state, parents, outer, B, N, row_bytes, used_bytes, st);
}
