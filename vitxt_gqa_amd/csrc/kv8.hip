// The 8-bit key / value cache of answer decoding and the attention that reads it, for gfx950.
//
//  * t2s_kv8_append      quantises new K / V rows into the cache, behind each sequence's length, and advances the length
//  * t2s_kv8_dequantize  what the cache holds, as [B, H, capacity, 64] rows in the operand dtype
//  * t2s_kv8_attn        softmax(scale q K^T) V of a few query rows per sequence over [cache | the row's own tail]
//
// The decode step these serve is T2S._forward_mmt_and_output's eval loop (pythia/models/t2s.py:315-354): the prefix
// [question; frames; OCR] of up to 10 120 rows is the same in every step and for every beam, the decoded tokens are few.
//
// Cache format.  Token t of a sequence lies in block t / 64; a block of one head is 4 096 bytes of keys and 4 096 of values with
// one fp32 scale each.  amax = largest magnitude of the block's tokens (at least 2^-100); int8: s = amax / 127; e4m3: s = the
// least power of two with amax <= 448 s.  An element x is the int8 / e4m3 number nearest to x r, r = 1 / s rounded to fp32, ties
// to even, of the EXACT product (int8: one fma against 1.5 2^23; e4m3: a power-of-two product is exact): the code does not
// depend on how the product is rounded.  A value that is not finite makes its block's scale NaN: visible, never a wrong number.
//   keys    byte token * 64 + dim
//   values  byte dim * 64 + p, position p = g * 16 + t * 4 + r holding token t * 16 + g * 4 + r
// The value order is what the attention's registers hold: S^T = K Q^T by 16x16x32 MFMAs leaves lane (n = lane & 15, g = lane >> 4)
// with the scores of query n against tokens t * 16 + g * 4 + r, and P^T is fed back as the B operand of O^T = V^T P^T without leaving the
// lane; the 16 bytes a lane loads of value row `dim` are then the A operand against exactly those tokens.  No LDS, no
// shuffles between the two products, and every load of the pass is 16 contiguous bytes per lane.
#include "common.h"
#include "lanes.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int KV_BLOCK = 64;                       // tokens per block
constexpr int KV_HD = 64;                          // head dimension
constexpr int KV_BYTES = KV_BLOCK * KV_HD;         // code bytes of a block (keys or values)
constexpr float KV_LOG2E = 1.4426950408889634f;
constexpr float KV_LN2 = 0.6931471805599453f;

constexpr int FMT_INT8 = T2S_KV_INT8, FMT_E4M3 = T2S_KV_E4M3;

// the block's scale from the bits of its largest magnitude (>= 0x7f800000: a value that is not finite -> NaN)
template <int FMT>
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return as_f(0x7fc00000u);
  const float a = fmaxf(as_f(amax_bits), 0x1p-100f);
  if (FMT == FMT_INT8) return a / 127.0f;
  const uint32_t u = as_u(a);                      // 448 = 1.75 * 2^8
  return as_f(((u >> 23) - 8u + ((u & 0x7fffffu) > 0x600000u ? 1u : 0u)) << 23);
}

// four elements -> four codes; r = 1 / scale (0 for a block without a finite scale)
template <int FMT>
__device__ __forceinline__ uint32_t encode4(const float* x, float r) {
  if (FMT == FMT_INT8) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (as_u(__builtin_fmaf(x[i], r, 12582912.0f)) & 0xffu) << (8 * i);      // nearest even of the exact product
    return w;
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * r, x[1] * r, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * r, x[3] * r, w, true);
}

template <int FMT>
__device__ __forceinline__ void decode4(uint32_t w, float* x) {
  if (FMT == FMT_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  } else {
    typedef __attribute__((ext_vector_type(2))) float f2;
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
  }
}

// eight codes -> the bf16 operand of an MFMA (exact: int8 and e4m3 fit bf16's eight significant bits)
template <int FMT>
__device__ __forceinline__ bf16x8 decode8(uint32_t lo, uint32_t hi) {
  if (FMT == FMT_INT8) {
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (bf16_t)(float)(int8_t)(lo >> (8 * i));
#pragma unroll
    for (int i = 0; i < 4; ++i) r[4 + i] = (bf16_t)(float)(int8_t)(hi >> (8 * i));
    return r;
  }
  typedef __attribute__((ext_vector_type(2))) __bf16 b2;
  const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// ... and the f16 operand (exact: eleven significant bits, e4m3's 2^-9 .. 448 within f16's range)
template <int FMT>
__device__ __forceinline__ f16x8 decode8_f16(uint32_t lo, uint32_t hi) {
  typedef __attribute__((ext_vector_type(2))) _Float16 h2;
  if (FMT == FMT_INT8) {
    // code + 128 as the low byte of an f16 is 1024 + 128 + code: two bytes a v_perm_b32, two subtractions an instruction
    const h2 off = {(_Float16)1152.f, (_Float16)1152.f};
    const uint32_t l = lo ^ 0x80808080u, h = hi ^ 0x80808080u;
    const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, l, 0x04010400u)) - off, b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, l, 0x04030402u)) - off;
    const h2 c = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, h, 0x04010400u)) - off, d = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, h, 0x04030402u)) - off;
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// word position of token group tg (tokens 4 tg .. 4 tg + 3) inside a value row: p / 4 of the order above
__device__ __forceinline__ int v_word(int tg) { return (tg & 3) * 4 + (tg >> 2); }

// ------------------------------------------------------------------------------------------------------------------------------------
// append.  One workgroup = one (sequence, head) walking the blocks that the new tokens touch; a thread owns 4 tokens x 4 dims of a block, of
// keys and of values, so both storage orders are 32-bit words of it, and the words go out through LDS images as contiguous blocks.  HBM
// bound: the rows of the next block are on their way (their numbers, where a list names them, one block further) while a block is encoded.
// 64 x 12 pairs, 7 000 of 10 120 listed bf16 rows of a fused projection: 458 us for 1.39 GB read and 0.70 GB written, 4.5 TB/s (keys and values in
// workgroups of their own, nothing ahead: 619).  One token behind 84 for 48 x 12 pairs: 9.6 us, of which a workgroup's own chain - the length, the
// rows, what the block holds, a barrier, the codes, a barrier, the store - is 5.
struct AppendArgs {
  const void* x[2];                                // K, V
  int64_t x_bs[2], x_ts[2], x_hs[2];
  const int32_t *rows, *counts;
  int64_t rows_bs;
  uint8_t* codes[2];
  float* scales[2];
  int32_t *lens, *ticket;
  int B, H, T, L, nblk;
};

template <typename TX, int FMT>
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendArgs a) {
  typedef TX Raw __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(16))) uint32_t img[2][KV_BYTES / 4];
  __shared__ uint32_t red[2][4];
  const int tid = threadIdx.x, tg = tid >> 4, dg = tid & 15;
  const int h = blockIdx.y, b = blockIdx.z;
  const int len = a.lens[b];
  // A workgroup draws a ticket of its sequence once all of its waves have read the length (behind its first barrier: the ticket is on its way
  // while the block is encoded); the one with the last ticket advances the length at its end.
  int ticket = 0;
  const int cap = a.nblk * KV_BLOCK;
  int n = a.counts ? a.counts[b] : a.T;
  n = n < 0 ? 0 : (n > a.T ? a.T : n);
  const bool poisoned = len < 0 || len > cap;
  const int room = poisoned ? 0 : cap - len;
  const bool over = n > room;
  if (over) n = room;
  int begin = 0;
  bool idle = true;
  if (!poisoned && n > 0) {
    const TX* x[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) x[w] = (const TX*)a.x[w] + (int64_t)b * a.x_bs[w] + (int64_t)h * a.x_hs[w] + dg * 4;
    const int32_t* rows = a.rows ? a.rows + (int64_t)b * a.rows_bs : nullptr;
    const int64_t base = ((int64_t)b * a.H + h) * a.nblk;
    const int first = len / KV_BLOCK, last = (len + n - 1) / KV_BLOCK, stride = gridDim.x;
    // row numbers of this thread's four tokens of a block: -1 where there is no new token, L where the list names a row that is not there
    auto numbers = [&](int blk, int (&r)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = blk * KV_BLOCK + tg * 4 + i - len;
        r[i] = -1;
        if (j >= 0 && j < n) {
          r[i] = rows ? rows[j] : j;
          if (r[i] < 0 || r[i] > a.L) r[i] = a.L;
        }
      }
    };
    auto fetch = [&](const int (&r)[4], Raw (&d)[2][4]) {
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d[w][i] = Raw{(TX)0.f, (TX)0.f, (TX)0.f, (TX)0.f};
          if (r[i] >= 0 && r[i] < a.L) d[w][i] = *(const Raw*)(x[w] + r[i] * a.x_ts[w]);
          else if (r[i] >= a.L) d[w][i][0] = (TX)as_f(0x7fc00000u);    // a row that is not there: the block turns NaN
        }
    };
    int r_next[4];
    Raw d_next[2][4];
    begin = first + blockIdx.x;
    idle = begin > last;
    int blk = begin;
    if (blk <= last) {
      numbers(blk, r_next);
      fetch(r_next, d_next);
      if (blk + stride <= last) numbers(blk + stride, r_next);
    }
    for (; blk <= last; blk += stride) {
      const bool joins = blk == first && len % KV_BLOCK != 0;          // the block holds tokens already
      float val[2][4][4];                                               // [K, V][token][dim]
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < 4; ++d) val[w][i][d] = (float)d_next[w][i][d];
      if (blk + stride <= last) {
        fetch(r_next, d_next);
        if (blk + 2 * stride <= last) numbers(blk + 2 * stride, r_next);
      }
      float s_old[2] = {0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < 4; ++d) mx = max(mx, as_u(val[w][i][d]) & 0x7fffffffu);
        mx = wave_max(mx);
        if ((tid & 63) == 0) red[w][tid >> 6] = mx;
        if (joins) {                                                    // what the block holds, read before anyone writes (barrier below)
          const uint32_t* src = (const uint32_t*)(a.codes[w] + (base + blk) * KV_BYTES);
          s_old[w] = a.scales[w][base + blk];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float old[4];
            if (w == 0) {
              decode4<FMT>(src[(tg * 4 + i) * 16 + dg], old);           // token tg * 4 + i, four dims
              if (blk * KV_BLOCK + tg * 4 + i < len)
#pragma unroll
                for (int d = 0; d < 4; ++d) val[w][i][d] = old[d] * s_old[w];
            } else {
              decode4<FMT>(src[(dg * 4 + i) * 16 + v_word(tg)], old);   // dim dg * 4 + i, four tokens
#pragma unroll
              for (int t = 0; t < 4; ++t)
                if (blk * KV_BLOCK + tg * 4 + t < len) val[w][t][i] = old[t] * s_old[w];
            }
          }
        }
      }
      __syncthreads();
      if (tid == 0 && blk == begin) ticket = atomicAdd(a.ticket + b, 1);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t mx = max(max(red[w][0], red[w][1]), max(red[w][2], red[w][3]));
        float s = scale_of<FMT>(mx);
        if (joins && !(s >= s_old[w])) s = s != s ? s : s_old[w];       // the larger of the two; a NaN on either side stays
        const float r = s == s ? 1.0f / s : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float col[4] = {val[w][0][i], val[w][1][i], val[w][2][i], val[w][3][i]};
          const uint32_t code = s == s ? encode4<FMT>(w == 0 ? val[w][i] : col, r) : 0u;
          img[w][w == 0 ? (tg * 4 + i) * 16 + dg : (dg * 4 + i) * 16 + v_word(tg)] = code;
        }
        if (tid == 0) a.scales[w][base + blk] = s;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 2; ++w) ((uint4*)(a.codes[w] + (base + blk) * KV_BYTES))[tid] = ((const uint4*)img[w])[tid];
      // (the next block's barrier behind `red` keeps its image writes behind this block's reads)
    }
  }
  if (idle) {
    __syncthreads();
    if (tid == 0) ticket = atomicAdd(a.ticket + b, 1);
  }
  if (tid == 0 && ticket == (int)(gridDim.x * gridDim.y) - 1) {
    a.ticket[b] = 0;
    a.lens[b] = poisoned || over ? -1 : len + n;
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// read-back: one workgroup per (block walk, head and K / V, sequence).  A block comes in as 16 bytes a thread, is taken apart from LDS in the 4 x 4
// tiles of the append, and the next block is on its way meanwhile (word by word from HBM: 585 us where this takes 501).
template <typename TX, int FMT>
__global__ __launch_bounds__(256) void kv8_dequantize_kernel(const uint8_t* __restrict__ k8, const uint8_t* __restrict__ v8,
                                                             const float* __restrict__ ks, const float* __restrict__ vs,
                                                             const int32_t* __restrict__ lens, TX* __restrict__ k, TX* __restrict__ v,
                                                             int H, int nblk) {
  __shared__ __attribute__((aligned(16))) uint32_t img[2][KV_BYTES / 4];
  const int tid = threadIdx.x, tg = tid >> 4, dg = tid & 15;
  const int which = blockIdx.y & 1, h = blockIdx.y >> 1, b = blockIdx.z;
  const int len = lens[b];
  const int64_t base = ((int64_t)b * H + h) * nblk;
  const bool bad = len < 0 || len > nblk * KV_BLOCK;
  const float none = bad ? as_f(0x7fc00000u) : 0.f;
  const int held = bad || len <= 0 ? 0 : (len + KV_BLOCK - 1) / KV_BLOCK;          // blocks that hold something
  const uint4* src = (const uint4*)((which ? v8 : k8) + base * KV_BYTES) + tid;
  const float* sc = (which ? vs : ks) + base;
  uint4 next = {0, 0, 0, 0};
  float s_next = 0.f;
  int turn = 0;
  if ((int)blockIdx.x < held) {
    next = src[(int64_t)blockIdx.x * (KV_BYTES / 16)];
    s_next = sc[blockIdx.x];
  }
  for (int blk = blockIdx.x; blk < nblk; blk += gridDim.x, turn ^= 1) {
    TX* out = (which ? v : k) + ((base + blk) * KV_BLOCK + tg * 4) * KV_HD + dg * 4;
    float val[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < 4; ++d) val[i][d] = none;
    if (blk < held) {                              // (the same for the whole workgroup)
      const float s = s_next;
      ((uint4*)img[turn])[tid] = next;
      if (blk + (int)gridDim.x < held) {
        next = src[(int64_t)(blk + gridDim.x) * (KV_BYTES / 16)];
        s_next = sc[blk + gridDim.x];
      }
      __syncthreads();                             // (two images in turn: one barrier a block)
      const int left = len - blk * KV_BLOCK - tg * 4;                     // tokens of this thread's four that are there
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float c[4];
        if (which == 0) {
          decode4<FMT>(img[turn][(tg * 4 + i) * 16 + dg], c);
#pragma unroll
          for (int d = 0; d < 4; ++d) val[i][d] = i < left ? c[d] * s : 0.f;
        } else {
          decode4<FMT>(img[turn][(dg * 4 + i) * 16 + v_word(tg)], c);
#pragma unroll
          for (int t = 0; t < 4; ++t) val[t][i] = t < left ? c[t] * s : 0.f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) Vec4<TX>::store(out + i * KV_HD, f32x4{val[i][0], val[i][1], val[i][2], val[i][3]});
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// attention.  R = N * G query rows (N rows of a sequence, G query heads per key head) share the keys of one (sequence, head).
struct AttnArgs {
  const void* q;
  int64_t q_bs, q_ns, q_hs;
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  const int32_t* lens;
  const void *tk, *tv;
  int64_t t_bs, t_ns, t_ts, t_hs;
  const int32_t* tail_len;
  int64_t tl_bs, tl_ns;
  int tail_T;
  void* out;
  float* lse;
  float* part_o;        // [B * H][nshare][R][64]
  float* part_ml;       // [B * H][nshare][R][2]: running maximum (log2 units), sum
  float scale;
  int B, N, H, G, nblk, row_tiles;
  int nsplit, nshare, tail_groups;      // shares of the cache; one more for the tails unless a single share does it all; workgroups for the tails
};

// x as a sum of TERMS bf16 numbers (8 significant bits each): 1 for what is bf16 already, 2 keep 16 bits, 3 the whole of an fp32
template <int TERMS>
__device__ __forceinline__ void split_bf16(float x, bf16_t (&o)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    o[i] = (bf16_t)x;
    x -= (float)o[i];
  }
}

// The second product of a block: V^T P^T, codes times probabilities, for the tokens of step s of a lane.  A bf16 result takes its
// probabilities as f16: eleven bits, off by 2^-12 at most (and by 2^-25 of the largest where they are that small) before the result
// is rounded to eight bits.  An fp32 result takes them as three bf16 terms, which are all of an fp32 number.
template <typename TQ, int FMT>
struct Second;
template <int FMT>
struct Second<bf16_t, FMT> {
  typedef f16x8 V;
  struct P { f16x8 s[2]; };
  static __device__ __forceinline__ V decode(uint32_t lo, uint32_t hi) { return decode8_f16<FMT>(lo, hi); }
  static __device__ __forceinline__ void put(P& p, int i, int r, float x) { p.s[i >> 1][(i & 1) * 4 + r] = (_Float16)x; }
  static __device__ __forceinline__ f32x4 mul(const V (&v)[2], const P& p) {
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(v[1], p.s[1], __builtin_amdgcn_mfma_f32_16x16x32_f16(v[0], p.s[0], z, 0, 0, 0), 0, 0, 0);
  }
};
template <int FMT>
struct Second<float, FMT> {
  typedef bf16x8 V;
  struct P { bf16x8 s[2][3]; };
  static __device__ __forceinline__ V decode(uint32_t lo, uint32_t hi) { return decode8<FMT>(lo, hi); }
  static __device__ __forceinline__ void put(P& p, int i, int r, float x) {
    bf16_t w[3];
    split_bf16<3>(x, w);
#pragma unroll
    for (int k = 0; k < 3; ++k) p.s[i >> 1][k][(i & 1) * 4 + r] = w[k];
  }
  static __device__ __forceinline__ f32x4 mul(const V (&v)[2], const P& p) {
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 2; k >= 0; --k)
#pragma unroll
      for (int s = 0; s < 2; ++s) z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[s], p.s[s][k], z, 0, 0, 0);
    return z;
  }
};

// A query row's own tail, by one wave: running maximum (log2 units), sum, and o[lane] of dim `lane`.  Sixteen tokens at a time, four lanes
// (16 dims each) to a token; the values of the sixteen are on their way while the scores are made.
template <typename TQ>
__device__ __forceinline__ void tail_row(const AttnArgs& a, int b, int n, int hq, int lane, float& m, float& l, float& o) {
  m = -INFINITY;
  l = o = 0.f;
  int T = a.tail_len ? a.tail_len[(int64_t)b * a.tl_bs + (int64_t)n * a.tl_ns] : a.tail_T;
  T = T < 0 ? 0 : (T > a.tail_T ? a.tail_T : T);
  const int part = (lane & 3) * 16, tok = lane >> 2, h = hq / a.G;
  const float to_log2 = a.scale * KV_LOG2E;
  const TQ* qp = (const TQ*)a.q + (int64_t)b * a.q_bs + (int64_t)n * a.q_ns + (int64_t)hq * a.q_hs + part;
  const int64_t t_at = (int64_t)b * a.t_bs + (int64_t)n * a.t_ns + (int64_t)h * a.t_hs;
  const TQ* tk = (const TQ*)a.tk + t_at + part;
  const TQ* tv = (const TQ*)a.tv + t_at + lane;
  f32x4 q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = Vec4<TQ>::load(qp + i * 4);
  // (whole sixteens of the tail's capacity are requested before the row's own length is there; what is behind the length is not used)
  for (int t0 = 0; t0 < a.tail_T; t0 += 16) {
    if (t0 > 0 && t0 >= T) break;
    float x = 0.f, v[16];
    if (t0 + tok < a.tail_T) {
      f32x4 k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = Vec4<TQ>::load(tk + (int64_t)(t0 + tok) * a.t_ts + i * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < 4; ++d) x = __builtin_fmaf(q[i][d], k[i][d], x);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = (float)tv[(int64_t)min(t0 + i, a.tail_T - 1) * a.t_ts];
    x += dpp<DPP_XOR1>(x);
    x += dpp<DPP_XOR2>(x);
    x = t0 + tok < T ? x * to_log2 : -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = t0 + i < T ? v[i] : 0.f;
    const float mn = fmaxf(m, quads_max(x)), mu = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - mu), p = __builtin_amdgcn_exp2f(x - mu);
    l = l * f + quads_sum(p);
    o *= f;
    m = mn;
#pragma unroll
    for (int i = 0; i < 16; ++i) o = __builtin_fmaf(as_f((uint32_t)__builtin_amdgcn_readlane((int)as_u(p), i * 4)), v[i], o);
  }
}

// the row's result: one rounding.  Nothing seen: zeros, lse = -inf; a length that is none (the sequence overflowed on the device): NaN
__device__ __forceinline__ bool no_length(const AttnArgs& a, int len) { return len < 0 || len > a.nblk * KV_BLOCK; }
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * KV_LN2; }

// HBM bound from a few sequences on: 64 x 12 pairs, 5 rows, 1 to 10 120 tokens: 97 to 102 us for 505 MB of codes, 5.0 TB/s, though only a third of
// the matrix pipe's 16-row tile is in use; 2 x 8 pairs of 131 017 tokens, 4 rows: 55 to 58 us for 269 MB, 4.8 TB/s.  One sequence of 20 tokens:
// 5.4 us, a chain of latencies.
// One workgroup: one (sequence, head), one group of 16 QT query rows, one share of the blocks; its four waves take the blocks in turn,
// each with its own running maximum / sum / O, and are joined through LDS at the end.  With more than one share the results go to the
// workspace (the rows' tails are one share more, with workgroups of their own); a single share takes the tails of a few rows in as well and
// writes the output itself.
template <typename TQ, int FMT, int QT>
__global__ __launch_bounds__(256, 2) void kv8_attn_kernel(AttnArgs a) {
  typedef Second<TQ, FMT> PV;
  constexpr int TQN = sizeof(TQ) == 4 ? 3 : 1;     // bf16 terms of a query element
  constexpr int ROWS = 16 * QT;
  __shared__ __attribute__((aligned(16))) float o_s[4][16][KV_HD + 4];
  __shared__ __attribute__((aligned(16))) float t_s[ROWS][KV_HD];       // tails
  __shared__ float m_s[5][ROWS], l_s[5][ROWS];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int pair = blockIdx.x, b = pair / a.H, h = pair - b * a.H;
  const int R = a.N * a.G, row0 = blockIdx.y * ROWS, nrow = min(ROWS, R - row0);
  const bool direct = a.nshare == 1;
  // (the tails go first: their workgroups, a row to a wave, are short and end long before the others)
  const int split = (int)blockIdx.z - a.tail_groups, share = split < 0 ? a.nsplit : split;
  if (split < 0 || (direct && a.tk)) {
    for (int r = direct ? wave : (int)blockIdx.z * 4 + wave; r < nrow; r += direct ? 4 : ROWS) {
      const int row = row0 + r;
      float m, l, o;
      tail_row<TQ>(a, b, row / a.G, h * a.G + row % a.G, lane, m, l, o);
      if (direct) {
        t_s[r][lane] = o;
        if (lane == 0) {
          m_s[4][r] = m;
          l_s[4][r] = l;
        }
      } else {
        const int64_t at = ((int64_t)pair * a.nshare + share) * R + row;
        a.part_o[at * KV_HD + lane] = o;
        if (lane == 0) {
          a.part_ml[at * 2] = m;
          a.part_ml[at * 2 + 1] = l;
        }
      }
    }
    if (!direct) return;
  }
  const int len = a.lens[b];
  const int blocks = no_length(a, len) ? 0 : (len + KV_BLOCK - 1) / KV_BLOCK;
  const int per = blocks / a.nsplit, over = blocks - per * a.nsplit;
  const int b0 = split * per + min(split, over), b1 = b0 + per + (split < over ? 1 : 0);

  // queries: B operand, lane (n, g) holds dims g * 16 + step * 8 .. + 7 of row n.  A negative scale's sign goes into them.
  const float to_log2 = fabsf(a.scale) * KV_LOG2E;
  bf16x8 qf[QT][2][TQN];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int row = row0 + t * 16 + n;
    const int rc = row < R ? row : R - 1;
    const TQ* qp = (const TQ*)a.q + (int64_t)b * a.q_bs + (int64_t)(rc / a.G) * a.q_ns + (int64_t)(h * a.G + rc % a.G) * a.q_hs + g * 16;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x4 f = Vec4<TQ>::load(qp + s * 8 + e * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bf16_t w[TQN];
          split_bf16<TQN>(a.scale < 0.f ? -f[i] : f[i], w);
#pragma unroll
          for (int k = 0; k < TQN; ++k) qf[t][s][k][e * 4 + i] = w[k];
        }
      }
  }
  f32x4 o[QT][4];
  float m[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int d = 0; d < 4; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int64_t base = (int64_t)pair * a.nblk;
  // A block's keys are requested while the block before them is worked on (8 sequences x 12 heads x 5 rows over 10 120 tokens 15.2 us, 16.1 without;
  // 64 x 3 heads x 80 rows 90 us, 106), its values at the head of its own step: their turn comes behind the scores.
  uint4 kr[4];
  float ks_next = 0.f, vs_next = 0.f;
  auto fetch_k = [&](const int blk) {
    const uint8_t* kp = a.k8 + (base + blk) * KV_BYTES + n * KV_HD + g * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) kr[i] = *(const uint4*)(kp + i * 16 * KV_HD);
    ks_next = a.ks[base + blk];
    vs_next = a.vs[base + blk];
  };
  // one block; `whole`: all of its tokens are there (only the last block of a sequence is masked, by code of its own)
  auto step = [&](const int blk, auto whole) {
    constexpr bool last = !decltype(whole)::value;
    const uint8_t* vp = a.v8 + (base + blk) * KV_BYTES + n * KV_BLOCK + g * 16;
    const float ks = ks_next * to_log2, vs = vs_next;
    uint4 vr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) vr[i] = *(const uint4*)(vp + i * 16 * KV_BLOCK);
    const int left = len - blk * KV_BLOCK;                  // tokens of the block that are there
    bf16x8 kf[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kf[i][0] = decode8<FMT>(kr[i].x, kr[i].y);
      kf[i][1] = decode8<FMT>(kr[i].z, kr[i].w);
    }
    if (blk + 4 < b1) fetch_k(blk + 4);
    // scores of all row tiles, then one look at their maxima, then the probabilities: independent work side by side in each phase
    f32x4 x[QT][4];
    float mx[QT];
    bool moves = false;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int k = TQN - 1; k >= 0; --k) x[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i][s], qf[t][s][k], x[t][i], 0, 0, 0);
      }
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      mx[t] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (last) x[t][i][r] = i * 16 + g * 4 + r < left ? x[t][i][r] : -INFINITY;
          mx[t] = fmaxf(mx[t], x[t][i][r]);
        }
      mx[t] = across_max(mx[t]) * ks;
      moves |= mx[t] > m[t] + 8.f;
    }
    // the maximum need not be exact: it moves only when a score exceeds it by 2^8 (probabilities then stay below 2^8: in range, and as
    // precise as below 1), which after the first block hardly happens
    if (__any(moves)) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float mn = fmaxf(m[t], mx[t]);
        const float f = m[t] == mn ? 1.f : __builtin_amdgcn_exp2f(m[t] - mn);      // (0 the first time: exp2(-inf))
        m[t] = mn;
        l[t] *= f;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[t][d] *= f;
      }
    }
    typename PV::P pf[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float ms = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float e = __builtin_fmaf(x[t][i][r], ks, -ms);
          if (last) e = i * 16 + g * 4 + r < left ? e : -INFINITY;                 // (-inf times a scale of 0)
          const float p = __builtin_amdgcn_exp2f(e);
          l[t] += p;
          PV::put(pf[t], i, r, p);
        }
    }
    if (last) {                                             // codes behind the length count as zeros (an e4m3 NaN there would outlive p = 0)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t* w = (uint32_t*)&vr[i];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int k = left - (t * 16 + g * 4);
          w[t] &= k >= 4 ? 0xffffffffu : (k <= 0 ? 0u : (1u << (8 * k)) - 1u);
        }
      }
    }
    // values: a tile of 16 dims at a time, codes times probabilities, then the block's scale
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const typename PV::V vf[2] = {PV::decode(vr[d].x, vr[d].y), PV::decode(vr[d].z, vr[d].w)};
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const f32x4 z = PV::mul(vf, pf[t]);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[t][d][r] = __builtin_fmaf(z[r], vs, o[t][d][r]);
      }
    }
  };
  const int whole1 = min(b1, len / KV_BLOCK);               // (b1 <= blocks: at most one block behind it)
  int blk = b0 + wave;
  if (blk < b1) fetch_k(blk);
  for (; blk < whole1; blk += 4) step(blk, std::true_type{});
  if (blk < b1) step(blk, std::false_type{});
  // ---- join the four waves (and the tails)
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const float ls = across_sum(l[t]);
    if (g == 0) {
      m_s[wave][t * 16 + n] = m[t];
      l_s[wave][t * 16 + n] = ls;
    }
  }
  for (int t = 0; t < QT; ++t) {
#pragma unroll
    for (int d = 0; d < 4; ++d) *(f32x4*)&o_s[wave][n][d * 16 + g * 4] = o[t][d];
    __syncthreads();
    const int r = tid >> 4, c = (tid & 15) * 4, rr = t * 16 + r, row = row0 + rr;
    const bool tail = direct && a.tk && rr < nrow;
    const float mt = tail ? m_s[4][rr] : -INFINITY;
    const float m0 = fmaxf(fmaxf(fmaxf(m_s[0][rr], m_s[1][rr]), fmaxf(m_s[2][rr], m_s[3][rr])), mt);
    const float ms = m0 == -INFINITY ? 0.f : m0;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    float ls = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(m_s[w][rr] - ms);
      sum += *(const f32x4*)&o_s[w][r][c] * f;
      ls += l_s[w][rr] * f;
    }
    if (tail) {
      const float f = __builtin_amdgcn_exp2f(mt - ms);
      sum += *(const f32x4*)&t_s[rr][c] * f;
      ls += l_s[4][rr] * f;
    }
    if (row < R) {
      if (direct) {
        const float nan = as_f(0x7fc00000u), inv = no_length(a, len) ? nan : (ls == 0.f ? 0.f : 1.f / ls);
        const int64_t at = ((int64_t)b * a.N + row / a.G) * a.H * a.G + h * a.G + row % a.G;
        Vec4<TQ>::store((TQ*)a.out + at * KV_HD + c, sum * inv);
        if (c == 0) a.lse[at] = no_length(a, len) ? nan : lse_of(m0, ls);
      } else {
        const int64_t at = ((int64_t)pair * a.nshare + share) * R + row;
        *(f32x4*)(a.part_o + at * KV_HD + c) = sum;
        if (c == 0) {
          a.part_ml[at * 2] = m0;
          a.part_ml[at * 2 + 1] = ls;
        }
      }
    }
    __syncthreads();
  }
}

// Joins the shares of an output row: WPR waves to a row, each with every WPR-th share; lane s weighs share s, then lane d sums dim d.  A chain of
// two loads.  Four waves to a row where there are many shares, us with four and with one: 4 rows of 256 shares 7.2 and 19.9, 60 of 20 3.7 and 4.6,
// 12 288 of 4 20.5 and 7.2.
template <typename TQ, int WPR>
__global__ __launch_bounds__(256) void kv8_attn_join_kernel(AttnArgs a) {
  __shared__ float o_s[4][KV_HD], m_s[4], l_s[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, sub = wave % WPR;
  const int HQ = a.H * a.G, R = a.N * a.G;
  const int64_t rows = (int64_t)a.B * a.N * HQ;
  const int64_t row = (int64_t)blockIdx.x * (4 / WPR) + wave / WPR;           // b, n, query head
  const int64_t rc = row < rows ? row : rows - 1;
  const int hq = (int)(rc % HQ), n = (int)(rc / HQ % a.N), b = (int)(rc / HQ / a.N);
  const int64_t at0 = ((int64_t)b * a.H + hq / a.G) * a.nshare * R + n * a.G + hq % a.G;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int s0 = sub; s0 < a.nshare; s0 += 64 * WPR) {
    const int s = s0 + lane * WPR;
    float ms = -INFINITY, ls = 0.f;
    if (s < a.nshare) {
      const float2 ml = *(const float2*)(a.part_ml + (at0 + (int64_t)s * R) * 2);
      ms = ml.x;
      ls = ml.y;
    }
    float mx = ms;
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) mx = fmaxf(mx, __shfl_xor(mx, i, 64));
    const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - mu), w = __builtin_amdgcn_exp2f(ms - mu);
    l = l * f + wave_sum(ls * w);
    o *= f;
    m = mn;
    const int cnt = min(64, (a.nshare - s0 + WPR - 1) / WPR);
    const float* po = a.part_o + (at0 + (int64_t)s0 * R) * KV_HD + lane;
    for (int i0 = 0; i0 < cnt; i0 += 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i0 + i < cnt ? po[(int64_t)(i0 + i) * WPR * R * KV_HD] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) o = __builtin_fmaf(as_f((uint32_t)__builtin_amdgcn_readlane((int)as_u(w), (i0 + i) & 63)), v[i], o);
    }
  }
  if (WPR > 1) {
    o_s[wave][lane] = o;
    if (lane == 0) {
      m_s[wave] = m;
      l_s[wave] = l;
    }
    __syncthreads();
    m = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3]));
    const float mu = m == -INFINITY ? 0.f : m;
    o = l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(m_s[w] - mu);
      o += o_s[w][lane] * f;
      l += l_s[w] * f;
    }
    if (sub) return;
  }
  if (row < rows) {
    const bool bad = no_length(a, a.lens[b]);
    const float nan = as_f(0x7fc00000u);
    ((TQ*)a.out)[row * KV_HD + lane] = (TQ)(bad ? nan : (l == 0.f ? 0.f : o / l));
    if (lane == 0) a.lse[row] = bad ? nan : lse_of(m, l);
  }
}

template <typename TQ, int FMT>
void launch_attn(const AttnArgs& a, int qt, hipStream_t st) {
  const dim3 grid((unsigned)(a.B * a.H), (unsigned)a.row_tiles, (unsigned)(a.nsplit + a.tail_groups));
  if (qt == 1) hipLaunchKernelGGL((kv8_attn_kernel<TQ, FMT, 1>), grid, dim3(256), 0, st, a);
  else if (qt == 2) hipLaunchKernelGGL((kv8_attn_kernel<TQ, FMT, 2>), grid, dim3(256), 0, st, a);
  else if constexpr (sizeof(TQ) == 2) {
    if (qt == 3) hipLaunchKernelGGL((kv8_attn_kernel<TQ, FMT, 3>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv8_attn_kernel<TQ, FMT, 4>), grid, dim3(256), 0, st, a);
  }
}

template <typename TQ>
void launch_join(const AttnArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.N * a.H * a.G;
  if (a.nshare > 16) hipLaunchKernelGGL((kv8_attn_join_kernel<TQ, 4>), dim3((unsigned)rows), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((kv8_attn_join_kernel<TQ, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
}

// rows of a (sequence, head) whose tails a single share still takes in: four waves, two rows each (12 rows over 600 tokens and a tail
// of 12, 16 sequences: 17.1 us in one launch, 14.3 with workgroups for the tails and a join; 5 rows: 12.9 and 14.1)
constexpr int DIRECT_ROWS = 8;

// Workgroups of an append (each draws a ticket of its sequence).  64 x 12 pairs of 7 000 tokens, us: 2 048 565, 6 144 490, 16 384 461 - 4.5 TB/s,
// what a large copy reaches.
constexpr int APPEND_WGS = 16384;
// Workgroups of a read-back.  The same cache (0.7 GB of codes, 2 GB of bf16 values), us: 4 096 525, 16 384 511, 40 960 501 - 5.4 TB/s
constexpr int DEQUANTIZE_WGS = 40960;

bool kv8_bad_fmt(int fmt) { return fmt != FMT_INT8 && fmt != FMT_E4M3; }

// what a grid axis of 256 threads a workgroup can count: pairs, and output rows (a join may take a workgroup to a row)
bool kv8_attn_shape(int B, int N, int H, int G) {
  constexpr int64_t most = (int64_t)1 << 24;
  if (B <= 0 || N <= 0 || H <= 0 || G <= 0 || (int64_t)B * H >= most || (int64_t)N * G >= most) return false;
  return (int64_t)B * H * ((int64_t)N * G) < most;
}

// Row groups of a (sequence, head), each of which reads its cache: as few as registers allow (64 rows; fp32, with three terms to everything,
// 32), of equal size; returns the 16-row tiles of a group.  Measured, us: 16 x 12 pairs of 4 000 tokens, bf16, 64 rows in groups of 64 30.5, 32 32.4, 16
// 42.8; fp32, 32 rows in groups of 32 30.9, 16 33.5.  (A few pairs of 1 000 tokens, which the second-level caches hold, would be quicker in groups of 16:
// 10.2 and 5.7.)
int attn_row_tiles(int rows, int dtype, int* groups) {
  const int most = dtype == T2S_BF16 ? 64 : 32;
  *groups = (rows + most - 1) / most;
  return ((rows + *groups - 1) / *groups + 15) / 16;
}

}  // namespace

extern "C" int t2s_kv8_append(const void* k, int64_t k_batch_stride, int64_t k_row_stride, int64_t k_head_stride, const void* v,
                              int64_t v_batch_stride, int64_t v_row_stride, int64_t v_head_stride, const int32_t* rows, int64_t rows_batch_stride, const int32_t* counts, void* k8, void* v8, float* k_scale,
                              float* v_scale, int32_t* lens, int32_t* ticket, int B, int H, int T, int L, int nblk, int dtype, int fmt,
                              t2s_stream_t stream) {
  T2S_CHECK_ARG(k && v && k8 && v8 && k_scale && v_scale && lens && ticket, "kv8_append: null pointer");
  T2S_CHECK_ARG(B > 0 && B <= 65535 && H > 0 && H <= 32767 && T > 0 && L > 0 && nblk > 0 && nblk < (1 << 25), "kv8_append: bad shape B=%d H=%d T=%d L=%d nblk=%d", B, H, T, L, nblk);
  T2S_CHECK_ARG(rows || T <= L, "kv8_append: %d tokens of %d rows", T, L);
  T2S_CHECK_ARG(dtype == T2S_F32 || dtype == T2S_BF16, "kv8_append: bad dtype %d", dtype);
  T2S_CHECK_ARG(!kv8_bad_fmt(fmt), "kv8_append: bad format %d", fmt);
  const int al = dtype == T2S_F32 ? 16 : 8;
  T2S_CHECK_ARG((uintptr_t)k % al == 0 && (uintptr_t)v % al == 0 && k_batch_stride % 4 == 0 && k_row_stride % 4 == 0 && k_head_stride % 4 == 0 &&
                    v_batch_stride % 4 == 0 && v_row_stride % 4 == 0 && v_head_stride % 4 == 0,
                "kv8_append: rows must be aligned to 4 elements");
  T2S_CHECK_ARG((uintptr_t)k8 % 16 == 0 && (uintptr_t)v8 % 16 == 0, "kv8_append: the cache must be aligned to 16 bytes");
  AppendArgs a{{k, v}, {k_batch_stride, v_batch_stride}, {k_row_stride, v_row_stride}, {k_head_stride, v_head_stride}, rows, counts, rows_batch_stride, {(uint8_t*)k8, (uint8_t*)v8},
               {k_scale, v_scale}, lens, ticket, B, H, T, L, nblk};
  const int touched = (int)((T + 62LL) / 64 + 1);
  // enough workgroups to fill the card (8 of them run on a CU), no more: each draws a ticket of its sequence when it ends
  const int64_t pairs = (int64_t)B * H;
  int64_t gx = (APPEND_WGS + pairs - 1) / pairs;
  if (gx > touched) gx = touched;
  dim3 grid((unsigned)gx, (unsigned)H, (unsigned)B), block(256);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == T2S_BF16 && fmt == FMT_INT8) hipLaunchKernelGGL((kv8_append_kernel<bf16_t, FMT_INT8>), grid, block, 0, st, a);
  else if (dtype == T2S_BF16) hipLaunchKernelGGL((kv8_append_kernel<bf16_t, FMT_E4M3>), grid, block, 0, st, a);
  else if (fmt == FMT_INT8) hipLaunchKernelGGL((kv8_append_kernel<float, FMT_INT8>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((kv8_append_kernel<float, FMT_E4M3>), grid, block, 0, st, a);
  T2S_CHECK_LAUNCH("kv8_append");
  return 0;
}

extern "C" int t2s_kv8_dequantize(const void* k8, const void* v8, const float* k_scale, const float* v_scale, const int32_t* lens, void* k,
                                  void* v, int B, int H, int nblk, int dtype, int fmt, t2s_stream_t stream) {
  T2S_CHECK_ARG(k8 && v8 && k_scale && v_scale && lens && k && v, "kv8_dequantize: null pointer");
  T2S_CHECK_ARG(B > 0 && B <= 65535 && H > 0 && H <= 32767 && nblk > 0 && nblk < (1 << 25), "kv8_dequantize: bad shape B=%d H=%d nblk=%d", B, H, nblk);
  T2S_CHECK_ARG(dtype == T2S_F32 || dtype == T2S_BF16, "kv8_dequantize: bad dtype %d", dtype);
  T2S_CHECK_ARG(!kv8_bad_fmt(fmt), "kv8_dequantize: bad format %d", fmt);
  T2S_CHECK_ARG((uintptr_t)k8 % 16 == 0 && (uintptr_t)v8 % 16 == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "kv8_dequantize: 16-byte alignment");
  const int64_t pairs = (int64_t)B * H * 2;
  int64_t gx = (DEQUANTIZE_WGS + pairs - 1) / pairs;
  if (gx > nblk) gx = nblk;
  dim3 grid((unsigned)gx, (unsigned)(2 * H), (unsigned)B), block(256);
  hipStream_t st = (hipStream_t)stream;
  const uint8_t *a = (const uint8_t*)k8, *c = (const uint8_t*)v8;
  if (dtype == T2S_BF16 && fmt == FMT_INT8)
    hipLaunchKernelGGL((kv8_dequantize_kernel<bf16_t, FMT_INT8>), grid, block, 0, st, a, c, k_scale, v_scale, lens, (bf16_t*)k, (bf16_t*)v, H, nblk);
  else if (dtype == T2S_BF16)
    hipLaunchKernelGGL((kv8_dequantize_kernel<bf16_t, FMT_E4M3>), grid, block, 0, st, a, c, k_scale, v_scale, lens, (bf16_t*)k, (bf16_t*)v, H, nblk);
  else if (fmt == FMT_INT8)
    hipLaunchKernelGGL((kv8_dequantize_kernel<float, FMT_INT8>), grid, block, 0, st, a, c, k_scale, v_scale, lens, (float*)k, (float*)v, H, nblk);
  else
    hipLaunchKernelGGL((kv8_dequantize_kernel<float, FMT_E4M3>), grid, block, 0, st, a, c, k_scale, v_scale, lens, (float*)k, (float*)v, H, nblk);
  T2S_CHECK_LAUNCH("kv8_dequantize");
  return 0;
}

extern "C" int t2s_kv8_attn_splits(int B, int N, int H, int G, int max_tokens, int dtype) {
  if (!kv8_attn_shape(B, N, H, G)) return 0;
  const int blocks = max_tokens > 0 ? (int)(((int64_t)max_tokens + KV_BLOCK - 1) / KV_BLOCK) : 1;
  int groups;
  attn_row_tiles(N * G, dtype, &groups);
  const int64_t pairs = (int64_t)B * H * groups;
  // Else, few pairs: as many shares as three workgroups to a CU, of 8 blocks (two to a wave) at least.  Many pairs: shares of 20 blocks, so that
  // short sequences leave no long ones to wait for.  Measured, us (5 rows, 10 120 tokens): 12 pairs 1 share 37, 20 shares 9.9, 64 13.7; 96 pairs
  // 1 share 37, 8 15.2, 32 17.7; 768 pairs of ragged lengths 1 share 113, 8 103, 32 120.
  // Short caches: one share, whose workgroups write the output themselves.  Measured, us with one share and with two and a join (and a launch less, 4 us of the
  // host's): 12 pairs, 5 rows, bf16, 1 020 tokens 6.9 and 8.4, 1 530 8.5 and 8.4, 2 040 10.0 and 8.5; 192 pairs, 1 530 tokens 9.8 and 13.3; 768 pairs 26 and 30;
  // fp32, 12 pairs, 1 020 tokens 8.9 and 9.6, 1 530 11.3 and 9.6.
  if (N * G <= DIRECT_ROWS && blocks <= (dtype == T2S_BF16 ? 24 : 16)) return 1;
  const int64_t s = 768 / pairs >= 2 ? std::min((int64_t)768 / pairs, (int64_t)(blocks + 7) / 8) : (int64_t)(blocks + 19) / 20;
  return (int)(s < 1 ? 1 : s);
}

extern "C" int64_t t2s_kv8_attn_workspace_bytes(int B, int N, int H, int G, int splits) {
  if (!kv8_attn_shape(B, N, H, G) || splits < 1) return 0;
  return splits > 1 || N * G > DIRECT_ROWS ? (int64_t)B * H * (splits + 1) * N * G * (KV_HD + 2) * 4 : 0;
}

extern "C" int t2s_kv8_attn(const void* q, int64_t q_batch_stride, int64_t q_row_stride, int64_t q_head_stride, const void* k8, const void* v8,
                            const float* k_scale, const float* v_scale, const int32_t* lens, const void* tail_k, const void* tail_v,
                            int64_t t_batch_stride, int64_t t_row_stride, int64_t t_token_stride, int64_t t_head_stride,
                            const int32_t* tail_len, int64_t tl_batch_stride, int64_t tl_row_stride, int tail_T, void* out, float* lse,
                            void* workspace, int64_t workspace_bytes, int splits, int B, int N, int H, int G, int nblk, float scale, int dtype,
                            int fmt, t2s_stream_t stream) {
  T2S_CHECK_ARG(q && k8 && v8 && k_scale && v_scale && lens && out && lse && (workspace || !workspace_bytes), "kv8_attn: null pointer");
  T2S_CHECK_ARG(kv8_attn_shape(B, N, H, G) && nblk > 0 && nblk < (1 << 25),
                "kv8_attn: bad shape B=%d N=%d H=%d G=%d nblk=%d", B, N, H, G, nblk);
  T2S_CHECK_ARG(dtype == T2S_F32 || dtype == T2S_BF16, "kv8_attn: bad dtype %d", dtype);
  T2S_CHECK_ARG(!kv8_bad_fmt(fmt), "kv8_attn: bad format %d", fmt);
  T2S_CHECK_ARG((tail_k == nullptr) == (tail_v == nullptr) && tail_T >= 0, "kv8_attn: tail keys and values come together");
  const int al = dtype == T2S_F32 ? 16 : 8;
  T2S_CHECK_ARG((uintptr_t)q % al == 0 && q_batch_stride % 4 == 0 && q_row_stride % 4 == 0 && q_head_stride % 4 == 0, "kv8_attn: query rows must be aligned to 4 elements");
  T2S_CHECK_ARG((uintptr_t)tail_k % al == 0 && (uintptr_t)tail_v % al == 0 && t_batch_stride % 4 == 0 && t_row_stride % 4 == 0 && t_token_stride % 4 == 0 &&
                    t_head_stride % 4 == 0, "kv8_attn: tail rows must be aligned to 4 elements");
  T2S_CHECK_ARG((uintptr_t)k8 % 16 == 0 && (uintptr_t)v8 % 16 == 0 && (uintptr_t)workspace % 16 == 0, "kv8_attn: cache and workspace must be aligned to 16 bytes");
  T2S_CHECK_ARG(splits >= 1 && workspace_bytes >= t2s_kv8_attn_workspace_bytes(B, N, H, G, splits), "kv8_attn: workspace of %lld bytes is too small for %d shares",
                (long long)workspace_bytes, splits);
  int groups;
  const int rows = N * G, qt = attn_row_tiles(rows, dtype, &groups);
  AttnArgs a;
  a.q = q; a.q_bs = q_batch_stride; a.q_ns = q_row_stride; a.q_hs = q_head_stride;
  a.k8 = (const uint8_t*)k8; a.v8 = (const uint8_t*)v8; a.ks = k_scale; a.vs = v_scale; a.lens = lens;
  a.tk = tail_T > 0 ? tail_k : nullptr; a.tv = tail_v; a.t_bs = t_batch_stride; a.t_ns = t_row_stride; a.t_ts = t_token_stride; a.t_hs = t_head_stride;
  a.tail_len = tail_len; a.tl_bs = tl_batch_stride; a.tl_ns = tl_row_stride; a.tail_T = tail_T;
  a.out = out; a.lse = lse;
  a.scale = scale; a.B = B; a.N = N; a.H = H; a.G = G; a.nblk = nblk; a.nsplit = splits; a.nshare = a.tk && (splits > 1 || rows > DIRECT_ROWS) ? splits + 1 : splits;
  a.tail_groups = a.nshare > splits ? (std::min(rows, 16 * qt) + 3) / 4 : 0;
  a.row_tiles = groups;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + (int64_t)B * H * a.nshare * rows * KV_HD;
  T2S_CHECK_ARG(a.row_tiles <= 65535 && splits <= 65000, "kv8_attn: too many rows or shares");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == T2S_BF16) {
    if (fmt == FMT_INT8) launch_attn<bf16_t, FMT_INT8>(a, qt, st);
    else launch_attn<bf16_t, FMT_E4M3>(a, qt, st);
  } else {
    if (fmt == FMT_INT8) launch_attn<float, FMT_INT8>(a, qt, st);
    else launch_attn<float, FMT_E4M3>(a, qt, st);
  }
  T2S_CHECK_LAUNCH("kv8_attn");
  if (a.nshare == 1) return 0;
  if (dtype == T2S_BF16) launch_join<bf16_t>(a, st);
  else launch_join<float>(a, st);
  T2S_CHECK_LAUNCH("kv8_attn_join");
  return 0;
}
