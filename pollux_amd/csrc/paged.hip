// The paged KV cache: keys and values of sequences of any length in pages that
// all of them share, as fp32, fp16 or INT8 with a scale per key (or value) and
// head, and attention of new tokens over it.
//
//   page layout: k, v [pages, H, page_size, 24]; INT8 with fp32 scales
//   [pages, H, page_size].  Position j of sequence r lies in page
//   table[r, j / page_size], slot j % page_size: the slots of a page are
//   consecutive rows of 24 values per head, so a head's keys are read in runs
//   of page_size rows.
//   The new tokens of a step are rows cu_q[r] .. cu_q[r+1]-1 of one flat array
//   and the last positions of their sequences: kv_len[r] counts them.
//
// paged_write_kernel / paged_read_kernel: the new tokens' keys (RMS-normalised)
//   and values into their slots, and back as fp32.
// paged_decode_kernel: attention of one new token per sequence.
// paged_chunk_kernel: attention of several, on fp16 MFMA.
// paged_combine_kernel: the softmax states of a row's key ranges joined.
//
// Lengths, offsets and page ids are read from device memory (a captured graph
// replays a step while they change), so nothing on the host has checked them:
// a sequence whose length or page leaves its bounds is written nowhere, and
// its outputs are NaN.

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "plx_device.h"

namespace plx {
namespace {

constexpr int kThreads = 256;
constexpr int kPart = 28;            // floats of a key range's softmax state: 24 sums, maximum, weight, unit, -
constexpr float kLow = -3.0e38f;     // a maximum before any key (finite: kLow - kLow is 0, not NaN)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInv127 = 1.0f / 127.0f;
constexpr float kTiny = 1.2037062152420224e-35f;  // 2^-116: 127 / |x| leaves fp32 below

struct Batch {
  const int32_t *table, *cu_q, *kv_len, *order;
  int64_t table_stride, tokens;
  int seqs, max_q, max_kv;
  int first, count;  // the part of the order that a launch takes
};

struct Pages {
  void *k, *v;
  float *k_scale, *v_scale;
  int64_t pages;
  int heads, shift;  // page_size = 1 << shift
};

// ---- 8 values of any type as floats ---------------------------------------

struct bf16_t {
  uint16_t bits;
};

template <class T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
  if constexpr (std::is_same_v<T, float>) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, bf16_t>) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      } else {
        x[2 * i] = __half2float(__ushort_as_half(static_cast<uint16_t>(w[i])));
        x[2 * i + 1] = __half2float(__ushort_as_half(static_cast<uint16_t>(w[i] >> 16)));
      }
    }
  }
}

// a NaN stays a NaN (the carry of its rounding could leave the exponent)
__device__ __forceinline__ uint32_t to_bf16(float f) { return f != f ? 0x7FC0u : bf16_rne_bits(f); }

template <class T>
__device__ __forceinline__ uint32_t bits16(float f) {
  if constexpr (std::is_same_v<T, bf16_t>) return to_bf16(f);
  else return __half_as_ushort(__float2half_rn(f));
}

// 4 values rounded once to T, 4 consecutive elements at p
template <class T>
__device__ __forceinline__ void store4(T *p, float a, float b, float c, float d) {
  if constexpr (std::is_same_v<T, float>)
    *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d);
  else
    *reinterpret_cast<uint2 *>(p) =
        make_uint2(bits16<T>(a) | bits16<T>(b) << 16, bits16<T>(c) | bits16<T>(d) << 16);
}

__device__ __forceinline__ float byte_of(uint32_t w, int i) {  // signed byte i of w
  return static_cast<float>(static_cast<int>(w << (24 - 8 * i)) >> 24);
}

// ---- where a sequence's tokens are ----------------------------------------

// The sequence at place i of a launch's part of the order; -1 where that names none.
__device__ __forceinline__ int sequence_at(const Batch &b, int i) {
  const int r = b.order ? b.order[b.first + i] : b.first + i;
  return r >= 0 && r < b.seqs ? r : -1;
}

// Sequence r: its first row, its new tokens, its length; false where they leave the batch's bounds.
__device__ __forceinline__ bool sequence(const Batch &b, int r, int &row0, int &n, int &len) {
  row0 = b.cu_q[r];
  n = b.cu_q[r + 1] - row0;
  len = b.kv_len[r];
  return row0 >= 0 && n >= 0 && static_cast<int64_t>(row0) + n <= b.tokens && n <= b.max_q && len >= 0 &&
         len <= b.max_kv;
}

// NaN into head h of all the rows that cu_q gives a sequence out of bounds (its new tokens may be more than max_q), as far
// as they are the batch's: those from `at` on, `step` apart.
template <class TX>
__device__ __forceinline__ void nan_rows(TX *out, const Batch &b, int heads, int h, int row0, int n, int64_t at,
                                         int64_t step) {
  if (row0 < 0) return;
  const float nan = __builtin_nanf("");
  for (int64_t i = at; i < n && row0 + i < b.tokens; i += step)
#pragma unroll 1
    for (int d = 0; d < kDim; d += 4) store4(out + ((row0 + i) * heads + h) * kDim + d, nan, nan, nan, nan);
}

// Page of position j (0 <= j < max_kv) or -1.
__device__ __forceinline__ int page_of(const Batch &b, const Pages &kv, int r, int j) {
  const int p = b.table[r * b.table_stride + (j >> kv.shift)];
  return p >= 0 && p < kv.pages ? p : -1;
}

// Row index (of 24 values) of position j in page p, head h.
__device__ __forceinline__ int64_t slot_of(const Pages &kv, int p, int h, int j) {
  return ((static_cast<int64_t>(p) * kv.heads + h) << kv.shift) + (j & ((1 << kv.shift) - 1));
}

// ---- write and read -------------------------------------------------------

constexpr int kWrTok = 16, kWrHeads = 16;  // tokens x heads per block

// One thread per key or value of a head: 16 heads of 16 tokens a block, so that reads run over neighbouring heads
// and writes over neighbouring slots.  The norm is taken in fp64 and rounded once: a code's border then does
// not depend on the order of the sum.
// Bound by bytes, 3.5 to 3.9 TB/s: 1.5 million fp32 rows into INT8 take 52 us (36 at a copy's rate; the norm and the codes issue
// for some 20 of them), 2.6 million bf16 rows into fp16 64 us.  A row by three threads, or loads by consecutive lanes
// through LDS, cost the INT8 case 80 and 60 us: sums and maxima then cross lanes, and barriers part loads from stores.
// 32 x 8 and 64 x 4 blocks gain 2 to 5% here but leave a decode step's single tokens on 8 or 4 lanes of a block.
template <class TX, class TKV>
__global__ __launch_bounds__(kThreads) void paged_write_kernel(const TX *__restrict__ k, const TX *__restrict__ v,
                                                               int64_t stride, const float *__restrict__ norm_w,
                                                               float eps, Pages kv, Batch b, int q_tiles,
                                                               int head_tiles) {
  int idx = blockIdx.x;
  const bool is_v = idx & 1;
  idx >>= 1;
  const int ht = idx % head_tiles;
  idx /= head_tiles;
  const int qt = idx % q_tiles, r = idx / q_tiles;
  int row0, n, len;
  if (!sequence(b, r, row0, n, len)) return;
  const int i = qt * kWrTok + (threadIdx.x >> 4), h = ht * kWrHeads + (threadIdx.x & 15);
  const int j = len - n + i;
  if (i >= n || h >= kv.heads || j < 0) return;
  const int page = page_of(b, kv, r, j);
  if (page < 0) return;
  const TX *src = (is_v ? v : k) + (row0 + i) * stride + h * kDim;
  float x[3][8];
#pragma unroll
  for (int o = 0; o < 3; ++o) load8(src + 8 * o, x[o]);
  if (!is_v && norm_w) {
    double ss = 0.0;
#pragma unroll
    for (int o = 0; o < 3; ++o)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fma(static_cast<double>(x[o][e]), static_cast<double>(x[o][e]), ss);
    const double f = 1.0 / sqrt(ss / kDim + static_cast<double>(eps));
#pragma unroll
    for (int o = 0; o < 3; ++o)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[o][e] = f32_kept(static_cast<float>(x[o][e] * f * static_cast<double>(norm_w[8 * o + e])));
  }
  const int64_t at = slot_of(kv, page, h, j);
  if constexpr (std::is_same_v<TKV, int8_t>) {
    float a = 0.f;
    bool finite = true;
#pragma unroll
    for (int o = 0; o < 3; ++o)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a = fmaxf(a, fabsf(x[o][e]));
        finite &= (__float_as_uint(x[o][e]) & 0x7F800000u) != 0x7F800000u;
      }
    const bool live = finite && a >= kTiny;
    const float inv = live ? 127.0f / a : 0.f;
    uint2 *dst = reinterpret_cast<uint2 *>(static_cast<int8_t *>(is_v ? kv.v : kv.k) + at * kDim);
#pragma unroll
    for (int o = 0; o < 3; ++o) {
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float c = live ? fminf(fmaxf(rintf(x[o][e] * inv), -127.f), 127.f) : 0.f;
        w[e >> 2] |= (static_cast<uint32_t>(static_cast<int>(c)) & 0xFFu) << (8 * (e & 3));
      }
      dst[o] = make_uint2(w[0], w[1]);
    }
    (is_v ? kv.v_scale : kv.k_scale)[at] = live ? a * kInv127 : finite ? 0.f : __builtin_nanf("");
  } else {
    TKV *dst = static_cast<TKV *>(is_v ? kv.v : kv.k) + at * kDim;
#pragma unroll
    for (int o = 0; o < 3; ++o) {
      store4(dst + 8 * o, x[o][0], x[o][1], x[o][2], x[o][3]);
      store4(dst + 8 * o + 4, x[o][4], x[o][5], x[o][6], x[o][7]);
    }
  }
}

// The same slots as fp32.  A thread per 8 values (three of a row), so that neighbouring lanes store neighbouring 32 bytes:
// with a row per thread, 96 bytes apart, 1.5 million INT8 rows took 52 us in place of 36 (5.1 TB/s).
template <class TKV>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(Pages kv, Batch b, int q_tiles, int head_tiles,
                                                              float *__restrict__ k_out, float *__restrict__ v_out) {
  int idx = blockIdx.x;
  const bool is_v = idx & 1;
  idx >>= 1;
  const int ht = idx % head_tiles;
  idx /= head_tiles;
  const int qt = idx % q_tiles, r = idx / q_tiles;
  int row0, n, len;
  if (!sequence(b, r, row0, n, len)) {
    const int h = ht * kWrHeads + (threadIdx.x & 15);
    if (h < kv.heads)
      nan_rows(is_v ? v_out : k_out, b, kv.heads, h, row0, n, qt * kWrTok + (threadIdx.x >> 4), int64_t{q_tiles} * kWrTok);
    return;
  }
#pragma unroll
  for (int u = threadIdx.x; u < kWrTok * kWrHeads * 3; u += kThreads) {  // 8 values each
    const int o = u % 3, i = qt * kWrTok + u / 3 / kWrHeads, h = ht * kWrHeads + u / 3 % kWrHeads;
    if (i >= n || h >= kv.heads) continue;
    const int j = len - n + i;
    const int page = j < 0 ? 0 : page_of(b, kv, r, j);
    float *dst = (is_v ? v_out : k_out) + ((static_cast<int64_t>(row0) + i) * kv.heads + h) * kDim + 8 * o;
    float x[8];
    if (page < 0 || j < 0) {  // no such page; a token before the sequence's first position
      const float fill = page < 0 ? __builtin_nanf("") : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fill;
    } else {
      const int64_t at = slot_of(kv, page, h, j);
      const TKV *src = static_cast<const TKV *>(is_v ? kv.v : kv.k) + at * kDim + 8 * o;
      if constexpr (std::is_same_v<TKV, int8_t>) {
        const float s = (is_v ? kv.v_scale : kv.k_scale)[at];
        const uint2 w = *reinterpret_cast<const uint2 *>(src);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = byte_of(e < 4 ? w.x : w.y, e & 3) * s;
      } else {
        load8(src, x);
      }
    }
    store4(dst, x[0], x[1], x[2], x[3]);
    store4(dst + 4, x[4], x[5], x[6], x[7]);
  }
}

// ---- attention of one token per sequence ----------------------------------

// The sums a[0 .. W-1] over the lanes that differ in the bits from OFF on: lane pairs split their sums between them until
// 3 are left (their first dim is returned), those are added up.
template <int W, int OFF, int D>
__device__ __forceinline__ int join_lanes(float (&a)[D], int lane, int first) {
  if constexpr (W > 3) {
    const bool up = lane & OFF;
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const float give = up ? a[i] : a[i + W / 2], keep = up ? a[i + W / 2] : a[i];
      a[i] = keep + __shfl_xor(give, OFF, 64);
    }
    return join_lanes<W / 2, OFF * 2>(a, lane, first + (up ? W / 2 : 0));
  } else if constexpr (OFF < 64) {
#pragma unroll
    for (int i = 0; i < 3; ++i) a[i] += __shfl_xor(a[i], OFF, 64);
    return join_lanes<W, OFF * 2>(a, lane, first);
  } else {
    return first;
  }
}

// o = sum_j 2^(s_j c - m c) V_j / sum_j 2^(s_j c - m c), s_j = q . K_j, c = log2(e) / sqrt 24, m the largest s_j so far.
// Bound by bytes where there are many: 64 sequences of up to 1,024 INT8 positions and 80 heads take 34 us (152 MB: 30 us
// at a copy's rate), 4 of up to 32,768 fp16 positions 111 us (588 MB: 115; a read alone is faster than a copy); one sequence of 777 positions 5.6 us, a chain
// of latencies (table, page, rows, joins).
// One item per (sequence, head, key range).  A key's row is read by sizeof(TKV) lanes, 24 bytes (3 loads of 8) each,
// so a wave's loads run over consecutive rows; a lane keeps its own online softmax over its keys (every 4 waves x
// 64 / sizeof(TKV) keys, kDecRounds of them at once: one maximum and one rescaling for all), and the lanes' states
// are joined at the end: their 24 / sizeof(TKV) sums are halved between lane pairs until 3 are left, which takes a
// quarter of the exchanges of a reduction of all.  W: waves per item; with 1 a block has four items of its own and no
// barrier, which is faster where items are many and short.  64 sequences of up to n positions, 80 heads, us by one wave and
// by four: INT8 n = 256 14.4 and 35.2, 1,024 30.9 and 44.2, 2,048 59.6 and 67.8, 4,096 109.5 and 113.0; fp16 256 16.0 and
// 25.0, 1,024 50.4 and 52.0, 2,048 94.2 and 94.0, 4,096 182 and 177; fp32 256 23.8 and 28.7, 512 50.2 and 50.7, 1,024 94.8
// and 93.4, 2,048 183 and 176.  (One wave from n * sizeof(TKV) of 1,024 down: up to 2,048 it would lose nowhere either.)
constexpr int kDecRounds = 4;
template <class TX, class TKV, int W>
__global__ __launch_bounds__(kThreads) void paged_decode_kernel(const TX *__restrict__ q, int64_t stride,
                                                                const float *__restrict__ norm_w, float eps, Pages kv,
                                                                Batch b, int alone, int range, int splits,
                                                                float cst, TX *__restrict__ out,
                                                                float *__restrict__ part) {
  constexpr int G = sizeof(TKV);          // lanes per key
  constexpr int D = kDim / G;             // dims per lane
  constexpr int K = 64 / G;               // keys per wave and round
  constexpr int kWaves = W;               // of an item
  __shared__ float red[kWaves][kDim + 2];
  const int lane = threadIdx.x & 63, block_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = block_wave % W, tid = 64 * wave + lane;  // in the item
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / 64 / W) + block_wave / W;
  if (item >= static_cast<int64_t>(b.count) * kv.heads * splits) return;
  const int sp = static_cast<int>(item % splits);
  const int pair = static_cast<int>(item / splits), r = sequence_at(b, pair / kv.heads), h = pair % kv.heads;
  if (r < 0) return;
  int row0, n, len;
  if (!sequence(b, r, row0, n, len) || (alone && n > 1)) {  // (not alone: the chunk kernel has all sequences and answers)
    if (alone && sp == 0) nan_rows(out, b, kv.heads, h, row0, n, tid, 64 * W);
    return;
  }
  if (n != 1) return;
  const int begin = sp * range, end = min(len, begin + range);
  if (begin >= end && sp > 0) return;  // (the range of an empty sequence still writes its zeros)

  // this lane's dims of the query, normalised
  const int d0 = (lane & (G - 1)) * D;
  float qv[D];
  {
    const TX *src = q + row0 * stride + h * kDim;
    float x[3][8], ss = 0.f;
#pragma unroll
    for (int o = 0; o < 3; ++o) load8(src + 8 * o, x[o]);
    float f = 1.f;
    if (norm_w) {
#pragma unroll
      for (int o = 0; o < 3; ++o)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[o][e], x[o][e], ss);
      f = 1.0f / sqrtf(ss / static_cast<float>(kDim) + eps);
#pragma unroll
      for (int o = 0; o < 3; ++o)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[o][e] = x[o][e] * f * norm_w[8 * o + e];
    }
#pragma unroll
    for (int i = 0; i < D; ++i) {
      float t = x[i / 8][i % 8];
#pragma unroll
      for (int g = 1; g < G; ++g) t = (lane & (G - 1)) == g ? x[(g * D + i) / 8][(g * D + i) % 8] : t;
      qv[i] = t;
    }
  }

  float m = kLow, l = 0.f, acc[D];
#pragma unroll
  for (int i = 0; i < D; ++i) acc[i] = 0.f;
  const int key0 = begin + wave * K + lane / G;
  const uint8_t *kb = static_cast<const uint8_t *>(kv.k) + (lane & (G - 1)) * 24;
  const uint8_t *vb = static_cast<const uint8_t *>(kv.v) + (lane & (G - 1)) * 24;
  auto value = [](const uint2 (&w)[3], int i) -> float {  // dim i of a lane's 24 bytes
    if constexpr (G == 1) return byte_of(i & 4 ? w[i >> 3].y : w[i >> 3].x, i & 3);
    else if constexpr (G == 2) {
      const uint32_t u = i & 2 ? w[i >> 2].y : w[i >> 2].x;
      return __half2float(__ushort_as_half(static_cast<uint16_t>(i & 1 ? u >> 16 : u)));
    } else return __uint_as_float(i & 1 ? w[i >> 1].y : w[i >> 1].x);
  };
  for (int base = begin; base < end; base += kDecRounds * kWaves * K) {
    uint2 kr[kDecRounds][3], vr[kDecRounds][3];
    float ks[kDecRounds], vs[kDecRounds], s[kDecRounds];
    int page[kDecRounds];
#pragma unroll
    for (int u = 0; u < kDecRounds; ++u) page[u] = page_of(b, kv, r, min(key0 + (base - begin) + u * kWaves * K, end - 1));
#pragma unroll
    for (int u = 0; u < kDecRounds; ++u) {
      const int j = min(key0 + (base - begin) + u * kWaves * K, end - 1);
      const int64_t at = slot_of(kv, max(page[u], 0), h, j);
      const uint2 *a = reinterpret_cast<const uint2 *>(kb + at * (kDim * G));
      const uint2 *c = reinterpret_cast<const uint2 *>(vb + at * (kDim * G));
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        kr[u][i] = a[i];
        vr[u][i] = c[i];
      }
      if constexpr (G == 1) {
        ks[u] = kv.k_scale[at];
        vs[u] = kv.v_scale[at];
      }
    }
    float mx = m;
#pragma unroll
    for (int u = 0; u < kDecRounds; ++u) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < D; ++i) t = fmaf(qv[i], value(kr[u], i), t);
      if constexpr (G >= 2) t += dpp_f32<0xB1>(t);
      if constexpr (G >= 4) t += dpp_f32<0x4E>(t);
      if constexpr (G == 1) t *= ks[u];
      if (page[u] < 0) t = __builtin_nanf("");
      if (key0 + (base - begin) + u * kWaves * K >= end) {  // past the range: its row stands for no key
        t = -INFINITY;
#pragma unroll
        for (int i = 0; i < 3; ++i) vr[u][i] = make_uint2(0u, 0u);
        if constexpr (G == 1) vs[u] = 0.f;
      }
      s[u] = t;
      mx = fmaxf(mx, t);
    }
    if (__any(mx > m)) {
      const float f = __builtin_amdgcn_exp2f((m - mx) * cst);
      l *= f;
#pragma unroll
      for (int i = 0; i < D; ++i) acc[i] *= f;
      m = mx;
    }
#pragma unroll
    for (int u = 0; u < kDecRounds; ++u) {
      float p = __builtin_amdgcn_exp2f((s[u] - m) * cst);
      l += p;
      if constexpr (G == 1) p *= vs[u];
#pragma unroll
      for (int i = 0; i < D; ++i) acc[i] = fmaf(p, value(vr[u], i), acc[i]);
    }
  }

  // the wave's states joined
  float bm[1] = {m};
  group_reduce<64, true>(bm);
  const float f = __builtin_amdgcn_exp2f((m - bm[0]) * cst);
  l *= f;
#pragma unroll
  for (int i = 0; i < D; ++i) acc[i] *= f;
  const int first = join_lanes<D, G>(acc, lane, d0);
#pragma unroll
  for (int o = G; o < 64; o *= 2) l += __shfl_xor(l, o, 64);
  float *p = part ? part + (static_cast<int64_t>(pair) * splits + sp) * kPart : nullptr;
  auto store = [&](int d, float y) {  // dim d of the output
    TX *dst = out + (static_cast<int64_t>(row0) * kv.heads + h) * kDim + d;
    if constexpr (std::is_same_v<TX, float>) *dst = y;
    else *reinterpret_cast<uint16_t *>(dst) = static_cast<uint16_t>(bits16<TX>(y));
  };
  if constexpr (W == 1) {
    if (lane < 8) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        if (p) p[first + i] = acc[i];
        else store(first + i, len == 0 ? 0.f : acc[i] / l);
      }
      if (p && lane == 0) store4(p + kDim, bm[0], l, cst, 0.f);
    }
  } else {
    if (lane < 8) {
#pragma unroll
      for (int i = 0; i < 3; ++i) red[wave][first + i] = acc[i];
      if (lane == 0) {
        red[wave][kDim] = bm[0];
        red[wave][kDim + 1] = l;
      }
    }
    __syncthreads();
    if (tid < kDim) {
      float gm = red[0][kDim];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) gm = fmaxf(gm, red[w][kDim]);
      float o = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float e = __builtin_amdgcn_exp2f((red[w][kDim] - gm) * cst);
        o = fmaf(red[w][tid], e, o);
        sum = fmaf(red[w][kDim + 1], e, sum);
      }
      if (p) {
        p[tid] = o;
        if (tid == 0) store4(p + kDim, gm, sum, cst, 0.f);
      } else {
        store(tid, len == 0 ? 0.f : o / sum);
      }
    }
  }
}

// Rows of a split step, o = sum_s 2^((m_s - m) c) o_s / sum_s 2^((m_s - m) c) l_s (bound by latency and by the states'
// bytes: 8 us for a mixed step of 32 sequences, 16 us for 2,045 queries in 4 ranges): 8 lanes per (row, head), 6 of them with 4 dims each, over the row's live key ranges.  Items:
// the only token of each sequence (ONE), or token i % max_q of the sequence at place i / max_q, but for sequences of one
// token where the decode kernel has those (skip_one).
constexpr int kJoinItems = kThreads / 8;
template <class TX, bool ONE>
__global__ __launch_bounds__(kThreads) void paged_combine_kernel(Batch b, int heads, int skip_one, int range,
                                                                 int splits, const float *__restrict__ part,
                                                                 TX *__restrict__ out) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kJoinItems + (threadIdx.x >> 3);
  const int d = 4 * (threadIdx.x & 7), h = static_cast<int>(item % heads);
  const int64_t i = item / heads;
  const int64_t place = ONE ? i : i / b.max_q;
  const int t = ONE ? 0 : static_cast<int>(i % b.max_q);
  if (place >= b.count || d >= kDim) return;
  const int r = sequence_at(b, static_cast<int>(place));
  int row0, n, len;
  if (r < 0 || !sequence(b, r, row0, n, len) || t >= n) return;
  if (ONE ? n != 1 : (n == 1 && skip_one)) return;
  const int seen = len - (n - 1 - t);  // keys of this token
  const int live = seen > 0 ? (seen - 1) / range + 1 : 0;
  const int64_t row = static_cast<int64_t>(row0) + t;
  const float *p = part + ((ONE ? place : row) * heads + h) * splits * kPart;
  float m = kLow, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < live; ++s) {
    const float4 x = *reinterpret_cast<const float4 *>(p + s * kPart + d);
    const float4 y = *reinterpret_cast<const float4 *>(p + s * kPart + kDim);  // maximum, weight, unit
    const float mn = fmaxf(m, y.x);
    const float f = __builtin_amdgcn_exp2f((m - mn) * y.z), e = __builtin_amdgcn_exp2f((y.x - mn) * y.z);
    m = mn;
    sum = fmaf(sum, f, y.y * e);
    o[0] = fmaf(o[0], f, x.x * e);
    o[1] = fmaf(o[1], f, x.y * e);
    o[2] = fmaf(o[2], f, x.z * e);
    o[3] = fmaf(o[3], f, x.w * e);
  }
  const float f = live == 0 ? 0.f : 1.f / sum;
  store4(out + (row * heads + h) * kDim + d, live ? o[0] * f : 0.f, live ? o[1] * f : 0.f, live ? o[2] * f : 0.f,
         live ? o[3] * f : 0.f);
}

// ---- attention of a chunk of new tokens -----------------------------------

// A block takes 32 WQ queries of one (sequence, head) against one key range: WQ of its 4 waves side by side over the
// queries (32 each), 4 / WQ over the keys (64 of each tile of 256 / WQ); the latter's softmax states are joined at
// the end.
//   Contractions: v_mfma_f32_32x32x16_f16 on fp16 parts.  A value is the sum of two parts to 22 bits or more
// (an fp16 key or value of one, itself), scaled by a power of two taken from the tile's largest (K, V) or the row's
// (q), so that no part leaves fp16's range; a product takes the three pairs of parts above 2^-22.
//   S^T = K Q^T: the pairs' 24 dims lie one after the other along the contraction, 72 of 80 (48 of 48 for fp16 keys),
// so no MFMA is half padding.  P^T comes out with lane l holding query l % 32 and, of 32 keys, those with bit 2 equal
// to l / 32: V^T is laid out in LDS so that the same lane's share of the next contraction is those keys, and P^T
// goes from register to register.  Dim 24 of V^T is a row of ones: it sums the probabilities.
//   Probabilities are 2^(s c - M), one FMA each: M, a scaled maximum less 10, is a rounded number, but the same one
// for every key, and sums are rescaled by differences of it.  Beside an M of 2^22 and more (a rounding of it would be
// as large as an exponent) the maximum is taken off before the scale.
//   A tile with a key or value that is not finite would reach queries that do not see it (0 * inf), and so would one far
// larger than the others, whose parts it would leave without bits: such a tile's keys, or those that it would, are taken
// one by one on the VALU.  (The look at each row's largest costs a mixed step over fp32 pages 1%, INT8 prompts nothing
// measured; one row of 64 a millionth of the others', in every tile, takes the prompts from 103 to 230 us, one row of 1,000
// a million times the others' to 810.)
//   Bound by VALU issue, not by the matrix products: an exponent, its FMA, its share of the maximum and its two parts are
// 5 instructions a score; with staging 7.5 (0.5 cycles of a SIMD) for keys of one part, and 12.3 (0.8) for two, against 0.22
// and 0.34 cycles of MFMA.  2,045 queries behind 14,339 fp16 keys, 80 heads: 829 us (2.5 billion scores, 73% of the cycles
// issue VALU work, 31% MFMA); 16 prompts of up to 1,024 tokens over INT8 pages 103 us (57% and 23%; 40% of the waves' time
// is waits).  Four waves per SIMD in place of three would spill 17 registers: 946 -> 1,050 us profiled.
//   QG groups of 32 queries per wave share a staged tile: the staging, a fifth of the instructions, is then paid half as
// often.  WQ: with 64 queries or fewer the other waves take other keys, so that none is idle (both sides measured at the rule).
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// the power of two that brings values below 2^(e + 1) under 2^15 (its own exponent kept where 2^-14 over it is normal)
__device__ __forceinline__ int part_scale(uint32_t maxbits, int extra) {
  const int e = static_cast<int>(maxbits >> 23) - 127 + extra;
  return max(min(14 - e, 112), -113);
}

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_halves(float a, float b) {  // rounded to nearest even
  const half2v h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
  return __builtin_bit_cast(uint32_t, h);
}
// p less a half of w (LOW: the low one), exactly
template <bool LOW>
__device__ __forceinline__ float less_half(float p, uint32_t w) {
  float r;
  if constexpr (LOW) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(p));
  else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(p));
  return r;
}

// 8 values as fp16 parts (kept as fp32 first: a product folded into the conversion would round apart from the one
// that the low part is taken from)
__device__ __forceinline__ void split8(float (&x)[8], uint4 &hi, uint4 &lo) {
  uint32_t a[4], c[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) asm("" : "+v"(x[i]));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = pack_halves(x[2 * i], x[2 * i + 1]);
    c[i] = pack_halves(less_half<true>(x[2 * i], a[i]), less_half<false>(x[2 * i + 1], a[i]));
  }
  hi = make_uint4(a[0], a[1], a[2], a[3]);
  lo = make_uint4(c[0], c[1], c[2], c[3]);
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = max(v, dpp_u32<0xB1>(v));
  v = max(v, dpp_u32<0x4E>(v));
  v = max(v, dpp_u32<0x141>(v));
  v = max(v, dpp_u32<0x140>(v));
  v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16, 64)));
  return max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32, 64)));
}

// The probabilities' room in fp16: 2^kLift for a key at the maximum that M was taken from, and 2^(kLift + kRise) for one
// above it, before M is taken anew: with 32 queries a wave one of them meets a larger key in most tiles, by little.
// Below 2^-14 a low part loses bits: an error of 2^-25 against the 2^10 of the largest.
constexpr float kLift = 10.f, kRise = 5.f;

constexpr uint32_t kInfBits = 0x7F800000u;
// Of two parts below 2^15 the lower has steps of 2^-24: a row's values keep 22 bits of its largest down to 2^-kDeep of
// what the parts are scaled by.  The sums of values are held in a unit up to kKeep above the tile's own, and kFall at most
// below the largest tile's: 2^30 keys of 2^15 times values of 2^15 stay in fp32.
constexpr int kDeep = 16, kKeep = 3, kFall = 60;
constexpr int kVRow = 72;  // halves between dims of V^T in LDS (64 keys; 16 rows of a read in distinct banks)

// The state of 32 queries of a wave: lane l holds query l % 32 and, of its sums, the dims with bit 2 equal to l / 32.
struct Queries {
  f32x16 o;      // dims 8 (i / 4) + 4 (l / 32) + i % 4; from 24 on the probabilities' sum
  float m, mb;   // a maximum; scaled, less kLift
  float cst, qf; // a score's factor in the exponent; 1 / rms
  int lfq;       // the power of two in the query's parts
};

// The queries, normalised, as their parts in LDS rows of kQRow halves: octets of dims, high parts, then low ones.
constexpr int kQRow = 56;  // (16 rows of a read in distinct banks)
template <class TX>
__device__ __forceinline__ void load_queries(const TX *src, const float *norm_w, float eps, float scale_log2, int hh,
                                             uint16_t *row, Queries &g) {
  float x[3][8], ss = 0.f;
  uint32_t mb = 0;
#pragma unroll
  for (int o = 0; o < 3; ++o) load8(src + 8 * o, x[o]);
  g.qf = 1.f;
  if (norm_w) {
#pragma unroll
    for (int o = 0; o < 3; ++o)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[o][e], x[o][e], ss);
    g.qf = 1.0f / sqrtf(ss / static_cast<float>(kDim) + eps);
#pragma unroll
    for (int o = 0; o < 3; ++o)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[o][e] = x[o][e] * g.qf * norm_w[8 * o + e];
  }
#pragma unroll
  for (int o = 0; o < 3; ++o)
#pragma unroll
    for (int e = 0; e < 8; ++e) mb = max(mb, __float_as_uint(x[o][e]) & 0x7FFFFFFFu);
  g.lfq = part_scale(mb, 0);
  g.cst = scale_log2 * pow2(14 - g.lfq);
#pragma unroll
  for (int o = 0; o < 3; ++o) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[o][e] *= pow2(g.lfq);
    uint4 hi, lo;
    split8(x[o], hi, lo);
    *reinterpret_cast<uint4 *>(row + 24 * hh + 8 * o) =  // (two lanes a query: one writes its high parts, one its low)
        make_uint4(hh ? lo.x : hi.x, hh ? lo.y : hi.y, hh ? lo.z : hi.z, hh ? lo.w : hi.w);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) g.o[i] = 0.f;
  g.m = g.mb = kLow;
}

template <class TX, class TKV, int WQ, int QG>
__global__ __launch_bounds__(kThreads, WQ == 4 ? (QG == 1 ? 4 : 3) : 2) void paged_chunk_kernel(const TX *__restrict__ q, int64_t stride,
                                                               const float *__restrict__ norm_w, float eps, Pages kv,
                                                               Batch b, int skip_one, int q_tiles, int range,
                                                               int splits, float scale_log2, TX *__restrict__ out,
                                                               float *__restrict__ part) {
  constexpr int KP = std::is_same_v<TKV, __half> ? 1 : 2;  // parts of a key or value
  constexpr int WK = 4 / WQ, kTile = 64 * WK, kQ = 32 * WQ * QG;
  static_assert(WK == 1 || QG == 1, "waves that share queries hold 32 of them");
  constexpr int kKRow = KP == 2 ? 56 : 24;                  // halves between keys in LDS
  constexpr int kUnits = kTile * 3;                         // (key, 8 dims)
  constexpr int UN = (kUnits + kThreads - 1) / kThreads;
  constexpr int kVec = sizeof(TKV) == 4 ? 4 : 2;            // 8 values of a row in words / 2
  constexpr int kStates = (WK - 1) * WQ * 64 * 14 * 2;      // halves of the states joined at the end
  __shared__ __align__(16) uint16_t ks[kTile * kKRow > kStates ? kTile * kKRow : kStates];
  __shared__ __align__(16) uint16_t vt[WK * KP * 25 * kVRow];
  __shared__ __align__(16) uint16_t qs[(kQ + 1) * kQRow];  // the last row: zeros
  __shared__ uint32_t red[2][kThreads / 64];
  constexpr int kOcts = sizeof(TKV) == 1 ? 1 : 3;         // units that say how large a row is (INT8: each has its scale)
  __shared__ uint16_t rows[KP == 2 ? kOcts * kTile : 1];  // exponents of a unit's largest: a key's | a value's << 8
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wq = wave % WQ, wk = wave / WQ;
  const int pairs = b.count * kv.heads;
  const int pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
  const int sp = rest % splits, qt = q_tiles - 1 - rest / splits;  // the queries with the most keys first
  const int r = sequence_at(b, pair / kv.heads), h = pair % kv.heads;
  if (r < 0) return;
  int row0, n, len;
  if (!sequence(b, r, row0, n, len)) {
    if (sp == 0)
      nan_rows(out, b, kv.heads, h, row0, n, int64_t{qt} * kThreads + tid, int64_t{q_tiles} * kThreads);
    return;
  }
  if (qt * kQ >= n || (n == 1 && skip_one)) return;
  const int begin = sp * range;
  const int end = min(begin + range, len - n + min(n, (qt + 1) * kQ));
  if (begin >= end && sp > 0) return;

  // this wave's queries: group i from index first(i) on, at positions from low(i) on
  const int p0 = len - n;
  auto first = [&](int i) { return qt * kQ + (i * WQ + wq) * 32; };
  auto source = [&](int i) {
    return q + (static_cast<int64_t>(row0) + min(first(i) + col, n - 1)) * stride + h * kDim;
  };
  // (waves that share queries write the same rows with the same values)
  Queries g[QG];
#pragma unroll
  for (int i = 0; i < QG; ++i)
    load_queries(source(i), norm_w, eps, scale_log2, hh, &qs[((i * WQ + wq) * 32 + col) * kQRow], g[i]);
  if (tid < kQRow / 8) *reinterpret_cast<uint4 *>(&qs[kQ * kQRow + 8 * tid]) = make_uint4(0u, 0u, 0u, 0u);
  for (int i = tid; i < WK * KP * 64; i += kThreads)  // the probabilities' sum: ones beside V's high part
    vt[((i >> 6) * 25 + 24) * kVRow + (i & 63)] = (i >> 6) % KP == 0 ? 0x3C00 : 0;

  // staging: unit u is 8 dims (u / kTile) of key u % kTile
  uint2 kraw[UN][kVec], vraw[UN][kVec];
  float kscale[UN], vscale[UN];
  int page[UN];
  auto pages = [&](int base) {
#pragma unroll
    for (int x = 0; x < UN; ++x) {
      const int u = tid + kThreads * x;
      page[x] = page_of(b, kv, r, min(base + u % kTile, end - 1));
    }
  };
  bool bad[UN];
  auto load = [&](int base) {
#pragma unroll
    for (int x = 0; x < UN; ++x) {
      const int u = tid + kThreads * x;
      const int j = min(base + u % kTile, end - 1), o = min(u / kTile, 2);
      const int64_t at = slot_of(kv, max(page[x], 0), h, j);
      bad[x] = page[x] < 0;
      const uint2 *a = reinterpret_cast<const uint2 *>(static_cast<const TKV *>(kv.k) + at * kDim + 8 * o);
      const uint2 *c = reinterpret_cast<const uint2 *>(static_cast<const TKV *>(kv.v) + at * kDim + 8 * o);
      if constexpr (sizeof(TKV) == 1) {
        kraw[x][0] = a[0];
        vraw[x][0] = c[0];
        kscale[x] = kv.k_scale[at];
        vscale[x] = kv.v_scale[at];
      } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
          const uint4 y = *reinterpret_cast<const uint4 *>(a + i), z = *reinterpret_cast<const uint4 *>(c + i);
          kraw[x][i] = make_uint2(y.x, y.y); kraw[x][i + 1] = make_uint2(y.z, y.w);
          vraw[x][i] = make_uint2(z.x, z.y); vraw[x][i + 1] = make_uint2(z.z, z.w);
        }
      }
    }
  };
  // the bits of a unit's largest |value| (INT8: of its scale; fp16: 0 if finite); not finite: kInfBits or more
  auto largest = [&](const uint2 (&w)[kVec], float s) {
    uint32_t mb = 0;
    if constexpr (sizeof(TKV) == 1) {
      mb = __float_as_uint(s) & 0x7FFFFFFFu;
    } else if constexpr (sizeof(TKV) == 2) {
      // a half's exponent of all ones overflows into bit 15 of its own word
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        mb |= ((w[i].x & 0x7C007C00u) + 0x04000400u) | ((w[i].y & 0x7C007C00u) + 0x04000400u);
      mb = mb & 0x80008000u ? kInfBits : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) mb = max(mb, max(w[i].x & 0x7FFFFFFFu, w[i].y & 0x7FFFFFFFu));
    }
    return mb;
  };
  auto values = [&](const uint2 (&w)[kVec], float s, float f, float (&x)[8]) {
    if constexpr (sizeof(TKV) == 1) {
      const float m = s * f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = byte_of(e < 4 ? w[0].x : w[0].y, e & 3) * m;
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        x[2 * i] = __uint_as_float(w[i].x) * f;
        x[2 * i + 1] = __uint_as_float(w[i].y) * f;
      }
    }
  };

  int ev = -98, ev_top = -98;  // KP == 2: the sums of values are in units of 2^(ev - 14); the largest ev so far
  if (begin < end) {
    pages(begin);
    load(begin);
    if (begin + kTile < end) pages(begin + kTile);
  }
  for (int base = begin; base < end; base += kTile) {
    uint32_t mk = 0, mv = 0;
#pragma unroll
    for (int x = 0; x < UN; ++x) {
      const int u = tid + kThreads * x;
      if (u >= (sizeof(TKV) == 1 ? kTile : kUnits)) continue;
      const uint32_t k1 = largest(kraw[x], kscale[x]), v1 = largest(vraw[x], vscale[x]);
      if constexpr (KP == 2) rows[u] = static_cast<uint16_t>(k1 >> 23 | v1 >> 23 << 8);
      if (base + u % kTile >= end) continue;
      mk = max(mk, bad[x] ? kInfBits : k1);
      mv = max(mv, v1);
    }
    if constexpr (KP == 2) {
      if (sizeof(TKV) != 1 || 64 * wave < kTile) {  // (INT8: the other waves' units have the same scales)
        mk = wave_umax(mk);
        mv = wave_umax(mv);
      }
    } else {
      mk = __any(max(mk, mv) != 0) ? kInfBits : 0u;
    }
    if (lane == 0) {
      red[0][wave] = mk;
      if constexpr (KP == 2) red[1][wave] = mv;
    }
    __syncthreads();  // the last tile is done with; the maxima are in LDS
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      mk = max(mk, red[0][w]);
      if constexpr (KP == 2) mv = max(mv, red[1][w]);
    }
    mk = __builtin_amdgcn_readfirstlane(mk);
    mv = __builtin_amdgcn_readfirstlane(mv);
    const bool finite = (KP == 2 ? max(mk, mv) : mk) < kInfBits;  // (block-uniform)
    int lfk = 0;
    if constexpr (KP == 2) {
      if (!finite) {  // the sums' unit then goes by the values that are
        mv = 0;
#pragma unroll
        for (int x = 0; x < UN; ++x) {
          const int u = tid + kThreads * x;
          if (u >= kUnits || base + u % kTile >= end) continue;
          if constexpr (sizeof(TKV) == 1) {
            const uint32_t y = largest(vraw[x], vscale[x]);
            mv = max(mv, y < kInfBits ? y : 0u);
          } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t y = (e ? vraw[x][i].y : vraw[x][i].x) & 0x7FFFFFFFu;
                mv = max(mv, y < kInfBits ? y : 0u);
              }
          }
        }
        mv = wave_umax(mv);
        __syncthreads();
        if (lane == 0) red[1][wave] = mv;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) mv = max(mv, red[1][w]);
        mv = __builtin_amdgcn_readfirstlane(mv);
      } else {
        lfk = part_scale(mk, sizeof(TKV) == 1 ? 7 : 0);
      }
      const int e = 14 - part_scale(mv, sizeof(TKV) == 1 ? 7 : 0);
      if (e > ev || (e < ev - kKeep && mv != 0)) {
        ev_top = max(ev_top, e);
        const int to = max(e, ev_top - kFall);
        const float f = pow2(max(ev - to, -126)), f2 = pow2(min(ev - to + 126, 0));
#pragma unroll
        for (int i = 0; i < QG; ++i)
#pragma unroll
          for (int d = 0; d < 12; ++d) g[i].o[d] = g[i].o[d] * f * f2;
        ev = to;
      }
    }
    // this wave's keys that are not taken as parts: rows, but those of zeros, kDeep below what their parts are scaled by
    uint64_t single = finite ? 0 : ~uint64_t{0};
    if constexpr (KP == 2) {
      const uint16_t *at = &rows[64 * wk + lane];
      int k1 = 0, v1 = 0;
#pragma unroll
      for (int x = 0; x < kOcts; ++x) {
        const int y = at[x * kTile];
        k1 = max(k1, y & 0xFF);
        v1 = max(v1, y >> 8);
      }
      constexpr int kUp = sizeof(TKV) == 1 ? 6 : 0;  // (the largest is 127 scales)
      const int k_least = 127 - kUp + 14 - lfk - kDeep, v_least = 127 - kUp + ev - kDeep;
      single |= __ballot(((k1 != 0) & (k1 < k_least)) | ((v1 != 0) & (v1 < v_least)));
    }
    if (finite) {
#pragma unroll
      for (int x = 0; x < UN; ++x) {
        const int u = tid + kThreads * x;
        if (u >= kUnits) continue;
        // (a key past the range holds its last one again: no query sees it, and its value is finite)
        const int key = u % kTile, oc = u / kTile;
        uint4 kh, kl, vh, vl;
        if constexpr (KP == 2) {
          float y[8];
          values(kraw[x], kscale[x], pow2(lfk), y);
          split8(y, kh, kl);
          values(vraw[x], vscale[x], pow2(14 - ev), y);
          split8(y, vh, vl);
          *reinterpret_cast<uint4 *>(&ks[key * kKRow + 24 + 8 * oc]) = kl;
        } else {
          kh = make_uint4(kraw[x][0].x, kraw[x][0].y, kraw[x][1].x, kraw[x][1].y);
          vh = make_uint4(vraw[x][0].x, vraw[x][0].y, vraw[x][1].x, vraw[x][1].y);
        }
        *reinterpret_cast<uint4 *>(&ks[key * kKRow + 8 * oc]) = kh;
        // key 16 s + 8 a + 4 g + c of its 64 at column 16 s + 8 g + 4 a + c
        const int sub = key >> 6, c = (key & 0x33) | ((key & 4) << 1) | ((key & 8) >> 1);
        uint16_t *dst = &vt[(sub * KP * 25 + 8 * oc) * kVRow + c];
        const uint32_t wh[4] = {vh.x, vh.y, vh.z, vh.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i * kVRow] = static_cast<uint16_t>(i & 1 ? wh[i >> 1] >> 16 : wh[i >> 1]);
        if constexpr (KP == 2) {
          const uint32_t wl[4] = {vl.x, vl.y, vl.z, vl.w};
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dst[(25 + i) * kVRow] = static_cast<uint16_t>(i & 1 ? wl[i >> 1] >> 16 : wl[i >> 1]);
        }
      }
    }
    if (base + kTile < end) {
      load(base + kTile);
      if (base + 2 * kTile < end) pages(base + 2 * kTile);
    }
    __syncthreads();  // the tile is in LDS
    const int wbase = base + 64 * wk;  // this wave's keys of the tile
    if (wbase >= end) continue;
#pragma unroll
    for (int i = 0; i < QG; ++i) {
      Queries &w = g[i];
      const int low = p0 + first(i), top = p0 + min(first(i) + 32, n) - 1;  // the group's positions
      const int pos = low + col;  // (past the last query: masks nothing that is stored)
      if (first(i) >= n || wbase > top) continue;
      if (finite) {
        const float kfac = pow2(-lfk - 14);
        // the B operands: octets of the query's parts along the contraction, lanes below 32 | from there
        constexpr int kB = KP == 2 ? 5 : 3;
        half8 qa[kB];
        {
          const uint16_t *row = &qs[((i * WQ + wq) * 32 + col) * kQRow];
#pragma unroll
          for (int x = 0; x < kB; ++x) {
            // KP 2: high 0 1 | 2 0 | 1 2, low 0 1 | 2 -; KP 1: high 0 1 | 2, low 0 | 1 2
            const int below = KP == 2 ? (x < 3 ? 2 * x % 3 : 2 * x - 3) : 2 * x;
            const int from = KP == 2 ? (x < 3 ? (2 * x + 1) % 3 : 2 * x - 2) : 2 * x + 1;
            const uint16_t *at = row + 8 * (hh ? from : below);
            if (x == 4 && hh) at = &qs[kQ * kQRow];
            qa[x] = *reinterpret_cast<const half8 *>(at);
          }
        }
        f32x16 s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const uint16_t *a = &ks[(64 * wk + 32 * kb + col) * kKRow];
          half8 ka[3];
#pragma unroll
          for (int x = 0; x < 3; ++x) {
            const int oc = (2 * x + hh) % (KP == 2 ? 6 : 3);
            ka[x] = *reinterpret_cast<const half8 *>(a + 8 * oc);
          }
#pragma unroll
          for (int x = 0; x < 16; ++x) s[kb][x] = 0.f;
          s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[0], qa[0], s[kb], 0, 0, 0);
          s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[1], qa[1], s[kb], 0, 0, 0);
          s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[2], qa[2], s[kb], 0, 0, 0);
          if constexpr (KP == 2) {
            s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[0], qa[3], s[kb], 0, 0, 0);
            s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[1], qa[4], s[kb], 0, 0, 0);
          }
        }
        if (wbase + 63 > low) {  // keys after a query
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int x = 0; x < 16; ++x)
              if (wbase + 32 * kb + 8 * (x / 4) + 4 * hh + x % 4 > pos) s[kb][x] = -INFINITY;
        }
        if (KP == 2 && single != 0) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            const uint32_t bits = static_cast<uint32_t>(single >> (32 * kb)) >> (4 * hh);
#pragma unroll
            for (int x = 0; x < 16; ++x)
              if (bits >> (8 * (x / 4) + x % 4) & 1u) s[kb][x] = -INFINITY;
          }
        }
        float mx = s[0][0];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int x = 0; x < 16; ++x) mx = fmaxf(mx, s[kb][x]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * kfac;
        const bool large = __any(fabsf(fmaxf(w.m, mx)) * w.cst >= 4194304.f);  // (m before any key: large as well)
        if (__any((mx - w.m) * w.cst > kRise)) {
          const float mn = fmaxf(w.m, mx), mbn = fmaf(mn, w.cst, -kLift);
          const float f = __builtin_amdgcn_exp2f(large ? (w.m - mn) * w.cst : w.mb - mbn);
#pragma unroll
          for (int x = 0; x < 16; ++x) w.o[x] *= f;
          w.m = mn;
          w.mb = mbn;
        }
        float c = kfac * w.cst, shift = -w.mb;  // a score's exponent: s c + shift
        if (large) {
          c = w.cst;
          shift = kLift;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int x = 0; x < 16; ++x) s[kb][x] = fmaf(s[kb][x], kfac, -w.m);
        }
        const uint16_t *va = &vt[(wk * KP * 25 + min(col, 24)) * kVRow + 8 * hh];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              float p[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[kb][8 * y + 2 * x + e], c, shift));
              ph[x] = pack_halves(p[0], p[1]);
              pl[x] = pack_halves(less_half<true>(p[0], ph[x]), less_half<false>(p[1], ph[x]));
            }
            const half8 bh = __builtin_bit_cast(half8, make_uint4(ph[0], ph[1], ph[2], ph[3]));
            const half8 bl = __builtin_bit_cast(half8, make_uint4(pl[0], pl[1], pl[2], pl[3]));
            const half8 vh = *reinterpret_cast<const half8 *>(va + 32 * kb + 16 * y);
            w.o = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, bh, w.o, 0, 0, 0);
            w.o = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, bl, w.o, 0, 0, 0);
            if constexpr (KP == 2) {
              const half8 vl = *reinterpret_cast<const half8 *>(va + 25 * kVRow + 32 * kb + 16 * y);
              w.o = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, bh, w.o, 0, 0, 0);
            }
          }
        if (KP == 1 || single == 0) continue;
      }
      {
        // key by key, each to the queries that see it
        const float vf = KP == 2 ? pow2(14 - ev) : 1.f;
        const TX *src = source(i);
#pragma unroll 1
        for (int j = wbase; j < min(min(wbase + 64, end), top + 1); ++j) {
          if (KP == 2 && (single >> (j - wbase) & 1) == 0) continue;
          const int pg = page_of(b, kv, r, j);
          const int64_t at = slot_of(kv, max(pg, 0), h, j);
          const TKV *kp = static_cast<const TKV *>(kv.k) + at * kDim, *vp = static_cast<const TKV *>(kv.v) + at * kDim;
          float kq = 1.f, vq = vf;
          if constexpr (sizeof(TKV) == 1) {
            kq = kv.k_scale[at];
            vq = kv.v_scale[at] * vf;
          }
          float t = pg < 0 ? __builtin_nanf("") : 0.f;
#pragma unroll 1
          for (int o = 0; o < kDim; o += 8) {
            float x[8], y[8];
            load8(src + o, x);
            if constexpr (sizeof(TKV) == 1) {
              const uint2 c = *reinterpret_cast<const uint2 *>(kp + o);
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = byte_of(e < 4 ? c.x : c.y, e & 3);
            } else {
              load8(kp + o, y);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (norm_w) x[e] = x[e] * w.qf * norm_w[o + e];
              t = fmaf(x[e] * pow2(w.lfq - 14), y[e] * kq, t);
            }
          }
          if (j > pos) continue;
          const float mn = fmaxf(w.m, t);
          const float f = __builtin_amdgcn_exp2f((w.m - mn) * w.cst);
          const float p = __builtin_amdgcn_exp2f(fmaf(t - mn, w.cst, kLift));
          w.m = mn;
          w.mb = fmaf(mn, w.cst, -kLift);
#pragma unroll
          for (int x = 0; x < 12; ++x)
            w.o[x] = fmaf(w.o[x], f, p * (static_cast<float>(vp[8 * (x / 4) + 4 * hh + x % 4]) * vq));
#pragma unroll
          for (int x = 12; x < 16; ++x) w.o[x] = fmaf(w.o[x], f, p);
        }
      }
    }
  }

  if constexpr (WK > 1) {  // the states of the waves that share these queries (the tile's LDS is done with)
    Queries &w = g[0];
    float *st = reinterpret_cast<float *>(ks);
    __syncthreads();
    if (wk > 0) {
      float *d = st + (((wk - 1) * WQ + wq) * 14) * 64 + lane;
#pragma unroll
      for (int i = 0; i < 13; ++i) d[64 * i] = w.o[i];
      d[64 * 13] = w.m;
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int x = 1; x < WK; ++x) {
      const float *d = st + (((x - 1) * WQ + wq) * 14) * 64 + lane;
      const float mn = fmaxf(w.m, d[64 * 13]);
      const float f = __builtin_amdgcn_exp2f((w.m - mn) * w.cst), y = __builtin_amdgcn_exp2f((d[64 * 13] - mn) * w.cst);
#pragma unroll
      for (int i = 0; i < 13; ++i) w.o[i] = fmaf(w.o[i], f, d[64 * i] * y);
      w.m = mn;
    }
  }
  const float unit = KP == 2 ? pow2(ev - 14) : 1.f;
#pragma unroll
  for (int i = 0; i < QG; ++i) {
    if (first(i) + col >= n) continue;
    Queries &w = g[i];
    const int64_t row = (static_cast<int64_t>(row0) + first(i) + col) * kv.heads + h;
    const bool sees = p0 + first(i) + col >= 0;
    if (part) {  // (without the lift, which would take sums of values of 10^33 out of fp32)
      float *p = part + (row * splits + sp) * kPart;
      const float f = pow2(KP == 2 ? ev - 14 - static_cast<int>(kLift) : -static_cast<int>(kLift));
#pragma unroll
      for (int x = 0; x < 3; ++x)
        store4(p + 8 * x + 4 * hh, w.o[4 * x] * f, w.o[4 * x + 1] * f, w.o[4 * x + 2] * f, w.o[4 * x + 3] * f);
      if (hh == 0) store4(p + kDim, w.m, w.o[12] * pow2(-static_cast<int>(kLift)), w.cst, 0.f);
    } else {
      const float f = 1.f / w.o[12];
#pragma unroll
      for (int x = 0; x < 3; ++x) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = sees ? w.o[4 * x + e] * f * unit : 0.f;
        store4(out + row * kDim + 8 * x + 4 * hh, y[0], y[1], y[2], y[3]);
      }
    }
  }
}

}  // namespace

// ---- launchers ------------------------------------------------------------

namespace {

struct Plan {  // how a call's rows are taken: the one-token kernel, the chunk kernel, or both
  bool decode, chunk;
  int64_t d_first, d_count, c_count;  // their parts of the order
  int d_waves, d_range, d_splits, wq, groups, q_tiles, c_range, c_splits;
  size_t d_floats, c_floats;  // the split states' room
};

int round_up(int64_t x, int64_t m) { return static_cast<int>((x + m - 1) / m * m); }

// lanes that an item's keys fill, up to which one wave takes it (both sides at paged_decode_kernel)
constexpr int64_t kShortItem = 1024;

Plan plan_of(const plx_paged_kv &kv, const plx_paged_batch &b) {
  Plan p = {};
  p.decode = b.max_q == 1 || b.singles > 0;
  p.chunk = b.max_q > 1;
  // with an order the two kernels take its two parts, without one each looks at every sequence
  const bool parts = b.order != nullptr && p.chunk;
  p.d_first = parts ? b.seqs - b.singles : 0;
  p.d_count = b.seqs - p.d_first;
  p.c_count = parts ? b.seqs - b.singles : b.seqs;
  const int64_t pairs = p.d_count * kv.heads;
  const int bytes = kv.kv_type == PLX_KV_INT8 ? 1 : kv.kv_type == PLX_KV_F16 ? 2 : 4;
  // Key ranges: as many as bring the launch to 2,048 items (8 a CU), each of `least` positions or more.
  //   One token: 2,048 lanes' worth of keys or more.  One sequence of 8,000 INT8 positions, 80 heads, 19.2 us whole and 16.4
  // in 3 ranges, of 4,000 12.5 either way; ranges of 1,024 lanes took the latter to 15.3, ranges of 4,096 the former to 19.1.
  //   Chunks: 512 positions, and 256 where a range is all four waves' and the blocks alone leave CUs idle.  256 tokens behind
  // 768, 80 heads: one sequence 45 us whole, 33 in 2 ranges, 30.5 in 4; eight of them (640 blocks) 95 in 2 and 108 in 4.
  auto split = [&](int64_t blocks, int64_t want, int64_t least, int &range, int &splits) {
    int64_t n = blocks > 0 ? (want + blocks - 1) / blocks : 1;
    n = std::min<int64_t>(std::min<int64_t>(n, b.max_kv / least), 64);
    if (n < 2) {
      range = 0x7FFFFFFF;
      splits = 1;
    } else {
      range = round_up((b.max_kv + n - 1) / n, 256);
      splits = static_cast<int>((b.max_kv + range - 1) / range);
    }
  };
  if (p.decode) {
    split(pairs, 2048, 2048 / bytes, p.d_range, p.d_splits);
    p.d_waves = pairs >= 2048 && b.max_kv * bytes <= kShortItem ? 1 : 4;
    if (p.d_splits > 1) p.d_floats = static_cast<size_t>(pairs) * p.d_splits * kPart;
  }
  if (p.chunk) {
    // As many waves over the queries as they fill: 8 sequences of up to 20 tokens behind 1,000, 80 heads, 26 us with 1 (30
    // with 2, 33 with 4), of up to 64 28 with 2 (37 with 1, 33 with 4); 64 of 100 tokens 354 with 4 (438 with 2).
    // Two groups of queries a wave above 128: 16 prompts of up to 1,024 109 us (114 with one); 64 of 100 354 with one (364).
    p.wq = b.max_q <= 32 ? 1 : b.max_q <= 64 ? 2 : 4;
    p.groups = b.max_q <= 128 ? 1 : 2;
    const int tile = 32 * p.wq * p.groups;
    p.q_tiles = static_cast<int>((b.max_q + tile - 1) / tile);
    const int64_t blocks = p.c_count * kv.heads * p.q_tiles;
    split(blocks, 2048, p.wq == 4 && blocks < 256 ? 256 : 512, p.c_range, p.c_splits);
    if (p.c_splits > 1) p.c_floats = static_cast<size_t>(b.tokens) * kv.heads * p.c_splits * kPart;
  }
  return p;
}

Pages pages_of(const plx_paged_kv &kv) {
  int shift = 0;
  while ((int64_t{1} << shift) < kv.page_size) ++shift;
  return Pages{kv.k, kv.v, kv.k_scale, kv.v_scale, kv.pages, static_cast<int>(kv.heads), shift};
}

Batch batch_of(const plx_paged_batch &b) {
  return Batch{b.table, b.cu_q, b.kv_len, b.order, b.table_stride, b.tokens,
               static_cast<int>(b.seqs), static_cast<int>(b.max_q), static_cast<int>(b.max_kv), 0, static_cast<int>(b.seqs)};
}

constexpr int64_t kMaxBlocks = 0xFFFFFFFFll / kThreads;  // (a grid's threads are counted in 32 bits)

template <class F>
int with_x(int x_type, F f) {
  if (x_type == PLX_DTYPE_F32) return f(float{});
  if (x_type == PLX_DTYPE_F16) return f(__half{});
  return f(bf16_t{});
}

template <class F>
int with_kv(int kv_type, F f) {
  if (kv_type == PLX_KV_F32) return f(float{});
  if (kv_type == PLX_KV_F16) return f(__half{});
  return f(int8_t{});
}

}  // namespace

int launch_paged_write(const plx_paged_kv &kv, const plx_paged_batch &b, const void *k, const void *v, int x_type,
                       int64_t stride, const float *norm_w, float eps, hipStream_t s) {
  const int64_t q_tiles = (b.max_q + kWrTok - 1) / kWrTok, head_tiles = (kv.heads + kWrHeads - 1) / kWrHeads;
  const int64_t each = 2 * q_tiles * head_tiles, blocks = each * b.seqs;
  if (each > kMaxBlocks || blocks > kMaxBlocks) return fail(PLX_EINVAL, "paged_write: too many sequences, tokens and heads for one call");
  return with_x(x_type, [&](auto x) {
    return with_kv(kv.kv_type, [&](auto c) {
      using TX = decltype(x);
      using TKV = decltype(c);
      hipLaunchKernelGGL((paged_write_kernel<TX, TKV>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s,
                         static_cast<const TX *>(k), static_cast<const TX *>(v), stride, norm_w, eps, pages_of(kv),
                         batch_of(b), static_cast<int>(q_tiles), static_cast<int>(head_tiles));
      return check_launch("paged_write_kernel");
    });
  });
}

int launch_paged_read(const plx_paged_kv &kv, const plx_paged_batch &b, float *k_out, float *v_out, hipStream_t s) {
  const int64_t q_tiles = (b.max_q + kWrTok - 1) / kWrTok, head_tiles = (kv.heads + kWrHeads - 1) / kWrHeads;
  const int64_t each = 2 * q_tiles * head_tiles, blocks = each * b.seqs;
  if (each > kMaxBlocks || blocks > kMaxBlocks) return fail(PLX_EINVAL, "paged_read: too many sequences, tokens and heads for one call");
  return with_kv(kv.kv_type, [&](auto c) {
    hipLaunchKernelGGL((paged_read_kernel<decltype(c)>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s,
                       pages_of(kv), batch_of(b), static_cast<int>(q_tiles), static_cast<int>(head_tiles), k_out,
                       v_out);
    return check_launch("paged_read_kernel");
  });
}

size_t paged_attention_workspace_bytes(const plx_paged_kv &kv, const plx_paged_batch &b) {
  const Plan p = plan_of(kv, b);
  return (p.d_floats + p.c_floats) * sizeof(float);
}

int launch_paged_attention(const plx_paged_kv &kv, const plx_paged_batch &b, const void *q, int x_type, int64_t stride,
                           const float *norm_w, float eps, void *out, void *workspace, size_t workspace_bytes,
                           hipStream_t s) {
  const Plan p = plan_of(kv, b);
  const int64_t pairs = p.d_count * kv.heads, c_pairs = p.c_count * kv.heads;
  if (pairs * p.d_splits > kMaxBlocks || c_pairs * p.q_tiles * p.c_splits > kMaxBlocks ||
      (p.c_splits > 1 && p.c_count * b.max_q * kv.heads / kJoinItems > kMaxBlocks))
    return fail(PLX_EINVAL, "paged_attention: too many sequences, tokens and heads for one call");
  const size_t need = (p.d_floats + p.c_floats) * sizeof(float);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr))
    return fail(PLX_EINVAL, "paged_attention: workspace of %zu bytes, need %zu", workspace_bytes, need);
  if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
    return fail(PLX_EINVAL, "paged_attention: the workspace must be 16-byte aligned");
  float *d_part = p.d_floats ? static_cast<float *>(workspace) : nullptr;
  float *c_part = p.c_floats ? static_cast<float *>(workspace) + p.d_floats : nullptr;
  const double scale = 1.0 / sqrt(static_cast<double>(kDim));
  const float cst = static_cast<float>(static_cast<double>(kLog2e) * scale);
  const Pages pages = pages_of(kv);
  Batch batch = batch_of(b), longer = batch;
  batch.first = static_cast<int>(p.d_first);
  batch.count = static_cast<int>(p.d_count);
  longer.count = static_cast<int>(p.c_count);
  const int skip_one = p.decode && b.order == nullptr;  // (the decode kernel has them)
  const int heads = static_cast<int>(kv.heads);
  return with_x(x_type, [&](auto xv) {
    return with_kv(kv.kv_type, [&](auto cv) {
      using TX = decltype(xv);
      using TKV = decltype(cv);
      const TX *qx = static_cast<const TX *>(q);
      TX *ox = static_cast<TX *>(out);
      const auto joined = [](int64_t items) { return dim3(static_cast<unsigned>((items + kJoinItems - 1) / kJoinItems)); };
      if (p.chunk && c_pairs > 0) {
        const auto run = [&](auto wq, auto groups) {
          hipLaunchKernelGGL((paged_chunk_kernel<TX, TKV, decltype(wq)::value, decltype(groups)::value>),
                             dim3(static_cast<unsigned>(c_pairs * p.q_tiles * p.c_splits)), dim3(kThreads), 0, s, qx,
                             stride, norm_w, eps, pages, longer, skip_one, p.q_tiles, p.c_range,
                             p.c_splits, cst, ox, c_part);
        };
        using std::integral_constant;
        if (p.wq == 1) run(integral_constant<int, 1>{}, integral_constant<int, 1>{});
        else if (p.wq == 2) run(integral_constant<int, 2>{}, integral_constant<int, 1>{});
        else if (p.groups == 1) run(integral_constant<int, 4>{}, integral_constant<int, 1>{});
        else run(integral_constant<int, 4>{}, integral_constant<int, 2>{});
        if (const int st = check_launch("paged_chunk_kernel"); st != PLX_OK) return st;
        if (c_part) {
          hipLaunchKernelGGL((paged_combine_kernel<TX, false>), joined(p.c_count * b.max_q * heads), dim3(kThreads), 0, s,
                             longer, heads, skip_one, p.c_range, p.c_splits, c_part, ox);
          if (const int st = check_launch("paged_combine_kernel"); st != PLX_OK) return st;
        }
      }
      if (p.decode) {
        const auto run = [&](auto waves) {
          constexpr int W = decltype(waves)::value, per = kThreads / 64 / W;
          hipLaunchKernelGGL((paged_decode_kernel<TX, TKV, W>),
                             dim3(static_cast<unsigned>((pairs * p.d_splits + per - 1) / per)), dim3(kThreads), 0, s, qx,
                             stride, norm_w, eps, pages, batch, static_cast<int>(!p.chunk || b.order != nullptr), p.d_range, p.d_splits, cst,
                             ox, d_part);
        };
        if (p.d_waves == 1) run(std::integral_constant<int, 1>{});
        else run(std::integral_constant<int, 4>{});
        if (const int st = check_launch("paged_decode_kernel"); st != PLX_OK) return st;
        if (d_part) {
          hipLaunchKernelGGL((paged_combine_kernel<TX, true>), joined(pairs), dim3(kThreads), 0, s, batch, heads, 0,
                             p.d_range, p.d_splits, d_part, ox);
          return check_launch("paged_combine_kernel");
        }
      }
      return PLX_OK;
    });
  });
}

}  // namespace plx
