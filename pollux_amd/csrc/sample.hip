// The next token of each row of logits, from a given uniform number
// (generate.py:286-336's repetition penalty, temperature, top-k, top-p and
// multinomial draw, with min-p beside them).
//
//   z_i: the logit as fp32; of a token seen before, z / penalty above 0 and
//   z * penalty below.  w_i = e^((z_i - max z) / T).  In the order (z falling,
//   index rising): top-k leaves the first k tokens; of those, top-p leaves a
//   token if the mass before it is below p times theirs; min-p leaves those of
//   w >= min_p.  The token is the first, by index, at which the summed mass of
//   what is left passes u times all of it.
//
//   Every rule cuts that order at one place, so the row is never sorted: a
//   histogram over 2,048 ranges of z (counts for top-k, masses for top-p) says in
//   which range the first rule cuts.  Where the tokens up to there are 1,024 or
//   fewer -- as with any of a user's usual settings -- they are listed, sorted
//   and cut by all rules at once: by one wave's registers up to 64 of them, by a
//   block's above.  Otherwise the tokens of that range alone are sorted to find
//   the cut, or, where even they are too many (equal logits), a histogram of the
//   range's keys narrows it until one key is left, of which the first by index
//   are taken.
//   A weight is an integer, w * 2^44 rounded: sums do not depend on the order of
//   additions, nor on atomics, so a row's token is the same every time, and in any
//   batch.  The exponential is taken in fp64 to 2^-44, as the error of a 32-bit
//   one moves borders between tokens by 2^-20 and more: a table of 2^(i / 256) and
//   a short polynomial (a polynomial alone, of degree 9, took 512 rows of 50,688
//   tokens 58 us in place of 51; an fp64 FMA issues as often as an fp32 one here:
//   29.5 and 32.7 * 10^12 a second measured).
//
//   What bounds it: one row is a chain of four launches (24 us for 50,257 tokens
//   with every rule, 5 to 8 us each); 512 rows by the pass that takes the exponentials,
//   32 of 51 us (52 MB of bf16 logits would take 10).  Before the passes had
//   many blocks, a block per row took 39 us for one row and 80 for the 512.

#include <type_traits>

#include "plx_device.h"

namespace plx {
namespace {

constexpr int kSmThreads = 1024;
constexpr int kSmWaves = kSmThreads / 64;
constexpr int kBins = 2048;
constexpr int kAhead = 2;         // chunks of a wave whose loads are in flight together, where the row is read again
constexpr int kSmMost = 524288;   // longest row (a bit per token in LDS)
constexpr int kList = kSmThreads; // tokens that are sorted: one per thread
constexpr double kWeightOne = 17592186044416.0;  // 2^44

// The kernel's lambdas are all inlined: one that is not would hold what it shares in memory.
#define PLX_FLAT __attribute__((always_inline))

struct SampleArgs {
  const void *logits;
  int64_t stride;
  int x_type, n, vec;
  const float *u;
  plx_sample_rules rules;
  int64_t *ids, *kept;
  float *logp;
};

// bits whose unsigned order is the order of the values (-0 as +0)
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// 2^44 2^(i / 256), i = 0 .. 255, in LDS: filled by the first 256 threads (a barrier before it is read).  2^f by
// interpolation at the Chebyshev nodes of [-1/2, 1/2], to 2^-46.
constexpr int kTable = 256;
__device__ __forceinline__ void fill_table(double *table) {
  const int i = threadIdx.x;
  if (i >= kTable) return;
  const int n = i >= kTable / 2;
  const double f = static_cast<double>(i) / kTable - n;
  double p = 0x1.b6571e720cb47p-24;
  p = fma(p, f, 0x1.63ef969801aa6p-20);
  p = fma(p, f, 0x1.ffcb7677f3128p-17);
  p = fma(p, f, 0x1.43088e25816a1p-13);
  p = fma(p, f, 0x1.5d87fe908fcc6p-10);
  p = fma(p, f, 0x1.3b2ab72b175ddp-7);
  p = fma(p, f, 0x1.c6b08d7044116p-5);
  p = fma(p, f, 0x1.ebfbdff8149f2p-3);
  p = fma(p, f, 0x1.62e42fefa39f7p-1);
  p = fma(p, f, 1.0);
  table[i] = p * kWeightOne * (n ? 2.0 : 1.0);
}

// 2^44 2^(d rate / 256), d rate / 256 from -80 to 0: the table's entry times e^x, x = f ln 2 / 256 with |f| <= 1/2.
// e^x - 1 is x and the rest, below 2^-20 and so good to 2^-44 from fp32: that takes 11 fp64 operations, conversions
// among them, six fewer than a polynomial alone.
__device__ __forceinline__ double exp2_scaled(const double *table, double d, double rate) {
  const double round = 6755399441055744.0;  // 1.5 * 2^52: its last bits then hold the rounded integer
  const double r = fma(d, rate, round);
  const double f = fma(d, rate, round - r);
  const int32_t j = static_cast<int32_t>(static_cast<uint32_t>(__double_as_longlong(r)));
  const float x = static_cast<float>(f) * 2.7076061740622863e-3f;  // ln 2 / 256
  const float rest = x * x * fmaf(x, 1.6666667163e-1f, 0.5f);
  const double e = fma(f, 2.707606174062286e-3, static_cast<double>(rest));
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(table[j & (kTable - 1)]));
  const uint32_t high = static_cast<uint32_t>(b >> 32) + (static_cast<uint32_t>(j >> 8) << 20);
  const double t = __longlong_as_double(static_cast<long long>((static_cast<uint64_t>(high) << 32) | (b & 0xFFFFFFFFu)));
  return fma(t, e, t);
}

__device__ __forceinline__ uint64_t to_weight(double w) {  // rounded: the low mantissa bits of 2^52 + w
  return static_cast<uint64_t>(__double_as_longlong(w + 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
}

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int o) {
  return __shfl_xor(static_cast<unsigned long long>(v), o, 64);
}
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) v += shfl_xor_u64(v, o);
  return v;
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const uint64_t w = __shfl_up(static_cast<unsigned long long>(v), o, 64);
    if (lane >= o) v += w;
  }
  return v;
}

// a row without a distribution
__device__ __forceinline__ void no_token(const SampleArgs &a, int64_t row) {
  a.ids[row] = -1;
  if (a.logp) a.logp[row] = __builtin_nanf("");
  if (a.kept) a.kept[row] = 0;
}

struct Shared {
  uint64_t mass[kBins];  // of the ranges (counts too); the sort's exchange
  uint32_t lo[kBins], hi[kBins];  // a range's keys; the list: keys, indices
  uint64_t wave[kSmWaves];
  float fwave[kSmWaves];
  uint64_t found_base, target, total;
  uint32_t found_bin, found_index;
  uint32_t flags, listed;
};

// A row: its rules, its logits with the penalty on them, and, once the maximum is known, their weights and ranges.
template <bool WIDE>
struct Row {
  // four logits as they lie in memory (converted later: no load waits for another's)
  using Raw = std::conditional_t<WIDE, uint4, uint2>;
  const float *x32;
  const uint16_t *x16;
  const uint32_t *seen;  // a bit per token (in LDS)
  float temp, pen, top_p, min_p, u;
  uint64_t first_k;      // top-k (T = 0: 1), 0 where it leaves everything
  int n;
  bool is_half, penal, greedy, sole;  // sole: all below the maximum weighs nothing
  const double *table;   // (in LDS)
  double inv_pen, rate, top, deep, least;
  float mx, per, near;

  __device__ __forceinline__ Row(const SampleArgs &a, int64_t row, const uint32_t *bits, const double *powers) {
    table = powers;
    const plx_sample_rules &ru = a.rules;
    x32 = static_cast<const float *>(a.logits) + row * a.stride;
    x16 = static_cast<const uint16_t *>(a.logits) + row * a.stride;
    seen = bits;
    n = a.n;
    is_half = a.x_type == PLX_DTYPE_F16;
    temp = ru.temperature_rows ? ru.temperature_rows[row] : ru.temperature;
    pen = ru.penalty_rows ? ru.penalty_rows[row] : ru.penalty;
    top_p = ru.top_p_rows ? ru.top_p_rows[row] : ru.top_p;
    min_p = ru.min_p_rows ? ru.min_p_rows[row] : ru.min_p;
    const int64_t top_k = ru.top_k_rows ? ru.top_k_rows[row] : ru.top_k;
    u = a.u[row];
    penal = ru.seen != nullptr && pen != 1.0f;
    greedy = temp == 0.f;
    first_k = greedy ? 1 : top_k > 0 && top_k < n ? static_cast<uint64_t>(top_k) : 0;
    // z / pen through fp64: a quotient of two 24-bit numbers lies 2^-49 of itself or more from the middle of two
    // fp32 numbers, the product with the rounded reciprocal 2^-52 from the quotient, so it rounds to the same
    inv_pen = 1.0 / static_cast<double>(pen);
    least = kWeightOne * static_cast<double>(fminf(fmaxf(min_p, 0.f), 1.f));
  }
  // The bits of the tokens seen before, by all `threads` of the block (a barrier before they are read).
  static __device__ __forceinline__ void mark_seen(const SampleArgs &a, int64_t row, uint32_t *bits, int threads) {
    const plx_sample_rules &ru = a.rules;
    const int tid = threadIdx.x;
    for (int i = tid; i < (a.n + 31) / 32; i += threads) bits[i] = 0;
    __syncthreads();
    const int64_t have = ru.seen_len ? ru.seen_len[ru.seen_len_stride * row] : ru.seen_cols;
    const int64_t count = have < 0 ? 0 : have < ru.seen_cols ? have : ru.seen_cols;
    for (int64_t i = tid; i < count; i += threads) {
      const int64_t t = ru.seen[row * ru.seen_stride + i];
      if (t >= 0 && t < a.n) atomicOr(&bits[t >> 5], 1u << (t & 31));
    }
  }
  __device__ __forceinline__ float of16(uint32_t b) const {
    return is_half ? __half2float(__ushort_as_half(static_cast<uint16_t>(b))) : bf16_bits_to_float(b & 0xFFFFu);
  }
  __device__ __forceinline__ float value(int i) const {  // without the penalty
    if constexpr (WIDE) return x32[i];
    else return of16(x16[i]);
  }
  __device__ __forceinline__ Raw load(int i) const {  // from index i, all in the row, aligned
    if constexpr (WIDE) return *reinterpret_cast<const uint4 *>(x32 + i);
    else return *reinterpret_cast<const uint2 *>(x16 + i);
  }
  __device__ __forceinline__ Raw gather(int i) const {  // at the row's end, or of no alignment; past the row: -inf
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = min(i + e, n - 1);  // (no branch holds a load)
      if constexpr (WIDE) w[e] = i + e < n ? __float_as_uint(x32[j]) : 0xFF800000u;
      else w[e] = i + e < n ? x16[j] : (is_half ? 0xFC00u : 0xFF80u);
    }
    if constexpr (WIDE) return make_uint4(w[0], w[1], w[2], w[3]);
    else return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
  }
  __device__ __forceinline__ float penalised(float z) const {
    const float less = f32_kept(static_cast<float>(static_cast<double>(z) * inv_pen)), more = z * pen;
    return z > 0.f ? less : more;  // (kept: a select, not a branch)
  }
  __device__ __forceinline__ void convert(const Raw &v, int i, float (&z)[4]) const {  // with the penalty
    if constexpr (WIDE) {
      z[0] = __uint_as_float(v.x); z[1] = __uint_as_float(v.y); z[2] = __uint_as_float(v.z); z[3] = __uint_as_float(v.w);
    } else {
      z[0] = of16(v.x); z[1] = of16(v.x >> 16); z[2] = of16(v.y); z[3] = of16(v.y >> 16);
    }
    if (!penal) return;
    const uint32_t bits = i < n ? seen[i >> 5] >> (i & 31) : 0;  // (i is a multiple of 4)
    if ((bits & 15u) == 0) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p = f32_kept(penalised(z[e]));
      z[e] = bits >> e & 1u ? p : z[e];
    }
  }
  // Takes the row's maximum; false where there is no distribution: NaN logits, none above -inf, settings that are none.
  __device__ __forceinline__ bool scale(float maximum, bool nan) {
    mx = maximum;
    sole = greedy || mx == INFINITY;
    rate = greedy ? 0.0 : kTable * 1.4426950408889634 / static_cast<double>(temp);
    top = sole ? 0.0 : static_cast<double>(mx);
    deep = -60.0 * kTable / rate;  // (weights below 2^-45 round to 0)
    // ranges of max - z: 30.5 T holds every weight that is not 0
    per = fminf(fmaxf(static_cast<float>(kBins - 1) / (30.5f * (greedy ? 1.f : temp)), 1e-30f), 3e38f);
    near = fminf(mx, 3.402823466e38f);  // (finite: the distance of +inf to it is below 0)
    return !(nan || mx == -INFINITY || !(temp >= 0.f) || !(top_p == top_p) || !(min_p == min_p) ||
             (penal && !(pen > 0.f)) || !(u == u));
  }
  __device__ __forceinline__ double power(float z) const {  // 2^44 e^((z - max) / T)
    const double w = exp2_scaled(table, fmax(static_cast<double>(z) - top, deep), rate);
    return sole ? (z == mx ? kWeightOne : 0.0) : w;
  }
  __device__ __forceinline__ float depth(float z) const { return (near - z) * per; }
  __device__ __forceinline__ int bin_of(float z) const {
    return static_cast<int>(__builtin_amdgcn_fmed3f(depth(z), 0.f, static_cast<float>(kBins - 1)));
  }
  __device__ __forceinline__ int min_p_bin() const {  // the ranges down to min_p's, and one for the roundings
    const float far = -logf(fminf(min_p, 1.f)) * (static_cast<float>(kBins - 1) / 30.5f) + 1.f;
    return static_cast<int>(fminf(far, static_cast<float>(kBins - 1)));
  }
  __device__ __forceinline__ uint64_t share(uint64_t all) const {  // the mass that top-p reaches for
    const double p = top_p > 0.f ? static_cast<double>(top_p) * static_cast<double>(all) : 0.0;
    const uint64_t t = static_cast<uint64_t>(ceil(p));
    return t < 1 ? uint64_t{1} : t < all ? t : all;
  }
  __device__ __forceinline__ uint64_t drawn(uint64_t total) const {  // what the token's running sum has to pass
    const double p = static_cast<double>(u) * static_cast<double>(total);
    const uint64_t t = p > 0.0 ? static_cast<uint64_t>(fmin(p, 9.0e18)) : 0;
    return t < total ? t : total - 1;
  }
  __device__ __forceinline__ float logit(int id) const {  // with the penalty
    const float z = value(id);
    return penal && (seen[id >> 5] >> (id & 31) & 1u) ? penalised(z) : z;
  }
  __device__ __forceinline__ float log_share(float z, uint64_t total) const {
    const double t = z == mx ? 0.0 : (static_cast<double>(z) - top) / static_cast<double>(temp);
    return static_cast<float>(t - log(static_cast<double>(total) / kWeightOne));
  }
};

// ---- the passes over the row, by many blocks ------------------------------
//
// A row of 50,000 tokens takes one CU some 6 us for a pass; so the passes over it are launches of their own, a row's
// blocks of 4 waves (as many as bring the launch to 1,024 blocks, 4 a CU; at least one group a wave) taking groups of
// 1,024 tokens: its maximum; the histogram that its first rule needs, or, without a
// rule, every group's mass; and the list of the tokens that are left, or the token itself.  sample_rows_kernel then
// sorts the list (or takes the row alone, as it does without a workspace, where the list does not hold what is left).
// One row 39 -> 29 us by this, 16 rows 54 -> 33, 512 rows 80 -> 58; shorter lists by one wave and the table 24, 31 and 51.

constexpr int kSlThreads = 256;
constexpr int kSlWaves = kSlThreads / 64;
constexpr int kGroup = 1024;  // tokens: 4 chunks of 256
constexpr int kMaxSlices = 64;

struct Scratch {  // one row's part of the workspace
  uint64_t *mass, *totals, *reach;
  uint32_t *keys, *indices, *counts, *listed;
  float *maxima;
};

struct ScratchShape {
  unsigned char *base;
  int slices, groups;
  int64_t row_bytes;

  __host__ __device__ __forceinline__ static ScratchShape of(void *workspace, int64_t rows, int n) {
    ScratchShape s;
    s.base = static_cast<unsigned char *>(workspace);
    s.groups = (n + kGroup - 1) / kGroup;
    const int64_t want = (1024 + rows - 1) / (rows > 0 ? rows : 1), most = (s.groups + kSlWaves - 1) / kSlWaves;
    s.slices = static_cast<int>(want < most ? want : most);
    if (s.slices > kMaxSlices) s.slices = kMaxSlices;
    if (s.slices < 1) s.slices = 1;
    s.row_bytes = (int64_t{8} * (kBins + s.groups + 1) + int64_t{4} * (2 * kList + s.groups + 1 + s.slices) + 15) / 16 * 16;
    return s;
  }
  __device__ __forceinline__ Scratch row(int64_t r) const {
    Scratch x;
    x.mass = reinterpret_cast<uint64_t *>(base + r * row_bytes);
    x.totals = x.mass + kBins;
    x.reach = x.totals + groups;
    x.keys = reinterpret_cast<uint32_t *>(x.reach + 1);
    x.indices = x.keys + kList;
    x.counts = x.indices + kList;
    x.listed = x.counts + groups;
    x.maxima = reinterpret_cast<float *>(x.listed + 1);
    return x;
  }
};

// The row's maximum from those of its blocks, NaN if any is; every lane of a wave.
__device__ __forceinline__ float maximum_of(const float *maxima, int slices, int lane, bool &nan) {
  const float v = lane < slices ? maxima[lane] : -INFINITY;
  nan = __any(v != v);
  float m[1] = {v};
  group_reduce<64, true>(m);
  return m[0];
}

// f(four logits, index of the first, group) for the chunks of the groups of this block's waves, done(group) after each.
template <bool WIDE, class F, class G>
__device__ __forceinline__ void each_group(const Row<WIDE> &rv, const ScratchShape &shape, bool vec, int slice, int wave,
                                           int lane, F f, G done) {
  for (int g = slice * kSlWaves + wave; g < shape.groups; g += shape.slices * kSlWaves) {
    const int i0 = g * kGroup + 4 * lane;
    typename Row<WIDE>::Raw raw[4];
    if (vec && (g + 1) * kGroup <= rv.n) {
#pragma unroll
      for (int c = 0; c < 4; ++c) raw[c] = rv.load(i0 + 256 * c);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) raw[c] = rv.gather(i0 + 256 * c);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float z[4];
      rv.convert(raw[c], i0 + 256 * c, z);
      f(z, i0 + 256 * c);
    }
    done(g);
  }
}

// Each slice's maximum (NaN if any logit is); the row's scratch cleared.  Bytes: 512 rows of 50,688 bf16 logits 12 us
// (4.3 TB/s).
template <bool WIDE>
__global__ __launch_bounds__(kSlThreads) void sample_max_kernel(SampleArgs a, ScratchShape shape) {
  extern __shared__ __align__(16) uint32_t seen[];
  __shared__ float waves[kSlWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x / shape.slices;
  const int slice = blockIdx.x % shape.slices;
  const Scratch sc = shape.row(row);
  for (int i = slice * kSlThreads + tid; i < kBins; i += shape.slices * kSlThreads) sc.mass[i] = 0;
  if (slice == 0 && tid == 0) *sc.listed = 0;
  const Row<WIDE> rv(a, row, seen, nullptr);
  if (rv.penal) {
    Row<WIDE>::mark_seen(a, row, seen, kSlThreads);
    __syncthreads();
  }
  float mx = -INFINITY;
  bool nan = false;
  each_group(rv, shape, a.vec, slice, wave, lane,
             [&](const float (&z)[4], int) PLX_FLAT {
               mx = fmaxf(fmaxf(mx, fmaxf(z[0], z[1])), fmaxf(z[2], z[3]));
#pragma unroll
               for (int e = 0; e < 4; ++e) nan |= z[e] != z[e];
             },
             [](int) PLX_FLAT {});
  float red[1] = {mx};
  group_reduce<64, true>(red);
  const bool any = __any(nan);
  if (lane == 0) waves[wave] = any ? __builtin_nanf("") : red[0];
  __syncthreads();
  if (wave == 0) {
    mx = maximum_of(waves, kSlWaves, lane, nan);
    if (lane == 0) sc.maxima[slice] = nan ? __builtin_nanf("") : mx;
  }
}

// The histogram (in LDS, then added up in the scratch: integers, so in any order) of counts for top-k or of weights for
// top-p; without a rule each group's weight.  32 us of the 512 rows': 33 VALU instructions a token, 11 of them fp64, take
// 59% of the issue cycles; 37% of the waves' time is waits, as a token above -inf is a branch with a table read of its own.
template <bool WIDE>
__global__ __launch_bounds__(kSlThreads) void sample_mass_kernel(SampleArgs a, ScratchShape shape) {
  extern __shared__ __align__(16) uint32_t seen[];
  __shared__ uint64_t mass[kBins];
  __shared__ double powers[kTable];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x / shape.slices;
  const int slice = blockIdx.x % shape.slices;
  const Scratch sc = shape.row(row);
  Row<WIDE> rv(a, row, seen, powers);
  bool nan;
  const float mx = maximum_of(sc.maxima, shape.slices, lane, nan);
  if (!rv.scale(mx, nan)) return;
  const bool count = rv.first_k > 0, share = !count && rv.top_p < 1.f;
  if (!count && !share && rv.min_p > 0.f) return;  // (min-p alone needs no sums)
  if (!count) fill_table(powers);
  if (rv.penal) Row<WIDE>::mark_seen(a, row, seen, kSlThreads);
  if (count || share)
    for (int i = tid; i < kBins; i += kSlThreads) mass[i] = 0;
  __syncthreads();
  if (count) {
    each_group(rv, shape, a.vec, slice, wave, lane,
               [&](const float (&z)[4], int) PLX_FLAT {
#pragma unroll
                 for (int e = 0; e < 4; ++e)
                   atomicAdd(reinterpret_cast<unsigned int *>(&mass[rv.bin_of(z[e])]), z[e] > -INFINITY ? 1u : 0u);
               },
               [](int) PLX_FLAT {});
  } else if (share) {
    each_group(rv, shape, a.vec, slice, wave, lane,
               [&](const float (&z)[4], int) PLX_FLAT {
#pragma unroll
                 for (int e = 0; e < 4; ++e)
                   atomicAdd(reinterpret_cast<unsigned long long *>(&mass[rv.bin_of(z[e])]),
                             static_cast<unsigned long long>(z[e] > -INFINITY ? to_weight(rv.power(z[e])) : 0));
               },
               [](int) PLX_FLAT {});
  } else {
    uint64_t sum = 0;
    uint32_t number = 0;
    each_group(rv, shape, a.vec, slice, wave, lane,
               [&](const float (&z)[4], int) PLX_FLAT {
#pragma unroll
                 for (int e = 0; e < 4; ++e) {
                   const bool is = z[e] > -INFINITY;
                   sum += is ? to_weight(rv.power(z[e])) : 0;
                   number += is;
                 }
               },
               [&](int g) PLX_FLAT {
                 const uint64_t s = wave_sum_u64(sum);
                 const uint32_t k = static_cast<uint32_t>(wave_sum_u64(number));
                 if (lane == 0) {
                   sc.totals[g] = s;
                   sc.counts[g] = k;
                 }
                 sum = 0;
                 number = 0;
               });
    return;
  }
  __syncthreads();
  for (int i = tid; i < kBins; i += kSlThreads)
    if (mass[i] != 0)
      atomicAdd(reinterpret_cast<unsigned long long *>(&sc.mass[i]), static_cast<unsigned long long>(mass[i]));
}

// Where the first rule cuts, by every block of the row from the same histogram, and the tokens up to there into the row's
// list, in any order; without a rule the token itself, by one block from the groups' weights (9 us for 512 rows, a
// chain of latencies).
template <bool WIDE>
__global__ __launch_bounds__(kSlThreads) void sample_pick_kernel(SampleArgs a, ScratchShape shape) {
  extern __shared__ __align__(16) uint32_t seen[];
  __shared__ double powers[kTable];
  __shared__ uint64_t waves[kSlWaves];
  __shared__ uint64_t found_base;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x / shape.slices;
  const int slice = blockIdx.x % shape.slices;
  const Scratch sc = shape.row(row);
  Row<WIDE> rv(a, row, seen, powers);
  bool nan;
  const float mx = maximum_of(sc.maxima, shape.slices, lane, nan);
  if (!rv.scale(mx, nan)) {
    if (slice == 0 && tid == 0) no_token(a, row);
    return;
  }
  const bool count = rv.first_k > 0, share = !count && rv.top_p < 1.f, floor = !count && !share && rv.min_p > 0.f;
  if (!count && !share && !floor) {
    if (slice != 0) return;
    fill_table(powers);
  }
  if (rv.penal) Row<WIDE>::mark_seen(a, row, seen, kSlThreads);
  __syncthreads();
  // the sum over the block's threads up to and with this one; of all
  auto block_scan = [&](uint64_t v, uint64_t &all) PLX_FLAT {
    const uint64_t scan = wave_scan_u64(v, lane);
    __syncthreads();
    if (lane == 63) waves[wave] = scan;
    __syncthreads();
    uint64_t before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kSlWaves; ++w) {
      before += w < wave ? waves[w] : 0;
      all += waves[w];
    }
    return before + scan;
  };
  uint64_t all;
  if (count || share || floor) {
    int bin = 0;
    uint64_t base = 0;
    if (floor) {
      bin = rv.min_p_bin();
    } else {
      constexpr int kEach = kBins / kSlThreads;
      uint64_t m[kEach], sum = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        m[i] = sc.mass[kEach * tid + i];
        sum += m[i];
      }
      const uint64_t after = block_scan(sum, all);
      const uint64_t target = share ? rv.share(all) : rv.first_k < all ? rv.first_k : all;
      uint64_t before = after - sum;
      if (before < target && after >= target) {
        int b = kEach * tid;
#pragma unroll
        for (int i = 0; i < kEach - 1; ++i)
          if (b == kEach * tid + i && before + m[i] < target) {
            before += m[i];
            ++b;
          }
        found = b;
        found_base = before;
      }
      __syncthreads();
      bin = found;
      base = found_base;
      if (slice == 0 && tid == 0) *sc.reach = target;
    }
    if (count && base > kList) {  // (what is left is more than the list holds)
      if (slice == 0 && tid == 0) atomicAdd(sc.listed, kList + 1u);
      return;
    }
    const float d1 = bin < kBins - 1 ? static_cast<float>(bin + 1) : INFINITY;
    each_group(rv, shape, a.vec, slice, wave, lane,
               [&](const float (&z)[4], int i) PLX_FLAT {
                 bool hit[4], any = false;
#pragma unroll
                 for (int e = 0; e < 4; ++e) {
                   hit[e] = ((rv.depth(z[e]) < d1) | (bin == kBins - 1)) & (z[e] > -INFINITY);
                   any |= hit[e];
                 }
                 if (!any) return;
#pragma unroll
                 for (int e = 0; e < 4; ++e) {
                   if (!hit[e]) continue;
                   const uint32_t at = atomicAdd(sc.listed, 1u);
                   if (at < kList) {
                     sc.keys[at] = key_of(z[e]);
                     sc.indices[at] = static_cast<uint32_t>(i + e);
                   }
                 }
               },
               [](int) PLX_FLAT {});
    return;
  }
  // no rule: the group, then the token, at which the running mass passes u of all
  uint64_t mine = 0, number = 0;
  const int per = (shape.groups + kSlThreads - 1) / kSlThreads;  // consecutive groups per thread
  for (int i = 0; i < per; ++i) {
    const int g = tid * per + i;
    if (g < shape.groups) {
      mine += sc.totals[g];
      number += sc.counts[g];
    }
  }
  uint64_t kept;
  block_scan(number, kept);
  const uint64_t after = block_scan(mine, all), target = rv.drawn(all);
  if (after > target && after - mine <= target) {
    uint64_t before = after - mine;
    int g = tid * per;
    while (before + sc.totals[g] <= target) before += sc.totals[g++];
    found = g;
    found_base = before;
  }
  __syncthreads();
  if (wave != 0) return;
  uint64_t before = found_base;
  typename Row<WIDE>::Raw raw[kGroup / 256];
#pragma unroll
  for (int c = 0; c < kGroup / 256; ++c) raw[c] = rv.gather(found * kGroup + 256 * c + 4 * lane);
#pragma unroll
  for (int c = 0; c < kGroup / 256; ++c) {
    if (before > target) break;
    const int i = found * kGroup + 256 * c + 4 * lane;
    float z[4];
    rv.convert(raw[c], i, z);
    uint64_t w[4], s = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = z[e] > -INFINITY ? to_weight(rv.power(z[e])) : 0;
      s += w[e];
    }
    const uint64_t scan = wave_scan_u64(s, lane);
    uint64_t sum = before + scan - s;
    if (sum <= target && sum + s > target) {  // one lane
      int at = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (sum <= target) at = e;  // (the last whose sum before it has not passed)
        sum += w[e];
      }
      a.ids[row] = i + at;
      if (a.logp) a.logp[row] = rv.log_share(rv.logit(i + at), all);
      if (a.kept) a.kept[row] = static_cast<int64_t>(kept);
    }
    before += __shfl(static_cast<unsigned long long>(scan), 63, 64);
  }
}

// ---- a row by one block ----------------------------------------------------

// One block per row.  Wave w holds elements of one run of the row, 256 at a time (4 a lane): index order is wave, chunk,
// lane, element.
template <bool WIDE>
__global__ __launch_bounds__(kSmThreads) void sample_rows_kernel(SampleArgs a, ScratchShape shape) {
  extern __shared__ __align__(16) uint32_t seen[];  // a bit per token (penalty)
  __shared__ Shared sh;
  __shared__ double powers[kTable];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x;
  const int run = ((a.n + kSmWaves - 1) / kSmWaves + 255) / 256;  // chunks of a wave that hold any of the row
  const int start = wave * run * 256 + lane * 4;
  Row<WIDE> rv(a, row, seen, powers);
  fill_table(powers);
  int count = kList + 1;  // listed tokens
  uint64_t reach = 0;     // top-p's mass, where the first rule is top-p
  float mx = -INFINITY;
  bool nan = false;
  if (shape.base) {  // after the passes of many blocks
    const Scratch sc = shape.row(row);
    mx = maximum_of(sc.maxima, shape.slices, lane, nan);
    if (!rv.scale(mx, nan) || (rv.first_k == 0 && !(rv.top_p < 1.f) && !(rv.min_p > 0.f))) return;  // (all done)
    const uint32_t listed = *sc.listed;
    if (listed <= 64) {  // one wave sorts and cuts them, a token per lane, without a barrier
      __syncthreads();   // (the table)
      if (wave != 0) return;
      const int many = static_cast<int>(listed);
      uint64_t v = ~uint64_t{0};
      if (lane < many) v = static_cast<uint64_t>(~sc.keys[lane]) << 32 | sc.indices[lane];
#pragma unroll
      for (int k = 2; k <= 64; k *= 2)
#pragma unroll
        for (int j = k / 2; j > 0; j /= 2) {
          const uint64_t o = shfl_xor_u64(v, j);
          v = (((lane & k) == 0) == ((lane & j) == 0)) == (v < o) ? v : o;
        }
      const float z = value_of(~static_cast<uint32_t>(v >> 32));
      const double w = lane < many ? rv.power(z) : 0.0;
      const uint64_t m = to_weight(w), after = wave_scan_u64(m, lane);
      bool stays = lane < many && (rv.first_k == 0 || static_cast<uint64_t>(lane) < rv.first_k) && w >= rv.least;
      if (rv.top_p < 1.f) {
        uint64_t goal;
        if (rv.first_k == 0) goal = *sc.reach;
        else goal = rv.share(__shfl(static_cast<unsigned long long>(after), min(many, static_cast<int>(rv.first_k)) - 1, 64));
        stays &= after - m < goal;
      }
      const int stay = __popcll(__ballot(stays));  // every rule cuts the order once: the first `stay`
      const uint64_t total = __shfl(static_cast<unsigned long long>(after), stay - 1, 64), target = rv.drawn(total);
      // by index, each with its place in the order
      uint32_t o = lane < stay ? static_cast<uint32_t>(v) << 6 | static_cast<uint32_t>(lane) : 0xFFFFFFFFu;
#pragma unroll
      for (int k = 2; k <= 64; k *= 2)
#pragma unroll
        for (int j = k / 2; j > 0; j /= 2) {
          const uint32_t y = static_cast<uint32_t>(__shfl_xor(static_cast<int>(o), j, 64));
          o = (((lane & k) == 0) == ((lane & j) == 0)) == (o < y) ? o : y;
        }
      uint64_t wi = __shfl(static_cast<unsigned long long>(m), static_cast<int>(o & 63u), 64);
      wi = lane < stay ? wi : 0;
      const uint64_t sum = wave_scan_u64(wi, lane);
      const uint64_t passed = __ballot(sum > target && sum - wi <= target);
      const int place = __shfl(static_cast<int>(o & 63u), __ffsll(static_cast<unsigned long long>(passed)) - 1, 64);
      if (lane == place) {
        a.ids[row] = static_cast<int64_t>(static_cast<uint32_t>(v));
        if (a.kept) a.kept[row] = stay;
        if (a.logp) a.logp[row] = rv.log_share(z, total);
      }
      return;
    }
    if (listed <= kList) {
      count = static_cast<int>(listed);
      reach = rv.first_k == 0 && rv.top_p < 1.f ? *sc.reach : 0;
      if (tid < count) {
        sh.lo[tid] = sc.keys[tid];
        sh.hi[tid] = sc.indices[tid];
      }
    }
  }
  if (tid == 0) sh.flags = 0;
  if (rv.penal && count > kList) Row<WIDE>::mark_seen(a, row, seen, kSmThreads);
  for (int i = tid; i < kBins; i += kSmThreads) sh.mass[i] = 0;
  __syncthreads();
  // f(four logits, index of the first) for the chunks of this thread: a pass over the row, from memory once, then from L2
  const int whole = a.vec ? (a.n - wave * run * 256) / 256 : 0;  // chunks of the run that the row fills
  auto each = [&](auto f) PLX_FLAT {
#pragma unroll 1
    for (int c0 = 0; c0 < run; c0 += kAhead) {
      typename Row<WIDE>::Raw raw[kAhead];
      const int i0 = start + 256 * c0;
      if (c0 < whole) {  // (from clamped addresses: no branch between the loads, which would make each wait for the last)
#pragma unroll
        for (int c = 0; c < kAhead; ++c) raw[c] = rv.load(start + 256 * min(c0 + c, whole - 1));
      }
#pragma unroll
      for (int c = 0; c < kAhead; ++c) {
        if (c0 + c < run) {
          if (c0 + c >= whole) raw[c] = rv.gather(i0 + 256 * c);
          float z[4];
          rv.convert(raw[c], i0 + 256 * c, z);
          f(z, i0 + 256 * c);
        }
        __builtin_amdgcn_sched_barrier(0);  // (chunks worked on together take more registers than there are)
      }
    }
  };

  if (!shape.base) {
    each([&](const float (&z)[4], int) PLX_FLAT {
      mx = fmaxf(fmaxf(mx, fmaxf(z[0], z[1])), fmaxf(z[2], z[3]));
#pragma unroll
      for (int e = 0; e < 4; ++e) nan |= z[e] != z[e];
    });
    float red[1] = {mx};
    group_reduce<64, true>(red);
    if (lane == 0) sh.fwave[wave] = red[0];
    if (__any(nan) && lane == 0) atomicOr(&sh.flags, 1u);
    __syncthreads();
    mx = sh.fwave[0];
#pragma unroll
    for (int w = 1; w < kSmWaves; ++w) mx = fmaxf(mx, sh.fwave[w]);
    if (!rv.scale(mx, sh.flags != 0)) {
      if (tid == 0) no_token(a, row);
      return;
    }
  }

  // what is left: values above `cut`, and of those equal to it the indices up to `last`
  float cut = -INFINITY;
  int last = -1;
  auto in = [&](float z, int i) PLX_FLAT { return (z > cut) | ((z == cut) & (i <= last)); };

  // v at every thread: the sum up to and with it, in `all` the sum of all
  auto block_scan = [&](uint64_t v, uint64_t &all) PLX_FLAT {
    const uint64_t scan = wave_scan_u64(v, lane);
    __syncthreads();
    if (lane == 63) sh.wave[wave] = scan;
    __syncthreads();
    uint64_t before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kSmWaves; ++w) {
      const uint64_t s = sh.wave[w];
      before += w < wave ? s : 0;
      all += s;
    }
    return before + scan;
  };
  // ascending over the first `size` threads (a power of two, 64 or more), one value each
  auto sort = [&](auto v, int size) PLX_FLAT {
    using V = decltype(v);
    V *ex = reinterpret_cast<V *>(sh.mass);
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        V o;
        if (j < 64) {
          if constexpr (sizeof(V) == 8) o = shfl_xor_u64(v, j);
          else o = static_cast<V>(__shfl_xor(static_cast<int>(v), j, 64));
        } else {
          __syncthreads();
          ex[tid] = v;
          __syncthreads();
          o = ex[tid ^ j];
        }
        const bool low = ((tid & k) == 0) == ((tid & j) == 0);
        v = low == (v < o) ? v : o;
      }
    return v;
  };
  auto pow2_above = [](int n) PLX_FLAT {
    int s = 64;
    while (s < n) s *= 2;
    return s;
  };
  // Tokens of the ranges from b0 to b1 that are left: (key, index) into the list; how many there are.
  auto list = [&](int b0, int b1) PLX_FLAT {
    __syncthreads();
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    const float d0 = b0 > 0 ? static_cast<float>(b0) : -INFINITY;
    const float d1 = b1 < kBins - 1 ? static_cast<float>(b1 + 1) : INFINITY;  // (-inf lies at INFINITY: in no list)
    each([&](const float (&z)[4], int i) PLX_FLAT {
      bool hit[4], any = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float d = rv.depth(z[e]);
        hit[e] = (d >= d0) & ((d < d1) | (b1 == kBins - 1));
        any |= hit[e];
      }
      if (!any) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!hit[e] || !in(z[e], i + e)) continue;
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kList) {
          sh.lo[at] = key_of(z[e]);
          sh.hi[at] = static_cast<uint32_t>(i + e);
        }
      }
    });
    __syncthreads();
    return static_cast<int>(sh.listed);
  };
  // the list in order, a token per thread: the key's complement, then the index
  auto listed = [&](int count) PLX_FLAT {
    uint64_t v = ~uint64_t{0};
    if (tid < count) v = static_cast<uint64_t>(~sh.lo[tid]) << 32 | sh.hi[tid];
    return sort(v, pow2_above(count));
  };

  // Sums over the ranges in order: the first where they reach the target (of the sum of all).
  auto crossing = [&](auto target_of, uint64_t base) PLX_FLAT {
    __syncthreads();
    const uint64_t s0 = sh.mass[2 * tid], s1 = sh.mass[2 * tid + 1];
    uint64_t all;
    const uint64_t after = base + block_scan(s0 + s1, all), before = after - s0 - s1;
    const uint64_t target = target_of(base + all);
    if (before < target && after >= target) {
      const bool second = before + s0 < target;
      sh.found_bin = static_cast<uint32_t>(2 * tid + second);
      sh.found_base = second ? before + s0 : before;
      sh.target = target;
      sh.total = base + all;
    }
    __syncthreads();
  };

  // The first index (by order of indices) at which the running sum of weight(z, i) passes target; all threads.
  auto locate = [&](auto weight, uint64_t mine, uint64_t target) PLX_FLAT {
    mine = wave_sum_u64(mine);
    __syncthreads();
    if (lane == 0) sh.wave[wave] = mine;
    __syncthreads();
    uint64_t before = 0;
    int at = -1;
#pragma unroll
    for (int w = 0; w < kSmWaves; ++w) {
      const uint64_t s = sh.wave[w];
      if (at < 0) {
        if (before + s > target) at = w;
        else before += s;
      }
    }
    // that wave's run, a chunk of it for every wave
    uint64_t *sums = sh.mass;
    const int from = at * run * 256 + lane * 4;
    auto chunk = [&](int c, float (&z)[4]) PLX_FLAT {
      rv.convert(rv.gather(from + 256 * c), from + 256 * c, z);
      uint64_t s = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) s += weight(z[e], from + 256 * c + e);
      return s;
    };
    float z[4];
    uint64_t s = 0;
    int mine_c = -1;
    for (int c = wave; c < run; c += kSmWaves) {
      mine_c = c;
      s = chunk(c, z);
      const uint64_t all = wave_sum_u64(s);
      if (lane == 0) sums[c] = all;
    }
    __syncthreads();
    int c = 0;
    while (c < run - 1) {  // (64 chunks at a time)
      const uint64_t v = c + lane < run ? sums[c + lane] : 0, scan = wave_scan_u64(v, lane);
      const uint64_t passed = __ballot(before + scan > target);
      const int n = passed ? __ffsll(static_cast<unsigned long long>(passed)) - 1 : 64;
      if (n > 0) before += __shfl(static_cast<unsigned long long>(scan), n - 1, 64);
      c += n;
      if (passed) break;
    }
    c = min(c, run - 1);
    if (wave == c % kSmWaves) {
      if (mine_c != c) s = chunk(c, z);
      const uint64_t scan = wave_scan_u64(s, lane);
      uint64_t sum = before + scan - s;
      if (sum <= target && sum + s > target) {  // one lane
        int found = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum += weight(z[e], from + 256 * c + e);
          if (found < 0 && sum > target) found = from + 256 * c + e;
        }
        sh.found_index = static_cast<uint32_t>(found);
      }
    }
    __syncthreads();
    return static_cast<int>(sh.found_index);
  };

  // Cuts what is left where the count (weight_of 1) or mass of the tokens in order reaches the target: range `bin` holds
  // the cut, `base` is what lies before it.
  // (`count` of them listed, if they fit).
  auto narrow = [&](auto weight_of, int count, int bin, uint64_t base, uint64_t target) PLX_FLAT {
    if (count <= kList) {
      const uint64_t v = listed(count);
      const float z = value_of(~static_cast<uint32_t>(v >> 32));
      const uint64_t w = tid < count ? weight_of(z) : 0;
      uint64_t all;
      const uint64_t after = base + block_scan(w, all);
      if (after >= target && after - w < target) {
        sh.fwave[0] = z;
        sh.found_index = static_cast<uint32_t>(v);
      }
      __syncthreads();
      cut = sh.fwave[0];
      last = static_cast<int>(sh.found_index);
      __syncthreads();
      return;
    }
    auto was = [&, cut, last](float z, int i) PLX_FLAT { return z > cut || (z == cut && i <= last); };
    if (tid == 0) {
      sh.flags = 0xFFFFFFFFu;
      sh.found_index = 0;
    }
    __syncthreads();
    uint32_t kl = 0xFFFFFFFFu, kh = 0;
    each([&](const float (&z)[4], int i) PLX_FLAT {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (was(z[e], i + e) && rv.bin_of(z[e]) == bin) {
          kl = min(kl, key_of(z[e]));
          kh = max(kh, key_of(z[e]));
        }
    });
    if (kl <= kh) {
      atomicMin(&sh.flags, kl);
      atomicMax(&sh.found_index, kh);
    }
    __syncthreads();
    uint32_t lo = sh.flags, hi = sh.found_index;
    while (lo != hi) {  // (a range of keys becomes one of its 2,048 parts, cut to the keys there are)
      __syncthreads();
      for (int i = tid; i < kBins; i += kSmThreads) {
        sh.mass[i] = 0;
        sh.lo[i] = 0xFFFFFFFFu;
        sh.hi[i] = 0;
      }
      __syncthreads();
      const double scale = static_cast<double>(kBins) / (static_cast<double>(hi - lo) + 1.0);
      each([&](const float (&z)[4], int i) PLX_FLAT {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k = key_of(z[e]);
          if (k >= lo && k <= hi && was(z[e], i + e)) {
            const int s = min(kBins - 1, static_cast<int>(static_cast<double>(hi - k) * scale));
            atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[s]),
                      static_cast<unsigned long long>(weight_of(z[e])));
            atomicMin(&sh.lo[s], k);
            atomicMax(&sh.hi[s], k);
          }
        }
      });
      crossing([&](uint64_t) PLX_FLAT { return target; }, base);
      base = sh.found_base;
      lo = sh.lo[sh.found_bin];
      hi = sh.hi[sh.found_bin];
    }
    // all of one value, as many of the first as the target needs
    const float z1 = value_of(lo);
    const uint64_t one = weight_of(z1);
    const uint64_t need = (target - base + one - 1) / one;
    auto tie = [&](float z, int i) PLX_FLAT -> uint64_t { return z == z1 && was(z, i); };
    uint64_t mine = 0;
    each([&](const float (&z)[4], int i) PLX_FLAT {
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += tie(z[e], i + e);
    });
    last = locate(tie, mine, need - 1);
    cut = z1;
  };

  auto mass_of = [&](float z) PLX_FLAT { return to_weight(rv.power(z)); };
  int id = -1;
  uint64_t total = 0, kept = 0;
  // the rules in turn, until the tokens that are left fit the list: top-k, top-p, min-p
#pragma unroll 1
  for (int rule = 0; rule < 3 && count > kList; ++rule) {
    const bool mass = rule == 1, first = rule == 0 || rv.first_k == 0;
    int bin;
    uint64_t base = 0, target = 0;
    if (rule == 2) {
      if (!(rv.min_p > 0.f) || rv.first_k > 0 || rv.top_p < 1.f) break;
      bin = rv.min_p_bin();
    } else {
      if (mass ? !(rv.top_p < 1.f) : rv.first_k == 0) continue;
      if (!first) {
        for (int i = tid; i < kBins; i += kSmThreads) sh.mass[i] = 0;
        __syncthreads();
      }
      if (mass) {
        each([&](const float (&z)[4], int i) PLX_FLAT {
          uint64_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = in(z[e], i + e) ? mass_of(z[e]) : 0;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[rv.bin_of(z[e])]), static_cast<unsigned long long>(w[e]));
        });
      } else {
        each([&](const float (&z)[4], int) PLX_FLAT {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            atomicAdd(reinterpret_cast<unsigned int *>(&sh.mass[rv.bin_of(z[e])]), z[e] > -INFINITY ? 1u : 0u);
        });
      }
      crossing([&](uint64_t all) PLX_FLAT { return mass ? rv.share(all) : rv.first_k < all ? rv.first_k : all; }, 0);
      bin = static_cast<int>(sh.found_bin);
      base = sh.found_base;
      target = sh.target;
      if (mass) reach = target;
    }
    // all up to the cut if they fit; the cut's range alone otherwise
    for (int b0 = first && (mass || base <= kList) ? 0 : bin;; b0 = bin) {
      const int found = list(b0, bin);
      if (b0 == 0 && first && found <= kList) {
        count = found;
        break;
      }
      if (b0 < bin && rule < 2) continue;
      if (rule < 2) narrow([&](float z) PLX_FLAT -> uint64_t { return mass ? mass_of(z) : 1; }, found, bin, base, target);
      break;
    }
  }
  if (count <= kList) {
    const uint64_t v = listed(count);
    const int index = static_cast<int>(static_cast<uint32_t>(v));
    const double w = tid < count ? rv.power(value_of(~static_cast<uint32_t>(v >> 32))) : 0.0;
    const uint64_t m = to_weight(w);
    uint64_t all;
    const uint64_t after = block_scan(m, all);
    bool stays = tid < count;
    if (rv.first_k > 0) {
      stays &= static_cast<uint64_t>(tid) < rv.first_k;
      if (rv.top_p < 1.f) {
        __syncthreads();
        if (tid == min(count, static_cast<int>(rv.first_k)) - 1) sh.total = after;
        __syncthreads();
        reach = rv.share(sh.total);
      }
    }
    if (rv.top_p < 1.f) stays &= after - m < reach;
    stays &= w >= rv.least;
    const int stay = __syncthreads_count(stays);  // every rule cuts the order once: the first `stay`
    if (tid == stay - 1) sh.total = after;
    uint64_t *weights = reinterpret_cast<uint64_t *>(sh.lo);
    static_assert(sizeof(sh.lo) >= kList * sizeof(uint64_t), "the list's weights");
    weights[tid] = m;
    __syncthreads();
    total = sh.total;
    kept = static_cast<uint64_t>(stay);
    // by index
    uint32_t o = tid < stay ? static_cast<uint32_t>(index) << 10 | static_cast<uint32_t>(tid) : 0xFFFFFFFFu;
    o = sort(o, pow2_above(stay));
    const uint64_t wi = tid < stay ? weights[o & 1023u] : 0;
    const uint64_t sum = block_scan(wi, all);
    const uint64_t target = rv.drawn(total);
    if (sum > target && sum - wi <= target) sh.found_index = o & 1023u;
    __syncthreads();
    if (tid == static_cast<int>(sh.found_index)) {  // the token's thread
      a.ids[row] = index;
      if (a.kept) a.kept[row] = static_cast<int64_t>(kept);
      if (a.logp) a.logp[row] = rv.log_share(value_of(~static_cast<uint32_t>(v >> 32)), total);
    }
    return;
  } else {
    auto weight = [&](float z, int i) PLX_FLAT -> uint64_t {
      const double w = rv.power(z);
      return (in(z, i) & (w >= rv.least)) ? to_weight(w) : 0;
    };
    uint64_t mine = 0;
    uint32_t number = 0;
    each([&](const float (&z)[4], int i) PLX_FLAT {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double w = rv.power(z[e]);
        const bool ok = in(z[e], i + e) & (w >= rv.least);
        mine += ok ? to_weight(w) : 0;
        number += ok;
      }
    });
    uint64_t all;
    block_scan(number, all);
    kept = all;
    block_scan(mine, total);
    id = locate(weight, mine, rv.drawn(total));
  }
  if (tid == 0) {
    a.ids[row] = id;
    if (a.kept) a.kept[row] = static_cast<int64_t>(kept);
    if (a.logp) a.logp[row] = rv.log_share(rv.logit(id), total);
  }
}

}  // namespace

size_t sample_rows_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kSmMost) return 0;
  return static_cast<size_t>(rows * ScratchShape::of(nullptr, rows, static_cast<int>(cols)).row_bytes);
}

int launch_sample_rows(const void *logits, int x_type, int64_t rows, int64_t cols, int64_t stride, const float *u,
                       const plx_sample_rules &rules, int64_t *ids, float *logp, int64_t *kept, void *workspace,
                       size_t workspace_bytes, hipStream_t s) {
  if (cols > kSmMost) return fail(PLX_EINVAL, "sample_rows: rows of %lld tokens (at most %d)", static_cast<long long>(cols), kSmMost);
  ScratchShape shape = ScratchShape::of(workspace, rows, static_cast<int>(cols));
  if (workspace) {
    if (workspace_bytes < static_cast<size_t>(rows * shape.row_bytes))
      return fail(PLX_EINVAL, "sample_rows: workspace of %zu bytes, need %zu", workspace_bytes,
                  static_cast<size_t>(rows * shape.row_bytes));
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
      return fail(PLX_EINVAL, "sample_rows: the workspace must be 16-byte aligned");
  }
  const bool wide = x_type == PLX_DTYPE_F32;
  const int size = wide ? 4 : 2;
  const int vec = stride % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % (4 * size) == 0;
  const SampleArgs a{logits, stride, x_type, static_cast<int>(cols), vec, u, rules, ids, kept, logp};
  const unsigned lds = rules.seen ? static_cast<unsigned>((a.n + 127) / 128 * 16) : 0;
  const auto launch = [&](auto *kernel, unsigned blocks, int threads, size_t fixed) {  // fixed: the kernel's own LDS
    if (fixed + lds > 65536) {  // (the longest row's for any: a call of another thread, of other rows, sets no other value)
      const int st = check_hip(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, kSmMost / 8),
                               "sample_rows: LDS");
      if (st != PLX_OK) return st;
    }
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), lds, s, a, shape);
    return check_launch("sample_rows");
  };
  if (workspace) {
    const unsigned blocks = static_cast<unsigned>(rows * shape.slices);
    int st = launch(wide ? &sample_max_kernel<true> : &sample_max_kernel<false>, blocks, kSlThreads, 64);
    if (st == PLX_OK)
      st = launch(wide ? &sample_mass_kernel<true> : &sample_mass_kernel<false>, blocks, kSlThreads, 8 * (kBins + kTable));
    if (st == PLX_OK)
      st = launch(wide ? &sample_pick_kernel<true> : &sample_pick_kernel<false>, blocks, kSlThreads, 8 * kTable + 64);
    // (rules that are known to leave every token: nothing to sort)
    const bool cuts = rules.top_k_rows || (rules.top_k > 0 && rules.top_k < cols) || rules.top_p_rows || rules.top_p < 1.f ||
                      rules.min_p_rows || rules.min_p > 0.f || rules.temperature_rows || rules.temperature == 0.f;
    if (st != PLX_OK || !cuts) return st;
  }
  return launch(wide ? &sample_rows_kernel<true> : &sample_rows_kernel<false>, static_cast<unsigned>(rows), kSmThreads,
                sizeof(Shared) + 8 * kTable);
}

}  // namespace plx
