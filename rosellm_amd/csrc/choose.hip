// Next tokens from given uniforms, every row with its own temperature, top-k, top-p and
// min-p, and their log-probs.
//
// Per row x_0..x_{V-1}, uniform u, m = max x, c = log2(e) / T:
//   w_v = 2^(c (x_v - m)),  p_v = w_v / sum w
//   1. the k largest are left (ties: lowest index first)
//   2. of these, in descending order, those up to which the sum of w is at most
//      top_p of theirs all (the first always)
//   3. of these, those with x_v - m >= T log(min_p)
//   token: the first v, in vocabulary order, whose running sum of what is left exceeds u
//   times its whole
// T <= 0: the first maximum, log-prob at T = 1.
//
// A cut and a token are decided by where a running sum passes a border, so weights are
// formed in float64 (1.1e-12) and added as integers, in units of 2^-44 of the largest
// one (2^-(62 - b) for rows of 2^b > 2^18 entries): integer sums are the same in any
// order, so that LDS atomics may form them.  An entry is off by up to half a unit, and
// entries below that count as none, so that a sum may be off by 2^-45 V of the largest
// weight (a border by 4.3e-9 for 150,000 entries that all are rounded the same way, 1e-11 where
// they are not); an error that a log-prob next to 0 would show.  Log-probs are formed from
// sums of the same weights in float64, which are the same in any order of a row's chunks too.
//
// What is left is always the entries above a place (x, v) in descending order.  Rows are
// cut into parts of 8192 entries or more, a workgroup each (a single row of 151,936 is 19
// of them, on as many of the 256 CUs), and read once a launch (from the caches, but for the
// first):
//   1. choose_max: the maximum of each part
//   2. choose_weigh: each part's sum, and where the row has a top-k or a top-p its
//      histogram, counts or sums in 1024 bins of 1/16 of a factor of two below m, of the
//      entries that a nucleus or the top k can hold at all; the latter are listed as well
//   3. choose_cut (only if there may be a top-k or top-p): a workgroup a row finds the bin
//      that holds the border, lists its entries, and finds the place among them
//   4. choose_left (as 3): the sum of what is left, of each quarter of a part
//   5. choose_draw: a workgroup a row finds the quarter, then the entry
//
// Times, us (bfloat16 rows of 151,936): one row with a nucleus 3 + 8 + 29 + 6 + 9, 64 rows
// without a filter 5 + 14 + 9, 256 rows with settings of their own 15 + 65 + 41 + 30 + 18.
// The second launch is bound by issue: 21 instructions an entry without a filter, 14 of them
// float64 (32 and 16 with a min-p), and the histograms' atomics; the third by the chain of
// some fifteen barriers of sixteen waves each (9 us a border) and a read of the row by one CU;
// the bytes of 256 rows are 16 us at a copy's rate.
#include "vocab_weights.hpp"

#include <type_traits>

namespace rrl {
namespace {

constexpr int kPT = 256, kPW = kPT / 64;   // threads and waves of a part
constexpr int kRT = 1024, kRW = kRT / 64;  // of a row
constexpr int kBins = 1024, kBinBits = 10;
constexpr int kListed = 4096, kPartListed = 2048;  // entries that are held in LDS
constexpr int kAhead = 4;                  // 16-byte vectors that a lane loads at once
constexpr int kNoIndex = 0x7fffffff;
static_assert(kBins == kRT, "a bin to a thread");

typedef unsigned long long u64;

// Entries are left where x > v, or x == v and their index is below n.
struct Cut {
  float v;
  int n;
  __device__ __forceinline__ bool keeps(float x, int i) const { return x > v || (x == v && i < n); }
};

struct ChooseArgs {
  const char* x;
  int64_t ld, V;
  const float* u;
  // one setting a row, or null: the number beside it
  const float *temperature, *top_p, *min_p;
  const void* top_k;
  int top_k_dt;
  double temperature_all, top_p_all, min_p_all;
  int64_t top_k_all;
  int parts, part;  // parts of a row, and their entries
  double magic;     // 2^(52 - F): a weight added to it stands in the low bits, in units of 2^-F
  int unit_log2;    // F
  int bins;         // of a histogram: kBins, or fewer where a row has fewer entries
  int list_room;    // kListed, or the row's length
  float* peak;      // [B, parts] a part's maximum; +inf: it holds NaN or +inf
  u64* whole;       // [B, parts] sum of all entries, where there is a top-p and no top-k
  u64* left;        // [B, parts, kPW] of those that are left, a wave's run of a part each
  struct Exact* all;   // [B, parts, kPW] the same two sums for log-probs; kept only where
  struct Exact* kept;  // a setting leaves out entries
  u64* sums;        // [B, parts, bins], where there may be a top-p
  uint32_t* counts; // [B, parts, bins], where there may be a top-k
  Cut* cut;         // [B], where there may be either
  float* tops;      // [B, parts, kPT] a lane's maximum, where there may be a top-k
  float* reach;     // [B] the least value that the top k can hold
  float* list_x;    // [B, list_room] entries that the top k can hold, in any order
  int *list_i, *listed;  // their places, and [B] their number (over kListed: not all are there)
  int64_t* token_out;
  float *logp_out, *logq_out;  // logq_out may be null
};

// Order of floats as that of unsigned numbers (-0 as +0).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}

// The bits of a key that a type's values differ in: bfloat16's lower 16 and float16's lower
// 13 are all zeros, or all ones below 0.
template <class Tag> constexpr int kKeyShift = 0;
template <> constexpr int kKeyShift<TagBF16> = 16;
template <> constexpr int kKeyShift<TagF16> = 13;
template <class Tag>
__device__ __forceinline__ uint32_t short_key(float x) { return key_of(x) >> kKeyShift<Tag>; }
template <class Tag>
__device__ __forceinline__ float short_value(uint32_t k) {
  constexpr int S = kKeyShift<Tag>;
  k <<= S;
  return value_of(k >> 31 ? k : k | ((1u << S) - 1u));
}

// `sh` holds a value for each of the NW waves.
template <int NW, class T, class Op>
__device__ __forceinline__ T block_reduce(T v, T* sh, Op op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int k = 1; k < NW; ++k) v = op(v, sh[k]);
  return v;
}
struct Add {
  __device__ __forceinline__ u64 operator()(u64 a, u64 b) const { return a + b; }
};
struct Max {
  template <class T>
  __device__ __forceinline__ T operator()(T a, T b) const { return a > b ? a : b; }
};
struct Min {
  template <class T>
  __device__ __forceinline__ T operator()(T a, T b) const { return a < b ? a : b; }
};

// A row's settings.
struct Settings {
  double T, top_p, min_p;
  int64_t top_k;  // 0: none
  bool greedy, bad, filtered;
  __device__ __forceinline__ Settings(const ChooseArgs& a, int64_t b) {
    T = a.temperature ? (double)a.temperature[b] : a.temperature_all;
    top_p = a.top_p ? (double)a.top_p[b] : a.top_p_all;
    min_p = a.min_p ? (double)a.min_p[b] : a.min_p_all;
    top_k = a.top_k ? load_index(a.top_k, a.top_k_dt, b) : a.top_k_all;
    greedy = T <= 0.0;
    bad = !(T < M<double>::inf());
    if (greedy) T = 1.0;
    if (T < 1e-290) T = 1e-290;  // has the distribution's limit already
    if (top_k < 0 || top_k >= a.V) top_k = 0;
    if (!(top_p > 0.0 && top_p < 1.0)) top_p = 0.0;
    filtered = !greedy && (top_k > 0 || top_p > 0.0);
  }
  __device__ __forceinline__ double c() const { return 1.4426950408889634074 / T; }
  // bins of 1/16 of a factor of two, by the distance to the maximum
  __device__ __forceinline__ float scale() const { return (float)fmin(16.0 * c(), 3e38); }
  // what min_p alone leaves
  __device__ __forceinline__ Cut least(float m) const {
    if (!(min_p > 0.0)) return Cut{-M<float>::inf(), 0};
    // the least float at no more than that distance, a step or two from this one
    const double far = T * log(fmin(min_p, 1.0));
    uint32_t k = key_of((float)((double)m + far));
    for (int n = 0; n < 4 && (double)value_of(k) - (double)m < far; ++n) ++k;
    for (int n = 0; n < 4 && (double)value_of(k - 1) - (double)m >= far; ++n) --k;
    return Cut{value_of(k), kNoIndex};
  }
};
// The last of `bins` takes all that lies below it.
__device__ __forceinline__ int bin_of(float x, float m, float scale, int bins) {
  return (int)fminf((m - x) * scale, (float)(bins - 1));
}

// The least float (by its key) that falls into a bin up to `bin`.  Whole waves look for the
// same, 64 places at a time.
__device__ __forceinline__ float bin_floor(int bin, float m, float scale, int bins) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t lo = key_of(-__FLT_MAX__), hi = key_of(m);  // hi does
  while (lo < hi) {
    const uint32_t step = (hi - lo) / 64 + 1;
    const uint32_t at = hi - lo > lane * step ? lo + lane * step : hi;
    const uint64_t in = __ballot(bin_of(value_of(at), m, scale, bins) <= bin);
    if (in) {
      const uint32_t first = (uint32_t)__ffsll((unsigned long long)in) - 1;
      const uint32_t found = hi - lo > first * step ? lo + first * step : hi;
      if (first > 0) lo += (first - 1) * step + 1;
      hi = found;
      if (first == 0) lo = hi;
    } else {
      lo += 63 * step + 1;
    }
  }
  return value_of(hi);
}

// The row's maximum; +inf where it has no distribution.
template <int NW>
__device__ __forceinline__ float row_peak(const ChooseArgs& a, int64_t b, float* sh) {
  float m = -M<float>::inf();
  for (int k = threadIdx.x; k < a.parts; k += NW * 64) m = fmaxf(m, a.peak[b * a.parts + k]);
  m = block_reduce<NW>(m, sh, Max());
  return m == -M<float>::inf() ? M<float>::inf() : m;
}

// The integer mass of an entry.
struct Mass {
  Weight w;
  double magic;
  u64 zero;  // the bits of magic
  __device__ __forceinline__ Mass(float m, double c, double magic_)
      : w(m, c, 1.0), magic(magic_), zero((u64)__double_as_longlong(magic_)) {}
  // of w.unscaled(x)
  template <bool DIRECT>
  __device__ __forceinline__ u64 of(double v) const {
    return (u64)__double_as_longlong(DIRECT ? fma(v, w.k, magic) : v + magic) - zero;
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    return w.direct ? of<true>(w.unscaled<true>(x)) : of<false>(w.unscaled<false>(x));
  }
};

// A sum of weights in units of 2^-90 of the largest, as two integers.
struct Exact {
  u64 coarse = 0, fine = 0;  // units of 2^-40; of 2^-90, signed
  // A chunk's sum, of at most 2^11 weights.  Its last bits are those of a 64-bit number of
  // its size, and nothing else is rounded: the order of the chunks changes nothing.
  __device__ __forceinline__ void add(double s) {
#pragma clang fp contract(off)  // s is a rounded product, as log_share's
    const double near = s + 0x1p12, rest = s - (near - 0x1p12);  // |rest| <= 2^-41
    coarse += (u64)__double_as_longlong(near) - (u64)__double_as_longlong(0x1p12);
    fine += (u64)__double_as_longlong(rest + 0x1.8p-38) - (u64)__double_as_longlong(0x1.8p-38);
  }
  __device__ __forceinline__ double value() const {
    return fma((double)(int64_t)fine, 0x1p-90, (double)coarse * 0x1p-40);
  }
};

// f(values, index of the first) for the 16-byte vectors of entries lo..hi-1 of a row, by
// NT threads of which this is the t-th; past the end of them -inf.  done() after each chunk
// of kAhead vectors a thread, by all of them.
struct Nothing {
  __device__ __forceinline__ void operator()() const {}
};
template <class Tag, int NT, class F, class D = Nothing>
__device__ __forceinline__ void sweep(const char* row, int64_t lo, int64_t hi, int t, F f, D done = D()) {
  constexpr int EPV = Pack16<Tag>::EPV, SZ = 16 / EPV;
  static_assert(kAhead * 64 * EPV <= 2048, "a chunk of a wave is one of Exact's");
  for (int64_t base = lo; base < hi; base += kAhead * NT * EPV) {
    const int64_t i0 = base + t * EPV;
    u32x4 raw[kAhead];
    if (base + kAhead * NT * EPV <= hi) {
#pragma unroll
      for (int s = 0; s < kAhead; ++s)
        raw[s] = reinterpret_cast<const Any16*>(row + (i0 + s * NT * EPV) * SZ)->v;
    } else {
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        float x[EPV];
        load_entries<Tag>(row, i0 + s * NT * EPV, hi, x);
        raw[s] = Pack16<Tag>::pack(x);
      }
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      float x[EPV];
      Pack16<Tag>::unpack(raw[s], x);
      f(x, (int)(i0 + s * NT * EPV));
    }
    done();
  }
}
// The same by a wave over its quarter of a part, which starts with a chunk.
template <class Tag, class F, class D = Nothing>
__device__ __forceinline__ void sweep_part(const ChooseArgs& a, const char* row, int64_t part, F f, D done = D()) {
  const int64_t lo = part * a.part + (threadIdx.x >> 6) * (a.part / kPW);
  sweep<Tag, 64>(row, lo, min(lo + a.part / kPW, a.V), threadIdx.x & 63, f, done);
}
template <class Tag>
__device__ __forceinline__ const char* row_at(const ChooseArgs& a, int64_t b) {
  return a.x + b * a.ld * (16 / Pack16<Tag>::EPV);
}

// ---- 1 ---------------------------------------------------------------------------------

template <class Tag>
__global__ __launch_bounds__(kPT) void choose_max_kernel(ChooseArgs a) {
  constexpr int EPV = Pack16<Tag>::EPV;
  const int64_t b = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  __shared__ float sh[kPW];
  float m = -M<float>::inf();
  bool nan = false;
  sweep_part<Tag>(a, row_at<Tag>(a, b), part, [&](const float (&x)[EPV], int) {
#pragma unroll
    for (int k = 0; k < EPV; k += 2) {
      // with NaN among them the result is not used
      asm("v_max3_f32 %0, %1, %2, %0" : "+v"(m) : "v"(x[k]), "v"(x[k + 1]));
      nan |= __builtin_isunordered(x[k], x[k + 1]);
    }
  });
  if (a.tops) {
    a.tops[(int64_t)blockIdx.x * kPT + threadIdx.x] = m;
    if (part == 0 && threadIdx.x == 0) a.listed[b] = 0;
  }
  m = block_reduce<kPW>(nan ? M<float>::inf() : m, sh, Max());
  if (threadIdx.x == 0) a.peak[blockIdx.x] = m;
}

// ---- 2 ---------------------------------------------------------------------------------

struct WeighShared {
  u64 sums[kBins];
  uint32_t counts[kBins];
  float list_x[kPartListed];
  int list_i[kPartListed];
  u64 wave[kPW];
  int listed, bin, base;
};

// The last bin that the top k reach at most: k lanes' maxima are that large or larger.
__device__ __forceinline__ int top_bin(const ChooseArgs& a, const Settings& set, float m, int64_t b, WeighShared& sh) {
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, n = a.parts * kPT;
  if (set.top_k > n) return a.bins - 1;
  const float scale = set.scale();
  constexpr int kTogether = 8;
  for (int k0 = t; k0 < n; k0 += kTogether * kPT) {
    float x[kTogether];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) x[k] = a.tops[b * n + min(k0 + k * kPT, n - 1)];
#pragma unroll
    for (int k = 0; k < kTogether; ++k)
      if (k0 + k * kPT < n && x[k] != -M<float>::inf()) atomicAdd(&sh.counts[bin_of(x[k], m, scale, a.bins)], 1u);
  }
  if (t == 0) sh.bin = a.bins - 1;
  __syncthreads();
  constexpr int kEach = kBins / kPT;
  uint32_t mine[kEach], sum = 0;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    mine[k] = sh.counts[t * kEach + k];
    sum += mine[k];
  }
  uint32_t upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(upto, o, 64);
    if (lane >= o) upto += y;
  }
  uint32_t* const sums = reinterpret_cast<uint32_t*>(sh.wave);
  if (lane == 63) sums[wv] = upto;
  __syncthreads();
  for (int k = 0; k < wv; ++k) upto += sums[k];
  uint32_t at = upto - sum;
  if (at < set.top_k && upto >= set.top_k) {  // one thread's
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (at < set.top_k && at + mine[k] >= set.top_k) sh.bin = t * kEach + k;
      at += mine[k];
    }
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) sh.counts[t * kEach + k] = 0;
  __syncthreads();
  return sh.bin;
}

// A sum is formed here and not later: where branches follow, the weights of all that a lane
// holds would wait for it in registers, which leaves two of three waves a SIMD (256 rows with
// a nucleus 148 us instead of 142, with settings of their own 173 instead of 166).
__device__ __forceinline__ void here(double& sum) { asm volatile("" : "+v"(sum)); }

// whole and left are this thread's, all and kept the wave's.
template <class Tag, bool DIRECT>
__device__ __forceinline__ void weigh(const ChooseArgs& a, const Settings& set, const Mass& mass, float m, int64_t b,
                                      int64_t part, float reach, WeighShared& sh, u64& whole, u64& left, Exact& all,
                                      Exact& kept) {
  constexpr int EPV = Pack16<Tag>::EPV;
  const char* row = row_at<Tag>(a, b);
  const float scale = set.scale();
  double sum = 0.0, some = 0.0;
  auto add = [&] {
    all.add(wave_sum_d(sum) * mass.w.template factor<DIRECT>());
    sum = 0.0;
  };
  if (set.filtered && set.top_k > 0) {
    sweep_part<Tag>(a, row, part, [&](const float (&x)[EPV], int i) {
#pragma unroll
      for (int k = 0; k < EPV; ++k) {
        const double v = mass.w.template unscaled<DIRECT>(x[k]);
        sum += v;
        if (x[k] >= reach) {
          const int bin = bin_of(x[k], m, scale, a.bins), at = atomicAdd(&sh.listed, 1);
          atomicAdd(&sh.counts[bin], 1u);
          if (set.top_p > 0.0) atomicAdd(&sh.sums[bin], mass.of<DIRECT>(v));
          if (at < kPartListed) {
            sh.list_x[at] = x[k];
            sh.list_i[at] = i + k;
          }
        }
      }
    }, add);
  } else if (set.filtered) {
    // Entries of at most (1 - top_p) / V of the largest make up no more than 1 - top_p of
    // the whole, so that the border lies above them.
    const u64 floor = (u64)ldexp((1.0 - set.top_p) / (double)a.V, a.unit_log2);
    sweep_part<Tag>(a, row, part, [&](const float (&x)[EPV], int) {
#pragma unroll
      for (int k = 0; k < EPV; ++k) {
        const double v = mass.w.template unscaled<DIRECT>(x[k]);
        const u64 w = mass.of<DIRECT>(v);
        sum += v;
        here(sum);
        whole += w;
        if (w > floor) atomicAdd(&sh.sums[bin_of(x[k], m, scale, a.bins)], w);
      }
    }, add);
  } else if (set.min_p > 0.0) {
    const Cut cut = set.least(m);
    sweep_part<Tag>(a, row, part, [&](const float (&x)[EPV], int) {
#pragma unroll
      for (int k = 0; k < EPV; ++k) {
        const double v = mass.w.template unscaled<DIRECT>(x[k]);
        const bool in = x[k] >= cut.v;
        sum += v;
        some += in ? v : 0.0;
        left += in ? mass.of<DIRECT>(v) : 0;
      }
    }, [&] {
      add();
      kept.add(wave_sum_d(some) * mass.w.template factor<DIRECT>());
      some = 0.0;
    });
  } else {
    sweep_part<Tag>(a, row, part, [&](const float (&x)[EPV], int) {
#pragma unroll
      for (int k = 0; k < EPV; ++k) {
        const double v = mass.w.template unscaled<DIRECT>(x[k]);
        sum += v;
        left += mass.of<DIRECT>(v);
      }
    }, add);
  }
}
__device__ __forceinline__ u64 wave_total(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <class Tag>
__global__ __launch_bounds__(kPT) void choose_weigh_kernel(ChooseArgs a) {
  const int64_t b = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int t = threadIdx.x;
  __shared__ WeighShared sh;
  const Settings set(a, b);
  const float m = row_peak<kPW>(a, b, reinterpret_cast<float*>(sh.wave));
  if (set.bad || !(m < M<float>::inf())) return;
  float reach = 0.0f;
  if (set.filtered) {
    for (int k = t; k < kBins; k += kPT) {
      sh.sums[k] = 0;
      sh.counts[k] = 0;
    }
    if (t == 0) sh.listed = 0;
    __syncthreads();
    if (set.top_k > 0) reach = bin_floor(top_bin(a, set, m, b, sh), m, set.scale(), a.bins);
  }
  const Mass mass(m, set.c(), a.magic);
  u64 whole = 0, left = 0;
  Exact all, kept;
  if (mass.w.direct) weigh<Tag, true>(a, set, mass, m, b, part, reach, sh, whole, left, all, kept);
  else weigh<Tag, false>(a, set, mass, m, b, part, reach, sh, whole, left, all, kept);
  const int64_t wave = (int64_t)blockIdx.x * kPW + (t >> 6);
  if ((t & 63) == 0) a.all[wave] = all;
  if (set.filtered) {
    whole = block_reduce<kPW>(whole, sh.wave, Add());
    if (t == 0) a.whole[blockIdx.x] = whole;
    const int64_t to = (int64_t)blockIdx.x * a.bins;
    if (set.top_p > 0.0)
      for (int k = t; k < a.bins; k += kPT) a.sums[to + k] = sh.sums[k];
    if (set.top_k > 0) {
      for (int k = t; k < a.bins; k += kPT) a.counts[to + k] = sh.counts[k];
      if (part == 0 && t == 0) a.reach[b] = reach;
      // a run of the row's list; beyond its end, or this part's, nothing is listed
      if (t == 0) sh.base = atomicAdd(&a.listed[b], min(sh.listed, kListed + 1) + (sh.listed > kPartListed ? kListed + 1 : 0));
      __syncthreads();
      for (int k = t; k < min(sh.listed, kPartListed) && sh.base + k < a.list_room; k += kPT) {
        a.list_x[b * a.list_room + sh.base + k] = sh.list_x[k];
        a.list_i[b * a.list_room + sh.base + k] = sh.list_i[k];
      }
    }
  } else {
    left = wave_total(left);
    if ((t & 63) == 0) {
      a.left[wave] = left;
      if (set.min_p > 0.0) a.kept[wave] = kept;
    }
  }
}

// ---- 3 ---------------------------------------------------------------------------------

struct CutShared {
  u64 hist[kBins];
  u64 wave[kRW];
  u64 above;  // of the bins before the one that holds the border
  float list_x[kListed];
  int list_i[kListed];
  int bin, listed;
};

// The bin at which the running sum, `above` before the first, exceeds target: -1 if none
// does.  `mine` is this thread's bin; `above` becomes the sum before that bin.
__device__ __forceinline__ int find_bin(CutShared& sh, u64 mine, u64& above, u64 target) {
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  u64 v = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (t == 0) sh.bin = -1;
  if (lane == 63) sh.wave[wv] = v;
  __syncthreads();
  u64 end = above + v;
#pragma unroll
  for (int k = 0; k < kRW; ++k) end += k < wv ? sh.wave[k] : 0;  // all read at once
  if (end - mine <= target && end > target) {  // one thread's
    sh.bin = t;
    sh.above = end - mine;
  }
  __syncthreads();
  const int bin = sh.bin;
  if (bin >= 0) above = sh.above;
  return bin;
}

__device__ __forceinline__ int bits_over(uint32_t n) {  // bits to drop so that numbers up to n fit the bins
  const int bits = 32 - __clz((int)n);
  return bits > kBinBits ? bits - kBinBits : 0;
}

// The entries of one bin that a cut leaves: in a list in LDS, or, if they are too many for
// that, looked for in the row each time.  The list is the row's if that is whole.
template <class Tag>
struct BinEntries {
  const char* row;
  int64_t V;
  float lo, hi;  // entries lo <= x < hi (hi: +inf for the first bin)
  Cut cut;
  CutShared* sh;
  int listed;
  __device__ __forceinline__ BinEntries(const ChooseArgs& a, int64_t b, float m, float scale, int bin, const Cut& cut_,
                                        bool have_list, CutShared& sh_)
      : row(row_at<Tag>(a, b)), V(a.V), cut(cut_), sh(&sh_), listed(kListed + 1) {
    lo = bin_floor(bin, m, scale, a.bins);
    hi = bin > 0 ? bin_floor(bin - 1, m, scale, a.bins) : M<float>::inf();  // (its key lies above all others)
    if (have_list) {
      listed = sh->listed;
      return;
    }
    __syncthreads();
    if (threadIdx.x == 0) sh->listed = 0;
    __syncthreads();
    constexpr int EPV = Pack16<Tag>::EPV;
    // a lane marks its entries, then lists them one after another, all lanes' at once
    for (int64_t base = 0; base < V; base += kAhead * kRT * EPV) {
      const int64_t i0 = base + threadIdx.x * EPV;
      uint32_t marks = 0;
      u32x4 raw[kAhead];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        const int64_t i = i0 + (int64_t)s * kRT * EPV;
        if (i + EPV <= V) {
          raw[s] = reinterpret_cast<const Any16*>(row + i * (16 / EPV))->v;
        } else {
          float x[EPV];
          load_entries<Tag>(row, i, V, x);
          raw[s] = Pack16<Tag>::pack(x);
        }
      }
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        float x[EPV];
        Pack16<Tag>::unpack(raw[s], x);
#pragma unroll
        for (int k = 0; k < EPV; ++k)
          marks |= (x[k] >= lo && x[k] < hi && x[k] != -M<float>::inf() ? 1u : 0u) << (s * EPV + k);
      }
      while (__any(marks != 0)) {
        const int k = __ffs((int)marks) - 1;
        const int64_t i = marks ? i0 + (int64_t)(k / EPV) * kRT * EPV + k % EPV : 0;
        const float x = marks ? load_entry<Tag>(row, i) : 0.0f;
        const bool in = marks && cut.keeps(x, (int)i);
        const uint64_t all = __ballot(in);
        int from = 0;
        if ((threadIdx.x & 63) == 0 && all) from = atomicAdd(&sh->listed, (int)__popcll(all));
        from = __builtin_amdgcn_readfirstlane(from);
        const int at = from + __popcll(all & (((uint64_t)1 << (threadIdx.x & 63)) - 1));
        if (in && at < kListed) {  // in any order: what follows does not depend on it
          sh->list_x[at] = x;
          sh->list_i[at] = (int)i;
        }
        marks &= marks - 1;
      }
    }
    __syncthreads();
    listed = sh->listed;
  }
  // f(whether there is one, value, index) with whole waves.  One loop for both kinds, and one
  // call of f: this kernel runs once over long code, which has to come from memory.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int EPV = Pack16<Tag>::EPV;
    const bool list = listed <= kListed;
    const int per = list ? kRT : kRT * EPV;
    const int64_t n = list ? listed : V;
    for (int64_t base = 0; base < n; base += per) {
      const int64_t i0 = base + (int64_t)threadIdx.x * (list ? 1 : EPV);
      uint32_t marks = 0;
      if (list) {
        marks = i0 < n && sh->list_x[i0] >= lo && sh->list_x[i0] < hi ? 1u : 0u;
      } else {
        float x[EPV];
        load_entries<Tag>(row, i0, V, x);
#pragma unroll
        for (int k = 0; k < EPV; ++k) marks |= (x[k] >= lo && x[k] < hi && x[k] != -M<float>::inf() ? 1u : 0u) << k;
      }
      while (__any(marks != 0)) {
        const int64_t at = marks ? i0 + __ffs((int)marks) - 1 : 0;
        const float x = list ? sh->list_x[at] : load_entry<Tag>(row, at);
        const int i = list ? sh->list_i[at] : (int)at;
        f(marks && cut.keeps(x, i), x, i);
        marks &= marks - 1;
      }
    }
  }
};

// Adds v to bins that hold equal values of v each; whole waves call it.  An LDS atomic on one
// address takes some 28 cycles a lane, and the entries of one bin have few values, so that
// up to eight of them are counted over the wave first.
__device__ __forceinline__ void add_equal(u64* hist, bool in, int bin, u64 v) {
  for (int k = 0; k < 8; ++k) {
    const uint64_t left = __ballot(in);
    if (!left) return;
    const bool mine = in && bin == __builtin_amdgcn_readlane(bin, __ffsll((unsigned long long)left) - 1);
    const uint64_t like = __ballot(mine);
    if (mine && (int)(threadIdx.x & 63) == __ffsll((unsigned long long)like) - 1)
      atomicAdd(&hist[bin], v * (u64)__popcll(like));
    in = in && !mine;
  }
  if (in) atomicAdd(&hist[bin], v);
}

// The longest run of these entries, in descending order, ties lowest index first, whose
// measure (1 or a mass), with `above` before them, sums to no more than target, which all
// of them exceed; at least one entry where nothing is above.
// With `want_rest`, `rest` becomes this thread's part of their masses.
template <class Tag>
__device__ __forceinline__ Cut select(const BinEntries<Tag>& in, bool by_mass, u64 above, u64 target, const Mass& mass,
                                      bool want_rest, u64& rest, CutShared& sh) {
  const int t = threadIdx.x;
  enum { KEYS, TIES, REST } phase = KEYS;
  uint32_t lo = short_key<Tag>(in.lo), hi = short_key<Tag>(in.hi);  // the border lies among these keys,
  uint32_t ilo = 0, ihi = (uint32_t)in.V;                           // the first that is not taken among these places
  u64 take = 0, seen = 0;
  float v = 0.0f;
  Cut out{0.0f, 0};
  for (;;) {
    const int shift = phase == KEYS ? bits_over(hi - lo) : bits_over(ihi - ilo);
    __syncthreads();
    sh.hist[t] = 0;
    __syncthreads();
    in.each([&](bool is, float x, int i) {
      if (phase == REST) {
        rest += is && out.keeps(x, i) ? mass(x) : 0;
        return;
      }
      const uint32_t at = phase == KEYS ? short_key<Tag>(x) : (uint32_t)i;
      const uint32_t from = phase == KEYS ? lo : ilo, to = phase == KEYS ? hi : ihi;
      is = is && at >= from && at <= to && (phase == KEYS || x == v);
      const int bin = (int)((phase == KEYS ? to - at : at - from) >> shift);
      const u64 w = !is ? 0 : (phase == KEYS && by_mass ? mass(x) : 1);
      if (phase == KEYS && shift == 0) add_equal(sh.hist, is, bin, w);
      else if (is) atomicAdd(&sh.hist[bin], w);
    });
    if (phase == REST) return out;
    __syncthreads();
    const int b = find_bin(sh, sh.hist[t], phase == KEYS ? above : seen, phase == KEYS ? target : take);
    if (phase == KEYS) {
      const u64 here = sh.hist[max(b, 0)];
      hi -= (uint32_t)max(b, 0) << shift;
      lo = max(lo, shift ? hi - ((1u << shift) - 1) : hi);
      if (lo < hi) continue;
      // the ties at that value: as many as the rest of the target holds
      v = short_value<Tag>(hi);
      const u64 each = by_mass ? mass(v) : 1;
      const u64 room = each ? (target - above) / each : ~(u64)0;
      take = above == 0 && room == 0 ? 1 : room;
      out = Cut{v, in.cut.v == v ? in.cut.n : kNoIndex};  // all of them
      if (take == 0) {
        out.n = 0;
      } else if (each != 0 && take * each < here) {
        phase = TIES;
        continue;
      }
    } else if (b >= 0) {
      ilo += (uint32_t)b << shift;
      ihi = min(ihi, ilo + (1u << shift) - 1);
      if (ilo < ihi) continue;
      out.n = (int)ilo;
    }
    if (!want_rest) return out;
    phase = REST;
  }
}

// One bin of every part.
template <class T>
__device__ __forceinline__ u64 over_parts(const T* all, int64_t b, int bin, int bins, int parts) {
  constexpr int kTogether = 10;
  u64 sum = 0;
  if (bin >= bins) return sum;
  const T* const of = all + b * parts * bins + bin;
  for (int k0 = 0; k0 < parts; k0 += kTogether) {
    T v[kTogether];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) v[k] = of[(int64_t)min(k0 + k, parts - 1) * bins];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) sum += k0 + k < parts ? v[k] : 0;
  }
  return sum;
}

template <class Tag>
__global__ __launch_bounds__(kRT) void choose_cut_kernel(ChooseArgs a) {
  __shared__ CutShared sh;
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x;
  const Settings set(a, b);
  if (!set.filtered || set.bad) return;
  const float m = row_peak<kRW>(a, b, reinterpret_cast<float*>(sh.wave));
  if (!(m < M<float>::inf())) return;
  const float scale = set.scale();
  const Mass mass(m, set.c(), a.magic);
  Cut cut{-M<float>::inf(), 0};
  u64 sum = 0;  // of this thread's bin
  if (set.top_p > 0.0) sum = over_parts(a.sums, b, t, a.bins, a.parts);
  bool have_list = false;
  if (set.top_k > 0) {
    const int n = a.listed[b];
    have_list = n <= kListed;
    if (have_list) {
      for (int k = t; k < n; k += kRT) {
        sh.list_x[k] = a.list_x[b * a.list_room + k];
        sh.list_i[k] = a.list_i[b * a.list_room + k];
      }
      if (t == 0) sh.listed = n;
    }
    __syncthreads();
  }
#pragma unroll 1
  for (int stage = set.top_k > 0 ? 0 : 1; stage < (set.top_p > 0.0 ? 2 : 1); ++stage) {
    const bool by_mass = stage == 1, both = stage == 0 && set.top_p > 0.0;
    u64 mine = sum, target = (u64)set.top_k, above = 0;
    if (by_mass) {
      u64 all = 0;
      if (set.top_k > 0) all = sum;
      else
        for (int k = t; k < a.parts; k += kRT) all += a.whole[b * a.parts + k];
      target = (u64)(set.top_p * (double)block_reduce<kRW>(all, sh.wave, Add()));
    } else {
      mine = over_parts(a.counts, b, t, a.bins, a.parts);
      cut = Cut{a.reach[b], kNoIndex};  // if these are k
    }
    const int bin = find_bin(sh, mine, above, target);
    if (bin < 0) continue;
    const BinEntries<Tag> in(a, b, m, scale, bin, by_mass ? cut : Cut{-M<float>::inf(), 0}, have_list, sh);
    u64 rest = 0;
    cut = select(in, by_mass, above, target, mass, both, rest, sh);
    if (both) {  // what is left of that bin, and nothing below it
      rest = block_reduce<kRW>(rest, sh.wave, Add());
      sum = t < bin ? sum : (t == bin ? rest : 0);
    }
  }
  const Cut least = set.least(m);
  if (least.v > cut.v) cut = least;
  if (t == 0) a.cut[b] = cut;
}

// ---- 4 ---------------------------------------------------------------------------------

// A nucleus is a few entries in a hundred, so a lane first marks those of its vectors,
// then weighs its marked ones, read again, one after another: as many turns as the lane
// with most of them has.  Where some lane has over a quarter, all are weighed in place.
template <class Tag, bool DIRECT>
__device__ __forceinline__ u64 weigh_left(const ChooseArgs& a, const char* row, int64_t part, const Cut& cut,
                                          const Mass& mass, Exact& kept) {
  constexpr int EPV = Pack16<Tag>::EPV;
  u64 left = 0;
  const int64_t quarter = a.part / kPW, lo = part * a.part + (threadIdx.x >> 6) * quarter;
  const int64_t hi = min(lo + quarter, a.V);
  const int lane = threadIdx.x & 63;
  for (int64_t i0 = lo; i0 < hi; i0 += kAhead * 64 * EPV) {
    u32x4 raw[kAhead];
    if (i0 + kAhead * 64 * EPV <= hi) {
#pragma unroll
      for (int s = 0; s < kAhead; ++s)
        raw[s] = reinterpret_cast<const Any16*>(row + (i0 + (s * 64 + lane) * EPV) * (16 / EPV))->v;
    } else {
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        float x[EPV];
        load_entries<Tag>(row, i0 + (s * 64 + lane) * EPV, hi, x);
        raw[s] = Pack16<Tag>::pack(x);
      }
    }
    uint32_t marks = 0;
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      float x[EPV];
      Pack16<Tag>::unpack(raw[s], x);
#pragma unroll
      for (int k = 0; k < EPV; ++k)
        marks |= (cut.keeps(x[k], (int)(i0 + (s * 64 + lane) * EPV) + k) ? 1u : 0u) << (s * EPV + k);
    }
    if (!__any(marks != 0)) continue;
    double sum = 0.0;  // in the same order either way
    if (__any(__popc(marks) > kAhead * EPV / 4)) {
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        float x[EPV];
        Pack16<Tag>::unpack(raw[s], x);
#pragma unroll
        for (int k = 0; k < EPV; ++k) {
          const double v = marks >> (s * EPV + k) & 1 ? mass.w.template unscaled<DIRECT>(x[k]) : 0.0;
          sum += v;
          left += mass.of<DIRECT>(v);
        }
      }
    } else {
      while (__any(marks != 0)) {
        if (marks) {
          const int k = __ffs((int)marks) - 1;
          marks &= marks - 1;
          const double v =
              mass.w.template unscaled<DIRECT>(load_entry<Tag>(row, i0 + (k / EPV * 64 + lane) * EPV + k % EPV));
          sum += v;
          left += mass.of<DIRECT>(v);
        }
      }
    }
    kept.add(wave_sum_d(sum) * mass.w.template factor<DIRECT>());
  }
  return left;
}

template <class Tag>
__global__ __launch_bounds__(kPT) void choose_left_kernel(ChooseArgs a) {
  const int64_t b = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  __shared__ float sh[kPW];
  const Settings set(a, b);
  if (!set.filtered || set.bad) return;
  const float m = row_peak<kPW>(a, b, sh);
  if (!(m < M<float>::inf())) return;
  const Cut cut = a.cut[b];
  u64 left = 0;
  Exact kept;
  if (a.peak[blockIdx.x] >= cut.v) {
    const Mass mass(m, set.c(), a.magic);
    const char* row = row_at<Tag>(a, b);
    left = mass.w.direct ? weigh_left<Tag, true>(a, row, part, cut, mass, kept)
                         : weigh_left<Tag, false>(a, row, part, cut, mass, kept);
    left = wave_total(left);
  }
  if ((threadIdx.x & 63) == 0) {
    const int64_t wave = (int64_t)blockIdx.x * kPW + (threadIdx.x >> 6);
    a.left[wave] = left;
    a.kept[wave] = kept;
  }
}

// ---- 5 ---------------------------------------------------------------------------------

// The log of an entry's share of a sum that holds it.  From the rest beside it where that is
// less than half, so that it is 0 where there is none.
__device__ __forceinline__ float log_share(const Weight& w, float x, double sum) {
#pragma clang fp contract(off)
  const double own = w.one(x);
  if (own > sum - own) return fminf((float)(0.0 - log1p((sum - own) / own)), 0.0f);
  return fminf((float)(((double)x - w.m) * w.c * 0.69314718055994530942 - log(sum)), 0.0f);
}

template <class Tag>
__global__ __launch_bounds__(kPT) void choose_draw_kernel(ChooseArgs a) {
  constexpr int EPV = Pack16<Tag>::EPV;
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  __shared__ u64 sh[kPW], sh_before;
  __shared__ int sh_quarter;
  int* const shi = reinterpret_cast<int*>(sh);
  const char* row = row_at<Tag>(a, b);
  const float* peak = a.peak + b * a.parts;
  const Settings set(a, b);
  const float m = row_peak<kPW>(a, b, reinterpret_cast<float*>(sh));
  if (set.bad || !(m < M<float>::inf())) {  // a row or a temperature without a distribution
    if (t == 0) {
      a.token_out[b] = -1;
      a.logp_out[b] = M<float>::nan();
      if (a.logq_out) a.logq_out[b] = M<float>::nan();
    }
    return;
  }
  u64 left = 0;
  // sums of what is left in their order, a run of quarters to a thread
  const int quarters = a.parts * kPW, run = (quarters + kPT - 1) / kPT;
  const int p0 = min(t * run, quarters), p1 = min(p0 + run, quarters);
  const u64* const lefts = a.left + b * quarters;
  if (!set.greedy)
    for (int p = p0; p < p1; ++p) left += lefts[p];
  double all = 0.0, kept = 0.0;  // the first wave's: for log-probs
  if (wv == 0) {
    auto row_sum = [&](const Exact* sums) {
      Exact s;
      for (int p = lane; p < quarters; p += 64) {
        s.coarse += sums[b * quarters + p].coarse;
        s.fine += sums[b * quarters + p].fine;
      }
      s.coarse = wave_total(s.coarse);
      s.fine = wave_total(s.fine);
      return s.value();
    };
    all = row_sum(a.all);
    kept = set.filtered || (!set.greedy && set.min_p > 0.0) ? row_sum(a.kept) : all;
  }
  const Mass mass(m, set.c(), a.magic);
  int token = kNoIndex;
  auto span = [&](int64_t lo, int64_t n, auto f) {
    sweep<Tag, kPT>(row, lo, min(lo + n, a.V), t, [&](const float (&x)[EPV], int i) {
#pragma unroll
      for (int k = 0; k < EPV; ++k) f(x[k], i + k);
    });
  };
  if (set.greedy) {
    int first = kNoIndex;
    for (int p = t; p < a.parts; p += kPT)
      if (peak[p] == m) first = min(first, p);
    first = min(block_reduce<kPW>(first, shi, Min()), a.parts - 1);
    span((int64_t)first * a.part, a.part, [&](float x, int i) { token = x == m ? min(token, i) : token; });
    token = block_reduce<kPW>(token, shi, Min());
  } else {
    const Cut cut = set.filtered ? a.cut[b] : set.least(m);
    u64 upto = left;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 y = __shfl_up(upto, o, 64);
      if (lane >= o) upto += y;
    }
    __syncthreads();
    if (lane == 63) sh[wv] = upto;
    __syncthreads();
    u64 total = 0;
    for (int k = 0; k < kPW; ++k) {
      if (k < wv) upto += sh[k];
      total += sh[k];
    }
    const double u = (double)a.u[b];
    const u64 border = u > 0.0 ? (u64)(fmin(u, 1.0) * (double)total) : 0;
    if (border == 0) {  // the first entry with any mass, be it less than a unit
      for (int p = 0; p < a.parts && token == kNoIndex; ++p) {
        if (peak[p] < cut.v) continue;
        span((int64_t)p * a.part, a.part, [&](float x, int i) {
          if (x != -M<float>::inf() && cut.keeps(x, i) && ((double)x - (double)m) * mass.w.c > -1000.0)
            token = min(token, i);
        });
        token = block_reduce<kPW>(token, shi, Min());
      }
    } else if (border >= total) {  // a uniform of 1: the last with any
      int last = -1;
      for (int p = p0; p < p1; ++p)
        if (lefts[p]) last = p;
      last = max(block_reduce<kPW>(last, shi, Max()), 0);
      token = -1;
      span((int64_t)last * (a.part / kPW), a.part / kPW, [&](float x, int i) {
        if (cut.keeps(x, i) && mass(x)) token = max(token, i);
      });
      token = block_reduce<kPW>(token, shi, Max());
    } else {
      if (upto > border && upto - left <= border) {  // one thread's
        u64 at = upto - left;
        int p = p0;
        for (; p < p1 - 1; ++p) {
          const u64 w = lefts[p];
          if (at + w > border) break;
          at += w;
        }
        sh_quarter = p;
        sh_before = at;
      }
      __syncthreads();
      // a run of the quarter's vectors to a thread
      const int vectors = a.part / (kPW * EPV * kPT) > 0 ? a.part / (kPW * EPV * kPT) : 1;
      const int64_t lo = (int64_t)sh_quarter * (a.part / kPW), hi = min(lo + a.part / kPW, a.V);
      const int64_t i0 = lo + (int64_t)t * vectors * EPV;
      auto weights = [&](int64_t i, u64 (&w)[EPV]) {
        float x[EPV];
        load_entries<Tag>(row, i, hi, x);
#pragma unroll
        for (int k = 0; k < EPV; ++k) w[k] = cut.keeps(x[k], (int)i + k) ? mass(x[k]) : 0;
      };
      u64 here = 0;
      for (int s = 0; s < vectors; ++s) {
        u64 w[EPV];
        weights(i0 + s * EPV, w);
#pragma unroll
        for (int k = 0; k < EPV; ++k) here += w[k];
      }
      u64 end = here;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const u64 y = __shfl_up(end, o, 64);
        if (lane >= o) end += y;
      }
      if (lane == 63) sh[wv] = end;
      __syncthreads();
      for (int k = 0; k < wv; ++k) end += sh[k];
      u64 at = sh_before + end - here;
      if (at <= border && at + here > border) {  // one thread's
        for (int s = 0; s < vectors; ++s) {
          u64 w[EPV];
          weights(i0 + s * EPV, w);
#pragma unroll
          for (int k = 0; k < EPV; ++k) {
            at += w[k];
            if (at > border) token = min(token, (int)(i0 + s * EPV) + k);
          }
        }
      }
      token = block_reduce<kPW>(token, shi, Min());
    }
  }
  if (t == 0) {
    // (there is a token, unless the logits changed meanwhile; then none is read for it)
    const bool some = token >= 0 && token < a.V;
    const float x = some ? load_entry<Tag>(row, token) : m;
    a.token_out[b] = some ? token : -1;
    a.logp_out[b] = some ? log_share(mass.w, x, all) : M<float>::nan();
    if (a.logq_out) a.logq_out[b] = !some ? M<float>::nan() : (set.greedy ? 0.0f : log_share(mass.w, x, kept));
  }
}

// ---- host ------------------------------------------------------------------------------

// Entries of a part: as many as leave a thousand workgroups.
inline int part_entries(int64_t B, int64_t V) {
  int part = 8192;
  while (part < 65536 && B * ((V + 2 * part - 1) / (2 * part)) >= 1024) part *= 2;
  return part;
}

struct ChooseLayout {
  int part, bins, list_room;
  int64_t parts;
  size_t peak, whole, left, all, kept, sums, counts, cut, tops, reach, list_x, list_i, listed, total;
};
inline ChooseLayout choose_layout(int64_t B, int64_t V, bool top_k, bool top_p) {
  ChooseLayout l;
  l.part = part_entries(B, V);
  l.parts = (V + l.part - 1) / l.part;
  // no more of either than a row has entries (131,072 rows of 9: 0.3 GB instead of 6)
  l.bins = 64;
  while (l.bins < kBins && l.bins < V) l.bins *= 2;
  l.list_room = (int)min(V, (int64_t)kListed);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t n = (size_t)(B * l.parts);
  l.peak = take(4 * n);
  l.whole = take(8 * n);
  l.left = take(8 * n * kPW);
  l.all = take(sizeof(Exact) * n * kPW);
  l.kept = take(sizeof(Exact) * n * kPW);
  l.sums = take(top_p ? 8 * n * l.bins : 0);
  l.counts = take(top_k ? 4 * n * l.bins : 0);
  l.cut = take(sizeof(Cut) * (size_t)B);
  l.tops = take(top_k ? 4 * n * kPT : 0);
  l.reach = take(top_k ? 4 * (size_t)B : 0);
  l.list_x = take(top_k ? 4 * (size_t)B * l.list_room : 0);
  l.list_i = take(top_k ? 4 * (size_t)B * l.list_room : 0);
  l.listed = take(top_k ? 4 * (size_t)B : 0);
  l.total = at;
  return l;
}

template <class Tag>
int launch_choose(const ChooseArgs& a, int64_t B, bool filters, hipStream_t st) {
  const dim3 parts((uint32_t)(B * a.parts)), rows((uint32_t)B);
  hipLaunchKernelGGL(choose_max_kernel<Tag>, parts, dim3(kPT), 0, st, a);
  if (int rc = check_launch("choose_max_kernel")) return rc;
  hipLaunchKernelGGL(choose_weigh_kernel<Tag>, parts, dim3(kPT), 0, st, a);
  if (int rc = check_launch("choose_weigh_kernel")) return rc;
  if (filters) {
    hipLaunchKernelGGL(choose_cut_kernel<Tag>, rows, dim3(kRT), 0, st, a);
    if (int rc = check_launch("choose_cut_kernel")) return rc;
    hipLaunchKernelGGL(choose_left_kernel<Tag>, parts, dim3(kPT), 0, st, a);
    if (int rc = check_launch("choose_left_kernel")) return rc;
  }
  hipLaunchKernelGGL(choose_draw_kernel<Tag>, rows, dim3(kPT), 0, st, a);
  return check_launch("choose_draw_kernel");
}

// Sizes whose index arithmetic and grids fit (a grid's threads are counted in 32 bits), and
// of rows whose sums are good enough to draw from: those of 2^20 entries, in units of 2^-42,
// are off by up to 2^-23 of the largest weight, a step or two of a float32 uniform; those of
// 2^30 would be by an eighth of it.
constexpr int64_t kMostEntries = (int64_t)1 << 20;
inline bool choose_fits(int64_t B, int64_t V) {
  return B >= 0 && V >= 1 && B < ((int64_t)1 << 22) && V <= kMostEntries &&
         B * ((V + part_entries(B, V) - 1) / part_entries(B, V)) < ((int64_t)1 << 24);
}
inline bool may_top_k(const rrl_sample_params& p, int64_t V) { return p.top_ks || (p.top_k > 0 && p.top_k < V); }
inline bool may_top_p(const rrl_sample_params& p) { return p.top_ps || (p.top_p > 0.0 && p.top_p < 1.0); }

}  // namespace
}  // namespace rrl

using namespace rrl;

extern "C" size_t rrl_sample_tokens_workspace_bytes(int64_t B, int64_t V, const rrl_sample_params* params) {
  if (!choose_fits(B, V)) return 0;
  return choose_layout(B, V, !params || may_top_k(*params, V), !params || may_top_p(*params)).total;
}

extern "C" int rrl_sample_tokens(const void* logits, int32_t dtype, int64_t B, int64_t V, int64_t row_stride,
                                 const float* uniforms, const rrl_sample_params* params, int64_t* token_out,
                                 float* logp_out, float* logq_out, void* workspace, void* stream) {
  clear_error();
  RRL_REQUIRE(dtype == RRL_F32 || dtype == RRL_BF16 || dtype == RRL_F16, RRL_EDTYPE,
              "rrl_sample_tokens: logits must be float32, bfloat16 or float16");
  RRL_REQUIRE(B >= 0, RRL_EINVAL, "rrl_sample_tokens: negative size");
  if (B == 0) return RRL_OK;
  RRL_REQUIRE(V >= 1, RRL_EINVAL, "rrl_sample_tokens: logits need at least one vocabulary entry");
  RRL_REQUIRE(choose_fits(B, V), RRL_EINVAL,
              "rrl_sample_tokens: 2^22 rows or more, 2^24 parts of them or more, or rows of over 2^20 entries (the "
              "sums of 2^30 would be too coarse to draw from)");
  RRL_REQUIRE(logits != nullptr && uniforms != nullptr && params != nullptr && token_out != nullptr &&
                  logp_out != nullptr && workspace != nullptr,
              RRL_EINVAL, "rrl_sample_tokens: null operand");
  RRL_REQUIRE(B <= 1 || row_stride >= 0, RRL_EINVAL, "rrl_sample_tokens: negative row stride");
  const rrl_sample_params& p = *params;
  RRL_REQUIRE(p.top_ks == nullptr || p.top_k_dtype == RRL_I32 || p.top_k_dtype == RRL_I64, RRL_EDTYPE,
              "rrl_sample_tokens: top_k must be int32 or int64");
  RRL_REQUIRE((uintptr_t)logits % dtype_size(dtype) == 0 && (uintptr_t)uniforms % 4 == 0 &&
                  (uintptr_t)p.temperatures % 4 == 0 && (uintptr_t)p.top_ps % 4 == 0 &&
                  (uintptr_t)p.min_ps % 4 == 0 && (uintptr_t)workspace % 16 == 0 &&
                  (p.top_ks == nullptr || (uintptr_t)p.top_ks % dtype_size(p.top_k_dtype) == 0),
              RRL_EALIGN, "rrl_sample_tokens: a pointer is not aligned (workspace: 16 bytes)");
  ChooseArgs a;
  a.x = static_cast<const char*>(logits);
  a.ld = row_stride;
  a.V = V;
  a.u = uniforms;
  a.temperature = p.temperatures;
  a.top_p = p.top_ps;
  a.min_p = p.min_ps;
  a.top_k = p.top_ks;
  a.top_k_dt = p.top_k_dtype;
  a.temperature_all = p.temperature;
  a.top_p_all = p.top_p;
  a.min_p_all = p.min_p;
  a.top_k_all = p.top_k;
  int bits = 0;
  while (((int64_t)1 << bits) < V) ++bits;
  a.unit_log2 = bits > 18 ? 62 - bits : 44;
  a.magic = ldexp(1.0, 52 - a.unit_log2);
  const bool top_k = may_top_k(p, V), top_p = may_top_p(p);
  const ChooseLayout l = choose_layout(B, V, top_k, top_p);
  char* w = static_cast<char*>(workspace);
  a.part = l.part;
  a.bins = l.bins;
  a.list_room = l.list_room;
  a.parts = (int)l.parts;
  a.peak = reinterpret_cast<float*>(w + l.peak);
  a.whole = reinterpret_cast<u64*>(w + l.whole);
  a.left = reinterpret_cast<u64*>(w + l.left);
  a.all = reinterpret_cast<Exact*>(w + l.all);
  a.kept = reinterpret_cast<Exact*>(w + l.kept);
  a.sums = reinterpret_cast<u64*>(w + l.sums);
  a.counts = reinterpret_cast<uint32_t*>(w + l.counts);
  a.cut = reinterpret_cast<Cut*>(w + l.cut);
  a.tops = top_k ? reinterpret_cast<float*>(w + l.tops) : nullptr;
  a.reach = reinterpret_cast<float*>(w + l.reach);
  a.list_x = reinterpret_cast<float*>(w + l.list_x);
  a.list_i = reinterpret_cast<int*>(w + l.list_i);
  a.listed = reinterpret_cast<int*>(w + l.listed);
  a.token_out = token_out;
  a.logp_out = logp_out;
  a.logq_out = logq_out;
  hipStream_t st = as_stream(stream);
  if (dtype == RRL_F32) return launch_choose<TagF32>(a, B, top_k || top_p, st);
  if (dtype == RRL_BF16) return launch_choose<TagBF16>(a, B, top_k || top_p, st);
  return launch_choose<TagF16>(a, B, top_k || top_p, st);
}
