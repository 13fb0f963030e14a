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
// order, so that LDS atomics may form them, and off by 2^-45 an entry, 1e-11 of the
// whole for 150,000 entries.
//
// What is left is always the entries above a place (x, v) in descending order, so a cut
// is found by histograms of 2048 bins: first of the distance to the maximum, then of the
// keys within the bin that holds the border, until that is one value; then, if it was
// only partly taken, of the indexes of its ties.
#include "vocab_weights.hpp"

namespace rrl {
namespace {

constexpr int kCT = 1024, kCW = kCT / 64;  // a workgroup's threads and waves
constexpr int kBins = 2048;                // two for each thread
constexpr int kNoIndex = 0x7fffffff;

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
  int slabs;     // 16-byte vectors of a lane: a wave's entries stand together
  double magic;  // 2^(52 - F): a weight added to it stands in the low bits, in units of 2^-F
  int unit_log2; // F
  int64_t* token_out;
  float *logp_out, *logq_out;  // logq_out may be null
};

typedef unsigned long long u64;

// Entries are left where x > v, or x == v and their index is below n.
struct Cut {
  float v;
  int n;
  __device__ __forceinline__ bool keeps(float x, int i) const { return x > v || (x == v && i < n); }
};

// Order of floats as that of unsigned numbers (-0 below +0, which are brought together
// before).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}

template <class T, class Op>
__device__ __forceinline__ T block_reduce(T v, T* sh, Op op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int k = 1; k < kCW; ++k) v = op(v, sh[k]);
  return v;
}
__device__ __forceinline__ u64 block_sum_u64(u64 v, u64* sh) {
  return block_reduce(v, sh, [](u64 a, u64 b) { return a + b; });
}

struct ChooseShared {
  u64 hist[kBins];
  u64 wave[kCW];
  u64 above;  // of the bins before the one that holds the border
  int bin;
  int slot;
};

template <class Tag>
struct Row {
  static constexpr int EPV = Pack16<Tag>::EPV;
  const char* p;
  int64_t V;
  int slabs;
  // f(value, index) for every entry of this lane that is above -inf
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int s = 0; s < slabs; ++s) {
      const int64_t i = (((int64_t)wv * slabs + s) * 64 + lane) * EPV;
      if (i >= V) break;
      float x[EPV];
      load_entries<Tag>(p, i, V, x);
#pragma unroll
      for (int k = 0; k < EPV; ++k)
        if (x[k] != -M<float>::inf()) f(x[k], (int)i + k);
    }
  }
};

// The integer mass of an entry.
struct Mass {
  Weight w;
  double magic;
  u64 zero;  // the bits of magic
  __device__ __forceinline__ Mass(const Weight& weight, double magic_)
      : w(weight), magic(magic_), zero((u64)__double_as_longlong(magic_)) {}
  __device__ __forceinline__ u64 operator()(float x) const {
    const double v = w.direct ? fma(w.template unscaled<true>(x), w.k, magic) : w.template unscaled<false>(x) + magic;
    return (u64)__double_as_longlong(v) - zero;
  }
};

// Clears the histogram; the workgroup may add to it afterwards.
__device__ __forceinline__ void clear_bins(ChooseShared& sh) {
  __syncthreads();
  for (int k = threadIdx.x; k < kBins; k += kCT) sh.hist[k] = 0;
  __syncthreads();
}

// The bin at which the running sum, `above` before the first, exceeds target: -1 if none
// does.  `above` becomes the sum before that bin.
__device__ __forceinline__ int find_bin(ChooseShared& sh, u64& above, u64 target) {
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  __syncthreads();
  const u64 a = sh.hist[2 * t], b = sh.hist[2 * t + 1];
  u64 v = a + b;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  if (t == 0) sh.bin = -1;
  if (lane == 63) sh.wave[wv] = v;
  __syncthreads();
  u64 before = above;
  for (int k = 0; k < wv; ++k) before += sh.wave[k];
  const u64 end = before + v, mid = end - b, start = mid - a;
  if (start <= target && end > target) {  // one thread's
    sh.bin = mid > target ? 2 * t : 2 * t + 1;
    sh.above = mid > target ? start : mid;
  }
  __syncthreads();
  const int bin = sh.bin;
  if (bin >= 0) above = sh.above;
  return bin;
}

__device__ __forceinline__ int bits_over(uint32_t n) {  // bits to drop so that numbers up to n fit the bins
  const int bits = 32 - __clz((int)n);
  return bits > 11 ? bits - 11 : 0;
}

// The longest run of the entries that `cut` leaves, in descending order, ties lowest
// index first, whose measure (1 or a mass) sums to no more than target; at least one entry.
template <class R, class Measure>
__device__ Cut select(const R& row, const Cut& cut, float m, float scale, u64 target, Measure measure,
                      ChooseShared& sh) {
  u64 above = 0;
  clear_bins(sh);
  auto bin_of = [&](float x) { return (int)fminf((m - x) * scale, (float)(kBins - 1)); };
  row.each([&](float x, int i) {
    if (cut.keeps(x, i)) atomicAdd(&sh.hist[bin_of(x)], measure(x));
  });
  const int bin = find_bin(sh, above, target);
  if (bin < 0) return cut;
  // the keys of that bin
  uint32_t lo = 0xffffffffu, hi = 0;
  row.each([&](float x, int i) {
    if (cut.keeps(x, i) && bin_of(x) == bin) {
      const uint32_t k = key_of(x);
      lo = min(lo, k);
      hi = max(hi, k);
    }
  });
  uint32_t* sh32 = reinterpret_cast<uint32_t*>(sh.wave);
  lo = block_reduce(lo, sh32, [](uint32_t a, uint32_t b) { return min(a, b); });
  hi = block_reduce(hi, sh32, [](uint32_t a, uint32_t b) { return max(a, b); });
  while (lo < hi) {
    const int shift = bits_over(hi - lo);
    clear_bins(sh);
    row.each([&](float x, int i) {
      const uint32_t k = key_of(x);
      if (k >= lo && k <= hi && cut.keeps(x, i)) atomicAdd(&sh.hist[(hi - k) >> shift], measure(x));
    });
    const int b = find_bin(sh, above, target);
    hi -= (uint32_t)b << shift;
    lo = max(lo, shift ? hi - ((1u << shift) - 1) : hi);
  }
  // the ties at that value: as many as the rest of the target holds
  const float v = value_of(hi);
  const u64 each = measure(v);
  const u64 room = each ? (target - above) / each : ~(u64)0;
  const u64 take = above == 0 && room == 0 ? 1 : room;
  u64 seen = 0;
  int ilo = 0, ihi = (int)min(row.V, (int64_t)kNoIndex - 1);  // the place of the first that is not taken
  if (take == 0) return Cut{v, 0};
  while (ilo < ihi) {
    const int shift = bits_over((uint32_t)(ihi - ilo));
    clear_bins(sh);
    row.each([&](float x, int i) {
      if (x == v && i >= ilo && i <= ihi && cut.keeps(x, i)) atomicAdd(&sh.hist[(i - ilo) >> shift], (u64)1);
    });
    const int b = find_bin(sh, seen, take);
    if (b < 0) return Cut{v, cut.v == v ? cut.n : kNoIndex};  // all of them
    ilo += b << shift;
    ihi = min(ihi, ilo + (1 << shift) - 1);
  }
  return Cut{v, ilo};
}

template <class Tag>
__global__ __launch_bounds__(kCT) void choose_kernel(ChooseArgs a) {
  __shared__ ChooseShared sh;
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  const Row<Tag> row{a.x + b * a.ld * (16 / Pack16<Tag>::EPV), a.V, a.slabs};
  double T = a.temperature ? (double)a.temperature[b] : a.temperature_all;
  const double top_p = a.top_p ? (double)a.top_p[b] : a.top_p_all;
  const double min_p = a.min_p ? (double)a.min_p[b] : a.min_p_all;
  const int64_t top_k = a.top_k ? load_index(a.top_k, a.top_k_dt, b) : a.top_k_all;
  const bool greedy = T <= 0.0;
  if (greedy) T = 1.0;

  float m = -M<float>::inf();
  int nan = 0;
  row.each([&](float x, int) {
    m = fmaxf(m, x);
    nan |= x != x;
  });
  float* shf = reinterpret_cast<float*>(sh.wave);
  m = block_reduce(m, shf, [](float p, float q) { return fmaxf(p, q); });
  nan = block_reduce(nan, reinterpret_cast<int*>(sh.wave), [](int p, int q) { return p | q; });
  // a row or a temperature without a distribution
  if (nan || !(fabsf(m) < M<float>::inf()) || !(T < M<double>::inf())) {
    if (t == 0) {
      a.token_out[b] = -1;
      a.logp_out[b] = M<float>::nan();
      if (a.logq_out) a.logq_out[b] = M<float>::nan();
    }
    return;
  }
  if (T < 1e-290) T = 1e-290;  // has the distribution's limit already
  const Weight weight(m, 1.4426950408889634074 / T, 1.0);
  const Mass mass(weight, a.magic);

  u64 whole = 0;
  row.each([&](float x, int) { whole += mass(x); });
  const double unit = ldexp(1.0, -a.unit_log2);
  const double norm = log((double)block_sum_u64(whole, sh.wave) * unit);

  int64_t token;
  double logq = 0.0;
  if (greedy) {
    int first = kNoIndex;
    row.each([&](float x, int i) { first = x == m ? min(first, i) : first; });
    token = block_reduce(first, reinterpret_cast<int*>(sh.wave), [](int p, int q) { return min(p, q); });
  } else {
    Cut cut{-M<float>::inf(), 0};
    // bins of 1/32 of a factor of two
    const float scale = (float)fmin(32.0 * weight.c, 3e38);
    if (top_k > 0 && top_k < a.V)
      cut = select(row, cut, m, scale, (u64)top_k, [](float) { return (u64)1; }, sh);
    if (top_p > 0.0 && top_p < 1.0) {
      u64 left = 0;
      row.each([&](float x, int i) { left += cut.keeps(x, i) ? mass(x) : 0; });
      left = block_sum_u64(left, sh.wave);
      cut = select(row, cut, m, scale, (u64)(top_p * (double)left), mass, sh);
    }
    if (min_p > 0.0) {
      const double far = T * log(fmin(min_p, 1.0));
      // the least float at no more than that distance, a step or two from this one
      uint32_t k = key_of((float)((double)m + far));
      for (int n = 0; n < 4 && (double)value_of(k) - (double)m < far; ++n) ++k;
      for (int n = 0; n < 4 && (double)value_of(k - 1) - (double)m >= far; ++n) --k;
      const float least = value_of(k);
      if (least > cut.v) cut = Cut{least, kNoIndex};
    }
    u64 mine = 0;
    row.each([&](float x, int i) { mine += cut.keeps(x, i) ? mass(x) : 0; });
    u64 sum = mine;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    __syncthreads();
    if (lane == 0) sh.wave[wv] = sum;
    if (t == 0) sh.slot = kNoIndex;
    __syncthreads();
    u64 total = 0, before = 0;
    for (int k = 0; k < kCW; ++k) {
      if (k < wv) before += sh.wave[k];
      total += sh.wave[k];
    }
    const double u = (double)a.u[b];
    const u64 border = u > 0.0 ? (u64)(fmin(u, 1.0) * (double)total) : 0;
    int found = kNoIndex;
    if (border == 0) {  // the first entry with any mass, be it less than a unit
      row.each([&](float x, int i) {
        if (cut.keeps(x, i) && ((double)x - (double)m) * weight.c > -1000.0) found = min(found, i);
      });
    } else if (border >= total) {  // a uniform of 1: the last with any
      int last = -1;
      row.each([&](float x, int i) {
        if (cut.keeps(x, i) && mass(x)) last = max(last, i);
      });
      found = block_reduce(last, reinterpret_cast<int*>(sh.wave), [](int p, int q) { return max(p, q); });
    } else if (before <= border && before + sum > border) {  // one wave's
      for (int s = 0; s < a.slabs; ++s) {
        constexpr int EPV = Row<Tag>::EPV;
        const int64_t i = (((int64_t)wv * a.slabs + s) * 64 + lane) * EPV;
        float x[EPV];
#pragma unroll
        for (int k = 0; k < EPV; ++k) x[k] = -M<float>::inf();
        if (i < a.V) load_entries<Tag>(row.p, i, a.V, x);
        u64 w[EPV], here = 0;
#pragma unroll
        for (int k = 0; k < EPV; ++k) {
          w[k] = x[k] != -M<float>::inf() && cut.keeps(x[k], (int)i + k) ? mass(x[k]) : 0;
          here += w[k];
        }
        u64 upto = here;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const u64 y = __shfl_up(upto, o, 64);
          if (lane >= o) upto += y;
        }
        u64 at = before + upto - here;
        if (at <= border && at + here > border) {
#pragma unroll
          for (int k = 0; k < EPV; ++k) {
            at += w[k];
            if (at > border) found = min(found, (int)i + k);
          }
        }
        before += __shfl(upto, 63, 64);
        if (before > border) break;
      }
    }
    token = block_reduce(found, reinterpret_cast<int*>(sh.wave), [](int p, int q) { return min(p, q); });
    logq = log((double)total * unit);
  }
  if (t == 0) {
    const double d = ((double)load_entry<Tag>(row.p, token) - (double)m) / T;
    a.token_out[b] = token;
    a.logp_out[b] = fminf((float)(d - norm), 0.0f);
    if (a.logq_out) a.logq_out[b] = greedy ? 0.0f : fminf((float)(d - logq), 0.0f);
  }
}

template <class Tag>
int launch_choose(ChooseArgs a, int64_t B, hipStream_t st) {
  constexpr int64_t step = (int64_t)kCT * Pack16<Tag>::EPV;
  a.slabs = (int)((a.V + step - 1) / step);
  hipLaunchKernelGGL(choose_kernel<Tag>, dim3((uint32_t)B), dim3(kCT), 0, st, a);
  return check_launch("choose_kernel");
}

}  // namespace
}  // namespace rrl

using namespace rrl;

extern "C" int rrl_sample_tokens(const void* logits, int32_t dtype, int64_t B, int64_t V, int64_t row_stride,
                                 const float* uniforms, const rrl_sample_params* params, int64_t* token_out,
                                 float* logp_out, float* logq_out, void* stream) {
  clear_error();
  RRL_REQUIRE(dtype == RRL_F32 || dtype == RRL_BF16 || dtype == RRL_F16, RRL_EDTYPE,
              "rrl_sample_tokens: logits must be float32, bfloat16 or float16");
  RRL_REQUIRE(B >= 0, RRL_EINVAL, "rrl_sample_tokens: negative size");
  if (B == 0) return RRL_OK;
  RRL_REQUIRE(V >= 1, RRL_EINVAL, "rrl_sample_tokens: logits need at least one vocabulary entry");
  // a grid's threads are counted in 32 bits, and an index with its bins in 31
  RRL_REQUIRE(B < ((int64_t)1 << 22) && V <= ((int64_t)1 << 30), RRL_EINVAL,
              "rrl_sample_tokens: 2^22 rows or more, or rows of over 2^30 entries");
  RRL_REQUIRE(logits != nullptr && uniforms != nullptr && params != nullptr && token_out != nullptr &&
                  logp_out != nullptr,
              RRL_EINVAL, "rrl_sample_tokens: null operand");
  RRL_REQUIRE(B <= 1 || row_stride >= 0, RRL_EINVAL, "rrl_sample_tokens: negative row stride");
  const rrl_sample_params& p = *params;
  RRL_REQUIRE(p.top_ks == nullptr || p.top_k_dtype == RRL_I32 || p.top_k_dtype == RRL_I64, RRL_EDTYPE,
              "rrl_sample_tokens: top_k must be int32 or int64");
  RRL_REQUIRE((uintptr_t)logits % dtype_size(dtype) == 0 && (uintptr_t)uniforms % 4 == 0 &&
                  (uintptr_t)p.temperatures % 4 == 0 && (uintptr_t)p.top_ps % 4 == 0 &&
                  (uintptr_t)p.min_ps % 4 == 0 &&
                  (p.top_ks == nullptr || (uintptr_t)p.top_ks % dtype_size(p.top_k_dtype) == 0),
              RRL_EALIGN, "rrl_sample_tokens: a pointer is not aligned to its element");
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
  a.token_out = token_out;
  a.logp_out = logp_out;
  a.logq_out = logq_out;
  hipStream_t st = as_stream(stream);
  if (dtype == RRL_F32) return launch_choose<TagF32>(a, B, st);
  if (dtype == RRL_BF16) return launch_choose<TagBF16>(a, B, st);
  return launch_choose<TagF16>(a, B, st);
}
