// The token embedding: scaled lookup of weight rows, and its gradient by sorted
// tokens.
//
//   out[i]     = scale * W[id_i]
//   dW[v]      = scale * sum_{i : id_i = v} g[i]       (float32 sums)
//
// A sum's order is decided by the ids alone: i ascending in runs of up to kPiece
// positions, and in longer ones within pieces of kPiece, which are then added up.
//
// A padding id takes a row of zeros and passes no gradient; any other id outside
// [0, V) takes a row of NaN (the host is not waited for) and passes none.
//
// Both are bound by memory: the lookup moves N rows in and out, the gradient
// reads N rows and writes V.  For the gradient the positions are sorted by id
// (stable least-significant-digit radix passes, in one workgroup's LDS while they
// fit), so that each row of dW is written once, zeros included, and no float is
// added by an atomic: equal inputs give equal bits.  A wave takes kRowsWave rows of dW,
// whose positions are neighbours in the sorted order, and streams through them.  Runs
// longer than kPiece positions, which one wave would follow for too long, are left to
// workgroups of their own: the positions are cut at multiples of kPiece, a piece that
// holds one id only is summed into a float32 row, and the run's workgroup adds those.
#include "wave_common.hpp"
#include "rrl_common.hpp"

namespace rrl {
namespace {

// ---- element vectors -----------------------------------------------------------

struct Bf16 {
  typedef uint16_t S;
  static __device__ __forceinline__ float up(uint16_t b) { return bf16_bits_to_f32(b); }
  static __device__ __forceinline__ uint16_t down(float f) { return f32_to_bf16_bits(f); }
};
struct F16 {
  typedef uint16_t S;
  static __device__ __forceinline__ float up(uint16_t b) { return f16_bits_to_f32(b); }
  static __device__ __forceinline__ uint16_t down(float f) { return f32_to_f16_bits(f); }
};
struct F32 {
  typedef float S;
  static __device__ __forceinline__ float up(float b) { return b; }
  static __device__ __forceinline__ float down(float f) { return f; }
};

template <typename S, int VEC>
struct alignas(sizeof(S) * VEC) Pack {
  S e[VEC];
};

// ---- ids -------------------------------------------------------------------------

struct Ids {
  const void* ptr;
  int dt;
  int64_t V, padding;
  int has_padding;
};
constexpr int64_t kIsPad = -1, kIsBad = -2;

// The row an id names, or kIsPad / kIsBad.
__device__ __forceinline__ int64_t id_row(const Ids& ids, int64_t i) {
  const int64_t v = load_index(ids.ptr, ids.dt, i);
  if (ids.has_padding && v == ids.padding) return kIsPad;
  return v >= 0 && v < ids.V ? v : kIsBad;
}

// ---- lookup ----------------------------------------------------------------------

constexpr int kThreads = 256;

// lpr lanes along a row, kThreads / lpr rows at a time, kFwdRows of each lane's in flight.
template <typename T, int VEC, int kFwdRows>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(Ids ids, int64_t N,
                                                             const typename T::S* __restrict__ w,
                                                             int64_t w_ld, int64_t H, float scale,
                                                             typename T::S* __restrict__ out,
                                                             int lpr) {
  typedef Pack<typename T::S, VEC> P;
  const int64_t rows = kThreads / lpr;
  for (int64_t i0 = blockIdx.x * rows * kFwdRows + threadIdx.x / lpr; i0 < N;
       i0 += gridDim.x * rows * kFwdRows) {
    int64_t v[kFwdRows];
#pragma unroll
    for (int r = 0; r < kFwdRows; ++r) v[r] = i0 + r * rows < N ? id_row(ids, i0 + r * rows) : kIsBad;
    for (int64_t c = (int64_t)(threadIdx.x % lpr) * VEC; c < H; c += (int64_t)lpr * VEC) {
      P x[kFwdRows];
#pragma unroll
      for (int r = 0; r < kFwdRows; ++r)
        if (v[r] >= 0) x[r] = *reinterpret_cast<const P*>(w + v[r] * w_ld + c);
#pragma unroll
      for (int r = 0; r < kFwdRows; ++r) {
        if (i0 + r * rows >= N) break;
        P o;
        const typename T::S f = T::down(v[r] == kIsPad ? 0.0f : __builtin_nanf(""));
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.e[k] = v[r] >= 0 ? T::down(T::up(x[r].e[k]) * scale) : f;
        *reinterpret_cast<P*>(out + (i0 + r * rows) * H + c) = o;
      }
    }
  }
}

// ---- the positions sorted by id ----------------------------------------------------

constexpr int kMaxDigit = 9;  // bits of one pass
constexpr int kBins = 1 << kMaxDigit;

struct SortShape {
  int passes, digit;  // digit bits of each pass
  int blocks;
  int64_t per;        // positions per block
};

// Key of position i: from the ids (first pass) or the last pass's order.
__device__ __forceinline__ uint32_t sort_key(const Ids& ids, const uint32_t* keys, int64_t i) {
  if (keys) return keys[i];
  const int64_t v = id_row(ids, i);
  return (uint32_t)(v >= 0 ? v : ids.V);
}

// Lanes of equal digit (all lanes that are `on`).
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int digit, bool on) {
  uint64_t same = __ballot(on);
  for (int b = 0; b < digit; ++b) {
    const uint64_t one = __ballot((d >> b) & 1);
    same &= ((d >> b) & 1) ? one : ~one;
  }
  return same;
}

// One pass over the ROUNDS x 64 keys that each wave of a workgroup holds, in order:
// at[r] becomes the place of lane's key r.  base: the place of the workgroup's first
// key of bin threadIdx.x (first kBins threads), advanced past its last.  Stable: the
// waves own consecutive stretches, and a wave goes through its own in order, lanes of
// equal digit ranked by lane.
template <int WAVES, int ROUNDS>
__device__ __forceinline__ void places(const uint32_t (&key)[ROUNDS], int count, int shift,
                                       uint32_t mask, int digit, uint32_t& base,
                                       uint32_t (&place)[WAVES][kBins], uint32_t (&at)[ROUNDS]) {
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  for (int k = t; k < WAVES * kBins; k += 64 * WAVES) (&place[0][0])[k] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (r * 64 + lane < count) atomicAdd(&place[wv][(key[r] >> shift) & mask], 1u);
  __syncthreads();
  if (t < kBins) {
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      const uint32_t c = place[k][t];
      place[k][t] = base;
      base += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    if (r * 64 >= count) break;
    const bool on = r * 64 + lane < count;
    const uint32_t d = (key[r] >> shift) & mask;
    const uint64_t same = same_digit(d, digit, on);
    const uint32_t rank = __popcll(same & (((uint64_t)1 << lane) - 1));
    at[r] = on ? place[wv][d] + rank : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (on && rank == 0) place[wv][d] += (uint32_t)__popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// Exclusive running sum over the first kBins threads of a workgroup.
__device__ __forceinline__ uint32_t bins_before(uint32_t v, uint32_t* sh) {
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  uint32_t incl = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 63 && t < kBins) sh[wv] = incl;
  __syncthreads();
  uint32_t before = incl - v;
  for (int k = 0; k < wv && k < kBins / 64; ++k) before += sh[k];
  return before;
}

// Few positions: every pass in one workgroup (4,097 of them, two passes: 17 us).
constexpr int kSmallWaves = 16, kSmallRounds = 8, kSmall = 64 * kSmallWaves * kSmallRounds;

__global__ __launch_bounds__(64 * kSmallWaves) void sort_small_kernel(Ids ids, int N, int passes,
                                                                      int digit,
                                                                      uint32_t* __restrict__ keys_out,
                                                                      uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t place[kSmallWaves][kBins];
  __shared__ uint32_t keys[kSmall], pos[kSmall], total[kBins], sh[kBins / 64];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  // a wave's stretch: as many rounds as all waves need
  const int rounds = (N + 64 * kSmallWaves - 1) / (64 * kSmallWaves), first = wv * rounds * 64;
  const int count = max(0, min(N - first, rounds * 64));
  const uint32_t mask = ((uint32_t)1 << digit) - 1;
  uint32_t key[kSmallRounds], p[kSmallRounds], at[kSmallRounds];
#pragma unroll
  for (int r = 0; r < kSmallRounds; ++r) {
    const int i = r * 64 + lane;
    p[r] = first + i;
    key[r] = i < count ? sort_key(ids, nullptr, first + i) : 0;
  }
  for (int pass = 0; pass < passes; ++pass) {
    if (t < kBins) total[t] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r)
      if (r * 64 + lane < count) atomicAdd(&total[(key[r] >> (pass * digit)) & mask], 1u);
    __syncthreads();
    uint32_t base = bins_before(t < kBins ? total[t] : 0, sh);
    places<kSmallWaves, kSmallRounds>(key, count, pass * digit, mask, digit, base, place, at);
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r)
      if (r * 64 + lane < count) {
        keys[at[r]] = key[r];
        pos[at[r]] = p[r];
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r)
      if (r * 64 + lane < count) {
        key[r] = keys[first + r * 64 + lane];
        p[r] = pos[first + r * 64 + lane];
      }
  }
#pragma unroll
  for (int r = 0; r < kSmallRounds; ++r)
    if (r * 64 + lane < count) {
      keys_out[first + r * 64 + lane] = key[r];
      pos_out[first + r * 64 + lane] = p[r];
    }
}

// More: a count, a scan and a scatter per pass (262,144 positions: 5 + 5 + 7 us).
constexpr int kSortThreads = 512;  // a thread per bin
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kRounds = 2;         // positions per lane in a tile
constexpr int kTile = kSortThreads * kRounds;
constexpr int kMaxBlocks = 512;
static_assert(kBins == kSortThreads, "a thread per bin");

inline SortShape sort_shape(int64_t N, int64_t V) {
  SortShape s;
  int bits = 1;
  while (((int64_t)1 << bits) < V + 1) ++bits;  // ids 0..V-1, and V: no row
  s.passes = (bits + kMaxDigit - 1) / kMaxDigit;
  s.digit = (bits + s.passes - 1) / s.passes;
  const int64_t tiles = (N + kTile - 1) / kTile;
  const int64_t per_block = (tiles + kMaxBlocks - 1) / kMaxBlocks;
  s.per = per_block * kTile;
  s.blocks = (int)((N + s.per - 1) / s.per);
  return s;
}

// hist[bin, block]
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(Ids ids,
                                                                  const uint32_t* __restrict__ keys,
                                                                  int64_t N, int64_t per, int shift,
                                                                  uint32_t mask,
                                                                  uint32_t* __restrict__ hist) {
  __shared__ uint32_t cnt[kBins];
  cnt[threadIdx.x] = 0;
  __syncthreads();
  const int64_t lo = blockIdx.x * per, hi = min(N, lo + per);
  for (int64_t i = lo + threadIdx.x; i < hi; i += kSortThreads)
    atomicAdd(&cnt[(sort_key(ids, keys, i) >> shift) & mask], 1u);
  __syncthreads();
  hist[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = cnt[threadIdx.x];
}

// A wave per bin: hist becomes each block's offset within the bin, total its sum.
__global__ __launch_bounds__(256) void sort_scan_kernel(uint32_t* __restrict__ hist, int blocks,
                                                        uint32_t* __restrict__ total) {
  const int lane = threadIdx.x & 63, bin = blockIdx.x * 4 + (threadIdx.x >> 6);
  uint32_t* row = hist + (int64_t)bin * blocks;
  constexpr int kEach = kMaxBlocks / 64;
  uint32_t h[kEach], sum = 0;
#pragma unroll
  for (int k = 0; k < kEach; ++k) h[k] = lane * kEach + k < blocks ? row[lane * kEach + k] : 0;
#pragma unroll
  for (int k = 0; k < kEach; ++k) sum += h[k];
  uint32_t incl = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  uint32_t at = incl - sum;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    if (lane * kEach + k < blocks) row[lane * kEach + k] = at;
    at += h[k];
  }
  if (lane == 63) total[bin] = incl;
}

// Moves a block's positions to their places.
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(
    Ids ids, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, int64_t N,
    int64_t per, int shift, uint32_t mask, int digit, const uint32_t* __restrict__ hist,
    const uint32_t* __restrict__ total, uint32_t* __restrict__ keys_out,
    uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t place[kSortWaves][kBins];
  __shared__ uint32_t sh[kBins / 64];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  const uint32_t within = hist[(int64_t)t * gridDim.x + blockIdx.x];
  uint32_t base = bins_before(total[t], sh) + within;
  const int64_t lo = blockIdx.x * per, hi = min(N, lo + per);
  for (int64_t tile = lo; tile < hi; tile += kTile) {
    const int64_t first = tile + (int64_t)wv * 64 * kRounds;
    const int count = (int)max((int64_t)0, min((int64_t)64 * kRounds, hi - first));
    uint32_t key[kRounds], p[kRounds], at[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int64_t i = first + r * 64 + lane;
      const bool on = r * 64 + lane < count;
      key[r] = on ? sort_key(ids, keys, i) : 0;
      p[r] = on && pos ? pos[i] : (uint32_t)i;
    }
    places<kSortWaves, kRounds>(key, count, shift, mask, digit, base, place, at);
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      if (r * 64 + lane < count) {
        keys_out[at[r]] = key[r];
        pos_out[at[r]] = p[r];
      }
    __syncthreads();
  }
}

// ---- gradient rows -----------------------------------------------------------------

constexpr int kPiece = 64;

// Adds rows g[pos[lo..hi)] in order, U packs of VEC elements per lane.
template <typename T, int VEC, int U>
__device__ __forceinline__ void add_rows(float (&acc)[U][VEC], const typename T::S* __restrict__ g,
                                         int64_t g_ld, const uint32_t* __restrict__ pos, int64_t lo,
                                         int64_t hi, int64_t c0, int64_t H) {
  typedef Pack<typename T::S, VEC> P;
  const int lane = threadIdx.x & 63;
  constexpr int kAhead = 8 / U;  // rows in flight
  for (int64_t b = lo; b < hi; b += 64) {
    const int n = (int)min((int64_t)64, hi - b);
    const uint32_t mine = lane < n ? pos[b + lane] : 0;
    for (int r = 0; r < n; r += kAhead) {
      P x[kAhead][U];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const uint32_t p = __builtin_amdgcn_readlane(mine, min(r + a, n - 1));
        const typename T::S* row = g + (int64_t)p * g_ld;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t c = c0 + (int64_t)(u * 64 + lane) * VEC;
          if (r + a < n && c < H) x[a][u] = *reinterpret_cast<const P*>(row + c);
        }
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        if (r + a < n) {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[u][k] += T::up(x[a][u].e[k]);
        }
    }
  }
}

// Piece blockIdx.x: its bounds of runs, and its sum where it holds one id only (a wave
// per chunk of columns).  Bound by reads of rows in no order: 79 us for about 125,000
// rows of 2 KB (3.2 TB/s).
template <typename T, int VEC, int U>
__global__ __launch_bounds__(64) void embed_piece_kernel(const uint32_t* __restrict__ keys,
                                                         const uint32_t* __restrict__ pos, int64_t N,
                                                         uint32_t V,
                                                         const typename T::S* __restrict__ g,
                                                         int64_t g_ld, int64_t H,
                                                         uint32_t* __restrict__ begin,
                                                         uint32_t* __restrict__ end,
                                                         float* __restrict__ partial) {
  const int lane = threadIdx.x;
  const int64_t i = (int64_t)blockIdx.x * kPiece + lane;
  const uint32_t k = i < N ? keys[i] : V;
  if (blockIdx.y == 0 && k < V) {
    if (i == 0 || keys[i - 1] != k) begin[k] = (uint32_t)i;
    if (i == N - 1 || keys[i + 1] != k) end[k] = (uint32_t)(i + 1);
  }
  const int64_t lo = (int64_t)blockIdx.x * kPiece;
  if (lo + kPiece > N) return;
  const uint32_t k0 = __builtin_amdgcn_readlane(k, 0), k1 = __builtin_amdgcn_readlane(k, 63);
  if (k0 != k1 || k0 >= V) return;
  const int64_t c0 = (int64_t)blockIdx.y * (64 * VEC * U);
  float acc[U][VEC] = {};
  add_rows<T, VEC, U>(acc, g, g_ld, pos, lo, lo + kPiece, c0, H);
  float* dst = partial + blockIdx.x * H;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t c = c0 + (int64_t)(u * 64 + lane) * VEC;
    if (c < H) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) dst[c + j] = acc[u][j];
    }
  }
}

template <typename T, int VEC, int U>
__device__ __forceinline__ void write_row(const float (&acc)[U][VEC], float scale,
                                          typename T::S* dst, int64_t c0, int64_t H) {
  typedef Pack<typename T::S, VEC> P;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t c = c0 + (int64_t)(u * 64 + (threadIdx.x & 63)) * VEC;
    if (c < H) {
      P o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.e[k] = T::down(acc[u][k] * scale);
      *reinterpret_cast<P*>(dst + c) = o;
    }
  }
}

constexpr int kRowWaves = 4, kRowsWave = 8;

// 151,936 rows of 1024 bfloat16 with about 110,000 positions take 188 us with the long
// runs beside them: 227 MB of rows in no order, and 311 MB of dW.
// A wave per (kRowsWave rows of dW, chunk of columns): zeros, and the runs of up to
// kPiece positions.  begin[v] is read before it is known to have been written: the key
// at its place tells (keys[begin[v]] == v only if v occurs, and then both bounds were
// written by this call).
template <typename T, int VEC, int U>
__device__ __forceinline__ void embed_rows(
    int64_t block, int chunk, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, int64_t N, int64_t V,
    const typename T::S* __restrict__ g, int64_t g_ld, int64_t H, float scale,
    const uint32_t* __restrict__ begin, const uint32_t* __restrict__ end,
    typename T::S* __restrict__ dw, int64_t dw_ld) {
  typedef Pack<typename T::S, VEC> P;
  const int lane = threadIdx.x & 63;
  const int64_t v0 = (block * kRowWaves + (threadIdx.x >> 6)) * kRowsWave;
  if (v0 >= V) return;
  const int64_t c0 = (int64_t)chunk * (64 * VEC * U);
  const int rows = (int)min((int64_t)kRowsWave, V - v0);
  // lane r: row r's run (an empty one where it does not occur)
  uint32_t b = 0, e = 0;
  if (lane < rows) {
    const uint32_t s = begin[v0 + lane];
    if (s < N && keys[s] == (uint32_t)(v0 + lane)) {
      b = s;
      e = end[v0 + lane];
    }
  }
  const bool longer = e - b > kPiece;
  const uint32_t occurs = (uint32_t)__ballot(e > b), skip = (uint32_t)__ballot(longer);
  float acc[U][VEC] = {};
  int cur = 0;  // the row that acc belongs to; rows before it are written
  auto finish = [&](int upto) {
    for (; cur < upto; ++cur) {
      if ((skip >> cur) & 1) continue;
      write_row<T, VEC, U>(acc, scale, dw + (v0 + cur) * dw_ld, c0, H);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[u][k] = 0.0f;
    }
  };
  // stretches of neighbouring positions: between runs that are skipped
  int r = 0;
  while (r < rows) {
    const uint32_t ahead = skip >> r;
    const int r1 = ahead ? r + __ffs(ahead) - 1 : rows;
    const uint32_t in = occurs & (((uint32_t)1 << r1) - 1) & ~(((uint32_t)1 << r) - 1);
    if (in) {
      const uint32_t lo = __builtin_amdgcn_readlane(b, __ffs(in) - 1);
      const uint32_t hi = __builtin_amdgcn_readlane(e, 31 - __clz(in));
      for (uint32_t w = lo; w < hi; w += 64) {
        const int n = (int)min(64u, hi - w);
        const uint32_t p = lane < n ? pos[w + lane] : 0;
        const uint32_t k = lane < n ? keys[w + lane] - (uint32_t)v0 : 0;
        constexpr int kAhead = 8 / U;  // positions in flight
        for (int i = 0; i < n; i += kAhead) {
          P x[kAhead][U];
#pragma unroll
          for (int a = 0; a < kAhead; ++a) {
            const typename T::S* row = g + (int64_t)__builtin_amdgcn_readlane(p, min(i + a, n - 1)) * g_ld;
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int64_t c = c0 + (int64_t)(u * 64 + lane) * VEC;
              if (c < H) x[a][u] = *reinterpret_cast<const P*>(row + c);
            }
          }
#pragma unroll
          for (int a = 0; a < kAhead; ++a)
            if (i + a < n) {
              finish((int)__builtin_amdgcn_readlane(k, i + a));
#pragma unroll
              for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[u][j] += T::up(x[a][u].e[j]);
            }
        }
      }
    }
    finish(min(r1 + 1, rows));
    r = r1 + 1;
  }
}

constexpr int kLongWaves = kRowWaves;

// Piece p, chunk of columns: the run of more than kPiece positions that begins in
// piece p, if there is one (there is at most one).  The waves take the run's pieces, and the
// positions before the first and behind the last, in turn; their sums are added in the
// waves' order.
template <typename T, int VEC, int U>
__device__ __forceinline__ void embed_long(
    int64_t piece, int chunk, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, int64_t N, uint32_t V,
    const typename T::S* __restrict__ g, int64_t g_ld, int64_t H, float scale,
    const uint32_t* __restrict__ begin, const uint32_t* __restrict__ end,
    const float* __restrict__ partial, typename T::S* __restrict__ dw, int64_t dw_ld) {
  __shared__ float sums[kLongWaves][64 * VEC];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int64_t c0 = (int64_t)chunk * (64 * VEC * U);
  const int64_t lo = piece * kPiece;
  if (lo + kPiece >= N) return;  // a run that begins in the last piece is no longer
  const uint32_t v = keys[lo + kPiece - 1];
  if (v >= V || keys[lo + kPiece] != v) return;
  const int64_t s = begin[v], e = end[v];
  if (s < lo || e - s <= kPiece) return;
  const int64_t p0 = (s + kPiece - 1) / kPiece, p1 = e / kPiece;
  float acc[U][VEC] = {};
  constexpr int kAhead = 8 / U;  // sums in flight
  for (int64_t p = p0 + wv; p < p1; p += kLongWaves * kAhead) {
    float x[kAhead][U][VEC] = {};
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t c = c0 + (int64_t)(u * 64 + lane) * VEC;
        if (p + a * kLongWaves < p1 && c < H) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) x[a][u][k] = partial[(p + a * kLongWaves) * H + c + k];
        }
      }
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[u][k] += x[a][u][k];
  }
  // the positions outside whole pieces, fewer than 2 kPiece: a stretch per wave
  const int64_t head = p0 < p1 ? p0 * kPiece - s : e - s, tail = p0 < p1 ? e - p1 * kPiece : 0;
  const int64_t each = (head + tail + kLongWaves - 1) / kLongWaves;
  const int64_t f0 = min(wv * each, head + tail), f1 = min(f0 + each, head + tail);
  if (f0 < head) add_rows<T, VEC, U>(acc, g, g_ld, pos, s + f0, s + min(f1, head), c0, H);
  if (f1 > head)
    add_rows<T, VEC, U>(acc, g, g_ld, pos, p1 * kPiece + max(f0, head) - head,
                        p1 * kPiece + f1 - head, c0, H);
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) sums[wv][k * 64 + lane] = acc[u][k];
    __syncthreads();
    if (wv == 0) {
      float one[1][VEC] = {};
      for (int x = 0; x < kLongWaves; ++x)
#pragma unroll
        for (int k = 0; k < VEC; ++k) one[0][k] += sums[x][k * 64 + lane];
      write_row<T, VEC, 1>(one, scale, dw + (int64_t)v * dw_ld, c0 + (int64_t)u * 64 * VEC, H);
    }
    __syncthreads();
  }
}

// Both, neither waiting for the other: the long runs first, then the rows.
template <typename T, int VEC, int U>
__global__ __launch_bounds__(64 * kRowWaves) void embed_grad_kernel(
    uint32_t pieces, uint32_t narrow, uint32_t chunks, const uint32_t* __restrict__ keys,
    const uint32_t* __restrict__ pos, int64_t N, int64_t V, const typename T::S* __restrict__ g,
    int64_t g_ld, int64_t H, float scale, const uint32_t* __restrict__ begin,
    const uint32_t* __restrict__ end, const float* __restrict__ partial,
    typename T::S* __restrict__ dw, int64_t dw_ld) {
  uint32_t id = blockIdx.x;
  if (id < pieces * narrow) {
    embed_long<T, VEC, 1>(id / narrow, id % narrow, keys, pos, N, (uint32_t)V, g, g_ld, H, scale, begin,
                          end, partial, dw, dw_ld);
  } else {
    id -= pieces * narrow;
    embed_rows<T, VEC, U>(id / chunks, id % chunks, keys, pos, N, V, g, g_ld, H, scale, begin, end, dw,
                          dw_ld);
  }
}

// ---- host ---------------------------------------------------------------------------

// Bytes of the widest access that every row start of `p` (rows ld elements
// apart) allows, for rows of H elements.
inline int access_bytes(const void* p, int64_t ld, int64_t H, size_t size) {
  for (int b = 16; b > (int)size; b >>= 1)
    if ((uintptr_t)p % b == 0 && (ld * size) % b == 0 && (H * size) % b == 0) return b;
  return (int)size;
}

struct BwdLayout {
  size_t keys[2], pos[2], hist, begin, end, partial, total;
};
inline BwdLayout bwd_layout(int64_t N, int64_t V, int64_t H) {
  BwdLayout l;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  for (int k = 0; k < 2; ++k) l.keys[k] = take(4 * (size_t)N);
  for (int k = 0; k < 2; ++k) l.pos[k] = take(4 * (size_t)N);
  l.hist = take(4 * (size_t)(kMaxBlocks + 1) * kBins);
  l.begin = take(4 * (size_t)V);
  l.end = take(4 * (size_t)V);
  l.partial = take(4 * (size_t)(N / kPiece) * (size_t)H);
  l.total = at;
  return l;
}

template <typename T, int VEC>
int launch_fwd(const Ids& ids, int64_t N, const void* w, int64_t w_ld, int64_t H, float scale,
               void* out, hipStream_t st) {
  const int64_t packs = (H + VEC - 1) / VEC;
  int lpr = 1;
  while (lpr < kThreads && lpr < packs) lpr <<= 1;
  const int64_t rows = kThreads / lpr;
  const typename T::S* src = static_cast<const typename T::S*>(w);
  typename T::S* dst = static_cast<typename T::S*>(out);
  // Four rows in flight where there are enough to fill the chip with them, one for a
  // decode step's few (320 rows of 2 KB: the kernel takes 2.8 against 4.1 us).  Calls of one
  // / four took, in us: 1024 bfloat16 (the border is at 16,384 rows): 8,192 rows 7.2 / 7.6,
  // 16,640 11.1 / 11.5, 24,576 14.7 / 14.8, 65,536 44.1 / 43.3, 262,144 208 / 197; 770
  // float32 (8,192 rows): 2,048 4.2 / 4.4, 8,192 10.8 / 9.4, 16,384 17.7 / 14.8, 65,536
  // 93.4 / 71.5.  A grid's threads are counted in 32 bits: past 2^22 workgroups they take
  // rows in turn.
  const int64_t groups = (N + rows - 1) / rows;
  if (groups <= 8192) {
    hipLaunchKernelGGL((embed_fwd_kernel<T, VEC, 1>), dim3((uint32_t)groups), dim3(kThreads), 0, st, ids,
                       N, src, w_ld, H, scale, dst, lpr);
  } else {
    hipLaunchKernelGGL((embed_fwd_kernel<T, VEC, 4>),
                       dim3((uint32_t)min((groups + 3) / 4, (int64_t)1 << 22)), dim3(kThreads), 0, st,
                       ids, N, src, w_ld, H, scale, dst, lpr);
  }
  return check_launch("embed_fwd_kernel");
}

// Elements of an access of `bytes` bytes: 16-bit types have 16-byte, 4-byte and single
// accesses only.
inline int access_elements(int bytes, size_t size) {
  if (size == 4) return bytes / 4;
  return bytes == 16 ? 8 : (bytes >= 4 ? 2 : 1);
}

// The gradient's grids with accesses of `vec` elements.
struct GradGrid {
  int u;                          // accesses of a lane along a row
  int64_t narrow, chunks;         // columns' shares for long runs (64 x vec elements), and for rows (u times that)
  int64_t pieces, rows, blocks;   // of kPiece positions, of a workgroup's rows of dW, and of embed_grad_kernel
};
inline GradGrid grad_grid(int64_t N, int64_t V, int64_t H, int vec) {
  GradGrid g;
  g.narrow = (H + 64 * vec - 1) / (64 * vec);
  g.u = g.narrow <= 1 ? 1 : 2;
  g.chunks = (g.narrow + g.u - 1) / g.u;
  // no run is longer than kPiece where the positions end with the first piece
  g.pieces = N / kPiece;
  g.rows = (V + kRowWaves * kRowsWave - 1) / (kRowWaves * kRowsWave);
  g.blocks = g.pieces * g.narrow + g.rows * g.chunks;
  return g;
}
// A grid's threads are counted in 32 bits.  (`narrow`, a second dimension, is at most the
// 2^16 that one may have: rows are shorter than 2^22.)
inline bool grad_fits(const GradGrid& g) { return g.blocks < ((int64_t)1 << 32) / (64 * kRowWaves); }

template <typename T, int VEC, int U>
int launch_rows(const BwdLayout& l, char* ws, int last, int64_t N, int64_t V, const void* g,
                int64_t g_ld, int64_t H, float scale, void* dw, int64_t dw_ld, const GradGrid& grid,
                hipStream_t st) {
  typedef typename T::S S;
  const uint32_t* keys = reinterpret_cast<uint32_t*>(ws + l.keys[last]);
  const uint32_t* pos = reinterpret_cast<uint32_t*>(ws + l.pos[last]);
  uint32_t* begin = reinterpret_cast<uint32_t*>(ws + l.begin);
  uint32_t* end = reinterpret_cast<uint32_t*>(ws + l.end);
  float* partial = reinterpret_cast<float*>(ws + l.partial);
  const uint32_t narrow = (uint32_t)grid.narrow;
  if (N > 0) {
    hipLaunchKernelGGL((embed_piece_kernel<T, VEC, 1>), dim3((uint32_t)((N + kPiece - 1) / kPiece), narrow),
                       dim3(64), 0, st, keys, pos, N, (uint32_t)V, static_cast<const S*>(g), g_ld, H,
                       begin, end, partial);
    if (int rc = check_launch("embed_piece_kernel")) return rc;
  }
  hipLaunchKernelGGL((embed_grad_kernel<T, VEC, U>), dim3((uint32_t)grid.blocks), dim3(64 * kRowWaves), 0, st,
                     (uint32_t)grid.pieces, narrow, (uint32_t)grid.chunks, keys, pos, N, V,
                     static_cast<const S*>(g), g_ld, H, scale, begin, end, partial, static_cast<S*>(dw), dw_ld);
  return check_launch("embed_grad_kernel");
}

template <typename T, int VEC>
int launch_rows_u(const BwdLayout& l, char* ws, int last, int64_t N, int64_t V, const void* g,
                  int64_t g_ld, int64_t H, float scale, void* dw, int64_t dw_ld, const GradGrid& grid,
                  hipStream_t st) {
  if (grid.u == 1)
    return launch_rows<T, VEC, 1>(l, ws, last, N, V, g, g_ld, H, scale, dw, dw_ld, grid, st);
  return launch_rows<T, VEC, 2>(l, ws, last, N, V, g, g_ld, H, scale, dw, dw_ld, grid, st);
}

int check_common(const char* what, int64_t N, int64_t V, int64_t H, int32_t ids_dtype,
                 int32_t dtype, double scale) {
  const std::string w(what);
  RRL_REQUIRE(dtype == RRL_F32 || dtype == RRL_BF16 || dtype == RRL_F16, RRL_EDTYPE,
              w + ": the weight must be float32, bfloat16 or float16");
  RRL_REQUIRE(ids_dtype == RRL_I32 || ids_dtype == RRL_I64, RRL_EDTYPE,
              w + ": ids must be int32 or int64");
  RRL_REQUIRE(N >= 0 && V >= 0 && H >= 0, RRL_EINVAL, w + ": negative size");
  // (its infinity would make NaN of zeros, and of the rows of dW that no id names)
  RRL_REQUIRE(!isinf((float)scale) || isinf(scale), RRL_EINVAL, w + ": the scale is past float32's range");
  // the gradient's grids (16 threads a position, 64 a row) are 32-bit
  RRL_REQUIRE(N < ((int64_t)1 << 28) && V < ((int64_t)1 << 26) && H < ((int64_t)1 << 22), RRL_EINVAL,
              w + ": at most 2^28 - 1 ids, and 2^26 - 1 rows of 2^22 - 1 elements");
  return RRL_OK;
}

}  // namespace
}  // namespace rrl

using namespace rrl;

extern "C" int rrl_embedding_fwd(const void* ids, int32_t ids_dtype, int64_t N, const void* weight,
                                 int32_t dtype, int64_t V, int64_t H, int64_t w_ld, double scale,
                                 int64_t padding_idx, int32_t has_padding, void* out, void* stream) {
  clear_error();
  if (int rc = check_common("rrl_embedding_fwd", N, V, H, ids_dtype, dtype, scale)) return rc;
  if (N == 0 || H == 0) return RRL_OK;
  RRL_REQUIRE(ids != nullptr && (weight != nullptr || V == 0) && out != nullptr, RRL_EINVAL,
              "rrl_embedding_fwd: null operand");
  RRL_REQUIRE(V <= 1 || w_ld >= H, RRL_EINVAL, "rrl_embedding_fwd: the row stride is shorter than a row");
  const size_t size = dtype_size(dtype);
  RRL_REQUIRE((uintptr_t)weight % size == 0 && (uintptr_t)out % size == 0 &&
                  (uintptr_t)ids % dtype_size(ids_dtype) == 0,
              RRL_EALIGN, "rrl_embedding_fwd: a pointer is not aligned to its element");
  const Ids d{ids, ids_dtype, V, padding_idx, has_padding};
  const int b = min(access_bytes(weight, w_ld, H, size), access_bytes(out, H, H, size));
  const float s = (float)scale;
  hipStream_t st = as_stream(stream);
  const int vec = access_elements(b, size);
#define RRL_FWD(T, VEC) return launch_fwd<T, VEC>(d, N, weight, w_ld, H, s, out, st)
  if (dtype == RRL_F32) {
    if (vec == 4) RRL_FWD(F32, 4);
    if (vec == 2) RRL_FWD(F32, 2);
    RRL_FWD(F32, 1);
  }
  if (dtype == RRL_BF16) {
    if (vec == 8) RRL_FWD(Bf16, 8);
    if (vec == 2) RRL_FWD(Bf16, 2);
    RRL_FWD(Bf16, 1);
  }
  if (vec == 8) RRL_FWD(F16, 8);
  if (vec == 2) RRL_FWD(F16, 2);
  RRL_FWD(F16, 1);
#undef RRL_FWD
}

extern "C" size_t rrl_embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t H) {
  if (N < 0 || V < 0 || H < 0) return 0;
  return bwd_layout(N, V, H).total;
}

extern "C" int rrl_embedding_bwd(const void* ids, int32_t ids_dtype, int64_t N, const void* grad,
                                 int32_t dtype, int64_t V, int64_t H, int64_t g_ld, double scale,
                                 int64_t padding_idx, int32_t has_padding, void* dweight,
                                 int64_t dw_ld, void* workspace, void* stream) {
  clear_error();
  if (int rc = check_common("rrl_embedding_bwd", N, V, H, ids_dtype, dtype, scale)) return rc;
  if (V == 0 || H == 0) return RRL_OK;
  RRL_REQUIRE((N == 0 || (ids != nullptr && grad != nullptr)) && dweight != nullptr &&
                  workspace != nullptr,
              RRL_EINVAL, "rrl_embedding_bwd: null operand");
  RRL_REQUIRE((N <= 1 || g_ld >= H) && (V <= 1 || dw_ld >= H), RRL_EINVAL,
              "rrl_embedding_bwd: a row stride is shorter than a row");
  const size_t size = dtype_size(dtype);
  RRL_REQUIRE((uintptr_t)grad % size == 0 && (uintptr_t)dweight % size == 0 &&
                  (uintptr_t)ids % dtype_size(ids_dtype) == 0 && (uintptr_t)workspace % 16 == 0,
              RRL_EALIGN, "rrl_embedding_bwd: a pointer is not aligned to its element");
  const int b = min(access_bytes(grad, g_ld, H, size), access_bytes(dweight, dw_ld, H, size));
  const int vec = access_elements(b, size);
  const GradGrid grid = grad_grid(N, V, H, vec);
  RRL_REQUIRE(grad_fits(grid), RRL_EINVAL, "rrl_embedding_bwd: too many ids or rows for their length");
  hipStream_t st = as_stream(stream);
  const Ids d{ids, ids_dtype, V, padding_idx, has_padding};
  const BwdLayout l = bwd_layout(N, V, H);
  char* ws = static_cast<char*>(workspace);
  int last = 0;
  if (N > 0) {
    const SortShape s = sort_shape(N, V);
    const uint32_t mask = ((uint32_t)1 << s.digit) - 1;
    uint32_t* hist = reinterpret_cast<uint32_t*>(ws + l.hist);
    uint32_t* total = hist + (size_t)kMaxBlocks * kBins;
    if (N <= kSmall) {
      hipLaunchKernelGGL(sort_small_kernel, dim3(1), dim3(64 * kSmallWaves), 0, st, d, (int)N, s.passes,
                         s.digit, reinterpret_cast<uint32_t*>(ws + l.keys[0]),
                         reinterpret_cast<uint32_t*>(ws + l.pos[0]));
      if (int rc = check_launch("sort_small_kernel")) return rc;
    }
    for (int p = 0; p < s.passes && N > kSmall; ++p) {
      const uint32_t* kin = p ? reinterpret_cast<uint32_t*>(ws + l.keys[last]) : nullptr;
      const uint32_t* pin = p ? reinterpret_cast<uint32_t*>(ws + l.pos[last]) : nullptr;
      const int to = p & 1;
      hipLaunchKernelGGL(sort_count_kernel, dim3(s.blocks), dim3(kSortThreads), 0, st, d, kin, N,
                         s.per, p * s.digit, mask, hist);
      if (int rc = check_launch("sort_count_kernel")) return rc;
      hipLaunchKernelGGL(sort_scan_kernel, dim3(kBins / 4), dim3(256), 0, st, hist, s.blocks, total);
      if (int rc = check_launch("sort_scan_kernel")) return rc;
      hipLaunchKernelGGL(sort_scatter_kernel, dim3(s.blocks), dim3(kSortThreads), 0, st, d, kin, pin,
                         N, s.per, p * s.digit, mask, s.digit, hist, total,
                         reinterpret_cast<uint32_t*>(ws + l.keys[to]),
                         reinterpret_cast<uint32_t*>(ws + l.pos[to]));
      if (int rc = check_launch("sort_scatter_kernel")) return rc;
      last = to;
    }
  }
  const float sc = (float)scale;
#define RRL_BWD(T, VEC) \
  return launch_rows_u<T, VEC>(l, ws, last, N, V, grad, g_ld, H, sc, dweight, dw_ld, grid, st)
  if (dtype == RRL_F32) {
    if (vec == 4) RRL_BWD(F32, 4);
    if (vec == 2) RRL_BWD(F32, 2);
    RRL_BWD(F32, 1);
  }
  if (dtype == RRL_BF16) {
    if (vec == 8) RRL_BWD(Bf16, 8);
    if (vec == 2) RRL_BWD(Bf16, 2);
    RRL_BWD(Bf16, 1);
  }
  if (vec == 8) RRL_BWD(F16, 8);
  if (vec == 2) RRL_BWD(F16, 2);
  RRL_BWD(F16, 1);
#undef RRL_BWD
}
