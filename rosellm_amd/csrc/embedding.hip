// The token embedding: scaled lookup of weight rows, and its gradient by sorted
// tokens.
//
//   out[i]     = scale * W[id_i]
//   dW[v]      = scale * sum_{i : id_i = v} g[i]       (float32 sums, i ascending)
//
// A padding id takes a row of zeros and passes no gradient; any other id outside
// [0, V) takes a row of NaN (the host is not waited for) and passes none.
//
// Both are bound by memory: the lookup moves N rows in and out, the gradient
// reads N rows and writes V.  For the gradient the positions are sorted by id
// (stable least-significant-digit radix passes), so that each row of dW is
// written once, by one wave, zeros included, and no float is added by an atomic:
// equal inputs give equal bits.  The runs of frequent ids, which one wave would
// follow for too long, are cut at multiples of kPiece sorted positions; a piece
// that holds one id only is summed by waves of its own into a float32 row that
// the id's wave then adds in place of its positions.
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

// kThreads / LPR rows per workgroup, LPR lanes along a row.
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(Ids ids, int64_t N,
                                                             const typename T::S* __restrict__ w,
                                                             int64_t w_ld, int64_t H, float scale,
                                                             typename T::S* __restrict__ out,
                                                             int lpr) {
  typedef Pack<typename T::S, VEC> P;
  const int64_t rows = kThreads / lpr;
  for (int64_t i = blockIdx.x * rows + threadIdx.x / lpr; i < N; i += gridDim.x * rows) {
    const int64_t v = id_row(ids, i);
    typename T::S* dst = out + i * H;
    for (int64_t c = (int64_t)(threadIdx.x % lpr) * VEC; c < H; c += (int64_t)lpr * VEC) {
      P o;
      if (v >= 0) {
        const P x = *reinterpret_cast<const P*>(w + v * w_ld + c);
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.e[k] = T::down(T::up(x.e[k]) * scale);
      } else {
        const typename T::S f = T::down(v == kIsPad ? 0.0f : __builtin_nanf(""));
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.e[k] = f;
      }
      *reinterpret_cast<P*>(dst + c) = o;
    }
  }
}

// ---- the positions sorted by id ----------------------------------------------------

constexpr int kMaxDigit = 9;               // bits of one pass
constexpr int kBins = 1 << kMaxDigit;
constexpr int kSortThreads = 512;          // a thread per bin
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kRounds = 8;                 // positions per lane in a tile
constexpr int kTile = kSortThreads * kRounds;
constexpr int kMaxBlocks = 128;
static_assert(kBins == kSortThreads, "a thread per bin");

struct SortShape {
  int passes, digit;   // digit bits of each pass
  int blocks;
  int64_t per;         // positions per block
};

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

// Key of position i: from the ids (first pass) or the last pass's order.
__device__ __forceinline__ uint32_t sort_key(const Ids& ids, const uint32_t* keys, int64_t i) {
  if (keys) return keys[i];
  const int64_t v = id_row(ids, i);
  return (uint32_t)(v >= 0 ? v : ids.V);
}

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
  hist[(int64_t)blockIdx.x * kBins + threadIdx.x] = cnt[threadIdx.x];
}

// Moves this block's positions to their places.  Stable: within a tile the
// waves own consecutive stretches, and a wave goes through its own in order,
// lanes of equal digit ranked by lane.
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(
    Ids ids, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, int64_t N,
    int64_t per, int shift, uint32_t mask, int digit, const uint32_t* __restrict__ hist,
    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t place[kSortWaves][kBins];
  __shared__ uint32_t wave_total[kSortWaves];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  // where this block's first position of bin t goes
  uint32_t before = 0, total = 0;
  for (int b = 0; b < (int)gridDim.x; ++b) {
    const uint32_t h = hist[(int64_t)b * kBins + t];
    before += b < (int)blockIdx.x ? h : 0;
    total += h;
  }
  uint32_t incl = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  if (lane == 63) wave_total[wv] = incl;
  __syncthreads();
  uint32_t base = incl - total + before;
  for (int k = 0; k < wv; ++k) base += wave_total[k];

  const int64_t lo = blockIdx.x * per, hi = min(N, lo + per);
  for (int64_t tile = lo; tile < hi; tile += kTile) {
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k) place[k][t] = 0;
    __syncthreads();
    uint32_t key[kRounds];
    const int64_t first = tile + (int64_t)wv * 64 * kRounds + lane;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int64_t i = first + r * 64;
      key[r] = i < hi ? sort_key(ids, keys, i) : 0;
      if (i < hi) atomicAdd(&place[wv][(key[r] >> shift) & mask], 1u);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k) {
      const uint32_t c = place[k][t];
      place[k][t] = base;
      base += c;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int64_t i = first + r * 64;
      const bool on = i < hi;
      const uint32_t d = (key[r] >> shift) & mask;
      uint64_t same = __ballot(on);
      for (int b = 0; b < digit; ++b) {
        const uint64_t one = __ballot((d >> b) & 1);
        same &= ((d >> b) & 1) ? one : ~one;
      }
      const uint32_t rank = __popcll(same & (((uint64_t)1 << lane) - 1));
      uint32_t at = 0;
      if (on) at = place[wv][d];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (on && rank == 0) place[wv][d] = at + (uint32_t)__popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (on) {
        keys_out[at + rank] = key[r];
        pos_out[at + rank] = pos ? pos[i] : (uint32_t)i;
      }
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
  constexpr int kAhead = 4;  // rows in flight
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

// Workgroup (p, chunk): piece p's bounds of runs (chunk 0), and its sum where the
// piece holds one id only.
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

constexpr int kRowWaves = 4;

// A wave per (row of dW, chunk of columns).  begin[v] is read before it is known
// to have been written: the key at its place tells (keys[begin[v]] == v only if
// v occurs, and then both bounds were written by this call).
template <typename T, int VEC, int U>
__global__ __launch_bounds__(64 * kRowWaves) void embed_rows_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, int64_t N, int64_t V,
    const typename T::S* __restrict__ g, int64_t g_ld, int64_t H, float scale,
    const uint32_t* __restrict__ begin, const uint32_t* __restrict__ end,
    const float* __restrict__ partial, typename T::S* __restrict__ dw, int64_t dw_ld) {
  typedef Pack<typename T::S, VEC> P;
  const int lane = threadIdx.x & 63;
  const int64_t v = (int64_t)blockIdx.x * kRowWaves + (threadIdx.x >> 6);
  if (v >= V) return;
  const int64_t c0 = (int64_t)blockIdx.y * (64 * VEC * U);
  float acc[U][VEC] = {};
  const int64_t s = begin[v];
  if (s < N && keys[s] == (uint32_t)v) {
    const int64_t e = end[v];
    const int64_t p0 = (s + kPiece - 1) / kPiece, p1 = e / kPiece;
    if (p0 < p1) {  // whole pieces [p0, p1) within the run
      add_rows<T, VEC, U>(acc, g, g_ld, pos, s, p0 * kPiece, c0, H);
      for (int64_t p = p0; p < p1; ++p) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t c = c0 + (int64_t)(u * 64 + lane) * VEC;
          if (c < H) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[u][k] += partial[p * H + c + k];
          }
        }
      }
      add_rows<T, VEC, U>(acc, g, g_ld, pos, p1 * kPiece, e, c0, H);
    } else {
      add_rows<T, VEC, U>(acc, g, g_ld, pos, s, e, c0, H);
    }
  }
  typename T::S* dst = dw + v * dw_ld;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t c = c0 + (int64_t)(u * 64 + lane) * VEC;
    if (c < H) {
      P o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.e[k] = T::down(acc[u][k] * scale);
      *reinterpret_cast<P*>(dst + c) = o;
    }
  }
}

// ---- host ---------------------------------------------------------------------------

// Bytes of the widest access that every row start of `p` (rows ld elements
// apart) allows, for rows of H elements.
inline int access_bytes(const void* p, int64_t ld, int64_t H, size_t size) {
  for (int b = 16; b > (int)size; b >>= 2)
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
  l.hist = take(4 * (size_t)kMaxBlocks * kBins);
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
  // a grid's threads are counted in 32 bits: past 2^22 workgroups they take rows in turn
  const int64_t blocks = min((N + rows - 1) / rows, (int64_t)1 << 22);
  hipLaunchKernelGGL((embed_fwd_kernel<T, VEC>), dim3((uint32_t)blocks), dim3(kThreads), 0, st, ids,
                     N, static_cast<const typename T::S*>(w), w_ld, H, scale,
                     static_cast<typename T::S*>(out), lpr);
  return check_launch("embed_fwd_kernel");
}

template <typename T, int VEC, int U>
int launch_rows(const BwdLayout& l, char* ws, int last, int64_t N, int64_t V, const void* g,
                int64_t g_ld, int64_t H, float scale, void* dw, int64_t dw_ld, hipStream_t st) {
  typedef typename T::S S;
  const uint32_t* keys = reinterpret_cast<uint32_t*>(ws + l.keys[last]);
  const uint32_t* pos = reinterpret_cast<uint32_t*>(ws + l.pos[last]);
  uint32_t* begin = reinterpret_cast<uint32_t*>(ws + l.begin);
  uint32_t* end = reinterpret_cast<uint32_t*>(ws + l.end);
  float* partial = reinterpret_cast<float*>(ws + l.partial);
  const int64_t chunk = 64 * VEC * U;
  const uint32_t chunks = (uint32_t)((H + chunk - 1) / chunk);
  if (N > 0) {
    hipLaunchKernelGGL((embed_piece_kernel<T, VEC, U>), dim3((uint32_t)((N + kPiece - 1) / kPiece), chunks),
                       dim3(64), 0, st, keys, pos, N, (uint32_t)V, static_cast<const S*>(g), g_ld, H,
                       begin, end, partial);
    if (int rc = check_launch("embed_piece_kernel")) return rc;
  }
  hipLaunchKernelGGL((embed_rows_kernel<T, VEC, U>),
                     dim3((uint32_t)((V + kRowWaves - 1) / kRowWaves), chunks), dim3(64 * kRowWaves), 0,
                     st, keys, pos, N, V, static_cast<const S*>(g), g_ld, H, scale, begin, end, partial,
                     static_cast<S*>(dw), dw_ld);
  return check_launch("embed_rows_kernel");
}

template <typename T, int VEC>
int launch_rows_u(const BwdLayout& l, char* ws, int last, int64_t N, int64_t V, const void* g,
                  int64_t g_ld, int64_t H, float scale, void* dw, int64_t dw_ld, hipStream_t st) {
  const int64_t packs = (H + 64 * VEC - 1) / (64 * VEC);
  if (packs <= 1) return launch_rows<T, VEC, 1>(l, ws, last, N, V, g, g_ld, H, scale, dw, dw_ld, st);
  return launch_rows<T, VEC, 2>(l, ws, last, N, V, g, g_ld, H, scale, dw, dw_ld, st);
}

int check_common(const char* what, int64_t N, int64_t V, int64_t H, int32_t ids_dtype,
                 int32_t dtype) {
  const std::string w(what);
  RRL_REQUIRE(dtype == RRL_F32 || dtype == RRL_BF16 || dtype == RRL_F16, RRL_EDTYPE,
              w + ": the weight must be float32, bfloat16 or float16");
  RRL_REQUIRE(ids_dtype == RRL_I32 || ids_dtype == RRL_I64, RRL_EDTYPE,
              w + ": ids must be int32 or int64");
  RRL_REQUIRE(N >= 0 && V >= 0 && H >= 0, RRL_EINVAL, w + ": negative size");
  // sorted positions and the gradient's grid (64 threads a row) are 32-bit
  RRL_REQUIRE(N < ((int64_t)1 << 31) && V < ((int64_t)1 << 26) && H < ((int64_t)1 << 22), RRL_EINVAL,
              w + ": at most 2^31 - 1 ids, and 2^26 - 1 rows of 2^22 - 1 elements");
  return RRL_OK;
}

}  // namespace
}  // namespace rrl

using namespace rrl;

extern "C" int rrl_embedding_fwd(const void* ids, int32_t ids_dtype, int64_t N, const void* weight,
                                 int32_t dtype, int64_t V, int64_t H, int64_t w_ld, double scale,
                                 int64_t padding_idx, int32_t has_padding, void* out, void* stream) {
  clear_error();
  if (int rc = check_common("rrl_embedding_fwd", N, V, H, ids_dtype, dtype)) return rc;
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
#define RRL_FWD(T, VEC) return launch_fwd<T, VEC>(d, N, weight, w_ld, H, s, out, st)
  if (dtype == RRL_F32) {
    if (b == 16) RRL_FWD(F32, 4);
    RRL_FWD(F32, 1);
  }
  if (dtype == RRL_BF16) {
    if (b == 16) RRL_FWD(Bf16, 8);
    if (b == 4) RRL_FWD(Bf16, 2);
    RRL_FWD(Bf16, 1);
  }
  if (b == 16) RRL_FWD(F16, 8);
  if (b == 4) RRL_FWD(F16, 2);
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
  if (int rc = check_common("rrl_embedding_bwd", N, V, H, ids_dtype, dtype)) return rc;
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
  hipStream_t st = as_stream(stream);
  const Ids d{ids, ids_dtype, V, padding_idx, has_padding};
  const BwdLayout l = bwd_layout(N, V, H);
  char* ws = static_cast<char*>(workspace);
  int last = 0;
  if (N > 0) {
    const SortShape s = sort_shape(N, V);
    const uint32_t mask = ((uint32_t)1 << s.digit) - 1;
    uint32_t* hist = reinterpret_cast<uint32_t*>(ws + l.hist);
    for (int p = 0; p < s.passes; ++p) {
      const uint32_t* kin = p ? reinterpret_cast<uint32_t*>(ws + l.keys[last]) : nullptr;
      const uint32_t* pin = p ? reinterpret_cast<uint32_t*>(ws + l.pos[last]) : nullptr;
      const int to = p & 1;
      hipLaunchKernelGGL(sort_count_kernel, dim3(s.blocks), dim3(kSortThreads), 0, st, d, kin, N,
                         s.per, p * s.digit, mask, hist);
      if (int rc = check_launch("sort_count_kernel")) return rc;
      hipLaunchKernelGGL(sort_scatter_kernel, dim3(s.blocks), dim3(kSortThreads), 0, st, d, kin, pin,
                         N, s.per, p * s.digit, mask, s.digit, hist,
                         reinterpret_cast<uint32_t*>(ws + l.keys[to]),
                         reinterpret_cast<uint32_t*>(ws + l.pos[to]));
      if (int rc = check_launch("sort_scatter_kernel")) return rc;
      last = to;
    }
  }
  const int b = min(access_bytes(grad, g_ld, H, size), access_bytes(dweight, dw_ld, H, size));
  const float sc = (float)scale;
#define RRL_BWD(T, VEC) return launch_rows_u<T, VEC>(l, ws, last, N, V, grad, g_ld, H, sc, dweight, dw_ld, st)
  if (dtype == RRL_F32) {
    if (b == 16) RRL_BWD(F32, 4);
    RRL_BWD(F32, 1);
  }
  if (dtype == RRL_BF16) {
    if (b == 16) RRL_BWD(Bf16, 8);
    if (b == 4) RRL_BWD(Bf16, 2);
    RRL_BWD(Bf16, 1);
  }
  if (b == 16) RRL_BWD(F16, 8);
  if (b == 4) RRL_BWD(F16, 2);
  RRL_BWD(F16, 1);
#undef RRL_BWD
}
