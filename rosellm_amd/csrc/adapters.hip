// Low-rank updates of many requests' adapters beside a shared projection, and their
// gradients.
//
//   y_n = base_n + scale_a up_a t_n,   t_n = down_a drop(x_n),   a = id_n
//   s_n = up_a^T g_n
//   dx_n = scale_a drop'(down_a^T s_n)
//   d down_a = scale_a sum_n s_n drop(x_n)^T,   d up_a = scale_a sum_n g_n t_n^T
//
// down_a [r, H] and up_a [O, r] are thin (r up to 128), so that all of this is bound by
// reading and writing the rows of N tokens: 2 r operations an entry.
//
// Rows of one adapter stand together only within a request, so a workgroup takes a
// window of 1024 tokens, sorts it by adapter in LDS (a counting sort; a window of one
// adapter needs none), and its tiles of 16 or 64 rows are of one adapter each, whatever
// the order of the ids: no other launch, no list kept between calls.
//
//   adapter_fused   few rows: t of 16 rows, the depth H split over four waves, and its product
//                   with a run of rows of up while it is there (64 rows of 16 adapters, 1024
//                   to 2048, rank 16: 9.7 us, a chain of four dependent loads)
//   adapter_shrink  t of many rows (131,072 x 1024 bfloat16: 57 us, 4.7 TB/s; with dropout 67,
//                   of which the generator's issue is 51)
//   adapter_expand  base + scale up t (131,072 x 2048 bfloat16: 246 us, 4.4 TB/s; a copy of
//                   that size reaches 4.7; dx, written only, 56 us, 4.8 TB/s)
//   adapter_outer   the factors' gradients over runs of tokens (g and x of the above: 148 us,
//                   5.4 TB/s; with dropout 173), adapter_join adds the runs (9 us)
// d x is adapter_shrink and adapter_expand on g with the transposes of up and down, which
// adapter_turn lays out.
//
// t is float32, and stays it: the second product's bfloat16 instruction takes it as the
// exact sum of three bfloat16 numbers of eight bits each.  With float16 operands, whose
// range t can leave, up is taken as the exact sum of two as well.  float32 operands take
// the float32 instruction.  An infinity times a part that is zero is NaN, which is what
// such a sum may become instead of infinite.  (With two parts of t, which hold 2^-17, both
// directions of 32,768 rows of 4 adapters, 1024 to 2048, took 287 us instead of 292 at rank 16
// and 455 instead of 486 at rank 64; float16 without the product of the low parts 322 instead
// of 331, and 498 instead of 555.)
#include "dropout_common.hpp"
#include "vocab_weights.hpp"

#include <type_traits>

namespace rrl {
namespace {

constexpr int kAT = 256, kAW = kAT / 64;  // a workgroup's threads and waves
constexpr int kWindow = 1024;             // tokens that a workgroup sorts
constexpr int kMostAdapters = 4096, kMostRank = 128;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mma_bf16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}

// Keeps the two arms of a choice between kinds of access from becoming one.
__device__ __forceinline__ void apart() { asm volatile("" ::: "memory"); }

// 16 bytes at any element's address.
typedef uint32_t AnyVec __attribute__((ext_vector_type(4), aligned(2)));

// The first n of 16 bytes' entries, zeros behind them; and their store.
template <class Tag>
__device__ __forceinline__ u32x4 load_part(const char* from, int64_t n) {
  constexpr int EPV = Pack16<Tag>::EPV;
  float x[EPV];
#pragma unroll
  for (int k = 0; k < EPV; ++k) x[k] = k < n ? load_entry<Tag>(from, k) : 0.0f;
  return Pack16<Tag>::pack(x);
}
template <class Tag>
__device__ __forceinline__ void store_part(char* to, const u32x4& v, int64_t n) {
  constexpr int EPV = Pack16<Tag>::EPV;
  float x[EPV];
  Pack16<Tag>::unpack(v, x);
#pragma unroll
  for (int k = 0; k < EPV; ++k)
    if (k < n) {
      if constexpr (EPV == 4) reinterpret_cast<float*>(to)[k] = x[k];
      else reinterpret_cast<uint16_t*>(to)[k] = (uint16_t)Pack16<Tag>::pack_one(x[k]);
    }
}

// Zeros where an entry's bit is not set.
template <class Tag>
__device__ __forceinline__ void keep_entries(u32x4& v, uint32_t bits) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    if constexpr (Pack16<Tag>::EPV == 4) {
      v[d] = bits >> d & 1 ? v[d] : 0u;
    } else {
      const uint32_t two = bits >> (2 * d) & 3;
      v[d] &= (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
    }
  }
}

// Eight consecutive entries as they stand in memory.
template <class Tag>
struct Frag {
  static constexpr int EPV = Pack16<Tag>::EPV, NV = 8 / EPV, SZ = 16 / EPV;
  u32x4 v[NV];
  // entries i..i+7 of a row that may start at any element, zeros from n on (WHOLE: there are
  // eight)
  template <bool WHOLE = false>
  __device__ __forceinline__ void load(const char* row, int64_t i, int64_t n) {
    if (WHOLE || i + 8 <= n) {
#pragma unroll
      for (int h = 0; h < NV; ++h) v[h] = reinterpret_cast<const AnyVec*>(row + i * SZ)[h];
      return;
    }
#pragma unroll
    for (int h = 0; h < NV; ++h) v[h] = load_part<Tag>(row + (i + h * EPV) * SZ, n - i - h * EPV);
  }
  // the same within the row, past the caches
  __device__ __forceinline__ void stream(const char* row, int64_t i) {
#pragma unroll
    for (int h = 0; h < NV; ++h) v[h] = __builtin_nontemporal_load(reinterpret_cast<const AnyVec*>(row + i * SZ) + h);
  }
  __device__ __forceinline__ void pack(const float (&x)[8]) {
#pragma unroll
    for (int h = 0; h < NV; ++h) {
      float part[EPV];
#pragma unroll
      for (int k = 0; k < EPV; ++k) part[k] = x[h * EPV + k];
      v[h] = Pack16<Tag>::pack(part);
    }
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
#pragma unroll
    for (int h = 0; h < NV; ++h) {
      float part[EPV];
      Pack16<Tag>::unpack(v[h], part);
#pragma unroll
      for (int k = 0; k < EPV; ++k) x[h * EPV + k] = part[k];
    }
  }
  __device__ __forceinline__ void store(char* row, int64_t i, int64_t n) const {
    if (i + 8 <= n) {
#pragma unroll
      for (int h = 0; h < NV; ++h) reinterpret_cast<AnyVec*>(row + i * SZ)[h] = v[h];
      return;
    }
#pragma unroll
    for (int h = 0; h < NV; ++h) store_part<Tag>(row + (i + h * EPV) * SZ, v[h], n - i - h * EPV);
  }
  // zeros where an entry is dropped
  __device__ __forceinline__ void keep(uint32_t bits) {
#pragma unroll
    for (int h = 0; h < NV; ++h) keep_entries<Tag>(v[h], bits >> (EPV * h));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int h = 0; h < NV; ++h) v[h] = u32x4{0, 0, 0, 0};
  }
};

// c += a b^T over the 32 entries of depth that the four groups of 16 lanes hold, eight
// each: rows of the result 4 (lane / 16) + i from a's lanes, columns lane % 16 from b's.
template <class Tag>
__device__ __forceinline__ f32x4 mma(const Frag<Tag>& a, const Frag<Tag>& b, f32x4 c) {
  if constexpr (std::is_same_v<Tag, TagBF16>) {
    return mma_bf16(a.v[0], b.v[0], c);
  } else if constexpr (std::is_same_v<Tag, TagF16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v[0]),
                                                  __builtin_bit_cast(f16x8, b.v[0]), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.v[k / 4][k % 4]), __uint_as_float(b.v[k / 4][k % 4]),
                                               c, 0, 0, 0);
    return c;
  }
}

// The upper halves of two numbers, cut off: bfloat16 numbers of their first eight bits, and
// what is left of them.  (Rounded, the largest would overflow.  An infinity leaves no rest.)
__device__ __forceinline__ uint32_t cut2(float& a, float& b) {
  const uint32_t bits = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  const float ha = __uint_as_float(bits << 16), hb = __uint_as_float(bits & 0xffff0000u);
  a = a == ha ? 0.0f : a - ha;
  b = b == hb ? 0.0f : b - hb;
  return bits;
}
// Eight numbers as exact sums of bfloat16 numbers: of N, which hold 8 N bits.
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], u32x4 (&part)[N]) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    float a = x[2 * d], b = x[2 * d + 1];
#pragma unroll
    for (int k = 0; k < N; ++k) part[k][d] = cut2(a, b);
  }
}

// The second product: rows of up against t, depth R = 16 R16.  16-bit operands take 32
// entries of depth at once: ranks up to 16 hold t's first parts in the first half of them
// and its second parts in the second, beside up's entries twice; then its last parts,
// beside both parts of a float16 up.
template <class Tag, int R16>
struct Thin {  // t of 16 tokens
  static constexpr bool F32 = std::is_same_v<Tag, TagF32>, F16 = std::is_same_v<Tag, TagF16>;
  static constexpr int KS = R16 == 1 ? 1 : R16 / 2;
  static constexpr int NF = F32 ? 4 * R16 : 0;
  u32x4 part[F32 ? 1 : KS][3];
  float f[F32 ? NF : 1];
  __device__ __forceinline__ void load(const float* t, int kb) {
    if constexpr (F32) {
#pragma unroll
      for (int k = 0; k < NF; ++k) f[k] = t[NF * kb + k];
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int at = R16 == 1 ? 8 * (kb & 1) : 32 * s + 8 * kb;
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = t[at + k];
        split8(x, part[s]);
        if constexpr (R16 == 1) {
          const u32x4 none = {0, 0, 0, 0};
          part[0][0] = kb < 2 ? part[0][0] : part[0][1];
          if constexpr (!F16) part[0][2] = kb < 2 ? part[0][2] : none;
        }
      }
    }
  }
};
template <class Tag, int R16>
struct UpRow {  // a lane's row of up; WHOLE: r is 16 R16
  using T = Thin<Tag, R16>;
  Frag<Tag> v[T::F32 ? (T::NF + 7) / 8 : T::KS];
  template <bool WHOLE = false>
  __device__ __forceinline__ void load(const char* row, int r, int kb) {
    if constexpr (T::F32) {
      if constexpr (T::NF >= 8) {
#pragma unroll
        for (int s = 0; s < T::NF / 8; ++s) v[s].template load<WHOLE>(row, T::NF * kb + 8 * s, r);
      } else if constexpr (WHOLE) {
        v[0].v[0] = reinterpret_cast<const AnyVec*>(row)[kb];
      } else {
        // four entries to a lane
        v[0].clear();
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (4 * kb + k < r) v[0].v[0][k] = reinterpret_cast<const uint32_t*>(row)[4 * kb + k];
      }
    } else {
#pragma unroll
      for (int s = 0; s < T::KS; ++s) v[s].template load<WHOLE>(row, R16 == 1 ? 8 * (kb & 1) : 32 * s + 8 * kb, r);
    }
  }
};
template <class Tag, int R16>
__device__ __forceinline__ f32x4 expand(const UpRow<Tag, R16>& u, const Thin<Tag, R16>& t, f32x4 c) {
  using T = Thin<Tag, R16>;
  if constexpr (T::F32) {
#pragma unroll
    for (int k = 0; k < T::NF; ++k)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(u.v[k / 8].v[k / 4 % 2][k % 4]), t.f[k], c, 0, 0, 0);
  } else {
#pragma unroll
    for (int s = 0; s < T::KS; ++s) {
      if constexpr (T::F16) {
        float x[8];
        u32x4 up[2];
        u.v[s].unpack(x);
        split8(x, up);
        c = mma_bf16(up[0], t.part[s][0], c);
        c = mma_bf16(up[1], t.part[s][0], c);
        if constexpr (R16 > 1) {
#pragma unroll
          for (int k = 1; k < 3; ++k) {
            c = mma_bf16(up[0], t.part[s][k], c);
            c = mma_bf16(up[1], t.part[s][k], c);
          }
        } else {
          c = mma_bf16((threadIdx.x & 63) < 32 ? up[0] : up[1], t.part[s][2], c);
        }
      } else {
        c = mma_bf16(u.v[s].v[0], t.part[s][0], c);
        if constexpr (R16 > 1) c = mma_bf16(u.v[s].v[0], t.part[s][1], c);
        c = mma_bf16(u.v[s].v[0], t.part[s][2], c);
      }
    }
  }
  return c;
}

struct AdapterIds {
  const void* ids;  // null: adapter 0 everywhere
  int dt, A;
  // the adapter, A for none (a negative id), or A + 1 for an id that there is none of
  __device__ __forceinline__ int at(int64_t n) const {
    if (!ids) return 0;
    const int64_t id = load_index(ids, dt, n);
    return id < 0 ? A : (id < A ? (int)id : A + 1);
  }
};

struct FusedArgs {
  const char *x, *down, *up, *base;  // base may be null
  int64_t x_ld, d_sa, d_sr, u_sa, u_so, b_ld;
  AdapterIds ids;
  const float* scales;  // null: 1
  char* out;            // contiguous [N, O]; null: t alone
  float* t;             // [N, 16 R16]
  int64_t N, K, O;
  int r;
  int groups;           // workgroups of a window
  int in_turn;          // 0: a window's workgroups are neighbours, else the windows, which take turns
  int slabs;            // runs of up's rows that a tile's work is cut into
  int64_t slab;         // their length
  Drop drop;
  int drop_in, drop_out;
  int nan_rows;         // rows of ids that there are none of: NaN, or zeros
  int stream_x, stream_out;  // x, and base and out, are larger than the memory-side cache
};

// The window that a workgroup belongs to, and which of the window's it is.  Windows that take
// turns start each turn one further, so that they do not stay on an XCD.
__device__ __forceinline__ int group_of(const FusedArgs& a) {
  return (int)(a.in_turn ? blockIdx.x / a.in_turn : blockIdx.x % a.groups);
}
__device__ __forceinline__ int64_t window_of(const FusedArgs& a) {
  return a.in_turn ? (blockIdx.x + blockIdx.x / a.in_turn) % a.in_turn : blockIdx.x / a.groups;
}

// The row of up that lane q holds of the i-th of tiles of 16 from column c on: pairs of
// tiles in an order that leaves eight consecutive columns to a lane of the result.
__device__ __forceinline__ int64_t up_row(int64_t c, int i, int q, int64_t O) {
  return min(c + 16 * (i & ~1) + 8 * (q >> 2) + 4 * (i & 1) + (q & 3), O - 1);
}

// A wave's exchange through LDS that is its own: the order of its accesses stays as written.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The rows of a window of 1024 tokens by adapter, in order, as tiles of up to TM rows of
// one: every workgroup of a window comes to the same tiles.  The whole workgroup takes part.
template <int TM>
struct Window {
  struct Tile {
    int ad, row0, here;  // ad: A for rows without an adapter, A + 1 for ids that there are none of
  };
  int64_t n0;
  int count, first, A2;
  bool one;  // one adapter's
  const uint16_t* order;
  const int *start, *tiles;
  int all;  // tiles

  static size_t lds(int A) { return (2 * sizeof(int) + kAW * sizeof(uint16_t)) * (size_t)(A + 3); }

  __device__ __forceinline__ Window(const FusedArgs& a, uint16_t* order_, int* scan, int* bins) {
    constexpr int kChunks = kWindow / kAT;
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    n0 = window_of(a) * kWindow;
    count = (int)min((int64_t)kWindow, a.N - n0);
    A2 = a.ids.A + 2;
    int* const start_ = bins;                // first place of each adapter, of none and bad, and the end
    int* const tiles_ = start_ + A2 + 1;     // first tile
    uint16_t* const seen = reinterpret_cast<uint16_t*>(tiles_ + A2 + 1);  // rows of each by wave
    order = order_;
    start = start_;
    tiles = tiles_;
    // a wave looks at a quarter of the rows
    int code[kChunks];
    bool same = true;
    const int i0 = wv * (kWindow / kAW) + lane;
    first = a.ids.at(n0);
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      code[k] = i0 + 64 * k < count ? a.ids.at(n0 + i0 + 64 * k) : first;
      same &= code[k] == first;
    }
    one = __syncthreads_and(same);
    all = (count + TM - 1) / TM;
    if (one) return;
    for (int k = t; k < kAW * A2; k += kAT) seen[k] = 0;
    __syncthreads();
    int rank[kChunks];  // among the wave's rows of the same adapter
    volatile uint16_t* const mine = seen + wv * A2;
    const int bits = 32 - __clz(A2);
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const bool in = i0 + 64 * k < count;
      uint64_t like = __ballot(in);
      for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot(code[k] >> b & 1);
        like &= code[k] >> b & 1 ? set : ~set;
      }
      rank[k] = 0;
      if (in) {
        rank[k] = mine[code[k]] + __popcll(like & (((uint64_t)1 << lane) - 1));
        if (lane == 63 - __clzll((long long)like)) mine[code[k]] = (uint16_t)(rank[k] + 1);
      }
    }
    __syncthreads();
    // exclusive sums of rows and tiles, a run of bins to a thread
    const int per = (A2 + kAT - 1) / kAT, lo = min(t * per, A2), hi = min(lo + per, A2);
    int rows = 0, tls = 0;
    for (int k = lo; k < hi; ++k) {
      int c = 0;
      for (int w = 0; w < kAW; ++w) c += seen[w * A2 + k];
      start_[k] = c;
      rows += c;
      tls += (c + TM - 1) / TM;
    }
    int rsum = rows, tsum = tls;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(rsum, o, 64), z = __shfl_up(tsum, o, 64);
      if (lane >= o) {
        rsum += y;
        tsum += z;
      }
    }
    if (lane == 63) {
      scan[wv] = rsum;
      scan[kAW + wv] = tsum;
    }
    __syncthreads();
    rsum -= rows;
    tsum -= tls;
    for (int k = 0; k < wv; ++k) {
      rsum += scan[k];
      tsum += scan[kAW + k];
    }
    for (int k = lo; k < hi; ++k) {
      const int c = start_[k];
      start_[k] = rsum;
      tiles_[k] = tsum;
      rsum += c;
      tsum += (c + TM - 1) / TM;
    }
    if (hi == A2 && lo < hi) {  // the thread of the last bin
      start_[A2] = rsum;
      tiles_[A2] = tsum;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kChunks; ++k)
      if (i0 + 64 * k < count) {
        int at = start_[code[k]] + rank[k];
        for (int w = 0; w < wv; ++w) at += seen[w * A2 + code[k]];
        order_[at] = (uint16_t)(i0 + 64 * k);
      }
    __syncthreads();
    all = tiles_[A2];
  }
  __device__ __forceinline__ Tile tile(int k) const {
    if (one) return Tile{first, k * TM, min(TM, count - k * TM)};
    // the last bin that starts at or before the tile and is not empty
    int lo = 0, hi = A2;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (tiles[mid] <= k) lo = mid;
      else hi = mid;
    }
    const int row0 = start[lo] + (k - tiles[lo]) * TM;
    return Tile{lo, row0, min(TM, start[lo + 1] - row0)};
  }
  // the i-th row of a tile, from the window's first; past its end the last again
  __device__ __forceinline__ int row(const Tile& k, int i) const {
    const int at = k.row0 + min(i, k.here - 1);
    return one ? at : (int)order[at];
  }
  __device__ __forceinline__ int64_t token(const Tile& k, int i) const { return n0 + row(k, i); }
};

// Columns c0..c1-1 of rows without an adapter.
template <class Tag, int TM>
__device__ __forceinline__ void plain_rows(const FusedArgs& a, const Window<TM>& w,
                                           const typename Window<TM>::Tile& tile, int64_t c0, int64_t c1) {
  constexpr int SZ = Frag<Tag>::SZ;
  const int per = (int)((c1 - c0 + 7) / 8);
  for (int64_t k = threadIdx.x; k < (int64_t)tile.here * per; k += kAT) {
    const int64_t n = w.token(tile, (int)(k / per)), c = c0 + k % per * 8;
    Frag<Tag> v;
    v.clear();
    if (tile.ad == a.ids.A) {
      if (a.base) v.load(a.base + n * a.b_ld * SZ, c, c1);
    } else if (a.nan_rows) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = M<float>::nan();
      v.pack(x);
    }
    v.store(a.out + n * a.O * SZ, c, c1);
  }
}

// Eight consecutive columns of a row: the product, scaled and dropped or added to base's.
template <class Tag>
__device__ __forceinline__ void finish(const FusedArgs& a, const f32x4& d0, const f32x4& d1, int64_t n, int64_t col,
                                       float scale, uint64_t at, Frag<Tag>& b) {
  float v[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = d0[k];
    v[4 + k] = d1[k];
  }
  if (a.drop_out) {
    const uint32_t keep = a.drop.keep_bits((uint64_t)(n * ((a.O + 7) / 8) + col / 8), at);
    const float s = scale * a.drop.scale;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = keep >> k & 1 ? v[k] * s : 0.0f;
  } else if (a.base) {
    float x[8];
    b.unpack(x);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __builtin_fmaf(v[k], scale, x[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= scale;
  }
  b.pack(v);
}

// Few rows, in tiles of 16: t with the depth split over the four waves, and (where out is
// not null) its product with a run of up's rows, 64 to a wave at a time.
template <class Tag, int R16>
__global__ __launch_bounds__(kAT) void adapter_fused_kernel(FusedArgs a) {
  constexpr int SZ = Frag<Tag>::SZ, R = 16 * R16, kAhead = 4, NC = 4;
  __shared__ uint16_t order[kWindow];
  __shared__ __attribute__((aligned(16))) float part[kAW][16][R + 4];
  __shared__ int scan[2 * kAW];
  extern __shared__ int bins[];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, kb = lane >> 4, q = lane & 15;
  const Window<16> w(a, order, scan, bins);
  const uint64_t at = a.drop_in || a.drop_out ? a.drop.counter() : 0;
  for (int64_t it = group_of(a); it < (int64_t)w.all * a.slabs; it += a.groups) {
    const Window<16>::Tile tile = w.tile((int)(it / a.slabs));
    const int slab = (int)(it % a.slabs);
    const int64_t c0 = slab * a.slab, c1 = min(c0 + a.slab, a.O);
    if (tile.ad >= a.ids.A) {
      if (a.out) plain_rows<Tag, 16>(a, w, tile, c0, c1);
      continue;
    }
    const int64_t n = w.token(tile, q);
    const char* xrow = a.x + n * a.x_ld * SZ;
    const char* down = a.down + tile.ad * a.d_sa * SZ;
    const int64_t steps = (a.K + 31) / 32, per_row = (a.K + 7) / 8;
    const int64_t s0 = steps * wv / kAW, s1 = steps * (wv + 1) / kAW;
    f32x4 acc[R16] = {};
    for (int64_t s = s0; s < s1; s += kAhead) {
      Frag<Tag> xf[kAhead], df[kAhead][R16];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        // past the wave's steps: zeros
        const int64_t k = s + e < s1 ? (s + e) * 32 + kb * 8 : a.K;
        xf[e].load(xrow, k, a.K);
#pragma unroll
        for (int j = 0; j < R16; ++j) {
          const int rr = 16 * j + q;
          df[e][j].load(down + min(rr, a.r - 1) * a.d_sr * SZ, rr < a.r ? k : a.K, a.K);
        }
      }
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        if (a.drop_in && s + e < s1) xf[e].keep(a.drop.keep_bits((uint64_t)(n * per_row + (s + e) * 4 + kb), at));
#pragma unroll
        for (int j = 0; j < R16; ++j) acc[j] = mma<Tag>(df[e][j], xf[e], acc[j]);
      }
    }
    __syncthreads();  // the last tile's t is read
#pragma unroll
    for (int j = 0; j < R16; ++j) *reinterpret_cast<f32x4*>(&part[wv][q][16 * j + 4 * kb]) = acc[j];
    __syncthreads();
    const float drop_scale = a.drop_in ? a.drop.scale : 1.0f;
    for (int k = t; k < 16 * R; k += kAT) {
      const int i = k / R, j = k % R;
      float v = (((part[0][i][j] + part[1][i][j]) + part[2][i][j]) + part[3][i][j]) * drop_scale;
      if (j >= a.r) v = 0.0f;  // not an infinity of x times a padding's zero
      part[0][i][j] = v;
      if (slab == 0 && i < tile.here) a.t[w.token(tile, i) * R + j] = v;
    }
    __syncthreads();
    if (!a.out) continue;
    Thin<Tag, R16> thin;
    thin.load(&part[0][q][0], kb);
    const float scale = a.scales ? a.scales[tile.ad] : 1.0f;
    const char* up = a.up + tile.ad * a.u_sa * SZ;
    for (int64_t c = c0 + 16 * NC * wv; c < c1; c += 16 * NC * kAW) {
      Frag<Tag> b[NC / 2];
      UpRow<Tag, R16> u[NC];
      if (a.base) {
#pragma unroll
        for (int p = 0; p < NC / 2; ++p) b[p].load(a.base + n * a.b_ld * SZ, c + 32 * p + 8 * kb, c1);
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) u[i].load(up + up_row(c, i, q, a.O) * a.u_so * SZ, a.r, kb);
#pragma unroll
      for (int p = 0; p < NC / 2; ++p) {
        const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
        const int64_t col = c + 32 * p + 8 * kb;
        finish<Tag>(a, expand<Tag, R16>(u[2 * p], thin, none), expand<Tag, R16>(u[2 * p + 1], thin, none), n, col, scale,
                    at, b[p]);
        if (q < tile.here) b[p].store(a.out + n * a.O * SZ, col, c1);
      }
    }
  }
}

// Eight KB of a matrix, ROWS rows of 8192 / ROWS bytes, staged in LDS by a wave: loaded and
// stored as whole 128-byte lines, read and written as the products hold them (16 rows of 64
// bytes to an instruction).  Matrices that are larger than the 256 MB memory-side cache are
// streamed past it, which only whole lines bear: 537 MB are read at 4.5 instead of 3.4 TB/s,
// and leave what other passes read again in it.
template <class Tag, int ROWS, bool WHOLE>
struct Stage {
  static constexpr int EPV = Pack16<Tag>::EPV, SZ = 16 / EPV, kBytes = 8192 / ROWS, kCols = kBytes / SZ;
  static constexpr int kPieces = kBytes / 16, kTogether = 64 / kPieces, kRow = kBytes + 16;  // rows to an instruction
  u32x4 raw[8];
  static __device__ __forceinline__ int piece() { return (threadIdx.x & 63) % kPieces; }
  static __device__ __forceinline__ int row(int i) { return kTogether * i + (threadIdx.x & 63) / kPieces; }
  // columns from c on of rows n[i], zeros from `end` on
  __device__ __forceinline__ void load(const char* base, int64_t ld, const int (&n)[8], int64_t c, int64_t end,
                                       bool stream) {
    const int64_t col = c + piece() * EPV;
    if (WHOLE || col + EPV <= end) {
      if (stream) {
        apart();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          raw[i] = __builtin_nontemporal_load(reinterpret_cast<const AnyVec*>(base + ((int64_t)n[i] * ld + col) * SZ));
        apart();
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = *reinterpret_cast<const AnyVec*>(base + ((int64_t)n[i] * ld + col) * SZ);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[i] = load_part<Tag>(base + ((int64_t)n[i] * ld + col) * SZ, end - col);
    }
  }
  __device__ __forceinline__ void put(char* stage) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<u32x4*>(stage + row(i) * kRow + piece() * 16) = raw[i];
  }
  __device__ __forceinline__ void get(const char* stage) {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = *reinterpret_cast<const u32x4*>(stage + row(i) * kRow + piece() * 16);
  }
  // the first `rows` of them
  __device__ __forceinline__ void store(char* base, int64_t ld, const int (&n)[8], int rows, int64_t c, int64_t end,
                                        bool stream) const {
    const int64_t col = c + piece() * EPV;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (row(i) >= rows) continue;
      char* to = base + ((int64_t)n[i] * ld + col) * SZ;
      if (WHOLE || col + EPV <= end) {
        if (stream) {
          apart();
          __builtin_nontemporal_store(raw[i], reinterpret_cast<AnyVec*>(to));
          apart();
        } else {
          *reinterpret_cast<AnyVec*>(to) = raw[i];
        }
      } else {
        store_part<Tag>(to, raw[i], end - col);
      }
    }
  }
  // eight columns of a row as the products hold them
  static __device__ __forceinline__ void read(const char* stage, int r, int col, Frag<Tag>& f) {
#pragma unroll
    for (int h = 0; h < Frag<Tag>::NV; ++h)
      f.v[h] = *reinterpret_cast<const u32x4*>(stage + r * kRow + col * SZ + 16 * h);
  }
  static __device__ __forceinline__ void write(char* stage, int r, int col, const Frag<Tag>& f) {
#pragma unroll
    for (int h = 0; h < Frag<Tag>::NV; ++h)
      *reinterpret_cast<u32x4*>(stage + r * kRow + col * SZ + 16 * h) = f.v[h];
  }
};

// t of many rows: 16 to a wave, over the whole depth.  WHOLE: the depth is stages, and r is
// 16 R16, so that no load looks for an end.
template <class Tag, int R16, bool WHOLE>
__global__ __launch_bounds__(kAT) void adapter_shrink_kernel(FusedArgs a) {
  using S = Stage<Tag, 16, WHOLE>;
  constexpr int SZ = S::SZ, R = 16 * R16;
  __shared__ uint16_t order[kWindow];
  __shared__ __attribute__((aligned(16))) char stages[kAW][16 * S::kRow];
  __shared__ int scan[2 * kAW];
  extern __shared__ int bins[];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, kb = lane >> 4, q = lane & 15;
  char* const stage = stages[wv];
  const Window<64> w(a, order, scan, bins);
  const uint64_t at = a.drop_in ? a.drop.counter() : 0;
  const float drop_scale = a.drop_in ? a.drop.scale : 1.0f;
  const char* const x0 = a.x + w.n0 * a.x_ld * SZ;
  for (int it = group_of(a); it < w.all; it += a.groups) {
    const Window<64>::Tile tile = w.tile(it);
    if (tile.ad >= a.ids.A || 16 * wv >= tile.here) continue;
    const int64_t n = w.token(tile, 16 * wv + q);
    int rows[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rows[i] = w.row(tile, 16 * wv + S::row(i));
    const char* down = a.down + tile.ad * a.d_sa * SZ;
    f32x4 acc[R16] = {};
    S in;
    in.load(x0, a.x_ld, rows, 0, a.K, a.stream_x);
    for (int64_t c = 0; c < a.K; c += S::kCols) {
      if (a.drop_in) {
        const int64_t col = c + S::piece() * S::EPV, per_row = (a.K + 7) / 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t bits = a.drop.keep_bits((uint64_t)((w.n0 + rows[i]) * per_row + col / 8), at);
          if constexpr (SZ == 4) bits >>= col & 4;
          keep_entries<Tag>(in.raw[i], bits);
        }
      }
      wave_fence();
      in.put(stage);
      wave_fence();
      if (c + S::kCols < a.K) in.load(x0, a.x_ld, rows, c + S::kCols, a.K, a.stream_x);
      constexpr int kSteps = S::kCols / 32, kAhead = R16 > 2 ? 2 : 4;
#pragma unroll
      for (int s0 = 0; s0 < kSteps; s0 += kAhead) {
        Frag<Tag> df[kAhead][R16];
#pragma unroll
        for (int e = 0; e < kAhead; ++e)
#pragma unroll
          for (int j = 0; j < R16; ++j) {
            const int rr = 16 * j + q;
            const int64_t k = c + (s0 + e) * 32 + 8 * kb;
            if constexpr (WHOLE) df[e][j].template load<true>(down + rr * a.d_sr * SZ, k, a.K);
            else df[e][j].load(down + min(rr, a.r - 1) * a.d_sr * SZ, rr < a.r ? k : a.K, a.K);
          }
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
          Frag<Tag> xf;
          S::read(stage, q, (s0 + e) * 32 + 8 * kb, xf);
#pragma unroll
          for (int j = 0; j < R16; ++j) acc[j] = mma<Tag>(df[e][j], xf, acc[j]);
        }
      }
    }
    if (16 * wv + q < tile.here) {
#pragma unroll
      for (int j = 0; j < R16; ++j) {
        f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k)  // padding: not an infinity of x times its zero
          v[k] = 16 * j + 4 * kb + k < a.r ? acc[j][k] * drop_scale : 0.0f;
        *reinterpret_cast<f32x4*>(a.t + n * R + 16 * j + 4 * kb) = v;
      }
    }
  }
}

// base + scale up t, a stage of all rows of a tile to a wave at a time, the waves side by
// side.  WHOLE: the columns are stages, and r is 16 R16.
template <class Tag, int R16, int TM, bool WHOLE>
__global__ __launch_bounds__(kAT, 2) void adapter_expand_kernel(FusedArgs a) {
  using S = Stage<Tag, TM, WHOLE>;
  constexpr int SZ = S::SZ, R = 16 * R16, MT = TM / 16;
  __shared__ uint16_t order[kWindow];
  __shared__ __attribute__((aligned(16))) char stages[kAW][TM * S::kRow];
  __shared__ int scan[2 * kAW];
  extern __shared__ int bins[];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, kb = lane >> 4, q = lane & 15;
  char* const stage = stages[wv];
  const Window<TM> w(a, order, scan, bins);
  const uint64_t at = a.drop_out ? a.drop.counter() : 0;
  const char* const base0 = a.base + w.n0 * a.b_ld * SZ;
  char* const out0 = a.out + w.n0 * a.O * SZ;
  for (int64_t it = group_of(a); it < (int64_t)w.all * a.slabs; it += a.groups) {
    const typename Window<TM>::Tile tile = w.tile((int)(it / a.slabs));
    const int slab = (int)(it % a.slabs);
    const int64_t c0 = slab * a.slab, c1 = min(c0 + a.slab, a.O);
    if (tile.ad >= a.ids.A) {
      plain_rows<Tag, TM>(a, w, tile, c0, c1);
      continue;
    }
    const int chunks = (int)((c1 - c0 + S::kCols - 1) / S::kCols);
    if (wv >= chunks) continue;
    int n[MT], rows[8];
    Thin<Tag, R16> thin[MT];
#pragma unroll
    for (int f = 0; f < MT; ++f) {
      n[f] = w.row(tile, 16 * f + q);
      thin[f].load(a.t + (w.n0 + n[f]) * R, kb);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) rows[i] = w.row(tile, S::row(i));
    const float scale = a.scales ? a.scales[tile.ad] : 1.0f;
    const char* up = a.up + tile.ad * a.u_sa * SZ;
    S in;
    if (a.base) in.load(base0, a.b_ld, rows, c0 + wv * S::kCols, c1, a.stream_out);
    for (int chunk = wv; chunk < chunks; chunk += kAW) {
      const int64_t c = c0 + chunk * S::kCols;
      if (a.base) {
        wave_fence();
        in.put(stage);
        if (chunk + kAW < chunks) in.load(base0, a.b_ld, rows, c + kAW * S::kCols, c1, a.stream_out);
      }
      wave_fence();
      // tiles of up's rows at once: with 16 rows of t, as many as 64 registers hold; with more
      // rows of a t of over 32 ranks in parts, two (four spill: 32,768 rows, 1024 to 2048, rank
      // 128, float16, both directions 1135 us instead of 1045)
      constexpr bool F32 = std::is_same_v<Tag, TagF32>;
      constexpr int kMost = TM > 16 ? (!F32 && R16 > 2 ? 2 : 4) : (F32 || R16 > 2 ? 32 / R16 : 16);
      constexpr int NC = S::kCols / 16 < kMost ? S::kCols / 16 : kMost;
#pragma unroll 1
      for (int i0 = 0; i0 < S::kCols / 16; i0 += NC) {
        if (c + 16 * i0 >= c1) break;
        UpRow<Tag, R16> u[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i)
          u[i].template load<WHOLE>(up + up_row(c + 16 * i0, i, q, a.O) * a.u_so * SZ, a.r, kb);
#pragma unroll
        for (int p = 0; p < NC / 2; ++p)
#pragma unroll
          for (int f = 0; f < MT; ++f) {
            const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
            const int col = 16 * i0 + 32 * p + 8 * kb;
            Frag<Tag> b;
            if (a.base) S::read(stage, 16 * f + q, col, b);
            finish<Tag>(a, expand<Tag, R16>(u[2 * p], thin[f], none), expand<Tag, R16>(u[2 * p + 1], thin[f], none),
                        w.n0 + n[f], c + col, scale, at, b);
            S::write(stage, 16 * f + q, col, b);
            // side by side, these would take the registers of more waves
            __builtin_amdgcn_sched_barrier(0);
          }
      }
      wave_fence();
      S out;
      out.get(stage);
      out.store(out0, a.O, rows, tile.here, c, c1, a.stream_out);
    }
  }
}

// ---- the weights' gradients ------------------------------------------------------------

// part[c, r] of an adapter and a run of tokens: sum over its tokens of wide[n, c] thin[n, r].
// A lane loads eight columns of eight tokens, which is what eight matrix instructions'
// fragments hold: the columns 8 (lane % 16) + j make up the j-th.
struct OuterJob {
  const char* wide;   // [N, C]; null: no such job
  int64_t ld, C;
  const float* thin;  // [N, R]
  float* part;        // [A, segments], each [C, R], or [R, C] where the gradient's rows are along C
  int32_t* seen;      // [A, segments]: whether the run holds any of its tokens
  char* out;          // the gradient: entry (a, c, r) at a * o_sa + c * o_sc + r * o_sr
  int64_t o_sa, o_sc, o_sr;
  int tiles;          // of kOuterCols columns
  int drop, stream;
};
struct OuterArgs {
  OuterJob job[2];
  AdapterIds ids;
  int64_t N;
  int r, R;           // R: r rounded up to a multiple of 16
  int rank_tiles;     // of 16 RT ranks
  int segments;
  Drop drop;
  const float* scales;
};
constexpr int kOuterCols = 128 * kAW;

// What a lane holds of 32 tokens: eight columns and RT ranks of eight of them.
template <class Tag, int RT>
struct OuterStep {
  Frag<Tag> x[8];
  float th[8][RT];
};

template <class Tag, int RT>
__global__ __launch_bounds__(kAT, RT <= 2 ? 3 : 2) void adapter_outer_kernel(OuterArgs a) {
  constexpr int SZ = 16 / Pack16<Tag>::EPV;
  constexpr bool F32 = std::is_same_v<Tag, TagF32>, F16 = std::is_same_v<Tag, TagF16>;
  __shared__ uint16_t list[kWindow];
  __shared__ int counts[kAW];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, kb = lane >> 4, q = lane & 15;
  uint32_t id = blockIdx.x;
  const uint32_t per = (uint32_t)((a.job[0].tiles + a.job[1].tiles) * a.rank_tiles);
  const uint32_t seg = id / per / a.ids.A, ad = id / per % a.ids.A;
  id %= per;
  const int rt = (int)(id % a.rank_tiles);
  int ct = (int)(id / a.rank_tiles);
  const bool second = ct >= a.job[0].tiles;
  if (second) ct -= a.job[0].tiles;
  const OuterJob& j = a.job[second];
  const int64_t col = (int64_t)ct * kOuterCols + wv * 128 + 8 * q;
  const bool whole = __all(col + 8 <= j.C);
  const int64_t per_row = (j.C + 7) / 8;
  const uint64_t at = j.drop ? a.drop.counter() : 0;
  const int r0 = rt * 16 * RT;

  f32x4 acc[8][RT] = {};
  bool any = false;
  // a run of tokens, from a multiple of 64 on
  const int64_t begin = a.N * seg / a.segments / 64 * 64;
  const int64_t end = seg + 1 == (uint32_t)a.segments ? a.N : a.N * (seg + 1) / a.segments / 64 * 64;
  for (int64_t n0 = begin; n0 < end; n0 += kWindow) {
    // the window's tokens of this adapter, in order: a wave looks at a quarter of it
    const int count = (int)min((int64_t)kWindow, end - n0);
    uint64_t mine[kWindow / kAT];
    int before = 0, sum = 0;
#pragma unroll
    for (int k = 0; k < kWindow / kAT; ++k) {
      const int i = wv * (kWindow / kAW) + 64 * k + lane;
      mine[k] = __ballot(i < count && a.ids.at(n0 + min(i, count - 1)) == (int)ad);
      sum += __popcll(mine[k]);
    }
    __syncthreads();  // the last window's list is read
    if (lane == 0) counts[wv] = sum;
    __syncthreads();
    int listed = 0;
    for (int k = 0; k < kAW; ++k) {
      if (k < wv) before += counts[k];
      listed += counts[k];
    }
#pragma unroll
    for (int k = 0; k < kWindow / kAT; ++k) {
      if (mine[k] >> lane & 1)
        list[before + __popcll(mine[k] & (((uint64_t)1 << lane) - 1))] =
            (uint16_t)(wv * (kWindow / kAW) + 64 * k + lane);
      before += __popcll(mine[k]);
    }
    __syncthreads();
    any |= listed > 0;
    if (listed == 0 || col - 8 * q >= j.C) continue;  // or this wave's columns are past the end
    for (int s = 0; s < listed; s += 32) {
      OuterStep<Tag, RT> in;
      const char* row[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = s + 8 * kb + i;
        const bool here = k < listed;
        const int64_t n = n0 + list[min(k, listed - 1)];
        row[i] = j.wide + n * j.ld * SZ;
#pragma unroll
        for (int e = 0; e < RT; ++e) in.th[i][e] = here ? j.thin[n * a.R + r0 + 16 * e + q] : 0.0f;
      }
      if (j.stream && s + 32 <= listed && whole) {
        apart();
#pragma unroll
        for (int i = 0; i < 8; ++i) in.x[i].stream(row[i], col);
        apart();
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) in.x[i].load(row[i], s + 8 * kb + i < listed ? col : j.C, j.C);
      }
      if (j.drop) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int64_t n = n0 + list[min(s + 8 * kb + i, listed - 1)];
          in.x[i].keep(a.drop.keep_bits((uint64_t)(n * per_row + col / 8), at));
        }
      }
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int e = 0; e < RT; ++e)
              acc[c][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(in.x[i].v[c / 4][c % 4]), in.th[i][e],
                                                               acc[c][e], 0, 0, 0);
      } else {
        u32x4 thin[RT][3];
#pragma unroll
        for (int e = 0; e < RT; ++e) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = in.th[i][e];
          split8(v, thin[e]);
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          u32x4 wide[F16 ? 2 : 1];
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            // column c of tokens 2d and 2d + 1
            const uint32_t two = __builtin_amdgcn_perm(in.x[2 * d + 1].v[0][c / 2], in.x[2 * d].v[0][c / 2],
                                                       c % 2 ? 0x07060302u : 0x05040100u);
            if constexpr (F16) {
              float p = f16_bits_to_f32((uint16_t)two), q = f16_bits_to_f32((uint16_t)(two >> 16));
              wide[0][d] = cut2(p, q);
              wide[1][d] = cut2(p, q);
            } else {
              wide[0][d] = two;
            }
          }
#pragma unroll
          for (int e = 0; e < RT; ++e)
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              acc[c][e] = mma_bf16(wide[0], thin[e][k], acc[c][e]);
              if constexpr (F16) acc[c][e] = mma_bf16(wide[1], thin[e][k], acc[c][e]);
            }
        }
      }
    }
  }
  const int64_t slot = (int64_t)ad * a.segments + seg;
  if (ct == 0 && rt == 0 && t == 0) j.seen[slot] = any;
  if (!any) return;
  // a lane's columns are 8 (4 kb + i) + c, its rank q; neighbours as in the gradient
  float* part = j.part + slot * j.C * a.R;
  const int64_t p_sc = j.o_sr == 1 ? a.R : 1, p_sr = j.o_sr == 1 ? 1 : j.C;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = (int64_t)ct * kOuterCols + wv * 128 + 8 * (4 * kb + i);
#pragma unroll
    for (int e = 0; e < RT; ++e) {
      float* at = part + o * p_sc + (r0 + 16 * e + q) * p_sr;
      if (p_sc == 1) {
        Frag<TagF32> v;
        float x[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) x[c] = acc[c][e][i];
        v.pack(x);
        v.store(reinterpret_cast<char*>(at), 0, j.C - o);
      } else {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (o + c < j.C) at[c * p_sc] = acc[c][e][i];
      }
    }
  }
}

// Joins the runs' sums, in order: a workgroup takes 64 entries at a time, a wave a quarter of
// the runs.
template <class Tag>
__global__ __launch_bounds__(kAT) void adapter_join_kernel(OuterArgs a) {
  __shared__ float quarter[kAW][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int64_t n0 = a.job[0].wide ? a.job[0].C * a.r : 0, n1 = a.job[1].wide ? a.job[1].C * a.r : 0;
  const int64_t b0 = (n0 + 63) / 64, b1 = (n1 + 63) / 64, blocks = (b0 + b1) * a.ids.A;
  const int begin = a.segments * wv / kAW, end = a.segments * (wv + 1) / kAW;
  for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    const int64_t ad = block / (b0 + b1);
    const bool second = block % (b0 + b1) >= b0;
    const int64_t k = (block % (b0 + b1) - (second ? b0 : 0)) * 64 + lane;
    const OuterJob& j = a.job[second];
    const bool in = k < (second ? n1 : n0);
    // neighbours in the gradient's rows
    const int64_t c = j.o_sr == 1 ? k / a.r : k % j.C, r = j.o_sr == 1 ? k % a.r : k / j.C;
    const int64_t size = j.C * a.R, slot0 = ad * a.segments;
    const float* part = j.part + slot0 * size + (j.o_sr == 1 ? c * a.R + r : r * j.C + c);
    constexpr int kTogether = 8;
    float sum = 0.0f;
    for (int s64 = begin; s64 < end; s64 += 64) {
      const uint64_t seen = __ballot(s64 + lane < end && j.seen[slot0 + min(s64 + lane, end - 1)]);
      for (int s0 = 0; s0 < 64 && seen >> s0; s0 += kTogether) {
        float v[kTogether];
#pragma unroll
        for (int s = 0; s < kTogether; ++s)
          v[s] = in && (seen >> (s0 + s) & 1) ? part[(s64 + s0 + s) * size] : 0.0f;
#pragma unroll
        for (int s = 0; s < kTogether; ++s) sum += v[s];
      }
    }
    __syncthreads();  // the last entries' sums are read
    quarter[wv][lane] = sum;
    __syncthreads();
    if (wv != 0 || !in) continue;
    sum = ((quarter[0][lane] + quarter[1][lane]) + quarter[2][lane]) + quarter[3][lane];
    sum *= (a.scales ? a.scales[ad] : 1.0f);
    if (j.drop) sum *= a.drop.scale;
    const int64_t o = ad * j.o_sa + c * j.o_sc + r * j.o_sr;
    if constexpr (std::is_same_v<Tag, TagF32>) reinterpret_cast<float*>(j.out)[o] = sum;
    else reinterpret_cast<uint16_t*>(j.out)[o] = (uint16_t)Pack16<Tag>::pack_one(sum);
  }
}

// up [A, O, r] as [A, R, P] (P: O rounded up to a multiple of 8) and down [A, r, H] as
// [A, H, R], zeros where there is nothing.
struct TurnArgs {
  const char *down, *up;
  int64_t d_sa, d_sr, u_sa, u_so, H, O, P;
  char *downt, *upt;
  int A, r, R;
};
template <class E>
__global__ __launch_bounds__(kAT) void adapter_turn_kernel(TurnArgs a) {
  const int64_t nu = (int64_t)a.R * a.P, nd = a.H * a.R;
  int64_t k = (int64_t)blockIdx.x * kAT + threadIdx.x;
  const int64_t ad = k / (nu + nd);
  if (ad >= a.A) return;
  k -= ad * (nu + nd);
  if (k < nu) {
    const int64_t r = k / a.P, o = k % a.P;
    reinterpret_cast<E*>(a.upt)[ad * nu + k] =
        r < a.r && o < a.O ? reinterpret_cast<const E*>(a.up)[ad * a.u_sa + o * a.u_so + r] : (E)0;
  } else {
    k -= nu;
    const int64_t h = k / a.R, r = k % a.R;
    reinterpret_cast<E*>(a.downt)[ad * nd + k] =
        r < a.r ? reinterpret_cast<const E*>(a.down)[ad * a.d_sa + r * a.d_sr + h] : (E)0;
  }
}

// ---- host ------------------------------------------------------------------------------

inline int rank_padded(int r) { return r <= 16 ? 16 : (r <= 32 ? 32 : (r <= 64 ? 64 : 128)); }

// Kernels for whole sizes leave out the looks for a row's end (131,072 rows of 1024 by rank
// 16: t 57 us instead of 64; sizes and ranks that are not whole take the others).
//
// The grid of tiles of TM rows, and with `wide` runs of columns: as many as make two
// workgroups to each of the 256 CUs, of `least` columns at least.
//
// How many tiles a window has its ids decide.  Up to a thousand workgroups each possible one
// gets its own; beyond that those that find nothing cost more (a window is sorted first) than
// the rounds of two workgroups to a CU: 16 rows of the LM head 26 -> 19 us, 8192 rows of 16
// adapters in any order, 1024 to 1024, 24 -> 18; with such rounds always, 8192 rows in runs of
// 700, 1024 to 4096, 37 -> 44.  Where workgroups may find nothing and a tile is not cut by
// columns, windows take turns, so that those come last: 32,768 rows of 4 adapters, 1024 to
// 2048, rank 64, a direction's two kernels 74 -> 57 us on average; with tiles that are cut,
// the 37 us above would be 47.
template <int TM>
dim3 tile_grid(FusedArgs& a, bool wide, int64_t least) {
  const int64_t windows = (a.N + kWindow - 1) / kWindow;
  const int rows = (int)min(a.N, (int64_t)kWindow);
  // tiles of a window if it is of one adapter, and at most
  const int64_t even = (rows + TM - 1) / TM, most = min((int64_t)rows, even + a.ids.A + 1);
  const int64_t cuts = wide ? max((int64_t)1, min((a.O + least - 1) / least, 512 / max((int64_t)1, windows * even))) : 1;
  a.slab = wide ? ((a.O + cuts - 1) / cuts + least - 1) / least * least : 1;
  a.slabs = wide ? (int)((a.O + a.slab - 1) / a.slab) : 1;
  a.groups = (int)(windows * most * a.slabs <= 1024 ? most * a.slabs
                                                    : min(most * a.slabs, max(even * a.slabs, 512 / windows)));
  // a grid's threads are counted in 32 bits (up to 2^30 rows: at least 15 workgroups a window)
  a.groups = (int)min((int64_t)a.groups, (((int64_t)1 << 32) / kAT - 1) / windows);
  a.in_turn = a.slabs == 1 && a.groups > even ? (int)windows : 0;
  return dim3((uint32_t)(windows * a.groups));
}

template <class Tag, int R16, int TM>
int launch_expand(FusedArgs a, int64_t least, size_t lds, hipStream_t st) {
  const dim3 grid = tile_grid<TM>(a, true, least);
  if (a.r == 16 * R16 && a.O % Stage<Tag, TM, true>::kCols == 0)
    hipLaunchKernelGGL((adapter_expand_kernel<Tag, R16, TM, true>), grid, dim3(kAT), lds, st, a);
  else hipLaunchKernelGGL((adapter_expand_kernel<Tag, R16, TM, false>), grid, dim3(kAT), lds, st, a);
  return check_launch("adapter_expand_kernel");
}

// Few rows take tiles of 16 with the depth split over the waves, and both products in one
// launch unless every workgroup would form t again for too few columns.  us with one / two
// launches: 64 rows of 16 adapters, 1024 to 2048 9.5 / 17.3, 4096 9.7 / 16.5, 8192 11.1 /
// 17.4, 16,384 17.8 / 17.7, 32,768 25.7 / 23.1; 320 rows, 1024 to 2048 11.1 / 21.8, 512 rows
// to 4096 15.7 / 24.7, 1000 rows to 2048 13.9 / 24.4; at rank 64 256 rows to 2048 15.2 / 33.5,
// 512 21.2 / 35.0, 1000 to 4096 42.5 / 39.9.
template <int R16> constexpr int64_t kFewRows = R16 <= 2 ? 1024 : 512;
constexpr int64_t kFusedColumns = 16384;
// Matrices of over half the memory-side cache are streamed past it: 268 and 537 MB are read
// in 65 and 118 us instead of 65 and 151, and what other passes read again stays in it (the
// factors' gradients over both: 147 us instead of 194).  67 MB, which stay there, are read in
// 52.8 us streamed and in 49.6 not.
constexpr int64_t kStreamed = (int64_t)128 << 20;
inline int larger_than_cache(int64_t rows, int64_t cols, size_t size) {
  return rows * cols * (int64_t)size > kStreamed;
}

template <class Tag, int R16>
int launch_fused(FusedArgs a, hipStream_t st) {
  constexpr int TM = R16 > 4 ? 32 : 64;  // (t of 64 rows of rank 128 would not stay in registers)
  a.stream_x = larger_than_cache(a.N, a.K, Frag<Tag>::SZ);
  a.stream_out = larger_than_cache(a.N, a.O, Frag<Tag>::SZ);
  const size_t lds = Window<64>::lds(a.ids.A);
  const bool few = a.N <= kFewRows<R16>, together = few && a.O <= kFusedColumns;
  if (few) {
    char* const out = a.out;
    if (!together) a.out = nullptr;
    const dim3 grid = tile_grid<16>(a, a.out != nullptr, 256);
    hipLaunchKernelGGL((adapter_fused_kernel<Tag, R16>), grid, dim3(kAT), lds, st, a);
    if (int rc = check_launch("adapter_fused_kernel")) return rc;
    a.out = out;
  } else {
    const dim3 grid = tile_grid<64>(a, false, 256);
    if (a.r == 16 * R16 && a.K % Stage<Tag, 16, true>::kCols == 0)
      hipLaunchKernelGGL((adapter_shrink_kernel<Tag, R16, true>), grid, dim3(kAT), lds, st, a);
    else hipLaunchKernelGGL((adapter_shrink_kernel<Tag, R16, false>), grid, dim3(kAT), lds, st, a);
    if (int rc = check_launch("adapter_shrink_kernel")) return rc;
  }
  if (together || !a.out) return RRL_OK;
  if (few) return launch_expand<Tag, R16, 16>(a, 1024, lds, st);
  return launch_expand<Tag, R16, TM>(a, 256, lds, st);
}
template <class Tag>
int launch_fused(const FusedArgs& a, hipStream_t st) {
  switch (rank_padded(a.r)) {
    case 16: return launch_fused<Tag, 1>(a, st);
    case 32: return launch_fused<Tag, 2>(a, st);
    case 64: return launch_fused<Tag, 4>(a, st);
    default: return launch_fused<Tag, 8>(a, st);
  }
}
int launch_fused(const FusedArgs& a, int32_t dtype, hipStream_t st) {
  if (a.N == 0) return RRL_OK;
  if (dtype == RRL_F32) return launch_fused<TagF32>(a, st);
  if (dtype == RRL_BF16) return launch_fused<TagBF16>(a, st);
  return launch_fused<TagF16>(a, st);
}

template <class Tag>
int launch_outer(const OuterArgs& a, hipStream_t st) {
  const int64_t blocks =
      (int64_t)a.segments * a.ids.A * (a.job[0].tiles + a.job[1].tiles) * a.rank_tiles;
  const dim3 grid((uint32_t)blocks), threads(kAT);
  if (a.R == 16) hipLaunchKernelGGL((adapter_outer_kernel<Tag, 1>), grid, threads, 0, st, a);
  else if (a.R == 32) hipLaunchKernelGGL((adapter_outer_kernel<Tag, 2>), grid, threads, 0, st, a);
  else hipLaunchKernelGGL((adapter_outer_kernel<Tag, 4>), grid, threads, 0, st, a);
  return check_launch("adapter_outer_kernel");
}
template <class Tag>
int launch_join(const OuterArgs& a, hipStream_t st) {
  const int64_t each = ((a.job[0].wide ? a.job[0].C * a.r : 0) + 63) / 64 + ((a.job[1].wide ? a.job[1].C * a.r : 0) + 63) / 64;
  // four threads an entry: of adapters of 2^30 weights more than a grid counts, so workgroups
  // take several turns from 2^22 on
  const int64_t blocks = min(each * a.ids.A, (int64_t)1 << 22);
  hipLaunchKernelGGL(adapter_join_kernel<Tag>, dim3((uint32_t)blocks), dim3(kAT), 0, st, a);
  return check_launch("adapter_join_kernel");
}

struct BackLayout {
  int R;
  int64_t P;
  int segments, rank_tiles;
  size_t upt, downt, s, part[2], seen[2], total;
};
inline BackLayout back_layout(int64_t N, int64_t H, int64_t O, int64_t A, int r, size_t size) {
  BackLayout l;
  l.R = rank_padded(r);
  l.P = (O + 7) / 8 * 8;
  l.rank_tiles = l.R > 64 ? 2 : 1;
  const int64_t tiles = ((H + kOuterCols - 1) / kOuterCols + (O + kOuterCols - 1) / kOuterCols) * l.rank_tiles;
  // runs of tokens so that there are four workgroups to each of the 256 CUs, of 64 tokens at least
  l.segments = (int)min((N + 63) / 64, max((int64_t)1, 1024 / (A * tiles)));
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.upt = take((size_t)(A * l.R * l.P) * size);
  l.downt = take((size_t)(A * l.R * H) * size);
  l.s = take((size_t)(N * l.R) * 4);
  l.part[0] = take((size_t)(A * l.segments * O * l.R) * 4);
  l.part[1] = take((size_t)(A * l.segments * H * l.R) * 4);
  l.seen[0] = take((size_t)(A * l.segments) * 4);
  l.seen[1] = take((size_t)(A * l.segments) * 4);
  l.total = at;
  return l;
}

// Sizes whose index arithmetic and grids fit.
inline bool adapter_fits(int64_t N, int64_t H, int64_t O, int64_t A, int64_t r) {
  if (N < 0 || H < 1 || O < 1 || A < 1 || r < 1) return false;
  if (N > ((int64_t)1 << 30) || H > ((int64_t)1 << 24) || O > ((int64_t)1 << 24) || A > kMostAdapters ||
      r > kMostRank)
    return false;
  return A * rank_padded((int)r) * (H + O + 8) < ((int64_t)1 << 32) - kAT;
}

int check_adapter(const char* who, int32_t dtype, int64_t N, int64_t H, int64_t O, int64_t A, int64_t r,
                  const void* ids, int32_t ids_dtype, const void* scales) {
  const std::string w(who);
  RRL_REQUIRE(dtype == RRL_F32 || dtype == RRL_BF16 || dtype == RRL_F16, RRL_EDTYPE,
              w + ": entries must be float32, bfloat16 or float16");
  RRL_REQUIRE(adapter_fits(N, H, O, A, r), RRL_EINVAL,
              w + ": a bad size (at most 4096 adapters of rank 1 to 128, 2^30 rows, 2^24 columns, and 2^32 "
                  "weights with ranks rounded up to 16, 32, 64 or 128)");
  RRL_REQUIRE(ids != nullptr || A == 1 || N == 0, RRL_EINVAL, w + ": ids are needed where there are several adapters");
  RRL_REQUIRE(ids == nullptr || ids_dtype == RRL_I32 || ids_dtype == RRL_I64, RRL_EDTYPE,
              w + ": adapter ids must be int32 or int64");
  RRL_REQUIRE((ids == nullptr || (uintptr_t)ids % dtype_size(ids_dtype) == 0) && (uintptr_t)scales % 4 == 0,
              RRL_EALIGN, w + ": a pointer is not aligned to its element");
  return RRL_OK;
}

}  // namespace
}  // namespace rrl

using namespace rrl;

extern "C" int64_t rrl_adapter_rank_padded(int64_t r) {
  return r < 1 || r > kMostRank ? 0 : rank_padded((int)r);
}

extern "C" int rrl_adapter_fwd(const rrl_adapter_params* p, const void* x, int64_t x_ld, const void* base,
                               int64_t base_ld, void* out, float* t_out, void* stream) {
  clear_error();
  RRL_REQUIRE(p != nullptr, RRL_EINVAL, "rrl_adapter_fwd: null operand");
  if (int rc = check_adapter("rrl_adapter_fwd", p->dtype, p->N, p->H, p->O, p->A, p->r, p->ids, p->ids_dtype,
                             p->scales))
    return rc;
  FusedArgs a = {};
  if (p->dropout)
    if (int rc = make_drop(p->dropout, a.drop, "rrl_adapter_fwd")) return rc;
  if (p->N == 0) return RRL_OK;
  RRL_REQUIRE(x != nullptr && p->down != nullptr && p->up != nullptr && out != nullptr && t_out != nullptr, RRL_EINVAL,
              "rrl_adapter_fwd: null operand");
  RRL_REQUIRE(p->N <= 1 || (x_ld >= 0 && base_ld >= 0), RRL_EINVAL, "rrl_adapter_fwd: negative row stride");
  const size_t size = dtype_size(p->dtype);
  RRL_REQUIRE((uintptr_t)x % size == 0 && (uintptr_t)p->down % size == 0 && (uintptr_t)p->up % size == 0 &&
                  (uintptr_t)base % size == 0 && (uintptr_t)out % size == 0 && (uintptr_t)t_out % 16 == 0,
              RRL_EALIGN, "rrl_adapter_fwd: a pointer is not aligned (t_out: 16 bytes)");
  a.x = static_cast<const char*>(x);
  a.x_ld = x_ld;
  a.down = static_cast<const char*>(p->down);
  a.d_sa = p->down_sa;
  a.d_sr = p->down_sr;
  a.up = static_cast<const char*>(p->up);
  a.u_sa = p->up_sa;
  a.u_so = p->up_so;
  a.base = static_cast<const char*>(base);
  a.b_ld = base_ld;
  a.ids = AdapterIds{p->ids, p->ids_dtype, (int)p->A};
  a.scales = p->scales;
  a.out = static_cast<char*>(out);
  a.t = t_out;
  a.N = p->N;
  a.K = p->H;
  a.O = p->O;
  a.r = (int)p->r;
  a.drop_in = p->dropout != nullptr;
  a.nan_rows = 1;
  return launch_fused(a, p->dtype, as_stream(stream));
}

extern "C" size_t rrl_adapter_bwd_workspace_bytes(int64_t N, int64_t H, int64_t O, int64_t A, int64_t r,
                                                  int32_t dtype) {
  if (!adapter_fits(N, H, O, A, r)) return 0;
  return back_layout(N, H, O, A, (int)r, dtype_size(dtype)).total;
}

extern "C" int rrl_adapter_bwd(const rrl_adapter_params* p, const void* x, int64_t x_ld, const void* grad,
                               int64_t g_ld, const float* t, void* dx, void* ddown, void* dup, void* workspace,
                               void* stream) {
  clear_error();
  RRL_REQUIRE(p != nullptr, RRL_EINVAL, "rrl_adapter_bwd: null operand");
  if (int rc = check_adapter("rrl_adapter_bwd", p->dtype, p->N, p->H, p->O, p->A, p->r, p->ids, p->ids_dtype,
                             p->scales))
    return rc;
  Drop drop = {};
  if (p->dropout)
    if (int rc = make_drop(p->dropout, drop, "rrl_adapter_bwd")) return rc;
  RRL_REQUIRE(workspace != nullptr && p->down != nullptr && p->up != nullptr &&
                  (p->N == 0 || (grad != nullptr && (ddown == nullptr || x != nullptr) &&
                                 (dup == nullptr || t != nullptr))),
              RRL_EINVAL, "rrl_adapter_bwd: null operand");
  RRL_REQUIRE(p->N <= 1 || (x_ld >= 0 && g_ld >= 0), RRL_EINVAL, "rrl_adapter_bwd: negative row stride");
  const size_t size = dtype_size(p->dtype);
  RRL_REQUIRE((uintptr_t)x % size == 0 && (uintptr_t)p->down % size == 0 && (uintptr_t)p->up % size == 0 &&
                  (uintptr_t)grad % size == 0 && (uintptr_t)dx % size == 0 && (uintptr_t)ddown % size == 0 &&
                  (uintptr_t)dup % size == 0 && (uintptr_t)t % 16 == 0 && (uintptr_t)workspace % 16 == 0,
              RRL_EALIGN, "rrl_adapter_bwd: a pointer is not aligned (t and workspace: 16 bytes)");
  hipStream_t st = as_stream(stream);
  const BackLayout l = back_layout(p->N, p->H, p->O, p->A, (int)p->r, size);
  char* w = static_cast<char*>(workspace);
  float* s = reinterpret_cast<float*>(w + l.s);
  const AdapterIds ids{p->ids, p->ids_dtype, (int)p->A};
  if (p->N > 0 && (dx || ddown)) {
    TurnArgs ta{static_cast<const char*>(p->down), static_cast<const char*>(p->up), p->down_sa, p->down_sr, p->up_sa,
                p->up_so, p->H, p->O, l.P, w + l.downt, w + l.upt, (int)p->A, (int)p->r, l.R};
    const dim3 grid((uint32_t)((p->A * l.R * (l.P + p->H) + kAT - 1) / kAT));
    if (size == 4) hipLaunchKernelGGL(adapter_turn_kernel<uint32_t>, grid, dim3(kAT), 0, st, ta);
    else hipLaunchKernelGGL(adapter_turn_kernel<uint16_t>, grid, dim3(kAT), 0, st, ta);
    if (int rc = check_launch("adapter_turn_kernel")) return rc;
    FusedArgs a = {};
    a.x = static_cast<const char*>(grad);
    a.x_ld = g_ld;
    a.down = w + l.upt;
    a.d_sa = l.R * l.P;
    a.d_sr = l.P;
    a.up = w + l.downt;
    a.u_sa = p->H * l.R;
    a.u_so = l.R;
    a.ids = ids;
    a.scales = p->scales;
    a.out = static_cast<char*>(dx);
    a.t = s;
    a.N = p->N;
    a.K = p->O;
    a.O = p->H;
    a.r = (int)p->r;
    a.drop = drop;
    a.drop_out = p->dropout != nullptr;
    if (int rc = launch_fused(a, p->dtype, st)) return rc;
  }
  if (!ddown && !dup) return RRL_OK;
  OuterArgs o = {};
  o.ids = ids;
  o.N = p->N;
  o.r = (int)p->r;
  o.R = l.R;
  o.rank_tiles = l.rank_tiles;
  o.segments = l.segments;
  o.drop = drop;
  o.scales = p->scales;
  if (dup) {
    o.job[0] = OuterJob{static_cast<const char*>(grad), g_ld, p->O, t, reinterpret_cast<float*>(w + l.part[0]),
                        reinterpret_cast<int32_t*>(w + l.seen[0]), static_cast<char*>(dup), p->O * p->r, p->r, 1,
                        (int)((p->O + kOuterCols - 1) / kOuterCols), 0, larger_than_cache(p->N, p->O, size)};
    o.job[0].wide = p->N ? o.job[0].wide : w;
  }
  if (ddown) {
    o.job[1] = OuterJob{static_cast<const char*>(x), x_ld, p->H, s, reinterpret_cast<float*>(w + l.part[1]),
                        reinterpret_cast<int32_t*>(w + l.seen[1]), static_cast<char*>(ddown), p->H * p->r, 1, p->H,
                        (int)((p->H + kOuterCols - 1) / kOuterCols), p->dropout != nullptr,
                        larger_than_cache(p->N, p->H, size)};
    o.job[1].wide = p->N ? o.job[1].wide : w;
  }
  if (p->N > 0) {
    int rc;
    if (p->dtype == RRL_F32) rc = launch_outer<TagF32>(o, st);
    else if (p->dtype == RRL_BF16) rc = launch_outer<TagBF16>(o, st);
    else rc = launch_outer<TagF16>(o, st);
    if (rc) return rc;
  }
  if (p->dtype == RRL_F32) return launch_join<TagF32>(o, st);
  if (p->dtype == RRL_BF16) return launch_join<TagBF16>(o, st);
  return launch_join<TagF16>(o, st);
}
