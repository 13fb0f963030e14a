// Microscaled 4-bit floating point (OCP MX, e2m1 elements with an e8m0 scale for
// each 32): quantisation, its inverse, and the product of a quantised activation
// matrix with a quantised weight on the scaled matrix instructions.
//
//   block of 32 entries x_i, amax = max |x_i|:  e = floor(log2 amax) - 2, at least -127
//   scale byte e + 127 (255, NaN, where the block holds NaN or infinity)
//   code_i = e2m1(x_i / 2^e): 0, 0.5, 1, 1.5, 2, 3, 4, 6 and signs, nearest, ties to
//            even, saturating at 6 (amax / 2^e < 8)
//
// Rows are padded to a multiple of kDepth = 128 entries (one matrix instruction's
// depth) with blocks of zeros: codes [R, P / 2] (two entries a byte, the first in
// the low half), scales [R, P / 32].
#include "rrl_common.hpp"
#include "slab_common.hpp"

#include <type_traits>

namespace rrl {
namespace {

constexpr int kBlock = 32, kDepth = 128;
constexpr int kQT = 256;

inline int64_t padded(int64_t H) { return (H + kDepth - 1) / kDepth * kDepth; }

struct __attribute__((packed, aligned(2))) Any16 {
  u32x4 v;
};

// Entries i..i+7 of a row of H, zeros past its end.
template <class Tag>
__device__ __forceinline__ void load8(const char* row, int64_t i, int64_t H, float (&x)[8]) {
  constexpr int EPV = Pack16<Tag>::EPV, SZ = 16 / EPV;
  if (i + 8 <= H) {
    if constexpr (EPV == 8) {
      Pack16<Tag>::unpack(reinterpret_cast<const Any16*>(row + i * SZ)->v, x);
    } else {
      float lo[4], hi[4];
      Pack16<Tag>::unpack(reinterpret_cast<const Any16*>(row + i * SZ)->v, lo);
      Pack16<Tag>::unpack(reinterpret_cast<const Any16*>(row + i * SZ + 16)->v, hi);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = lo[k];
        x[4 + k] = hi[k];
      }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    x[k] = 0.0f;
    if (i + k < H) {
      if constexpr (SZ == 4) x[k] = reinterpret_cast<const float*>(row)[i + k];
      else x[k] = Pack16<Tag>::one(reinterpret_cast<const uint16_t*>(row)[i + k]);
    }
  }
}

// The scale byte of a block whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255 ? 255 : (e > 2 ? e - 2 : 0);
}

// Eight entries as codes, entry 0 in the low four bits.
__device__ __forceinline__ uint32_t codes8(const float (&x)[8], uint32_t byte) {
  if (byte == 255) return 0;
  const float unit = __uint_as_float(byte << 23);  // the instruction takes the exponent field
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], unit, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], unit, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], unit, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], unit, 3);
  return c;
}

// Where block `b` of row `r` goes, in units of 16 bytes of codes and bytes of scales.
// Rows: as MxFp4 keeps them.
struct RowOrder {
  uint32_t blocks;
  __device__ __forceinline__ int64_t codes(int64_t r, uint32_t b) const { return r * blocks + b; }
  __device__ __forceinline__ int64_t scale(int64_t r, uint32_t b) const { return r * blocks + b; }
};
// Fragments: as the product's waves read their activations.  16 rows of 128 entries
// (a step) are 1 KB, lane 16 (b % 4) + r % 16 after lane; four steps (a stage) of a
// lane's scales are one dword, which the matrix instruction picks its byte from.
struct FragmentOrder {
  uint32_t steps, stages;
  __device__ __forceinline__ int64_t codes(int64_t r, uint32_t b) const {
    return ((r >> 4) * steps + (b >> 2)) * 64 + (b & 3) * 16 + (r & 15);
  }
  __device__ __forceinline__ int64_t scale(int64_t r, uint32_t b) const {
    return (((r >> 4) * stages + (b >> 4)) * 64 + (b & 3) * 16 + (r & 15)) * 4 + ((b >> 2) & 3);
  }
};

// Four lanes per block, eight entries each: 16-byte loads, a block's maximum by two
// exchanges within the quad.  Bound by memory: 151,936 x 1024 bfloat16 take 82 us
// (4.8 TB/s), and 68 us back (5.8 TB/s).
template <class Tag, class Order>
__global__ __launch_bounds__(kQT) void mxfp4_quantize_kernel(const char* __restrict__ x, int64_t R,
                                                             int64_t H, int64_t ld, uint32_t blocks,
                                                             Order order,
                                                             uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales) {
  constexpr int SZ = 16 / Pack16<Tag>::EPV;
  const uint32_t id = (blockIdx.x * kQT + threadIdx.x) / 4;  // below 2^30 (blocks_fit)
  const int part = threadIdx.x & 3;
  if (id >= R * blocks) return;
  const int64_t r = id / blocks;
  const uint32_t b = id % blocks;
  float v[8];
  load8<Tag>(x + r * ld * SZ, (int64_t)b * kBlock + part * 8, H, v);
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
  m = max(m, (uint32_t)dpp_i<kDppXor1>((int)m));
  m = max(m, (uint32_t)dpp_i<kDppXor2>((int)m));
  const uint32_t byte = scale_byte(m);
  reinterpret_cast<uint32_t*>(codes)[order.codes(r, b) * 4 + part] = codes8(v, byte);
  if (part == 0) scales[order.scale(r, b)] = (uint8_t)byte;
}

// Eight codes as the numbers they stand for.
__device__ __forceinline__ void values8(uint32_t word, uint32_t byte, float (&v)[8]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  // the instruction takes the exponent field; of 255, NaN, it would make an infinity
  const float unit = __uint_as_float(byte << 23);
  const f2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 0),
                   __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 1),
                   __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 2),
                   __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 3)};
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = byte == 255 ? __builtin_nanf("") : p[k / 2][k % 2];
}

template <class Tag>
__global__ __launch_bounds__(kQT) void mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales,
                                                               int64_t R, int64_t H, uint32_t blocks,
                                                               char* __restrict__ out, int vec) {
  constexpr int EPV = Pack16<Tag>::EPV, SZ = 16 / EPV;
  const uint32_t id = (blockIdx.x * kQT + threadIdx.x) / 4;
  const int part = threadIdx.x & 3;
  if (id >= R * blocks) return;
  const int64_t r = id / blocks, c = (int64_t)(id % blocks) * kBlock + part * 8;
  if (c >= H) return;
  const uint32_t word = reinterpret_cast<const uint32_t*>(codes)[(int64_t)id * 4 + part];
  const uint32_t byte = scales[id];
  float v[8];
  values8(word, byte, v);
  char* dst = out + (r * H + c) * SZ;
  if (vec) {  // whole vectors, every one 16-byte aligned
#pragma unroll
    for (int p = 0; p < 8 / EPV; ++p) {
      float w[EPV];
#pragma unroll
      for (int k = 0; k < EPV; ++k) w[k] = v[p * EPV + k];
      *reinterpret_cast<u32x4*>(dst + 16 * p) = Pack16<Tag>::pack(w);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < H) {
        if constexpr (SZ == 4) reinterpret_cast<float*>(dst)[k] = v[k];
        else reinterpret_cast<uint16_t*>(dst)[k] = (uint16_t)Pack16<Tag>::pack_one(v[k]);
      }
  }
}

// ---- product -------------------------------------------------------------------------

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// (Alone, two waves on a SIMD, this instruction reached 4.3 PFLOP/s and the 32 x 32 x 64
// one 8.3; but its outputs leave in runs of 32 bytes a row, and the product was slower
// on it.)
// D += A B^T over 128 entries: lane l holds 32 consecutive entries (block l / 16)
// of row l % 16 of each operand, and their scales in byte T of a dword; it receives
// rows 4 (l / 16) + i of A, row l % 16 of B.
template <int T>
__device__ __forceinline__ f32x4 mfma_fp4(const u32x4& a, uint32_t sa, const u32x4& b, uint32_t sb,
                                          const f32x4& c) {
  const i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8 bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, T, (int)sa, T, (int)sb);
}

// Lambdas that hold their captures in registers only if they are inlined.
#define RRL_INLINE __attribute__((always_inline))

constexpr int kLinWaves = 4, kStage = 4;  // steps of 128 entries in a stage

struct LinearArgs {
  const u32x4* ac;      // activations in fragment order: [fragments, steps, 64]
  const uint32_t* as;   // [fragments, stages, 64]
  const uint8_t* wc;    // weight codes [N, P / 2]
  const uint8_t* ws;    // weight scales [N, P / 32]
  int64_t M, N;
  int32_t steps, stages, fragments;
  int32_t tiles, groups;  // tiles of NT fragments, and the workgroups that share a slab's
  char* out;
  int32_t out_dtype;
  int32_t aligned;  // outputs are rows of whole, 16-byte aligned vectors of 8
};

// 8 outputs of one row.  store8: 16 bytes at any address, or one by one at the row's
// end.  store8_buffer: rows of whole, aligned vectors, dropped where `off` is past the
// buffer's end.
struct __attribute__((packed, aligned(2))) Out16 {
  u32x4 v;
};
template <class Tag>
__device__ __forceinline__ void store8(char* row, int64_t n, int64_t N, const float (&v)[8]) {
  constexpr int EPV = Pack16<Tag>::EPV, SZ = 16 / EPV;
  if (n + 8 <= N) {
#pragma unroll
    for (int p = 0; p < 8 / EPV; ++p) {
      float w[EPV];
#pragma unroll
      for (int k = 0; k < EPV; ++k) w[k] = v[p * EPV + k];
      reinterpret_cast<Out16*>(row + n * SZ + 16 * p)->v = Pack16<Tag>::pack(w);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (n + k < N) {
      if constexpr (SZ == 4) reinterpret_cast<float*>(row)[n + k] = v[k];
      else reinterpret_cast<uint16_t*>(row)[n + k] = (uint16_t)Pack16<Tag>::pack_one(v[k]);
    }
}
template <class Tag>
__device__ __forceinline__ void store8_buffer(__amdgpu_buffer_rsrc_t out, int off,
                                              const float (&v)[8]) {
  constexpr int EPV = Pack16<Tag>::EPV;
#pragma unroll
  for (int p = 0; p < 8 / EPV; ++p) {
    float w[EPV];
#pragma unroll
    for (int k = 0; k < EPV; ++k) w[k] = v[p * EPV + k];
    // cached: a non-temporal half line is written by itself, at 3.1 TB/s instead of 5.1
    __builtin_amdgcn_raw_buffer_store_b128(Pack16<Tag>::pack(w), out, off + 16 * p, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 1");  // as in store_b128_nt
    __builtin_amdgcn_sched_barrier(0);
  }
}

// A workgroup: a slab of 4 x VT x 16 weight rows (a wave's own VT x 16 each, in
// registers) against tile after tile of NT x 16 activation rows (shared, through LDS
// a stage ahead).  Two stages of weights are held: with up to 1024 entries a row
// (RESIDENT) they are loaded once and stay, beyond that each step's registers are
// refilled for the stage after next as soon as its products are issued.  Tiles and
// stages are one sequence of turns with a barrier each, so that loads run ahead over
// tile borders and a tile's stores leave while the next one's products run; a turn
// issues its loads before its stores, for a wait on a load waits for what was issued
// before it.  All loads are unconditional (past an end they read the last fragment or
// step again, or zeros past the buffer; scalar offsets stay within it, for the bounds
// check subtracts them): behind a branch the compiler would wait for all of them.
// 2,048 x 151,936 x 1024 bfloat16 takes 217 us: the matrix instructions alone 147, the
// same without its stores 170, stores like its own alone 122 (5.1 TB/s).  8 rows take
// 15 us, the head's 83 MB at 5.5 TB/s.
// A wave's weight rows are dealt to its fragments so that the 4 x VT outputs a
// lane receives are runs of 8 neighbours: fragment i, row 4 b + k is weight row
// 32 (i / 2) + 8 b + 4 (i % 2) + k of the wave's.
template <int VT, int NT, int STAGES>
__global__ __launch_bounds__(64 * kLinWaves, 2) void mxfp4_linear_kernel(LinearArgs a) {
  constexpr int kRows = 16 * VT, kSlab = kRows * kLinWaves;
  constexpr bool RESIDENT = STAGES > 0;
  const int stages = RESIDENT ? STAGES : a.stages;
  // with two stages a tile has two buffers, and a barrier serves both
  constexpr int kBuffers = STAGES == 2 ? 4 : 2;
  __shared__ u32x4 lds_c[kBuffers][kStage][NT][64];
  __shared__ uint32_t lds_a[kBuffers][NT][64];
  __shared__ uint32_t lds_w[2][kLinWaves][VT][64];
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r16 = lane & 15, blk = lane >> 4;
  // a slab's workgroups follow each other on one XCD (they go to the eight in turn),
  // so that its L2 reads the slab once
  const uint32_t xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
  const int64_t base = ((int64_t)(slot / a.groups) * 8 + xcd) * kSlab;
  if (base >= a.N) return;
  const int group = (int)(slot % a.groups);
  const int tile0 = (int)((int64_t)a.tiles * group / a.groups);
  const int tile1 = (int)((int64_t)a.tiles * (group + 1) / a.groups);
  const int turns = (tile1 - tile0) * stages;

  const int64_t P = (int64_t)a.steps * kDepth;
  const uint32_t rows = (uint32_t)min((int64_t)kSlab, a.N - base);
  const __amdgpu_buffer_rsrc_t crsrc = row_rsrc(a.wc + base * (P / 2), rows * (uint32_t)(P / 2));
  const __amdgpu_buffer_rsrc_t srsrc =
      row_rsrc(a.ws + base * (P / kBlock), rows * (uint32_t)(P / kBlock));
  int wrow[VT];
#pragma unroll
  for (int i = 0; i < VT; ++i)
    wrow[i] = (wv * kRows + 32 * (i / 2) + 8 * (r16 >> 2) + 4 * (i % 2) + (r16 & 3)) * (int)(P / 2) +
              blk * 16;
  u32x4 w[2][kStage][VT];
  auto weights = [&](auto bc, auto tc, int stage) RRL_INLINE {
    constexpr int B = decltype(bc)::value, T = decltype(tc)::value;
#pragma unroll
    for (int i = 0; i < VT; ++i)
      w[B][T][i] = __builtin_amdgcn_raw_buffer_load_b128(crsrc, wrow[i],
                                                         min(stage * kStage + T, a.steps - 1) * (kDepth / 2), 0);
  };

  // what a turn needs in LDS, through registers: activations (a wave's own step),
  // their scales, and the weights' scales (a thread's own row)
  u32x4 turn_c[NT], turn_w;
  constexpr int kOwn = (NT + kLinWaves - 1) / kLinWaves;
  uint32_t turn_a[kOwn];
  // the fragments whose scales this wave takes along
  auto own = [&](int e) RRL_INLINE { return min(wv + e * kLinWaves, NT - 1); };
  auto fetch = [&](int tl, int st) RRL_INLINE {
    // past the end the last fragment and step are read again
    const int f0 = min(tl * NT, a.fragments - 1), count = min(NT, a.fragments - f0);
    const __amdgpu_buffer_rsrc_t cr =
        row_rsrc(a.ac + (int64_t)f0 * a.steps * 64, (uint32_t)(count * a.steps) * 1024);
    const __amdgpu_buffer_rsrc_t ar =
        row_rsrc(a.as + (int64_t)f0 * stages * 64, (uint32_t)(count * stages) * 256);
#pragma unroll
    for (int j = 0; j < NT; ++j)
      turn_c[j] = __builtin_amdgcn_raw_buffer_load_b128(
          cr, lane * 16, (min(j, count - 1) * a.steps + min(st * kStage + wv, a.steps - 1)) * 1024, 0);
#pragma unroll
    for (int e = 0; e < kOwn; ++e)
      turn_a[e] = __builtin_amdgcn_raw_buffer_load_b32(
          ar, lane * 4, (min(own(e), count - 1) * stages + st) * 256, 0);
  };
  auto fetch_scales = [&](int stage) RRL_INLINE {
    // a row's last stage may hold fewer than 16 bytes: a dword past the end reads as zeros
    const int row = (t % kSlab) * (int)(P / kBlock) + stage * 16;
#pragma unroll
    for (int d = 0; d < 4; ++d)
      turn_w[d] = __builtin_amdgcn_raw_buffer_load_b32(srsrc, row + 4 * d, 0, 0);
  };
  auto put = [&](int B) RRL_INLINE {
#pragma unroll
    for (int j = 0; j < NT; ++j) lds_c[B][wv][j][lane] = turn_c[j];
#pragma unroll
    for (int e = 0; e < kOwn; ++e) lds_a[B][own(e)][lane] = turn_a[e];
  };
  auto put_scales = [&](int B) RRL_INLINE {
    // byte T of lane 16 b + r's dword: block b of step T
    const int local = t % kRows;
    const int i = 2 * (local / 32) + ((local >> 2) & 1), r = 4 * ((local >> 3) & 3) + (local & 3);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const uint32_t sel = (uint32_t)b | (uint32_t)(4 + b) << 8;
      const uint32_t lo = __builtin_amdgcn_perm(turn_w.y, turn_w.x, sel);
      const uint32_t hi = __builtin_amdgcn_perm(turn_w.w, turn_w.z, sel);
      lds_w[B][t % kSlab / kRows][i][16 * b + r] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
  };

  f32x4 acc[VT][NT] = {};
  int tile = tile0, stage = 0, half = 0;    // this turn, and its tile's buffers
  int next_tile = tile0, next_stage = 0;    // the one whose loads go out next
  auto advance = [&](int& tl, int& st) RRL_INLINE {
    const bool wrap = st + 1 == stages;
    st = wrap ? 0 : st + 1;
    tl += wrap;
  };
  const int64_t size = a.out_dtype == RRL_F32 ? 4 : 2;
  const int64_t column = base + wv * kRows + 8 * blk;  // of the first of a lane's runs
  auto store = [&]() RRL_INLINE {
    if (a.aligned) {
      // no branch: a lane whose row or column is past the end stores past the buffer's
      const int64_t m0 = (int64_t)tile * (NT * 16);
      const uint32_t here = (uint32_t)min((int64_t)NT * 16, a.M - m0);
      const __amdgpu_buffer_rsrc_t out =
          row_rsrc(a.out + m0 * a.N * size, here * (uint32_t)(a.N * size));
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < VT / 2; ++h) {
          const int64_t n = column + 32 * h;
          const uint32_t row = 16 * j + r16;
          const int off = n < a.N && row < here ? (int)((row * a.N + n) * size) : -64;
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = acc[2 * h + k / 4][j][k % 4];
          if (a.out_dtype == RRL_F32) store8_buffer<TagF32>(out, off, v);
          else if (a.out_dtype == RRL_BF16) store8_buffer<TagBF16>(out, off, v);
          else store8_buffer<TagF16>(out, off, v);
        }
    } else {
      const int64_t m0 = (int64_t)tile * (NT * 16) + r16;
      char* row = a.out + m0 * a.N * size;
#pragma unroll
      for (int j = 0; j < NT; ++j, row += 16 * a.N * size)
        if (m0 + 16 * j < a.M) {
#pragma unroll
          for (int h = 0; h < VT / 2; ++h) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = acc[2 * h + k / 4][j][k % 4];
            if (a.out_dtype == RRL_F32) store8<TagF32>(row, column + 32 * h, a.N, v);
            else if (a.out_dtype == RRL_BF16) store8<TagBF16>(row, column + 32 * h, a.N, v);
            else store8<TagF16>(row, column + 32 * h, a.N, v);
          }
        }
    }
    if constexpr (!RESIDENT) {  // a resident tile's first products take zeros for it
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < VT; ++i) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  };
  uint32_t sw[2][VT];
  auto turn = [&](auto bc) RRL_INLINE {
    constexpr int B = decltype(bc)::value;
    const int st = STAGES == 2 ? B : (STAGES == 1 ? 0 : stage);
    // this turn's buffer, and where the data loaded during it go
    const int from = STAGES == 2 ? 2 * half + B : B, to = STAGES == 2 ? from ^ 2 : from ^ 1;
    if (STAGES != 2 || B == 0) lds_barrier();
    if constexpr (!RESIDENT) {
#pragma unroll
      for (int i = 0; i < VT; ++i) sw[B][i] = lds_w[B][wv][i][lane];
    }
    uint32_t sa[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) sa[j] = lds_a[from][j][lane];
    // a fragment is read while the products of the one before run
    u32x4 x = lds_c[from][0][0][lane];
    auto step = [&](auto tc) RRL_INLINE {
      constexpr int T = decltype(tc)::value;
      if (st * kStage + T < a.steps) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const u32x4 next = lds_c[from][j + 1 < NT ? T : (T + 1) % kStage][(j + 1) % NT][lane];
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < VT; ++i)
            acc[i][j] = mfma_fp4<T>(w[B][T][i], sw[B][i], x, sa[j],
                                    RESIDENT && T == 0 && (STAGES == 1 || B == 0)
                                        ? f32x4{0.0f, 0.0f, 0.0f, 0.0f}
                                        : acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
          x = next;
        }
      }
      if constexpr (!RESIDENT) weights(bc, tc, next_stage);
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
    // what is in flight arrived during the products
    put(to);
    if constexpr (!RESIDENT) put_scales(B ^ 1);
    fetch(next_tile, next_stage);
    if constexpr (!RESIDENT) fetch_scales(next_stage);
    advance(next_tile, next_stage);
    if (st == stages - 1) store();
    advance(tile, stage);
    if (STAGES == 2 && B == 1) half ^= 1;
  };

  const std::integral_constant<int, 0> c0;
  const std::integral_constant<int, 1> c1;
  const std::integral_constant<int, 2> c2;
  const std::integral_constant<int, 3> c3;
  const int second = stages > 1 ? 1 : 0;
  fetch(tile0, 0);
  fetch_scales(0);
  weights(c0, c0, 0), weights(c0, c1, 0), weights(c0, c2, 0), weights(c0, c3, 0);
  put(0);
  put_scales(0);
  advance(next_tile, next_stage);
  fetch(next_tile, next_stage);
  fetch_scales(second);
  advance(next_tile, next_stage);
  if constexpr (STAGES == 2) {
    put(1);
    fetch(next_tile, next_stage);
    advance(next_tile, next_stage);
  }
  weights(c1, c0, second), weights(c1, c1, second), weights(c1, c2, second), weights(c1, c3, second);
  if constexpr (RESIDENT) {
    put_scales(1);
    lds_barrier();
#pragma unroll
    for (int B = 0; B < 2; ++B)
#pragma unroll
      for (int i = 0; i < VT; ++i) sw[B][i] = lds_w[B][wv][i][lane];
  }
  for (int it = 0; it < turns; it += 2) {
    turn(c0);
    if (it + 1 < turns) turn(c1);
  }
}

// ---- host ------------------------------------------------------------------------------

inline bool float_rows(int32_t dt) { return dt == RRL_F32 || dt == RRL_BF16 || dt == RRL_F16; }

// A grid's threads are counted in 32 bits.
inline bool blocks_fit(int64_t R, int64_t H) {
  return R <= ((int64_t)1 << 31) && H <= ((int64_t)1 << 31) &&
         R * (padded(H) / kBlock) < ((int64_t)1 << 30) - kQT;
}

template <class Tag, class Order>
int launch_quantize(const void* x, int64_t R, int64_t H, int64_t ld, const Order& order,
                    uint8_t* codes, uint8_t* scales, hipStream_t st) {
  const int64_t blocks = padded(H) / kBlock;
  hipLaunchKernelGGL((mxfp4_quantize_kernel<Tag, Order>),
                     dim3((uint32_t)((R * blocks * 4 + kQT - 1) / kQT)), dim3(kQT), 0, st,
                     static_cast<const char*>(x), R, H, ld, (uint32_t)blocks, order, codes, scales);
  return check_launch("mxfp4_quantize_kernel");
}

template <class Order>
int quantize_any(const void* x, int32_t dt, int64_t R, int64_t H, int64_t ld, const Order& order,
                 uint8_t* codes, uint8_t* scales, hipStream_t st) {
  if (dt == RRL_F32) return launch_quantize<TagF32>(x, R, H, ld, order, codes, scales, st);
  if (dt == RRL_BF16) return launch_quantize<TagBF16>(x, R, H, ld, order, codes, scales, st);
  return launch_quantize<TagF16>(x, R, H, ld, order, codes, scales, st);
}

template <class Tag>
int launch_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t R, int64_t H, void* out,
                      hipStream_t st) {
  constexpr int SZ = 16 / Pack16<Tag>::EPV;
  const int64_t blocks = padded(H) / kBlock;
  const int vec = (uintptr_t)out % 16 == 0 && H % 8 == 0 && H * SZ % 16 == 0;
  hipLaunchKernelGGL(mxfp4_dequantize_kernel<Tag>,
                     dim3((uint32_t)((R * blocks * 4 + kQT - 1) / kQT)), dim3(kQT), 0, st, codes,
                     scales, R, H, (uint32_t)blocks, static_cast<char*>(out), vec);
  return check_launch("mxfp4_dequantize_kernel");
}

struct LinearLayout {
  int64_t fragments, steps, stages;
  size_t scales, total;
};
inline LinearLayout linear_layout(int64_t M, int64_t H) {
  LinearLayout l;
  l.fragments = (M + 15) / 16;
  l.steps = padded(H) / kDepth;
  l.stages = (l.steps + kStage - 1) / kStage;
  l.scales = (size_t)(l.fragments * l.steps) * 1024;
  l.total = l.scales + (size_t)(l.fragments * l.stages) * 256;
  return l;
}

template <int VT, int NT>
int launch_linear(LinearArgs a, hipStream_t st) {
  const int64_t slabs = (a.N + 16 * VT * kLinWaves - 1) / (16 * VT * kLinWaves);
  a.tiles = (a.fragments + NT - 1) / NT;
  // workgroups for four rounds of two on each of the 256 CUs
  a.groups = (int32_t)max((int64_t)1, min((int64_t)a.tiles, 2048 / slabs));
  const int64_t blocks = (slabs + 7) / 8 * 8 * a.groups;
  RRL_REQUIRE(blocks < ((int64_t)1 << 32) / (64 * kLinWaves), RRL_EINVAL,
              "rrl_mxfp4_linear: too many weight rows");
  const dim3 grid((uint32_t)blocks), threads(64 * kLinWaves);
  if (a.stages == 1) hipLaunchKernelGGL((mxfp4_linear_kernel<VT, NT, 1>), grid, threads, 0, st, a);
  else if (a.stages == 2 && NT <= 4)  // four buffers of more fragments leave room for one workgroup
    hipLaunchKernelGGL((mxfp4_linear_kernel<VT, NT <= 4 ? NT : 1, 2>), grid, threads, 0, st, a);
  else hipLaunchKernelGGL((mxfp4_linear_kernel<VT, NT, 0>), grid, threads, 0, st, a);
  return check_launch("mxfp4_linear_kernel");
}

// Activation fragments of a tile: with narrow slabs as many as make the tiles even, for
// each tile reads the slab again (130 x 50,257 x 2080, nine fragments: 64, 46 and 37 us
// with 1, 2 and 4).
template <int VT>
int launch_linear(const LinearArgs& a, hipStream_t st) {
  if (a.fragments <= 1) return launch_linear<VT, 1>(a, st);
  if (a.fragments <= 2) return launch_linear<VT, 2>(a, st);
  if constexpr (VT == 2) {
    const int tiles = (a.fragments + 5) / 6, need = (a.fragments + tiles - 1) / tiles;
    if (need == 3) return launch_linear<VT, 3>(a, st);
    if (need == 5) return launch_linear<VT, 5>(a, st);
    if (need == 6) return launch_linear<VT, 6>(a, st);
  }
  return launch_linear<VT, 4>(a, st);
}

}  // namespace
}  // namespace rrl

using namespace rrl;

extern "C" int rrl_mxfp4_quantize(const void* x, int32_t dtype, int64_t R, int64_t H, int64_t ld,
                                  uint8_t* codes, uint8_t* scales, void* stream) {
  clear_error();
  RRL_REQUIRE(float_rows(dtype), RRL_EDTYPE,
              "rrl_mxfp4_quantize: entries must be float32, bfloat16 or float16");
  RRL_REQUIRE(R >= 0 && H >= 0, RRL_EINVAL, "rrl_mxfp4_quantize: negative size");
  if (R == 0 || H == 0) return RRL_OK;
  RRL_REQUIRE(blocks_fit(R, H), RRL_EINVAL, "rrl_mxfp4_quantize: 2^30 blocks of 32 or more");
  RRL_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr, RRL_EINVAL,
              "rrl_mxfp4_quantize: null operand");
  RRL_REQUIRE(R <= 1 || ld >= 0, RRL_EINVAL, "rrl_mxfp4_quantize: negative row stride");
  RRL_REQUIRE((uintptr_t)x % dtype_size(dtype) == 0 && (uintptr_t)codes % 16 == 0, RRL_EALIGN,
              "rrl_mxfp4_quantize: a pointer is not aligned (codes: 16 bytes)");
  return quantize_any(x, dtype, R, H, ld, RowOrder{(uint32_t)(padded(H) / kBlock)}, codes, scales,
                      as_stream(stream));
}

extern "C" int rrl_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t R,
                                    int64_t H, void* out, int32_t dtype, void* stream) {
  clear_error();
  RRL_REQUIRE(float_rows(dtype), RRL_EDTYPE,
              "rrl_mxfp4_dequantize: values must be float32, bfloat16 or float16");
  RRL_REQUIRE(R >= 0 && H >= 0, RRL_EINVAL, "rrl_mxfp4_dequantize: negative size");
  if (R == 0 || H == 0) return RRL_OK;
  RRL_REQUIRE(blocks_fit(R, H), RRL_EINVAL, "rrl_mxfp4_dequantize: 2^30 blocks of 32 or more");
  RRL_REQUIRE(out != nullptr && codes != nullptr && scales != nullptr, RRL_EINVAL,
              "rrl_mxfp4_dequantize: null operand");
  RRL_REQUIRE((uintptr_t)out % dtype_size(dtype) == 0 && (uintptr_t)codes % 16 == 0, RRL_EALIGN,
              "rrl_mxfp4_dequantize: a pointer is not aligned (codes: 16 bytes)");
  hipStream_t st = as_stream(stream);
  if (dtype == RRL_F32) return launch_dequantize<TagF32>(codes, scales, R, H, out, st);
  if (dtype == RRL_BF16) return launch_dequantize<TagBF16>(codes, scales, R, H, out, st);
  return launch_dequantize<TagF16>(codes, scales, R, H, out, st);
}

extern "C" size_t rrl_mxfp4_linear_workspace_bytes(int64_t M, int64_t H) {
  if (M < 0 || H < 0 || !blocks_fit(M, H)) return 0;
  return linear_layout(M, H).total;
}

extern "C" int rrl_mxfp4_linear(const void* x, int32_t dtype, int64_t M, int64_t H, int64_t x_ld,
                                const uint8_t* codes, const uint8_t* scales, int64_t N, void* out,
                                int32_t out_dtype, void* workspace, void* stream) {
  clear_error();
  RRL_REQUIRE(float_rows(dtype) && float_rows(out_dtype), RRL_EDTYPE,
              "rrl_mxfp4_linear: activations and outputs must be float32, bfloat16 or float16");
  RRL_REQUIRE(M >= 0 && H >= 1 && N >= 0, RRL_EINVAL, "rrl_mxfp4_linear: bad size");
  if (M == 0 || N == 0) return RRL_OK;
  // a slab's offsets are 32-bit
  RRL_REQUIRE(blocks_fit(M, H) && blocks_fit(N, H) && H <= (1 << 22), RRL_EINVAL,
              "rrl_mxfp4_linear: 2^30 blocks of 32 or more, or rows of over 2^22 entries");
  RRL_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr && out != nullptr &&
                  workspace != nullptr,
              RRL_EINVAL, "rrl_mxfp4_linear: null operand");
  RRL_REQUIRE(M <= 1 || x_ld >= 0, RRL_EINVAL, "rrl_mxfp4_linear: negative row stride");
  RRL_REQUIRE((uintptr_t)x % dtype_size(dtype) == 0 && (uintptr_t)out % dtype_size(out_dtype) == 0 &&
                  (uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 4 == 0 &&
                  (uintptr_t)workspace % 16 == 0,
              RRL_EALIGN, "rrl_mxfp4_linear: a pointer is not aligned (codes: 16 bytes, scales: 4)");
  hipStream_t st = as_stream(stream);
  const LinearLayout l = linear_layout(M, H);
  uint8_t* ac = static_cast<uint8_t*>(workspace);
  uint8_t* as = ac + l.scales;
  const FragmentOrder order{(uint32_t)l.steps, (uint32_t)l.stages};
  if (int rc = quantize_any(x, dtype, M, H, x_ld, order, ac, as, st)) return rc;
  LinearArgs a;
  a.ac = reinterpret_cast<const u32x4*>(ac);
  a.as = reinterpret_cast<const uint32_t*>(as);
  a.wc = codes;
  a.ws = scales;
  a.M = M;
  a.N = N;
  a.steps = (int32_t)l.steps;
  a.stages = (int32_t)l.stages;
  a.fragments = (int32_t)l.fragments;
  a.out = static_cast<char*>(out);
  a.out_dtype = out_dtype;
  // a tile's rows are addressed with 32 bits: up to 64 of these, or up to 96 with slabs of
  // 128 weight rows, which are taken for tiles of over 64 only while N is under 2^19
  const int64_t row = N * (int64_t)dtype_size(out_dtype);
  a.aligned = N % 8 == 0 && (uintptr_t)out % 16 == 0 && row < (1 << 25);
  // 128 weight rows to a workgroup, or 256 where those make work enough for rounds of
  // them.  Us with 128 / 256, by activation rows: 151,936 x 1024: 16 17.4 / 19.9, 128 32.8 /
  // 37.0, 256 68.3 / 59.5, 384 87.2 / 68.0, 400 (the border) 96.1 / 73.8, 1024 204 / 128;
  // 50,257 x 1024: 512 62.8 / 51.8, 2048 171 / 130; 151,936 x 2048, whose weights do not
  // stay in registers: 64 53.0 / 60.3, 256 116 / 145, 400 168 / 209, 512 203 / 234.  The
  // border lies late for weights that stay, and early for those that do not.
  return N * ((l.fragments + 3) / 4) < (1 << 20) ? launch_linear<2>(a, st) : launch_linear<4>(a, st);
}
