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

// Four lanes per block, eight entries each.
template <class Tag>
__global__ __launch_bounds__(kQT) void mxfp4_quantize_kernel(const char* __restrict__ x, int64_t R,
                                                             int64_t H, int64_t ld, uint32_t blocks,
                                                             uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales) {
  constexpr int SZ = 16 / Pack16<Tag>::EPV;
  const int64_t id = ((int64_t)blockIdx.x * kQT + threadIdx.x) / 4;
  const int part = threadIdx.x & 3;
  if (id >= R * blocks) return;
  const int64_t r = id / blocks, b = id % blocks;
  float v[8];
  load8<Tag>(x + r * ld * SZ, b * kBlock + part * 8, H, v);
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
  m = max(m, (uint32_t)dpp_i<kDppXor1>((int)m));
  m = max(m, (uint32_t)dpp_i<kDppXor2>((int)m));
  const uint32_t byte = scale_byte(m);
  reinterpret_cast<uint32_t*>(codes)[id * 4 + part] = codes8(v, byte);
  if (part == 0) scales[id] = (uint8_t)byte;
}

// The value of a code times 2^(byte - 127).
__device__ __forceinline__ float code_value(uint32_t code, uint32_t byte) {
  const uint32_t mag = code & 7;
  // e2m1: exponent bias 1, one bit of mantissa; twice the value is a whole number
  const int twice = mag < 2 ? (int)mag : (2 + (int)(mag & 1)) << ((mag >> 1) - 1);
  const float v = ldexpf((float)twice, (int)byte - 128);
  return byte == 255 ? __builtin_nanf("") : ((code & 8) ? -v : v);
}

template <class Tag>
__global__ __launch_bounds__(kQT) void mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales,
                                                               int64_t R, int64_t H, uint32_t blocks,
                                                               char* __restrict__ out, int vec) {
  constexpr int EPV = Pack16<Tag>::EPV, SZ = 16 / EPV;
  const int64_t id = ((int64_t)blockIdx.x * kQT + threadIdx.x) / 4;
  const int part = threadIdx.x & 3;
  if (id >= R * blocks) return;
  const int64_t r = id / blocks, c = (id % blocks) * kBlock + part * 8;
  if (c >= H) return;
  const uint32_t word = reinterpret_cast<const uint32_t*>(codes)[id * 4 + part];
  const uint32_t byte = scales[id];
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = code_value((word >> (4 * k)) & 15, byte);
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

// D += A B^T over 128 entries: lane l holds 32 consecutive entries (block l / 16)
// of row l % 16 of each operand and their scale; it receives rows 4 (l / 16) + i
// of A, row l % 16 of B.
__device__ __forceinline__ f32x4 mfma_fp4(const u32x4& a, uint32_t sa, const u32x4& b, uint32_t sb,
                                          const f32x4& c) {
  const i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8 bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

constexpr int kLinWaves = 4;

// A wave: VT x 16 weight rows times NT x 16 activation rows.
template <class Out, int VT, int NT>
__global__ __launch_bounds__(64 * kLinWaves) void mxfp4_linear_kernel(
    const uint8_t* __restrict__ ac, const uint8_t* __restrict__ as, int64_t M,
    const uint8_t* __restrict__ wc, const uint8_t* __restrict__ wsc, int64_t N, int64_t P,
    char* __restrict__ out) {
  constexpr int SZ = 16 / Pack16<Out>::EPV;
  const int lane = threadIdx.x & 63, r16 = lane & 15, blk = lane >> 4;
  const int64_t n0 = ((int64_t)blockIdx.x * kLinWaves + (threadIdx.x >> 6)) * (16 * VT);
  const int64_t m0 = (int64_t)blockIdx.y * (16 * NT);
  if (n0 >= N) return;
  int64_t wr[VT], ar[NT];  // rows past the end read the last one, and are not stored
#pragma unroll
  for (int i = 0; i < VT; ++i) wr[i] = min(n0 + 16 * i + r16, N - 1);
#pragma unroll
  for (int j = 0; j < NT; ++j) ar[j] = min(m0 + 16 * j + r16, M - 1);
  f32x4 acc[VT][NT] = {};
  for (int64_t k = 0; k < P; k += kDepth) {
    u32x4 w[VT], a[NT];
    uint32_t sw[VT], sa[NT];
    const int64_t kb = k / kBlock + blk;
#pragma unroll
    for (int i = 0; i < VT; ++i) {
      w[i] = *reinterpret_cast<const u32x4*>(wc + wr[i] * (P / 2) + kb * 16);
      sw[i] = wsc[wr[i] * (P / kBlock) + kb];
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      a[j] = *reinterpret_cast<const u32x4*>(ac + ar[j] * (P / 2) + kb * 16);
      sa[j] = as[ar[j] * (P / kBlock) + kb];
    }
#pragma unroll
    for (int i = 0; i < VT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = mfma_fp4(w[i], sw[i], a[j], sa[j], acc[i][j]);
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t m = m0 + 16 * j + r16;
    if (m >= M) continue;
#pragma unroll
    for (int i = 0; i < VT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t n = n0 + 16 * i + 4 * blk + k;
        if (n >= N) continue;
        char* dst = out + (m * N + n) * SZ;
        if constexpr (SZ == 4) *reinterpret_cast<float*>(dst) = acc[i][j][k];
        else *reinterpret_cast<uint16_t*>(dst) = (uint16_t)Pack16<Out>::pack_one(acc[i][j][k]);
      }
  }
}

// ---- host ------------------------------------------------------------------------------

inline bool float_rows(int32_t dt) { return dt == RRL_F32 || dt == RRL_BF16 || dt == RRL_F16; }

// A grid's threads are counted in 32 bits.
inline bool blocks_fit(int64_t R, int64_t H) {
  return R <= ((int64_t)1 << 31) && H <= ((int64_t)1 << 31) &&
         R * (padded(H) / kBlock) < ((int64_t)1 << 30) - kQT;
}

template <class Tag>
int launch_quantize(const void* x, int64_t R, int64_t H, int64_t ld, uint8_t* codes, uint8_t* scales,
                    hipStream_t st) {
  const int64_t blocks = padded(H) / kBlock;
  hipLaunchKernelGGL(mxfp4_quantize_kernel<Tag>, dim3((uint32_t)((R * blocks * 4 + kQT - 1) / kQT)),
                     dim3(kQT), 0, st, static_cast<const char*>(x), R, H, ld, (uint32_t)blocks, codes,
                     scales);
  return check_launch("mxfp4_quantize_kernel");
}

int quantize_any(const void* x, int32_t dt, int64_t R, int64_t H, int64_t ld, uint8_t* codes,
                 uint8_t* scales, hipStream_t st) {
  if (dt == RRL_F32) return launch_quantize<TagF32>(x, R, H, ld, codes, scales, st);
  if (dt == RRL_BF16) return launch_quantize<TagBF16>(x, R, H, ld, codes, scales, st);
  return launch_quantize<TagF16>(x, R, H, ld, codes, scales, st);
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

template <class Out>
int launch_linear(const uint8_t* ac, const uint8_t* as, int64_t M, const uint8_t* wc,
                  const uint8_t* wsc, int64_t N, int64_t P, void* out, hipStream_t st) {
  auto grid = [&](int vt, int nt) {
    const int64_t rows = 16 * vt * kLinWaves;
    return dim3((uint32_t)((N + rows - 1) / rows), (uint32_t)((M + 16 * nt - 1) / (16 * nt)));
  };
  if (M <= 16) {
    hipLaunchKernelGGL((mxfp4_linear_kernel<Out, 2, 1>), grid(2, 1), dim3(64 * kLinWaves), 0, st, ac,
                       as, M, wc, wsc, N, P, static_cast<char*>(out));
  } else {
    hipLaunchKernelGGL((mxfp4_linear_kernel<Out, 4, 4>), grid(4, 4), dim3(64 * kLinWaves), 0, st, ac,
                       as, M, wc, wsc, N, P, static_cast<char*>(out));
  }
  return check_launch("mxfp4_linear_kernel");
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
  return quantize_any(x, dtype, R, H, ld, codes, scales, as_stream(stream));
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
  const int64_t P = padded(H);
  return (size_t)(M * (P / 2) + (M * (P / kBlock) + 255) / 256 * 256);
}

extern "C" int rrl_mxfp4_linear(const void* x, int32_t dtype, int64_t M, int64_t H, int64_t x_ld,
                                const uint8_t* codes, const uint8_t* scales, int64_t N, void* out,
                                int32_t out_dtype, void* workspace, void* stream) {
  clear_error();
  RRL_REQUIRE(float_rows(dtype) && float_rows(out_dtype), RRL_EDTYPE,
              "rrl_mxfp4_linear: activations and outputs must be float32, bfloat16 or float16");
  RRL_REQUIRE(M >= 0 && H >= 1 && N >= 0, RRL_EINVAL, "rrl_mxfp4_linear: bad size");
  if (M == 0 || N == 0) return RRL_OK;
  RRL_REQUIRE(blocks_fit(M, H) && blocks_fit(N, H) && M <= 65535 * 16, RRL_EINVAL,
              "rrl_mxfp4_linear: 2^30 blocks of 32 or more, or over 1,048,560 activation rows");
  RRL_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr && out != nullptr &&
                  workspace != nullptr,
              RRL_EINVAL, "rrl_mxfp4_linear: null operand");
  RRL_REQUIRE(M <= 1 || x_ld >= 0, RRL_EINVAL, "rrl_mxfp4_linear: negative row stride");
  RRL_REQUIRE((uintptr_t)x % dtype_size(dtype) == 0 && (uintptr_t)out % dtype_size(out_dtype) == 0 &&
                  (uintptr_t)codes % 16 == 0 && (uintptr_t)workspace % 16 == 0,
              RRL_EALIGN, "rrl_mxfp4_linear: a pointer is not aligned (codes: 16 bytes)");
  hipStream_t st = as_stream(stream);
  const int64_t P = padded(H);
  uint8_t* ac = static_cast<uint8_t*>(workspace);
  uint8_t* as = ac + M * (P / 2);
  if (int rc = quantize_any(x, dtype, M, H, x_ld, ac, as, st)) return rc;
  if (out_dtype == RRL_F32) return launch_linear<TagF32>(ac, as, M, codes, scales, N, P, out, st);
  if (out_dtype == RRL_BF16) return launch_linear<TagBF16>(ac, as, M, codes, scales, N, P, out, st);
  return launch_linear<TagF16>(ac, as, M, codes, scales, N, P, out, st);
}
