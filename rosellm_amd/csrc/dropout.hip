// Dropout from a counter-based generator: y = residual + kept ? x / (1 - p) : 0, the
// mask drawn where it is needed (dropout_common.hpp) and never stored.  The gradient is
// the same kernel on d y.
//
// A thread takes one group of eight entries.  131,072 x 1024 bfloat16: 87 us without a
// residual (537 MB, 6.2 TB/s) and 143 with one (805 MB, 5.6 TB/s), bound by memory; the
// generator's 51 us of issue run beside it.  Loads and stores past the caches
// measured the same (90 and 122 to 125 us within a step, 15 to 17 for 16,384 rows).
#include "dropout_common.hpp"
#include "vocab_weights.hpp"

namespace rrl {
namespace {

constexpr int kDT = 256;

struct DropArgs {
  const char *x, *res;  // res may be null
  char* out;            // contiguous [rows, cols]
  int64_t cols, x_ld, r_ld;
  int64_t groups, per_row;
  Drop drop;
};

// Entries i..i+7 of a row of n, zeros past its end; any element may be the first.
template <class Tag>
__device__ __forceinline__ void load_group(const char* row, int64_t i, int64_t n, float (&v)[8]) {
  constexpr int EPV = Pack16<Tag>::EPV, SZ = 16 / EPV;
  if (i + 8 <= n) {
#pragma unroll
    for (int h = 0; h < 8 / EPV; ++h) {
      float part[EPV];
      Pack16<Tag>::unpack(reinterpret_cast<const Any16*>(row + i * SZ)[h].v, part);
#pragma unroll
      for (int k = 0; k < EPV; ++k) v[h * EPV + k] = part[k];
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = i + k < n ? load_entry<Tag>(row, i + k) : 0.0f;
}
template <class Tag>
__device__ __forceinline__ void store_group(char* row, int64_t i, int64_t n, const float (&v)[8]) {
  constexpr int EPV = Pack16<Tag>::EPV, SZ = 16 / EPV;
  if (i + 8 <= n) {
#pragma unroll
    for (int h = 0; h < 8 / EPV; ++h) {
      float part[EPV];
#pragma unroll
      for (int k = 0; k < EPV; ++k) part[k] = v[h * EPV + k];
      reinterpret_cast<Any16*>(row + i * SZ)[h].v = Pack16<Tag>::pack(part);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (i + k < n) {
      if constexpr (SZ == 4) reinterpret_cast<float*>(row)[i + k] = v[k];
      else reinterpret_cast<uint16_t*>(row)[i + k] = (uint16_t)Pack16<Tag>::pack_one(v[k]);
    }
}

template <class Tag>
__global__ __launch_bounds__(kDT) void dropout_kernel(DropArgs a) {
  constexpr int SZ = 16 / Pack16<Tag>::EPV;
  const int64_t g = (int64_t)blockIdx.x * kDT + threadIdx.x;
  if (g >= a.groups) return;
  const int64_t row = (uint32_t)g / (uint32_t)a.per_row;  // there are fewer than 2^32
  const int64_t i = (g - row * a.per_row) * 8;
  float v[8];
  load_group<Tag>(a.x + row * a.x_ld * SZ, i, a.cols, v);
  const uint32_t keep = a.drop.keep_bits((uint64_t)g, a.drop.counter());
  if (a.res) {
    float r[8];
    load_group<Tag>(a.res + row * a.r_ld * SZ, i, a.cols, r);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = keep >> k & 1 ? __builtin_fmaf(v[k], a.drop.scale, r[k]) : r[k];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = keep >> k & 1 ? v[k] * a.drop.scale : 0.0f;
  }
  store_group<Tag>(a.out + row * a.cols * SZ, i, a.cols, v);
}

template <class Tag>
int launch_dropout(const DropArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(dropout_kernel<Tag>, dim3((uint32_t)((a.groups + kDT - 1) / kDT)), dim3(kDT), 0, st, a);
  return check_launch("dropout_kernel");
}

}  // namespace
}  // namespace rrl

using namespace rrl;

extern "C" int rrl_dropout(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t x_ld,
                           const void* residual, int64_t r_ld, const rrl_dropout_params* params,
                           void* out, void* stream) {
  clear_error();
  RRL_REQUIRE(dtype == RRL_F32 || dtype == RRL_BF16 || dtype == RRL_F16, RRL_EDTYPE,
              "rrl_dropout: entries must be float32, bfloat16 or float16");
  RRL_REQUIRE(rows >= 0 && cols >= 0, RRL_EINVAL, "rrl_dropout: negative size");
  RRL_REQUIRE(params != nullptr, RRL_EINVAL, "rrl_dropout: null operand");
  DropArgs a;
  if (int rc = make_drop(params, a.drop, "rrl_dropout")) return rc;
  if (rows == 0 || cols == 0) return RRL_OK;
  RRL_REQUIRE(x != nullptr && out != nullptr, RRL_EINVAL, "rrl_dropout: null operand");
  RRL_REQUIRE(rows <= 1 || (x_ld >= 0 && r_ld >= 0), RRL_EINVAL, "rrl_dropout: negative row stride");
  // a grid's threads are counted in 32 bits
  const int64_t most = ((int64_t)1 << 32) - kDT;
  RRL_REQUIRE(cols <= 8 * most && rows <= most / ((cols + 7) / 8), RRL_EINVAL,
              "rrl_dropout: 2^32 groups of eight entries or more");
  const size_t size = dtype_size(dtype);
  RRL_REQUIRE((uintptr_t)x % size == 0 && (uintptr_t)residual % size == 0 && (uintptr_t)out % size == 0,
              RRL_EALIGN, "rrl_dropout: a pointer is not aligned to its element");
  a.x = static_cast<const char*>(x);
  a.res = static_cast<const char*>(residual);
  a.out = static_cast<char*>(out);
  a.cols = cols;
  a.x_ld = x_ld;
  a.r_ld = r_ld;
  a.per_row = (cols + 7) / 8;
  a.groups = rows * a.per_row;
  hipStream_t st = as_stream(stream);
  if (dtype == RRL_F32) return launch_dropout<TagF32>(a, st);
  if (dtype == RRL_BF16) return launch_dropout<TagBF16>(a, st);
  return launch_dropout<TagF16>(a, st);
}
