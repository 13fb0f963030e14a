// Which entries dropout keeps: shared by dropout.hip and adapters.hip, whose input
// is dropped within the product.
//
// The last dimension of x is cut into groups of eight; group i (counted in order, each
// row starting a new one) takes the four words of Philox4x32-10 at counter {i, offset}
// under the key `seed`, 16 bits an entry, the low half of a word first.  An entry is
// kept where its number is at least cut = round(65536 p), and scaled by
// 65536 / (65536 - cut): the probability is p to 2^-17, and the expectation exact.
// With 32 bits an entry the generator alone (about 120 issue slots a call, most of them the
// quarter-rate multiplications) would take longer than the entries' bytes.
#pragma once

#include "philox.hpp"
#include "rrl_common.hpp"

namespace rrl {
namespace {

struct Drop {
  uint64_t offset;
  const int64_t* offset_device;  // added to offset, or null
  uint32_t k0, k1, cut;
  float scale;  // 0 where nothing is kept
  __device__ __forceinline__ uint64_t counter() const {
    return offset + (offset_device ? (uint64_t)*offset_device : 0u);
  }
  // a bit for each of the eight entries of a group: set where it is kept
  __device__ __forceinline__ uint32_t keep_bits(uint64_t group, uint64_t at) const {
    uint32_t c[4] = {(uint32_t)group, (uint32_t)(group >> 32), (uint32_t)at, (uint32_t)(at >> 32)};
    philox4x32_10(c, k0, k1);
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      bits |= (((c[i / 2] >> (16 * (i % 2))) & 0xffffu) >= cut ? 1u : 0u) << i;
    return bits;
  }
};

inline int make_drop(const rrl_dropout_params* p, Drop& d, const char* who) {
  RRL_REQUIRE(p->p >= 0.0 && p->p <= 1.0, RRL_EINVAL,
              std::string(who) + ": the dropout probability must be in [0, 1]");
  RRL_REQUIRE((uintptr_t)p->offset_device % 8 == 0, RRL_EALIGN,
              std::string(who) + ": a pointer is not aligned to its element");
  d.offset = p->offset;
  d.offset_device = p->offset_device;
  d.k0 = (uint32_t)p->seed;
  d.k1 = (uint32_t)(p->seed >> 32);
  d.cut = (uint32_t)nearbyint(p->p * 65536.0);
  d.scale = d.cut < 65536u ? 65536.0f / (float)(65536u - d.cut) : 0.0f;
  return RRL_OK;
}

}  // namespace
}  // namespace rrl
