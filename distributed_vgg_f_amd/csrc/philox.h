// The counter-based generator of dropout: Philox4x32-10. Element i of a
// tensor (row-major order) takes word i & 3 of the block at counter
// (i >> 2, offset) under key (seed), so a mask is a function of (i, p, seed,
// offset) alone: the backward pass and any fused epilogue draw the same one
// again and nothing is stored.
#pragma once

#include "common.h"

namespace dvgg {

// One round is two 32x32 -> 64 products. Written as 64-bit products so that
// each becomes one v_mad_u64_u32 (high and low word together) instead of a
// v_mul_hi_u32 and a v_mul_lo_u32, which run at the same quarter rate.
DEV void philox_round(u32& c0, u32& c1, u32& c2, u32& c3, u32 k0, u32 k1) {
  unsigned long long a = (unsigned long long)c0 * 0xD2511F53u;
  unsigned long long b = (unsigned long long)c2 * 0xCD9E8D57u;
  c0 = u32(b >> 32) ^ c1 ^ k0;
  c2 = u32(a >> 32) ^ c3 ^ k1;
  c1 = u32(b);
  c3 = u32(a);
}

DEV u32x4 philox(u32 lo, u32 hi, u32 key0, u32 key1) {
  u32 c0 = lo, c1 = hi, c2 = key1, c3 = 0x243F6A88u;
  u32 k0 = key0, k1 = 0xBB67AE85u;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    philox_round(c0, c1, c2, c3, k0, k1);
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}

// What a kernel needs to draw a mask. An element stays where its word, as a
// 32-bit float times 2^-32, is not below p; that test is monotone in the
// word, so the host turns p into the first word that stays and the kernels
// compare whole numbers.
struct DropArgs {
  u32 first;              // first word that stays
  float scale;            // 1 / (1 - p)
  u32 seed, offset;
  const i64* offset_ptr;  // read on the device in place of `offset` if given

  DEV u32 off() const { return offset_ptr ? u32(*offset_ptr) : offset; }
};

// Bits 0..3: which of the elements 4*block .. 4*block+3 stay.
DEV u32 keep4(const DropArgs& d, u32 off, i64 block) {
  u32x4 r = philox(u32(block), u32(block >> 32), d.seed, off);
  return u32(r[0] >= d.first) | u32(r[1] >= d.first) << 1 |
         u32(r[2] >= d.first) << 2 | u32(r[3] >= d.first) << 3;
}

inline DropArgs drop_args(double p, i64 seed, i64 offset,
                          const i64* offset_ptr) {
  float pf = float(p);
  u32 lo = 0, hi = 0xFFFFFFFFu;           // hi stays for every p < 1
  while (lo < hi) {
    u32 mid = lo + (hi - lo) / 2;
    if (float(mid) * 2.3283064365386963e-10f >= pf) hi = mid;
    else lo = mid + 1;
  }
  return DropArgs{hi, float(1.0 / (1.0 - p)), u32(seed), u32(offset),
                  offset_ptr};
}

}  // namespace dvgg
