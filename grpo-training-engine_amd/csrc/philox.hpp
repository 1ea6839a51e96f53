// Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011, "Parallel random numbers: as easy
// as 1, 2, 3") and the dropout mask drawn from it.
//
// Element e of a tensor (its row-major index) is dropped iff u(e) < threshold, where
// u(e) are 16 bits of the block with counter (e / 8, offset) and key seed: word
// e % 8 / 2, low half first. Kept elements are scaled by 65536 / (65536 - threshold),
// the inverse of the share that is kept. 16 bits an element make one block serve the
// eight values of a 16-byte load; p is met to within 2^-17. The mask depends on (seed,
// offset) and e alone, so every kernel that needs it makes it again.
#pragma once

#include "common.hpp"

namespace grpo {

struct Dropout {
  const int64_t* rng;  // device: seed, offset
  uint32_t threshold;  // of 65536; 0: nothing is dropped
  float scale;         // 65536 / (65536 - threshold)
};

// seed and offset, wave-uniform
struct DropKey {
  uint32_t k0, k1, o0, o1;
};

__device__ __forceinline__ DropKey drop_key(const int64_t* rng) {
  const uint64_t seed = (uint64_t)load_uniform(rng), off = (uint64_t)load_uniform(rng + 1);
  return DropKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)off, (uint32_t)(off >> 32)};
}

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);  // one instruction of gfx950
}

// The four words of block i: twenty 32 x 32 -> 64 products (a quarter of the full rate) and
// twenty three-way xors.
__device__ __forceinline__ uint4 philox(uint64_t i, const DropKey& key) {
  uint32_t c0 = (uint32_t)i, c1 = (uint32_t)(i >> 32), c2 = key.o0, c3 = key.o1;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = xor3((uint32_t)(q >> 32), c1, k0);
    c1 = (uint32_t)q;
    c2 = xor3((uint32_t)(p >> 32), c3, k1);
    c3 = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Whether element j (0..7) of the block is kept. Both halves are compared in the high
// 16 bits: w >= t << 16 is (w >> 16) >= t.
__device__ __forceinline__ bool drop_keeps(const uint4& w, int j, uint32_t threshold) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  return (j & 1 ? v[j >> 1] : v[j >> 1] << 16) >= threshold << 16;
}

// Eight 16-bit values: dt(x * scale), or 0 (whatever the value) where dropped.
template <bool F16>
__device__ __forceinline__ uint4 drop8(uint4 x, const uint4& w, uint32_t threshold, float scale) {
  const uint32_t d[4] = {x.x, x.y, x.z, x.w};
  uint32_t o[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float lo = e2f<F16>((uint16_t)d[q]) * scale;
    const float hi = e2f<F16>((uint16_t)(d[q] >> 16)) * scale;
    o[q] = pack_e2<F16>(drop_keeps(w, 2 * q, threshold) ? lo : 0.f,
                        drop_keeps(w, 2 * q + 1, threshold) ? hi : 0.f);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Eight 16-bit values, 0 (whatever the value) where dropped and unscaled where kept, for a
// threshold above 0. Two halves at once: w >= t is w - (t - 1) >= 1 in saturating 16 bits.
__device__ __forceinline__ uint4 mask8(uint4 x, const uint4& w, uint32_t threshold) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const u16x2 below = (u16x2)(uint16_t)(threshold - 1), one = (u16x2)(uint16_t)1;
  auto kept = [&](uint32_t v, uint32_t u) __attribute__((always_inline)) {
    const u16x2 on = __builtin_elementwise_min(
        __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, u), below), one);
    return v & __builtin_bit_cast(uint32_t, (u16x2)(-on));
  };
  return make_uint4(kept(x.x, w.x), kept(x.y, w.y), kept(x.z, w.z), kept(x.w, w.w));
}

// Checks of a C entry point; *out is valid when it returns GRPO_OK.
inline int drop_args(const int64_t* rng, double p, Dropout* out) {
  if (!(p >= 0.0 && p < 1.0)) return einval("dropout p must lie in [0, 1)");
  const uint32_t t = (uint32_t)(p * 65536.0 + 0.5);
  if (t >= 65536u) return einval("dropout p too close to 1 (it is met to within 2^-17)");
  if (t && (!rng || (reinterpret_cast<uintptr_t>(rng) & 7u)))
    return einval("dropout needs two 8-byte aligned int64 (seed, offset) on the device");
  *out = Dropout{rng, t, (float)(65536.0 / (65536.0 - t))};
  return GRPO_OK;
}

}  // namespace grpo
