// Counter-based generator of the sampled training paths (PreNet / conv dropout, zoneout, stochastic rounding): a 32-bit word
// per (seed, stream, step, row, column), and 24 uniform bits of it.  TensorFlow's stateful random ops cannot be reproduced;
// the oracle uses this same function (oracle/t2_oracle.py:rng_u01), TF's arithmetic around it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

__host__ __device__ inline uint32_t t2_mix32(uint32_t x) {
    x ^= x >> 16; x *= 0x7FEB352Du; x ^= x >> 15; x *= 0x846CA68Bu; x ^= x >> 16;
    return x;
}
// the part of the word that does not depend on the column
__host__ __device__ inline uint32_t t2_row_key(uint32_t seed, uint32_t stream, uint32_t t, uint32_t row) {
    uint32_t h = t2_mix32(seed ^ (stream * 0x9E3779B9u));
    h = t2_mix32(h ^ (t * 0x85EBCA6Bu + 0x165667B1u));
    return t2_mix32(h ^ (row * 0xC2B2AE35u + 0x27D4EB2Fu));
}
__host__ __device__ inline uint32_t t2_word(uint32_t row_key, uint32_t col) { return t2_mix32(row_key ^ (col * 0x9E3779B1u + 0x85EBCA77u)); }
__host__ __device__ inline float t2_u01(uint32_t seed, uint32_t stream, uint32_t t, uint32_t row, uint32_t col) {
    return (float)(t2_word(t2_row_key(seed, stream, t, row), col) >> 8) * (1.0f / 16777216.0f);
}
