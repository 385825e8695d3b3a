// What choosing a token from a row of logits is made of, shared by the kernel that takes them as they are (sampling.hip) and the
// one that applies a request's rules on the way (logit_rules.hip): the noise and the comparison of one candidate.
#pragma once
#include "common.hpp"

__device__ __forceinline__ uint32_t fmix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x85EBCA6Bu;
  x ^= x >> 13;
  x *= 0xC2B2AE35u;
  x ^= x >> 16;
  return x;
}

// A candidate's value after temperature and noise.
__device__ __forceinline__ float sample_value(float z, int v, bool noisy, float inv_t, uint32_t key) {
  if (noisy) {
    const uint32_t x = fmix32(key ^ fmix32((uint32_t)v + 0x9E3779B9u));
    const float u = ((float)(x >> 9) + 0.5f) * 1.1920928955078125e-07f;   // 2^-23
    z = fmaf(z, inv_t, -logf(-logf(u)));
  }
  return z;
}

// One candidate, kept if it beats the best so far.
__device__ __forceinline__ void sample_consider(float z, int v, bool noisy, float inv_t, uint32_t key, float& bv, int& bi) {
  z = sample_value(z, v, noisy, inv_t, key);
  if (z > bv || (z == bv && v < bi)) { bv = z; bi = v; }
}

// (seed, counter) to what the noise of a row is drawn with
__device__ __forceinline__ uint32_t sample_key(unsigned long long seed, int counter) {
  return fmix32(fmix32(fmix32((uint32_t)seed) ^ (uint32_t)(seed >> 32)) ^ (uint32_t)counter);
}

// the better of two candidates: the larger value, the lower index among equals
__device__ __forceinline__ void sample_better(float ov, int oi, float& bv, int& bi) {
  if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
}
