// Helpers shared by the tensor-core attention kernels: packed fp32 arithmetic
// of their softmax passes and the position in a ring of pipeline stages.
#pragma once

#include <stdint.h>

namespace nf {

// Pairs of fp32 values in one 64-bit register, for the packed fp32x2
// instructions of sm_100 (two FMAs or adds per issue).
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A ring position: stage index and the parity of its current fill.
struct Ring {
  int st = 0;
  uint32_t ph = 0;
  __device__ void next(int n) {
    if (++st == n) {
      st = 0;
      ph ^= 1;
    }
  }
  __device__ Ring ahead(int k, int n) const {  // the position k fills later
    Ring r;
    const int t = st + k;
    r.st = t % n;
    r.ph = ph ^ ((uint32_t)(t / n) & 1u);
    return r;
  }
};

}  // namespace nf
