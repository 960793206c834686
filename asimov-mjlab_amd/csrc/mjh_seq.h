// mjh_seq.h — what the policy-memory kernels share (mjh_scan.hip, mjh_resnorm.hip):
// element types, vector loads, exp / sigmoid in float32, the dropout bits, host-side checks.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/mjh_abi.h"
#include "mjh_rng.h"

namespace mjh_seq {

using bf16 = __bf16;
using f16 = _Float16;
typedef long long ll;

// the last refusal of a call into these files, for mjh_seq_last_error (a literal: nothing allocates)
extern thread_local const char* g_why;
inline int refuse(const char* why) {
  g_why = why;
  return 1;
}
inline int launched() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return 0;
  g_why = hipGetErrorString(e);
  return 2;
}

template <class T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ Pack<T, V> load(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <class T, int V>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  Pack<T, V> o;
#pragma unroll
  for (int k = 0; k < V; k++) o.v[k] = (T)f[k];  // to nearest even, the one rounding of an output
  *reinterpret_cast<Pack<T, V>*>(p) = o;
}

// The exponential below: the hardware's 2^x of x log2(e), whose rounding error and the constant's own tail are
// carried along and applied to first order (x log2(e) alone would lose |x| 2^-24 relative).

// The smaller of sigmoid(g) and sigmoid(-g), to full relative precision; the larger is 1 - it. The sum 1 + e
// cannot overflow since e = e^-|g| <= 1. Beyond |g| = 87 the correction is left out (inf * 0 at |g| = inf):
// e < 2^-125 there, and an infinite gate gives exactly 0 and 1.
__device__ __forceinline__ float sigmoid_small(float g) {
  constexpr float kLog2e = 1.44269502e+0f, kLog2eTail = 1.92596299e-8f, kLn2 = 0.693147182f;
  const float x = -fabsf(g);
  const float hi = x * kLog2e;
  const float lo = __builtin_fmaf(x, kLog2eTail, __builtin_fmaf(x, kLog2e, -hi));
  const float p = __builtin_amdgcn_exp2f(hi);
  const float e = __builtin_fmaf(p, x < -87.f ? 0.f : lo * kLn2, p);
  return e * __builtin_amdgcn_rcpf(1.f + e);
}

// ---- dropout bits ----------------------------------------------------------------
// Element i keeps its value iff its 32 random bits are >= p 2^32. Two elements share one 64-bit word of the
// env layer's counter-based stream (mjh_rng.h): word i / 2 of the (seed, key, *counter) stream, its high half
// for even i, its low half for odd i. Nothing is stored: the backward pass forms the same words again.
struct Drop {
  unsigned long long seed, key;
  const mjh_i64* ctr;     // device step counter or NULL
  unsigned long long thr;  // round(p 2^32); 0: keep all, 2^32: drop all
  float scale;
};
__device__ __forceinline__ unsigned long long drop_word(unsigned long long base, unsigned long long pair) {
  return mjh::mix64(base + (pair + 1ull) * 0x9e3779b97f4a7c15ull);
}
__device__ __forceinline__ bool drop_keep(unsigned long long word, int odd, unsigned long long thr) {
  return (unsigned long long)(odd ? (unsigned)word : (unsigned)(word >> 32)) >= thr;
}

// Neighbouring elements at any element's address: gfx950 takes 16-byte global accesses at any alignment, so a row
// of an odd length is read as wide as an aligned one.
template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_loose(const T* p) {
  return __builtin_bit_cast(Pack<T, V>, *reinterpret_cast<const Loose<T, V>*>(p));
}
template <class T, int V>
__device__ __forceinline__ void store_loose(T* p, const float (&f)[V]) {
  Pack<T, V> o;
#pragma unroll
  for (int k = 0; k < V; k++) o.v[k] = (T)f[k];
  *reinterpret_cast<Loose<T, V>*>(p) = __builtin_bit_cast(Loose<T, V>, o);
}

// Waits for the loads issued so far. Before a loop that keeps a block of loads under way: a load of the first block
// that may still be under way at the loop's entry costs a wait for every load at its use in each turn (scan, backward,
// 16,384 x 2,048 bfloat16: 43 us, 47 so; norm's columns, 2,048 x 8,192: 56, 60).
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt 0; the others untouched

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace mjh_seq
