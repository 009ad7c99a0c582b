// What the sequence operators (selective scan, short convolution, residual norm) share: element types, wave-uniform
// loads, and the walk over the borders of packed sequences.
#pragma once
#include "common.h"
#include "../../include/dvae_hip.h"

#define ST(s) ((hipStream_t)(s))

// A launch holds fewer than 2^32 threads.
static inline bool launch_fits(int64_t groups, int threads) { return groups * threads < (1ll << 32); }
// Most tokens: positions are int, and those of the last workgroups run past the end by less than this margin.
#define SEQ_MAX_TOKENS ((1ll << 31) - (1ll << 16))

enum bf16_t : uint16_t {};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float((uint32_t)v << 16); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) {      // round to nearest even
  return (bf16_t)__builtin_bit_cast(uint16_t, (__bf16)v);
}

// V consecutive elements, moved as accesses of up to 16 bytes (V > 1 only where the host checked alignment)
template <typename T, int V> struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack { T v[V]; };
// The same as it lies in memory, in whole registers (an array of 16-bit values would take one each)
template <typename T, int V> struct Packed {
  static constexpr int K = sizeof(T) * V < 4 ? 1 : sizeof(T) * V / 4;
  uint32_t w[K];
  __device__ __forceinline__ void load(const T* p) {
    if (sizeof(T) * V < 4) {
      w[0] = (uint32_t)*(const uint16_t*)p;
    } else {
      const Pack<uint32_t, K> r = *reinterpret_cast<const Pack<uint32_t, K>*>(p);
#pragma unroll
      for (int i = 0; i < K; ++i) w[i] = r.v[i];
    }
  }
  __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i)
      v[i] = sizeof(T) == 4 ? __uint_as_float(w[i < K ? i : 0])
                            : __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};
template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, float (&v)[V]) {
  const Pack<T, V> r = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f32(r.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&v)[V]) {
  Pack<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = r;
}

#define LOG2E_F 1.44269504088896341f
#define LN2_F 0.693147180559945309f

// exp(x) through the hardware's 2^x (1 ulp; results below 2^-126 become 0)
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float sigmoid_hw(float x) { return __builtin_amdgcn_rcpf(1.f + exp2_hw(-LOG2E_F * x)); }

// softplus(x) = max(x, 0) + log(1 + e^-|x|).  The logarithm of 1 + e loses the low bits of a small e when the sum is
// rounded; multiplying by e / ((1 + e) - 1), the ratio of what was meant to what was added, puts them back.
__device__ __forceinline__ float softplus_hw(float x) {
  const float e = exp2_hw(-LOG2E_F * fabsf(x));
  const float w = 1.f + e;
  const float r = w - 1.f;
  const float l = LN2_F * __builtin_amdgcn_logf(w) * (e * __builtin_amdgcn_rcpf(r));
  return fmaxf(x, 0.f) + (r == 0.f ? e : l);
}

// softplus and its derivative, the sigmoid: 1 / (1 + e^-x), with e as above and x < 0 turned round
__device__ __forceinline__ float softplus_hw(float x, float& slope) {
  const float e = exp2_hw(-LOG2E_F * fabsf(x));
  const float w = 1.f + e;
  const float r = w - 1.f;
  const float l = LN2_F * __builtin_amdgcn_logf(w) * (e * __builtin_amdgcn_rcpf(r));
  slope = (x < 0.f ? e : 1.f) * __builtin_amdgcn_rcpf(w);
  return fmaxf(x, 0.f) + (r == 0.f ? e : l);
}

// NaN has to come out as NaN: fmaxf(NaN, 0) is 0, but e and with it l are NaN.

// Sum over `parts` rows of column `col` of part[parts][stride], for the 64 columns of a workgroup of SUM_WAVES waves: a
// wave adds every SUM_WAVES-th row, eight loads in flight, and the waves' sums are added in their order, so the result
// does not depend on timing.  Valid in wave 0; every thread takes part.
#define SUM_WAVES 16
__device__ __forceinline__ float column_sum(const float* part, int64_t parts, int64_t stride, int64_t col, bool ok) {
  __shared__ float red[SUM_WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float s = 0.f;
  if (ok) {
    int64_t k = wave;
    for (; k + 7 * SUM_WAVES < parts; k += 8 * SUM_WAVES) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = part[(k + i * SUM_WAVES) * stride + col];
      s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    for (; k < parts; k += SUM_WAVES) s += part[k * stride + col];
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave > 0) return 0.f;
  s = red[0][lane];
#pragma unroll
  for (int i = 1; i < SUM_WAVES; ++i) s += red[i][lane];
  return s;
}

// Wave-uniform reads of data that no kernel in flight writes go through the constant address space: the compiler then
// uses the scalar unit and its registers for them, whatever it knows about the kernel's other pointers.
#define DVAE_UNIFORM __attribute__((address_space(4)))
template <typename V> __device__ __forceinline__ V uniform_load(const V* p, int64_t i) {
  return ((const DVAE_UNIFORM V*)p)[i];
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The sequence that a walk over tokens is in.  With `off`, sequence s is [off[s], off[s + 1]) of S ascending int32
// positions; without, all S sequences have L tokens.  Wrong offsets give wrong results but never an access out of range:
// positions are clamped to the tokens there are, a sequence whose end does not lie behind its begin has no tokens, and the
// sequence that the walk is in always has some, the last of them at or behind the token it was looked for (what the rows of
// carried states are computed from).  Every loop here ends: the index only moves one way.
struct SeqWalk {
  const int32_t* off;
  int S, L;     // number of sequences; tokens of each (off == nullptr)
  int tokens;   // all tokens
  int s;        // current sequence; S (forward) or -1 (backward): none left
  int b, e;     // its borders

  __device__ __forceinline__ int at(int i) const {
    return off ? min(max(uniform_load(off, i), 0), tokens) : i * L;
  }
  __device__ __forceinline__ void load() {
    if (s >= 0 && s < S) { b = at(s); e = at(s + 1); } else { b = e = tokens; }
  }
  // the current sequence as an index that exists, also where wrong offsets have led the walk past the last one
  __device__ __forceinline__ int64_t seq() const { return min(max(s, 0), S - 1); }
  // first sequence that ends behind token t (empty ones are skipped).  The wave's 64 lanes, all of which have to be
  // there, probe 64 ends at once, so that up to 64 sequences take one wait for memory and 4096 two.
  __device__ __forceinline__ void seek(int t) {
    if (!off) {
      s = t / L;
    } else {
      int lo = 0, hi = S;                     // the answer is one of lo ... hi
      while (lo < hi) {
        const int step = (hi - lo + 63) >> 6;
        const int64_t probe = lo + ((int64_t)(threadIdx.x & 63) + 1) * step - 1;
        const bool past = probe < hi && lane_at(probe < hi ? probe + 1 : hi) <= t;
        const int n = __popcll(__ballot(past));
        lo = uniform(lo + n * step);
        hi = uniform(min(hi, lo + step - 1));
      }
      s = lo;
    }
    load();
    settle(t);
  }
  // f(s) for the sequences s without tokens: every of-th 64 of all from the part-th 64 on, looked at by 64 lanes at once
  template <typename F> __device__ __forceinline__ void for_empty(int part, int of, F f) const {
    for (int64_t s0 = (int64_t)part * 64; s0 < S; s0 += (int64_t)of * 64) {
      const int64_t i = s0 + (threadIdx.x & 63);
      uint64_t left = __ballot(i < S && lane_at(i < S ? i + 1 : S) <= lane_at(i < S ? i : S));
      while (left) {
        f(uniform((int)s0 + __builtin_ctzll(left)));
        left &= left - 1;
      }
    }
  }
  __device__ __forceinline__ int lane_at(int64_t i) const { return min(max(off[i], 0), tokens); }
  // forward: the next sequence with tokens from t on
  __device__ __forceinline__ void next(int t) {
    step();
    settle(t);
  }
  __device__ __forceinline__ void step() {
    ++s;
    b = e;
    if (s < S) e = at(s + 1); else b = e = tokens;
  }
  __device__ __forceinline__ void settle(int t) {
    while (s < S && (e <= t || e <= b)) step();
  }
  // backward: the last sequence that starts at or before token t and has tokens
  __device__ __forceinline__ void prev(int t) {
    do { --s; } while (s >= 0 && (at(s) > t || at(s + 1) <= at(s)));
    load();
  }
};
