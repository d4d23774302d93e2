// What the short convolution and the selective scan share: where a sequence's
// tokens and its state row lie, and 32-bit activation functions.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace wkvm {

// Sequences of one call: a batch [nseq, T] (cu null), or packed along one
// token axis of T tokens in all (cu: nseq + 1 ascending offsets).
struct Seqs {
  const int64_t* cu;
  int32_t nseq;
  int32_t T;
};

struct SeqSpan {
  int64_t bos, len;  // first token on the flattened token axis, token count
  bool ok;           // false: offsets that leave the token axis or descend
};

__device__ __forceinline__ SeqSpan seq_span(const Seqs& s, int n) {
  if (!s.cu) return {(int64_t)n * s.T, s.T, true};
  const int64_t b = s.cu[n], e = s.cu[n + 1];
  const bool ok = b >= 0 && e >= b && e <= s.T;
  return {ok ? b : 0, ok ? e - b : 0, ok};
}

// An activation tensor: element (sequence n, its token t, channel c) at
// p[n * bs + t * ts + c], or p[(bos + t) * ts + c] when packed.
struct Act {
  const void* p;
  int64_t bs, ts;  // elements
};

// Strides of axes with one element (or, packed, of the batch) never reach an
// address; as 0 they do not stand in the way of whole-vector accesses either.
inline Act plain_strides(Act a, const Seqs& s) {
  if (s.cu || s.nseq <= 1) a.bs = 0;
  if (s.T <= 1) a.ts = 0;
  return a;
}

__device__ __forceinline__ int64_t act_row(const Seqs& s, const Act& a, int n, int64_t bos) {
  return s.cu ? bos * a.ts : n * a.bs;
}

// The row of the state tensor that sequence n reads and writes: its slot, or
// n itself without slot ids. A slot id outside the bank is reported and its
// sequence skipped.
__device__ __forceinline__ bool state_row(const int32_t* ids, int64_t num_slots, int n,
                                          int64_t* row) {
  *row = ids ? (int64_t)ids[n] : n;
  return !ids || (*row >= 0 && *row < num_slots);
}

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// x * sigmoid(x). EXACT: the 32-bit functions (fp32 outputs); otherwise the
// hardware approximations, whose 2^-21 is far below a 16-bit output's
// rounding.
template <bool EXACT>
__device__ __forceinline__ float silu(float x) {
  if constexpr (EXACT) return x / (1.0f + expf(-x));
  return x * rcp(1.0f + ex2(-kLog2e * x));
}

// log(1 + e^x) = max(x, 0) + log1p(e^-|x|) in 32 bits, to 2^-20 (1 + |x| / 8)
// relative: log1p(e) on [0, 1] is e times a polynomial of degree 8, minimax in
// the relative error (Remez exchange, 3e-8; 2^-22.2 with fp32 rounding), ex2
// holds 2^-22, and the rounded exponent |x| 2^-23.7. log1pf of expf would hold
// some 2^-22 throughout; what is lost beside it is below the rounding of a
// 16-bit dt, and for fp32 within a few steps of the result.
__host__ __device__ constexpr float log1p_coeff(int i) {
  return i == 0 ? 0.99999994f : i == 1 ? -0.49999493f : i == 2 ? 0.33319098f : i == 3 ? -0.24842982f
       : i == 4 ? 0.19106007f : i == 5 ? -0.13663246f : i == 6 ? 0.078225955f : i == 7 ? -0.029505240f
       : 0.0052326931f;
}

__device__ __forceinline__ float softplus(float x) {
  const float e = ex2(-kLog2e * fabsf(x));
  float p = log1p_coeff(8);
#pragma unroll
  for (int i = 7; i >= 0; --i) p = fmaf(p, e, log1p_coeff(i));
  return fmaf(p, e, fmaxf(x, 0.0f));
}

// Two fp32 in one 64-bit register pair (one instruction for both).
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float x, float y) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// V elements as they lie in memory, held as words: elements of 16 bits kept
// apart would be taken apart, and so waited for, right after the load.
template <typename T, int V>
struct alignas(sizeof(T) * V >= 16 ? 16 : sizeof(T) * V <= 4 ? 4 : 8) Raw {
  static constexpr int kBytes = sizeof(T) * V, kWords = (kBytes + 3) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ float f32(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      // byte permutes: the compiler's shifts by multiplication would crowd the
      // fp32 pipe
      uint32_t x;
      if (i % 2)
        asm("prmt.b32 %0, %1, 0, 0x3244;" : "=r"(x) : "r"(w[i / 2]));
      else
        asm("prmt.b32 %0, %1, 0, 0x1044;" : "=r"(x) : "r"(w[i / 2]));
      return __uint_as_float(x);
    } else {
      const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
      return to_f32(*reinterpret_cast<const T*>(&h));
    }
  }
  __device__ __forceinline__ void set2(int i, float x, float y) {  // elements i and i + 1, i even
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(x);
      w[i + 1] = __float_as_uint(y);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(x, y);
      w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ void move(Raw<T, V>* dst, const Raw<T, V>* src) {  // one access each way
  constexpr int B = Raw<T, V>::kBytes;
  if constexpr (B >= 16) {
#pragma unroll
    for (int i = 0; i < B / 16; ++i) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
  } else if constexpr (B == 8) {
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(src);
  } else if constexpr (B == 4) {
    *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
  } else {
    *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src);
  }
}

inline bool aligned_to(const void* p, uintptr_t n) {
  return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

}  // namespace wkvm
