// Selective state space scan over sequences whose state [D, N] fp32 lives in
// a bank slot (or in a plain tensor). Per token t, channel d, state n:
//
//   delta = dt[t][d] + dt_bias[d], through softplus when asked
//   h[d][n] = exp(delta A[d][n]) h[d][n] + delta x[t][d] B[t][g][n]
//   y[t][d] = sum_n C[t][g][n] h[d][n] + D[d] x[t][d]
//   o[t][d] = y silu(z[t][d])                    (z optional)
//
// with g = d / (D / G): G groups of channels share B and C. The state, the
// step and every sum are fp32; only o is rounded to the activation dtype.
#include <cooperative_groups.h>
#include <float.h>

#include <type_traits>

#include "ssm_common.cuh"

namespace wkvm {
namespace {

struct ScanArgs {
  Act x, dt, z, B, C;  // z.p may be null
  const float* A;      // [D, N]
  const float* skip;   // [D] or null
  const float* bias;   // [D] or null
  void* o;             // [tokens, D]
  const float* h_in;   // rows of [D, N]; null: zeros
  float* h_out;        // null: not wanted
  const int32_t* ids;
  int64_t num_slots;
  Seqs seqs;
  int32_t D, G;
  int32_t softplus;
  int* status;
};

// ---------------------------------------------------------------------------
// Row kernel: the states of a block of channels of one sequence stream through
// registers once, T tokens applied in order. A single token moves 8 N bytes of
// state per channel against some 8 bytes of activations, so HBM bounds it.
// Four states (16 bytes) of J channels a thread: a warp's accesses are
// contiguous, J loads of state are in flight, and a thread's B and C serve its
// J channels. What is per channel (step, gate) is computed once, by one thread,
// and read from shared memory by the N/4 lanes that need it. Blocks of the same
// channels are neighbours, so A comes from L1 and L2.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 128;

// A as a power of two's exponent; -FLT_MAX for -inf, so that a step of zero
// keeps the state there too. NaN stays NaN (fmaxf would drop it). A decay is
// 2^(delta (A log2 e)) with both products rounded: |delta A| 2^-23 of it beside
// ex2's 2^-22. e^(delta A) would round one product only, for one more in the
// inner loop of every state.
__device__ __forceinline__ float scaled(float a) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a * kLog2e), "f"(-FLT_MAX));
  return r;
}

// 2^e h + y for the decay 2^e over many tokens. Steps without softplus may have
// any sign, so 2^e may leave fp32's range on either side where 2^e h does not:
// then half of e at a time, and a state of nothing stays nothing.
__device__ __forceinline__ float decayed(float e, float h, float y) {
  if (fabsf(e) <= 126.0f) return fmaf(ex2(e), h, y);
  if (h == 0.0f && e == e) return y;
  const float f = ex2(0.5f * e);
  return fmaf(h * f, f, y);
}

template <typename T, int N, int J>
__global__ void __launch_bounds__(kRowThreads, 8) scan_rows_kernel(ScanArgs p) {
  constexpr int LPC = N / 4;  // lanes of a channel
  constexpr int STEP = kRowThreads / LPC, CPB = STEP * J;
  constexpr int CPT = (CPB + kRowThreads - 1) / kRowThreads;  // channels whose step a thread computes
  __shared__ float4 s_ch[CPB];  // delta, delta x, D x, gate
  __shared__ float s_y[CPB];
  const int n = blockIdx.x % p.seqs.nseq, c0 = blockIdx.x / p.seqs.nseq * CPB;
  const int tid = threadIdx.x, lane = tid % LPC, ch = tid / LPC;
  const int live = p.D - c0 < CPB ? p.D - c0 : CPB;  // channels of this block
  // everything that needs no slot id goes out ahead of the state
  const T* xp = static_cast<const T*>(p.x.p) + n * p.x.bs + c0 + tid;
  const T* dp = static_cast<const T*>(p.dt.p) + n * p.dt.bs + c0 + tid;
  const T* zp = static_cast<const T*>(p.z.p) + n * p.z.bs + c0 + tid;
  T xr[CPT], dr[CPT], zr[CPT];
  auto load_token = [&](int t) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      if (tid + i * kRowThreads >= live) break;
      xr[i] = xp[t * p.x.ts + i * kRowThreads];
      dr[i] = dp[t * p.dt.ts + i * kRowThreads];
      if (p.z.p) zr[i] = zp[t * p.z.ts + i * kRowThreads];
    }
  };
  if (p.seqs.T > 0) load_token(0);
  int64_t row;
  if (!state_row(p.ids, p.num_slots, n, &row)) {
    if (tid == 0) report(p.status, WKVM_ERR_SLOT_RANGE);
    return;
  }
  const int64_t hoff = (row * p.D + c0 + ch) * N + lane * 4;
  float4 h[J], a[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    h[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.h_in && ch + j * STEP < live) h[j] = ld_stream_f4(p.h_in + hoff + j * STEP * N);
  }
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (ch + j * STEP < live)
      a[j] = *reinterpret_cast<const float4*>(p.A + (int64_t)(c0 + ch + j * STEP) * N + lane * 4);
  const int per_group = p.D / p.G;
  const T* bp = static_cast<const T*>(p.B.p) + n * p.B.bs + lane * 4;
  const T* cp = static_cast<const T*>(p.C.p) + n * p.C.bs + lane * 4;
  T* op = static_cast<T*>(p.o) + (int64_t)n * p.seqs.T * p.D + c0;
  const bool one_group = c0 / per_group == (c0 + live - 1) / per_group;
  for (int t = 0; t < p.seqs.T; ++t) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = tid + i * kRowThreads;
      if (c >= live) break;
      const float x = to_f32(xr[i]);
      float delta = to_f32(dr[i]) + (p.bias ? p.bias[c0 + c] : 0.f);
      if (p.softplus) delta = softplus(delta);
      const float gate = p.z.p ? silu<true>(to_f32(zr[i])) : 1.f;
      s_ch[c] = make_float4(delta, delta * x, p.skip ? p.skip[c0 + c] * x : 0.f, gate);
    }
    if (t + 1 < p.seqs.T) load_token(t + 1);
    __syncthreads();
    float bv[4], cv[4];
    int g = c0 / per_group;
    auto read_bc = [&] {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bv[i] = to_f32(bp[t * p.B.ts + g * N + i]);
        cv[i] = to_f32(cp[t * p.C.ts + g * N + i]);
      }
    };
    if (one_group) read_bc();
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = ch + j * STEP;
      float y = 0.f;
      if (c < live) {
        if (!one_group) {
          g = (c0 + c) / per_group;
          read_bc();
        }
        const float2 s = *reinterpret_cast<const float2*>(&s_ch[c]);
        h[j].x = fmaf(ex2(s.x * scaled(a[j].x)), h[j].x, s.y * bv[0]);
        h[j].y = fmaf(ex2(s.x * scaled(a[j].y)), h[j].y, s.y * bv[1]);
        h[j].z = fmaf(ex2(s.x * scaled(a[j].z)), h[j].z, s.y * bv[2]);
        h[j].w = fmaf(ex2(s.x * scaled(a[j].w)), h[j].w, s.y * bv[3]);
        y = fmaf(h[j].x, cv[0], h[j].y * cv[1]) + fmaf(h[j].z, cv[2], h[j].w * cv[3]);
      }
#pragma unroll
      for (int off = LPC / 2; off > 0; off >>= 1) y += __shfl_xor_sync(0xffffffffu, y, off);
      if (lane == 0) s_y[c] = y;
    }
    __syncthreads();
    for (int c = tid; c < live; c += kRowThreads) {
      const float2 s = reinterpret_cast<const float2*>(&s_ch[c])[1];
      op[(int64_t)t * p.D + c] = from_f32<T>((s_y[c] + s.x) * s.y);
    }
  }
  if (!p.h_out) return;
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (ch + j * STEP < live) st_stream_f4(p.h_out + hoff + j * STEP * N, h[j]);
}

// ---------------------------------------------------------------------------
// Tile kernel, for prompts. Its floor is T D N exponentials at 16 a clock and
// SM (4.65e12 / s; 231 us for 32768 x 2048 x 16) rather than the 8 bytes of
// activations per N of them (83 us). Other instructions come to some nine an
// exponential. Sixteen packed prompts of that size take 607 us (two channels to
// a register pair took it from 880, straight-line tile phases and byte permutes
// to this). Nothing is saturated there: the exponentials' pipe is half busy, and
// a scheduler issues 0.6 instructions a clock from three warps, which wait for
// their operands; the longest prompt's tail runs with fewer.
//
// One CTA walks one sequence for CB channels, TT tokens at a time. A thread
// keeps NS states of CH channels; the L = N / NS threads of a channel leave
// their partial sums of C h in shared memory and the thread that owns the
// output element adds them. What is per (token, channel) - softplus, the
// skip, the gate, conversions - is done once by the owner of the element, not
// by the L threads: they read (delta, delta x) pairs. Shared memory gives
// 128 bytes a clock however many lanes read the same word, so a thread's
// share of B and C (kept in the inputs' dtype) is read once for its CH
// channels. The next tile's inputs are copied into shared memory while this one
// runs, asynchronously where both sides are aligned.
//
// Few rows (a long prompt alone, few channels): the CTAs of a cluster split
// the sequence's tiles between them. Each first runs its part from a zero
// state for its final state and the sum of its steps (whose exponential is
// the part's whole decay, A being constant), then takes the parts before it
// from its peers' shared memory and runs its part again from its true start.
// The sum of n steps is held in fp32: n 2^-24 of it at most, as much as the n
// products of the tokens one by one lose.
// ---------------------------------------------------------------------------
// softplus() of two
__device__ __forceinline__ f32x2 softplus2(f32x2 x) {
  const float2 v = unpack2(x);
  const f32x2 e = pack2(ex2(-kLog2e * fabsf(v.x)), ex2(-kLog2e * fabsf(v.y)));
  f32x2 q = pack2(log1p_coeff(8), log1p_coeff(8));
#pragma unroll
  for (int i = 7; i >= 0; --i) q = fma2(q, e, pack2(log1p_coeff(i), log1p_coeff(i)));
  return fma2(q, e, pack2(fmaxf(v.x, 0.0f), fmaxf(v.y, 0.0f)));
}

// V elements at p, of which the first `n` exist (the others read as zero).
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_some(const T* p, int n) {
  Raw<T, V> r;
#pragma unroll
  for (int i = 0; i < Raw<T, V>::kWords; ++i) r.w[i] = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i >= n) continue;
    if constexpr (sizeof(T) == 4)
      r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    else
      r.w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i % 2));
  }
  return r;
}

// V elements from global to shared memory, zeros unless `have`: asynchronous,
// for copies_done() to wait for, where both sides are aligned to the vector.
template <typename T, int V>
__device__ __forceinline__ void copy_async(uint32_t dst, const T* src, bool have) {
  const int size = have ? Raw<T, V>::kBytes : 0;
  if constexpr (Raw<T, V>::kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(Raw<T, V>::kBytes), "r"(size) : "memory");
}
// The first n of V elements one by one, zeros for the others.
template <typename T, int V>
__device__ __forceinline__ void copy_some(T* dst, const T* src, int n) {
  const Raw<T, V> r = load_some<T, V>(src, n);
  move<T, V>(reinterpret_cast<Raw<T, V>*>(dst), &r);
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

constexpr int min_i(int a, int b) { return a < b ? a : b; }

// 4 floats of padding behind every 32 keep 16-byte accesses of neighbouring
// threads off each other's banks
__host__ __device__ constexpr int padded(int i) { return i + (i >> 5) * 4; }

// N states; NP pairs of channels and NS states a thread; NT threads; tiles of
// TT tokens.
template <typename T, int N, int NP, int NS, int NT, int TT>
struct Tile {
  static constexpr int L = N / NS;                        // threads of a channel
  static constexpr int CBP = NT / L, CB = 2 * CBP * NP;   // a thread's pairs: ch + j CBP, j < NP
  static constexpr int EPT = TT * CB / NT;                // elements of x a thread owns
  static constexpr int VE = min_i(EPT, 16 / (int)sizeof(T)), RV = EPT / VE;
  static constexpr int BPT = TT * N / NT;                 // elements of B a thread loads
  static constexpr int VB = min_i(BPT, 16 / (int)sizeof(T)), RB = BPT / VB;
  static constexpr int DROW = padded(2 * CB), YROW = padded(2 * NP * NT);
  // shared memory, in bytes
  static constexpr int XB = sizeof(T) * TT * CB, BB = sizeof(T) * TT * N;
  static constexpr int oD = 0;                      // [TT][pair] (delta, delta, delta x, delta x)
  static constexpr int oY = oD + 4 * TT * DROW;     // [TT][pair][L][2] partial sums
  static constexpr int oX = oY + 4 * TT * YROW;     // two stages of x, dt, z [TT][CB] and B, C [TT][N]
  static constexpr int kStage = 3 * XB + 2 * BB;
  static constexpr int oP = oX + 2 * kStage;        // dt_bias and D of the channels
  static constexpr int oH = oP + 8 * CB;            // cluster: final states, step sums
  static constexpr int bytes(bool cluster) { return oH + (cluster ? 8 * NP * (NS + 1) * NT : 0); }
  static_assert(EPT >= 2 && BPT >= 2 && NT * VB % N == 0 && TT * NT % CB == 0 && XB % 16 == 0 && BB % 16 == 0, "tile too small for the block");
};

struct TileArgs {
  ScanArgs s;
  int32_t cblocks;   // channel blocks of a group
  int32_t parts;     // CTAs of a cluster (1: none)
  bool vec_x, vec_b; // whole-vector accesses to x, dt, z, o and to B, C
  bool longest_first;
};

template <typename T, int N, int NP, int NS, int NT, int TT, bool CLUSTER>
__global__ void __launch_bounds__(NT) scan_tiles_kernel(TileArgs q) {
  using K = Tile<T, N, NP, NS, NT, TT>;
  constexpr int L = K::L, CB = K::CB, CBP = K::CBP, VE = K::VE, RV = K::RV, VB = K::VB, RB = K::RB;
  constexpr int CBV = CB / VE, TS = NT / CBV;
  extern __shared__ __align__(16) uint8_t smem[];
  float* sD = reinterpret_cast<float*>(smem + K::oD);
  float* sY = reinterpret_cast<float*>(smem + K::oY);
  float* sP = reinterpret_cast<float*>(smem + K::oP);
  auto meet = [] {
    if constexpr (NT == 32) __syncwarp(); else __syncthreads();
  };
  const ScanArgs& p = q.s;
  const int tid = threadIdx.x, lane = tid % L, ch = tid / L;
  const int part = CLUSTER ? (int)(blockIdx.x % q.parts) : 0;
  const int job = blockIdx.x / q.parts;
  const int blocks = q.cblocks * p.G;
  int n = job / blocks;
  const int blk = job - n * blocks, g = blk / q.cblocks;
  const int per_group = p.D / p.G;
  const int c0 = g * per_group + (blk - g * q.cblocks) * CB;  // first channel
  const int cn = min_i((g + 1) * per_group - c0, CB);         // channels of this CTA

  if (q.longest_first) {
    // the n-th longest sequence: the long ones start first and the short ones
    // fill the gaps
    __shared__ int s_n;
    for (int i = tid; i < p.seqs.nseq; i += NT) {
      const int64_t len = seq_span(p.seqs, i).len;
      int rank = 0;
      for (int j = 0; j < p.seqs.nseq; ++j) {
        const int64_t o = seq_span(p.seqs, j).len;
        rank += o > len || (o == len && j < i);
      }
      if (rank == n) s_n = i;
    }
    meet();
    n = s_n;
  }
  int64_t row;
  const SeqSpan sp = seq_span(p.seqs, n);
  if (!state_row(p.ids, p.num_slots, n, &row)) {
    if (tid == 0) report(p.status, WKVM_ERR_SLOT_RANGE);
    return;
  }
  if (!sp.ok) {
    if (tid == 0) report(p.status, WKVM_ERR_INVALID_ARG);
    return;
  }

  // ---- this thread's states and their A, two channels in a register pair
  f32x2 h[NP][NS], a[NP][NS];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int c = 2 * (ch + j * CBP);
    const float* ap = p.A + (int64_t)(c0 + c) * N + lane * NS;
    const float* hp = p.h_in + (row * p.D + c0 + c) * N + lane * NS;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      a[j][i] = pack2(c < cn ? scaled(ap[i]) : 0.f, c + 1 < cn ? scaled(ap[N + i]) : 0.f);
      h[j][i] = pack2(p.h_in && c < cn ? hp[i] : 0.f, p.h_in && c + 1 < cn ? hp[N + i] : 0.f);
    }
  }

  // ---- the elements of a tile this thread owns: channels ce..ce+VE-1 of
  //      tokens te + r * TS
  const int te = tid / CBV, ce = (tid % CBV) * VE;
  const int nv = cn - ce;  // channels of the vector that exist
  for (int i = tid; i < CB; i += NT) {
    sP[i] = p.bias && i < cn ? p.bias[c0 + i] : 0.f;
    sP[CB + i] = p.skip && i < cn ? p.skip[c0 + i] : 0.f;
  }
  const T* xp = static_cast<const T*>(p.x.p) + act_row(p.seqs, p.x, n, sp.bos) + c0 + ce;
  const T* dp = static_cast<const T*>(p.dt.p) + act_row(p.seqs, p.dt, n, sp.bos) + c0 + ce;
  const T* zp = p.z.p ? static_cast<const T*>(p.z.p) + act_row(p.seqs, p.z, n, sp.bos) + c0 + ce : nullptr;
  const T* bp = static_cast<const T*>(p.B.p) + act_row(p.seqs, p.B, n, sp.bos) + g * N;
  const T* cp = static_cast<const T*>(p.C.p) + act_row(p.seqs, p.C, n, sp.bos) + g * N;
  T* op = static_cast<T*>(p.o) + sp.bos * p.D + c0 + ce;

  // A thread copies in the elements it owns and is their only reader, so it
  // waits for its own copies alone; B and C, read by all, are also behind the
  // barrier ahead of the main loop. Pointers run along with the tiles, which
  // are fetched in order; past the end they stay on the tile's first token.
  const int len = (int)sp.len;
  constexpr int BT = NT * VB / N;  // tokens of one round of copies of B and C
  const int tb = tid * VB / N;
  const T *fx, *fd, *fz, *fb, *fc;
  T* out;
  int left;  // tokens from the next tile's start to the sequence's end
  auto aim = [&](int t0) {
    fx = xp + (int64_t)t0 * p.x.ts;
    fd = dp + (int64_t)t0 * p.dt.ts;
    fz = zp ? zp + (int64_t)t0 * p.z.ts : nullptr;
    fb = bp + (int64_t)t0 * p.B.ts + tid * VB % N;
    fc = cp + (int64_t)t0 * p.C.ts + tid * VB % N;
    out = op + ((int64_t)t0 + te) * p.D;
    left = len - t0;
  };
  auto fetch = [&](int stage, bool emit) {
    T* sx = reinterpret_cast<T*>(smem + K::oX + stage * K::kStage) + te * CB + ce;
    T* sb = reinterpret_cast<T*>(smem + K::oX + stage * K::kStage) + 3 * TT * CB + tid * VB;
    if (q.vec_x) {
      const uint32_t d = (uint32_t)__cvta_generic_to_shared(sx);
#pragma unroll
      for (int r = 0; r < RV; ++r) {
        const bool have = te + r * TS < left && nv > 0;
        const int t = have ? te + r * TS : 0;
        const uint32_t at = d + r * TS * CB * (int)sizeof(T);
        copy_async<T, VE>(at, nv > 0 ? fx + t * p.x.ts : xp - ce, have);
        copy_async<T, VE>(at + K::XB, nv > 0 ? fd + t * p.dt.ts : dp - ce, have);
        if (emit && zp) copy_async<T, VE>(at + 2 * K::XB, nv > 0 ? fz + t * p.z.ts : zp - ce, have);
      }
    } else {
#pragma unroll
      for (int r = 0; r < RV; ++r) {
        const int64_t t = te + r * TS;
        const int k = t < left ? nv : 0;
        copy_some<T, VE>(sx + r * TS * CB, fx + t * p.x.ts, k);
        copy_some<T, VE>(sx + TT * CB + r * TS * CB, fd + t * p.dt.ts, k);
        if (emit && zp) copy_some<T, VE>(sx + 2 * TT * CB + r * TS * CB, fz + t * p.z.ts, k);
      }
    }
    if (q.vec_b) {
      const uint32_t d = (uint32_t)__cvta_generic_to_shared(sb);
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const bool have = tb + r * BT < left;
        const int t = have ? tb + r * BT : 0;
        copy_async<T, VB>(d + r * NT * VB * (int)sizeof(T), fb + t * p.B.ts, have);
        if (emit) copy_async<T, VB>(d + K::BB + r * NT * VB * (int)sizeof(T), fc + t * p.C.ts, have);
      }
    } else {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const int64_t t = tb + r * BT;
        const int k = t < left ? VB : 0;
        copy_some<T, VB>(sb + r * NT * VB, fb + t * p.B.ts, k);
        if (emit) copy_some<T, VB>(sb + TT * N + r * NT * VB, fc + t * p.C.ts, k);
      }
    }
    fx += TT * p.x.ts;
    fd += TT * p.dt.ts;
    if (zp) fz += TT * p.z.ts;
    fb += TT * p.B.ts;
    fc += TT * p.C.ts;
    left -= TT;
  };

  f32x2 steps[NP];  // sums of delta over the part (first pass of a cluster)
#pragma unroll
  for (int j = 0; j < NP; ++j) steps[j] = 0;
  const float* sp0 = sP + ce;
  const float* dp0 = sD + padded(4 * ch);
  float* dst0 = sD + te * K::DROW + padded(2 * ce);
  const float* src0 = sY + te * K::YROW + padded(ce * L);
  float* y0 = sY + padded(2 * tid);
  // (unsigned: a tile's end may lie past the last int32. Counting down instead
  // takes 9 % longer, sixteen packed prompts 663 us against 607)
  auto run = [&](uint32_t t0, uint32_t t1, bool emit) {
    if (t0 >= t1) return;
    aim((int)t0);
    fetch(0, emit);
    meet();  // sP; the tiles of an earlier run
    for (int stage = 0; t0 < t1; t0 += TT, stage ^= 1) {
      const T* sX = reinterpret_cast<const T*>(smem + K::oX + stage * K::kStage);
      const T* own = sX + te * CB + ce;
      const T* sB = sX + 3 * TT * CB;
      const T* sC = sB + TT * N;
      copies_done();
      {
        // tokens behind the end give any numbers here; the main loop stops
        // ahead of them
        Raw<T, VE> rx[RV], rd[RV];
#pragma unroll
        for (int r = 0; r < RV; ++r) {
          move<T, VE>(&rx[r], reinterpret_cast<const Raw<T, VE>*>(own + r * TS * CB));
          move<T, VE>(&rd[r], reinterpret_cast<const Raw<T, VE>*>(own + TT * CB + r * TS * CB));
        }
#pragma unroll
        for (int i = 0; i < VE; i += 2) {
          const f32x2 bias = *reinterpret_cast<const f32x2*>(sp0 + i);
#pragma unroll
          for (int r = 0; r < RV; ++r) {
            f32x2 d = add2(pack2(rd[r].f32(i), rd[r].f32(i + 1)), bias);
            if (p.softplus) d = softplus2(d);
            *reinterpret_cast<ulonglong2*>(dst0 + r * TS * K::DROW + 2 * i) =
                make_ulonglong2(d, mul2(d, pack2(rx[r].f32(i), rx[r].f32(i + 1))));
          }
        }
      }
      meet();
      if (t0 + TT < t1) fetch(stage ^ 1, emit);
      const int live = min_i(len - (int)t0, TT);
      // Software pipeline: while token t is accumulated, the decays of t + 1 are
      // computed (the exponentials' pipe is the scarce one) and the operands of
      // t + 2 read. Reads past the tile wrap around; nothing uses them.
      const T* bp0 = sB + lane * NS;
      const T* cp0 = sC + lane * NS;
      ulonglong2 nd[NP];       // (delta, delta x) of t + 1
      f32x2 dx[NP], e[NP][NS]; // delta x and decays of t
      Raw<T, NS> nb, nc;       // B, C of t
      auto read_d = [&](int t, ulonglong2 (&d)[NP]) {
#pragma unroll
        for (int j = 0; j < NP; ++j)
          d[j] = *reinterpret_cast<const ulonglong2*>(dp0 + t * K::DROW + padded(4 * j * CBP));
      };
      auto read_bc = [&](int t, Raw<T, NS>& b, Raw<T, NS>& c) {
        move<T, NS>(&b, reinterpret_cast<const Raw<T, NS>*>(bp0 + t * N));
        if (emit) move<T, NS>(&c, reinterpret_cast<const Raw<T, NS>*>(cp0 + t * N));
      };
      read_d(0, nd);
      read_bc(0, nb, nc);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        dx[j] = nd[j].y;
        if (!emit) steps[j] = add2(steps[j], nd[j].x);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const float2 v = unpack2(mul2(a[j][i], nd[j].x));
          e[j][i] = pack2(ex2(v.x), ex2(v.y));
        }
      }
      read_d(1, nd);
#pragma unroll 4
      for (int t = 0; t < live; ++t) {
        const Raw<T, NS> kb = nb, kc = nc;
        ulonglong2 kd[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) kd[j] = nd[j];
        read_bc((t + 1) % TT, nb, nc);
        read_d((t + 2) % TT, nd);
        f32x2 y[NP];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const f32x2 b2 = pack2(kb.f32(i), kb.f32(i));
          const f32x2 c2 = emit ? pack2(kc.f32(i), kc.f32(i)) : 0;
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            const float2 v = unpack2(mul2(a[j][i], kd[j].x));
            h[j][i] = fma2(e[j][i], h[j][i], mul2(dx[j], b2));
            e[j][i] = pack2(ex2(v.x), ex2(v.y));
            if (emit) y[j] = i ? fma2(h[j][i], c2, y[j]) : mul2(h[j][i], c2);
          }
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          dx[j] = kd[j].y;
          if (emit)
            *reinterpret_cast<f32x2*>(y0 + t * K::YROW + padded(2 * j * NT)) = y[j];
          else if (t + 1 < live)
            steps[j] = add2(steps[j], kd[j].x);
        }
      }
      meet();
      if (!emit) continue;
      Raw<T, VE> rx[RV], rz[RV], ry[RV];
#pragma unroll
      for (int r = 0; r < RV; ++r) {
        move<T, VE>(&rx[r], reinterpret_cast<const Raw<T, VE>*>(own + r * TS * CB));
        if (zp) move<T, VE>(&rz[r], reinterpret_cast<const Raw<T, VE>*>(own + 2 * TT * CB + r * TS * CB));
      }
#pragma unroll
      for (int i = 0; i < VE; i += 2) {
        const f32x2 skip = *reinterpret_cast<const f32x2*>(sp0 + CB + i);
#pragma unroll
        for (int r = 0; r < RV; ++r) {
          const float* src = src0 + r * TS * K::YROW;
          f32x2 sum = 0;
          if constexpr (L >= 2) {
#pragma unroll
            for (int j = 0; j < L; j += 2) {
              const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(src + padded(i * L + 2 * j));
              sum = j ? add2(sum, add2(f.x, f.y)) : add2(f.x, f.y);
            }
          } else {
            sum = *reinterpret_cast<const f32x2*>(src + padded(i));
          }
          float2 y = unpack2(fma2(skip, pack2(rx[r].f32(i), rx[r].f32(i + 1)), sum));
          if (zp) {
            y.x *= silu<sizeof(T) == 4>(rz[r].f32(i));
            y.y *= silu<sizeof(T) == 4>(rz[r].f32(i + 1));
          }
          ry[r].set2(i, y.x, y.y);
        }
      }
#pragma unroll
      for (int r = 0; r < RV; ++r) {
        if (te + r * TS >= live) continue;
        T* dst = out + (int64_t)(r * TS) * p.D;
        if (q.vec_x) {
          if (nv > 0) move<T, VE>(reinterpret_cast<Raw<T, VE>*>(dst), &ry[r]);
        } else {
#pragma unroll
          for (int i = 0; i < VE; ++i)
            if (i < nv) dst[i] = from_f32<T>(ry[r].f32(i));
        }
      }
      out += TT * (int64_t)p.D;
    }
  };

  if constexpr (CLUSTER) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int64_t each = (((int64_t)len + TT - 1) / TT + q.parts - 1) / q.parts * TT;
    const int b0 = (int)(part * each < len ? part * each : len);
    const int b1 = (int)(b0 + each < len ? b0 + each : len);
    f32x2 start[NP][NS];
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        start[j][i] = h[j][i];
        h[j][i] = 0;
      }
    if (part + 1 < q.parts) run(b0, b1, false);  // nobody follows the last part
    f32x2* sH = reinterpret_cast<f32x2*>(smem + K::oH);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
#pragma unroll
      for (int i = 0; i < NS; ++i) sH[(j * NS + i) * NT + tid] = h[j][i];
      sH[(NP * NS + j) * NT + tid] = steps[j];
    }
    cluster.sync();
    for (int k = 0; k < part; ++k) {
      const f32x2* peer = cluster.map_shared_rank(sH, k) + tid;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const f32x2 sum = peer[(NP * NS + j) * NT];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const float2 e = unpack2(mul2(a[j][i], sum));
          const float2 x = unpack2(start[j][i]), y = unpack2(peer[(j * NS + i) * NT]);
          start[j][i] = pack2(decayed(e.x, x.x, y.x), decayed(e.y, x.y, y.y));
        }
      }
    }
    cluster.sync();  // peers have read; the state row may be written now
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
      for (int i = 0; i < NS; ++i) h[j][i] = start[j][i];
    run(b0, b1, true);
    if (part + 1 < q.parts) return;
  } else {
    run(0, len, true);
  }
  if (!p.h_out) return;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int c = 2 * (ch + j * CBP);
    float* hp = p.h_out + (row * p.D + c0 + c) * N + lane * NS;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const float2 v = unpack2(h[j][i]);
      if (c < cn) hp[i] = v.x;
      if (c + 1 < cn) hp[N + i] = v.y;
    }
  }
}

template <typename T, int N, int J>
int launch_rows(const ScanArgs& a, cudaStream_t st) {
  constexpr int CPB = kRowThreads / (N / 4) * J;
  const int64_t blocks = (int64_t)a.seqs.nseq * ((a.D + CPB - 1) / CPB);
  if (blocks > INT32_MAX) return WKVM_ERR_SHAPE;
  scan_rows_kernel<T, N, J><<<(unsigned)blocks, kRowThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? WKVM_OK : WKVM_ERR_CUDA;
}

template <typename T, int N, int NP, int NS, int NT, int TT, bool CLUSTER>
int launch_tiles(const ScanArgs& s, int parts, cudaStream_t st) {
  using K = Tile<T, N, NP, NS, NT, TT>;
  TileArgs q{s, 0, parts, false, false, false};
  const int per_group = s.D / s.G;
  q.cblocks = (per_group + K::CB - 1) / K::CB;
  const int64_t jobs = (int64_t)s.seqs.nseq * q.cblocks * s.G;
  constexpr uintptr_t ax = sizeof(T) * K::VE, ab = sizeof(T) * K::VB;
  auto even = [](const Act& a, int v) { return a.bs % v == 0 && a.ts % v == 0; };
  q.vec_x = per_group % K::VE == 0 && even(s.x, K::VE) && even(s.dt, K::VE) && aligned_to(s.x.p, ax) &&
            aligned_to(s.dt.p, ax) && aligned_to(s.o, ax) &&
            (!s.z.p || (even(s.z, K::VE) && aligned_to(s.z.p, ax)));
  q.vec_b = even(s.B, K::VB) && even(s.C, K::VB) && aligned_to(s.B.p, ab) && aligned_to(s.C.p, ab);
  // Every CTA compares all pairs of sequences for it, so it is for few and long
  // ones: 16 unequal ones of 32768 x 2048 in all take 595 us against 837 without,
  // 64 of them 579 against 605; but 64 of 2,048 tokens in all 85 against 66, 128
  // of 32768 789 against 662, and 256 of 16 tokens each 2,281 against 157.
  q.longest_first = s.seqs.cu && s.seqs.nseq > 1 && s.seqs.nseq <= 64 && s.seqs.T >= 4 * s.seqs.nseq * s.seqs.nseq;
  if (jobs * parts > INT32_MAX) return WKVM_ERR_SHAPE;
  constexpr auto kern = scan_tiles_kernel<T, N, NP, NS, NT, TT, CLUSTER>;
  constexpr int bytes = K::bytes(CLUSTER);
  WKVM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (CLUSTER)  // of 16
    WKVM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(jobs * parts));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, q) == cudaSuccess ? WKVM_OK : WKVM_ERR_CUDA;
}

template <typename T, int N>
int launch_scan_n(const ScanArgs& a, cudaStream_t st) {
  // a few tokens of every row: the state's traffic decides, so the row kernel
  if (!a.seqs.cu && a.seqs.T <= 8) {
    // Four channels a thread once that still gives every SM a thousand threads.
    // 512 rows of 4096 x 16, bf16, on the device: 60 us with four (4.7 TB/s, 72 %
    // of the measured HBM rate), 75 with two, 112 with one, 86 with eight, which
    // do not fit the 64 registers that eight blocks an SM leave. Few rows go the
    // other way: one 2.9 us with one channel a thread, 3.5 with four; eight rows
    // 3.7 and 4.1; sixteen 5.7 and 4.6.
    if ((int64_t)a.seqs.nseq * a.D * N / 16 >= 148 * 1024) return launch_rows<T, N, 4>(a, st);
    return launch_rows<T, N, 1>(a, st);
  }
  // Warps that four states (two channels) a thread give, of 592 schedulers.
  // Few: sequences are split in time over clusters (one of 8192 x 4096: 461 us
  // in eight parts, 528 in four, 590 whole in the fine form, 892 in the wide). A
  // split pays twice for the exponentials, so it takes four parts at least and
  // room for them. It goes by the average length, as the host knows no other:
  // one prompt of 8,192 beside 31 of four tokens stays whole (2048 channels: 594
  // us, 315 in eight parts). Packed sequences, or not enough rows for two waves:
  // the fine form, fewer states a thread and so more warps (sixteen unequal
  // prompts of 32768 x 2048 in all: 607 us against 788 wide; sixteen equal ones,
  // which the host cannot tell from them, 599 against 495). A batch of enough
  // rows is of equal length: the wide form. From 64 states on B and C outweigh a
  // CTA's channels, so the fine form keeps four or eight states (three sequences
  // of 666 x 1002 x 64, fp32: 104 us; 103 in the wide form).
  constexpr int kWide = N == 128 ? 8 : 4;
  const int64_t warps = (int64_t)a.seqs.nseq * a.D * N / (kWide * 2 * 32);
  const int64_t tokens = a.seqs.cu ? a.seqs.T / a.seqs.nseq : a.seqs.T;
  int parts = 1;
  while (parts < 16 && warps * parts * 2 <= 2048 && tokens >= parts * 8 * 16) parts *= 2;
  if (warps <= 256 && parts >= 4) return launch_tiles<T, N, 1, kWide, 64, 16, true>(a, parts, st);
  if constexpr (N < 128) {
    if (a.seqs.cu || warps < 2048) {
      if constexpr (N == 64) return launch_tiles<T, N, 1, 4, 128, 32, false>(a, 1, st);
      else return launch_tiles<T, N, 1, 2, 64, 32, false>(a, 1, st);
    }
  }
  return launch_tiles<T, N, 1, kWide, 64, 16, false>(a, 1, st);
}

template <typename T>
int launch_scan(const ScanArgs& a, int N, cudaStream_t st) {
  switch (N) {
    case 8: return launch_scan_n<T, 8>(a, st);
    case 16: return launch_scan_n<T, 16>(a, st);
    case 32: return launch_scan_n<T, 32>(a, st);
    case 64: return launch_scan_n<T, 64>(a, st);
    case 128: return launch_scan_n<T, 128>(a, st);
    default: return WKVM_ERR_SHAPE;
  }
}

int run_scan(const ScanArgs& a, int N, int dtype, cudaStream_t st) {
  if (a.seqs.nseq < 0 || a.seqs.T < 0 || a.D <= 0 || a.G <= 0 || N <= 0) return WKVM_ERR_INVALID_ARG;
  if (a.D % a.G || (N != 8 && N != 16 && N != 32 && N != 64 && N != 128)) return WKVM_ERR_SHAPE;
  if (dtype != WKVM_DTYPE_F32 && dtype != WKVM_DTYPE_BF16 && dtype != WKVM_DTYPE_F16)
    return WKVM_ERR_DTYPE;
  if (a.seqs.nseq == 0) return WKVM_OK;
  if (!a.A) return WKVM_ERR_INVALID_ARG;
  if (a.seqs.T > 0 && (!a.x.p || !a.dt.p || !a.B.p || !a.C.p || !a.o)) return WKVM_ERR_INVALID_ARG;
  if (!aligned_to(a.A, 16) || !aligned_to(a.h_in, 16) || !aligned_to(a.h_out, 16))
    return WKVM_ERR_ALIGN;
  switch (dtype) {
    case WKVM_DTYPE_F32: return launch_scan<float>(a, N, st);
    case WKVM_DTYPE_BF16: return launch_scan<__nv_bfloat16>(a, N, st);
    default: return launch_scan<__half>(a, N, st);
  }
}

Act act(const void* p, const int64_t* s, const int64_t* cu, int32_t nseq, int32_t T) {
  return plain_strides({p, s[0], s[1]}, {cu, nseq, T});
}

ScanArgs scan_args(const void* x, const void* dt, const float* A, const void* B, const void* C,
                   const float* skip, const void* z, const float* dt_bias, void* o,
                   const int64_t* s, const int64_t* cu, int32_t nseq, int32_t T, int32_t D,
                   int32_t G, int32_t softplus, int32_t* status) {
  return {act(x, s, cu, nseq, T), act(dt, s + 2, cu, nseq, T), act(z, s + 4, cu, nseq, T),
          act(B, s + 6, cu, nseq, T), act(C, s + 8, cu, nseq, T), A, skip, dt_bias, o, nullptr, nullptr, nullptr, 0, {cu, nseq, T}, D, G, softplus, status};
}

}  // namespace
}  // namespace wkvm

extern "C" int wkvm_selective_scan(
    const void* x, const void* dt, const float* A, const void* Bm, const void* Cm,
    const float* D_skip, const void* z, const float* dt_bias, void* o, const int64_t* strides,
    const float* h0, float* ht, const int64_t* cu_seqlens, int32_t B, int32_t T, int32_t D,
    int32_t N, int32_t G, int32_t softplus, int32_t dtype, int32_t* status,
    wkvm_stream_t stream) {
  if (!strides) return WKVM_ERR_INVALID_ARG;
  wkvm::ScanArgs a = wkvm::scan_args(x, dt, A, Bm, Cm, D_skip, z, dt_bias, o, strides, cu_seqlens,
                                     B, T, D, G, softplus, status);
  a.h_in = h0;
  a.h_out = ht;
  return wkvm::run_scan(a, N, dtype, (cudaStream_t)stream);
}

extern "C" int wkvm_selective_scan_slots(
    const void* x, const void* dt, const float* A, const void* Bm, const void* Cm,
    const float* D_skip, const void* z, const float* dt_bias, void* o, const int64_t* strides,
    float* bank_layer, int64_t num_slots, const int32_t* slot_ids, const int64_t* cu_seqlens,
    int32_t B, int32_t T, int32_t D, int32_t N, int32_t G, int32_t softplus, int32_t dtype,
    int32_t* status, wkvm_stream_t stream) {
  if (!strides) return WKVM_ERR_INVALID_ARG;
  if (B > 0 && (!bank_layer || !slot_ids || num_slots <= 0)) return WKVM_ERR_INVALID_ARG;
  wkvm::ScanArgs a = wkvm::scan_args(x, dt, A, Bm, Cm, D_skip, z, dt_bias, o, strides, cu_seqlens,
                                     B, T, D, G, softplus, status);
  a.h_in = a.h_out = bank_layer;
  a.ids = slot_ids;
  a.num_slots = num_slots;
  return wkvm::run_scan(a, N, dtype, (cudaStream_t)stream);
}
